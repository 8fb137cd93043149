"""policy_loss where a token's ratio is larger than its type holds: the CPU and the kernel give the same."""

import math

import pytest
import torch

from dtensor_muon_b200.ops import model_ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _call(device, gap, adv, dtype=torch.float32, vocab=4, rows=1, **kw):
    """One token of probability 1 / vocab under the model and exp(-gap) of it under the old one, next to ordinary ones."""
    x = torch.zeros(1, rows, vocab, device=device, dtype=dtype, requires_grad=True)
    old = torch.full((1, rows), -math.log(vocab), device=device)
    old[0, 0] -= gap
    a = torch.ones(1, rows, device=device)
    a[0, 0] = adv
    p = model_ops.policy_loss(x, torch.zeros(1, rows, dtype=torch.int64, device=device), old, a, **kw)
    return p, torch.autograd.grad(p.loss, x)[0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gap", [5.0, 89.0, 200.0, 700.0, 1000.0, math.inf])
@pytest.mark.parametrize("rows,vocab", [(1, 4), (3, 4), (2, 70000), (1300, 4)])
def test_a_clipped_token_has_no_gradient(device, dtype, gap, rows, vocab):
    p, grad = _call(device, gap, 1.0, dtype, vocab, rows)
    # the others' ratio is 1 up to 2^-22 (log vocab and the log-probability, each half a step of up to 16 in fp32)
    assert float(p.loss.detach()) == pytest.approx(-(1.2 + rows - 1) / rows, abs=2e-6)
    assert float(p.clipped) == pytest.approx(1 / rows, rel=1e-6)
    assert not grad[0, 0].any() and not grad.isnan().any()
    assert rows == 1 or all(g.any() for g in grad[0, 1:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gap", [89.0, 200.0, 700.0])
def test_a_token_without_advantage_gives_nothing(device, gap):
    p, grad = _call(device, gap, 0.0, rows=2, vocab=8)
    assert float(p.loss.detach()) == pytest.approx(-0.5, abs=2e-6) and float(p.clipped) == 0
    assert not grad[0, 0].any() and grad[0, 1].any() and not grad.isnan().any()


@pytest.mark.parametrize("device", DEVICES)
def test_the_kl_term_of_a_clipped_token_stays(device):
    ref = torch.full((1, 1), -math.log(4) + 0.5, device=device)
    p, grad = _call(device, 200.0, 1.0, ref_logp=ref, kl_coef=0.1)
    assert float(p.loss.detach()) == pytest.approx(-1.2 + 0.1 * (math.exp(0.5) - 1.5), abs=2e-6)
    c = 0.1 * (1 - math.exp(0.5))
    want = torch.tensor([[[0.75 * c, -0.25 * c, -0.25 * c, -0.25 * c]]])
    torch.testing.assert_close(grad.cpu(), want, rtol=1e-5, atol=1e-8)


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_not_clipped_grows(device):
    """A negative advantage holds nothing back: the loss is what the formula says, as far as fp32 goes."""
    p, grad = _call(device, 50.0, -1.0)
    assert float(p.loss.detach()) == pytest.approx(math.exp(50.0), rel=1e-4)  # the gap itself is off by 2^-19
    assert float(grad[0, 0, 0]) == pytest.approx(0.75 * math.exp(50.0), rel=1e-4)
    p, grad = _call(device, 200.0, -1.0)
    assert float(p.loss.detach()) == math.inf
