"""Log-probabilities do not lean to one side: a sequence's sum of them shows it where one token does not."""

import math

import pytest
import torch

from dtensor_muon_b200.ops import _ext, model_ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    _ext.check_device_errors("cuda")


def _errors(rows, vocab, dtype, scale, calls):
    out = []
    for seed in range(calls):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(rows, vocab, generator=g, device="cuda") * scale
        y = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        likely = math.log(vocab) + 2 * torch.randn(rows, generator=g, device="cuda")
        x = x.scatter(1, y[:, None], likely[:, None]).to(dtype)
        out.append(model_ops.token_logprobs(x, y).double() - torch.log_softmax(x.double(), -1).gather(-1, y[:, None])[:, 0])
    return torch.cat(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [2.0, 0.5])
@pytest.mark.parametrize("rows,vocab,calls", [
    (258, 64, 40), (258, 1024, 40), (258, 1031, 40), (258, 4096, 40), (2048, 1024, 20), (2048, 4096, 10), (258, 32000, 20),
])
def test_the_mean_error_is_near_zero(rows, vocab, calls, scale, dtype):
    off = _errors(rows, vocab, dtype, scale, calls)
    # 1e-8, a sixth of half a step of fp32, and three standard errors of the mean
    assert abs(float(off.mean())) <= 1e-8 + 3 * float(off.std()) / math.sqrt(off.numel())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(3, 1), (3, 9), (3, 5000), (1300, 600), (2, 200000)])
def test_a_sure_token_is_exact(rows, vocab, dtype):
    """Where one logit is left the sum is that one's exponential of 0, and nothing is lost."""
    x = torch.full((rows, vocab), -math.inf, device="cuda", dtype=dtype)
    y = torch.randint(0, vocab, (rows,), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    x.scatter_(1, y[:, None], torch.linspace(-7, 7, rows, device="cuda").to(dtype)[:, None])
    assert not model_ops.token_logprobs(x, y).any()
    x[x.isinf()] = torch.finfo(dtype).min
    assert not model_ops.token_logprobs(x, y).any()


@pytest.mark.parametrize("rows,vocab", [(3, 8), (3, 4096), (1300, 512)])
def test_equal_logits_are_exact(rows, vocab):
    x = torch.full((rows, vocab), 2.5, device="cuda")
    y = torch.zeros(rows, dtype=torch.int64, device="cuda")
    want = torch.tensor(-math.log(vocab), dtype=torch.float64).float().item()
    assert set(model_ops.token_logprobs(x, y).tolist()) == {want}


@pytest.mark.parametrize("n,vocab", [(1, 64), (400, 64), (2, 65536)])
def test_losses_that_cancel(n, vocab):
    """Pairs of tokens whose losses cancel to a rounding of the advantage: nothing of a token's loss is lost before the sum."""
    logits = torch.zeros(n, 2, vocab, device="cuda", requires_grad=True)
    targets = torch.zeros(n, 2, dtype=torch.int64, device="cuda")
    old = (-math.log(vocab) - torch.tensor([0.09, -0.11], device="cuda")).expand(n, 2)
    ratio = torch.exp(-math.log(vocab) - old.double())  # the logits are alike: a log-probability has no error
    adv = torch.stack([torch.ones(n, device="cuda"), -(ratio[:, 0] / ratio[:, 1]).float()], 1)
    want = -(ratio * adv.double()).mean()
    assert 0 < abs(float(want)) < 1e-7
    p = model_ops.policy_loss(logits, targets, old, adv)
    # a few steps of the 64-bit logarithm, exponential and sums (1.2e-15 of the largest term), then one rounding to fp32
    assert float(p.loss.detach()) == pytest.approx(float(want), abs=20 * 2**-52, rel=2**-24)
    assert float(p.clipped) == 0
