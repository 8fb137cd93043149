"""policy_loss at a loss gradient of 1, for which the forward kernel itself writes the logits' gradient: every form of that
kernel against 64 bits, over the sizes, layouts, masks and logits where it could go wrong."""

import pytest
import torch
import train_ops_reference as ref
from test_train_ops_gpu import _gen, _randn, _tokens

from dtensor_muon_b200.ops import _ext, model_ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    _ext.check_device_errors("cuda")


def _check(logits, targets, mask, old, adv, frozen, what=""):
    """Both ways to the gradient: at 1, and from a graph whose early gradient is spent."""
    x = logits.detach().requires_grad_()
    for kl, frozen_ in ((0.1, frozen), (0.0, frozen), (0.0, None)):
        p = model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen_, mask=mask, clip_low=0.1, clip_high=0.3, kl_coef=kl)
        (grad,) = torch.autograd.grad(p.loss, x, retain_graph=True)
        assert grad.is_contiguous() and grad.dtype == logits.dtype
        want = ref.policy_loss(logits, targets, old, adv, frozen_, mask, 0.1, 0.3, kl)
        ref.check(dict(p._asdict(), grad=grad), want, what)
        (again,) = torch.autograd.grad(p.loss, x)
        assert again.data_ptr() != grad.data_ptr()
        ref.check(dict(grad=again), want, what + " again")
    with torch.no_grad():  # the loss alone, from the kernel without a gradient
        q = model_ops.policy_loss(logits, targets, old, adv, ref_logp=None, mask=mask, clip_low=0.1, clip_high=0.3)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("b,s,v", [
    (2, 1, 1), (2, 3, 7), (2, 37, 1024), (4, 9, 2048), (4, 9, 2049), (2, 5, 2056), (2, 1, 128256), (2, 7, 32001), (2, 150, 16383),
    (2, 33, 40000), (2, 301, 2500), (1, 3, 65537), (1, 2, 300001),
])
def test_sizes(b, s, v, dtype):
    args = _tokens(b, s, v, dtype)
    _check(*args)
    _check(args[0], args[1], None, *args[3:], "no mask")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("v", [5, 1000, 1025, 8192])
def test_a_warp_for_each_row(v, dtype):
    logits, targets, mask, old, adv, frozen = _tokens(4, 400, v, dtype)
    mask[1] = False
    _check(logits, targets, mask, old, adv, frozen)
    if v == 1025:  # rows that lie on other boundaries than the gradient's
        _check(logits[:, :-1, 1:1001], targets[:, :-1] % 1000, *(t[:, :-1] for t in (mask, old, adv, frozen)), "cut")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("v", [4100, 40002])
def test_layouts(v, dtype):
    logits, targets, mask, old, adv, frozen = _tokens(4, 9, v, dtype)
    rest = (targets[:, :-1], mask[:, :-1], old[:, :-1], adv[:, :-1], frozen[:, :-1])
    _check(logits[:, :-1], *rest, "without the last")
    _check(logits[:, :-1, 3:-99], targets[:, :-1] % (v - 102), *rest[1:], "odd offset")
    _check(logits.transpose(0, 1).contiguous().transpose(0, 1), targets, mask, old, adv, frozen, "sequence first")
    _check(logits.transpose(1, 2).contiguous().transpose(1, 2), targets, mask, old, adv, frozen, "vocabulary first")
    _check(*(t.reshape(36, *t.shape[2:]) for t in (logits, targets, mask, old, adv, frozen)), "two dims")
    _check(*(t.reshape(2, 2, *t.shape[1:]) for t in (logits, targets, mask, old, adv, frozen)), "four dims")
    wide = torch.zeros(4, 9, v + 4, device="cuda", dtype=dtype)[..., :v]
    wide.copy_(logits)
    _check(wide, targets, mask, old, adv, frozen, "padded rows")
    _check(logits[:1, :1].expand(4, 9, v), targets, mask, old, adv, frozen, "one row for all")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("b,v", [(2, 1000), (2, 70000), (260, 1000)])
def test_masks(b, v, dtype):
    logits, targets, mask, old, adv, frozen = _tokens(b, 11, v, dtype)
    mask[1] = False
    bad = [t.clone() for t in (logits, targets, old, adv, frozen)]
    bad[0][~mask] = float("nan")  # what does not count may hold anything
    bad[1][~mask] = -100
    for t in bad[2:]:
        t[~mask] = float("inf")
    _check(bad[0], bad[1], mask, *bad[2:])
    _check(bad[0], bad[1], torch.zeros_like(mask), *bad[2:], "nothing counts")
    one = torch.zeros_like(mask)
    one[-1, -1] = mask[-1, -1] = True
    _check(logits, targets, one, old, adv, frozen, "one token")


@pytest.mark.parametrize("b,v", [(2, 1000), (2, 5000), (2, 70000), (260, 1000)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_unusual_logits(b, v, dtype):
    logits, targets, mask, old, adv, frozen = _tokens(b, 6, v, dtype)
    low = torch.finfo(dtype).min
    logits[:, 0, v // 2 :] = -torch.inf  # half of the vocabulary is masked
    targets[:, 0] = 3
    logits[:, 1, : v - 1] = low
    targets[:, 1] = v - 1
    logits[:, 2] = low  # all alike
    logits[:, 3, 1:] = -torch.inf  # one is left
    targets[:, 3] = 0
    logits[:, 4] += 3e4
    logits[:, 5] *= 20
    clean = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0].float()
    _check(logits, targets, None, clean + 0.1, adv, clean - 0.1)
    x = logits.clone()
    x[0, 0] = -torch.inf  # no distribution: NaN, and nothing else of the gradient is touched
    x[0, 1, 7] = float("nan")
    x[1, 2, 5] = torch.inf
    x.requires_grad_()
    p = model_ops.policy_loss(x, targets, clean + 0.1, adv)
    (grad,) = torch.autograd.grad(p.loss, x)
    dirty = torch.zeros_like(targets, dtype=torch.bool)
    dirty[0, :2] = dirty[1, 2] = True
    assert torch.isnan(p.loss) and torch.equal(torch.isnan(p.logp), dirty)
    assert torch.isnan(grad[dirty]).any(-1).all() and not torch.isnan(grad[~dirty]).any()
    want = ref.policy_loss(logits, targets, clean + 0.1, adv)["grad"]
    ref.check(dict(grad=grad[~dirty]), dict(grad=tuple(t[~dirty] for t in want)))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_every_place_of_the_target(dtype):
    """In the head, each of a vector's eight places, the tail, and the last part of a split row."""
    v = 40003
    places = list(range(12)) + [v // 2 + i for i in range(9)] + [v - 1 - i for i in range(12)]
    n = len(places)
    logits, _, _, old, adv, frozen = _tokens(1, n, v, dtype)
    targets = torch.tensor([places], device="cuda")
    logp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0].float()
    _check(logits, targets, None, logp + 0.05 * _randn(1, n, g=_gen(9)), adv, logp - 0.1)
    _check(logits[..., 1:], targets.clamp(max=v - 2), None, logp, adv, logp - 0.1, "odd offset")
