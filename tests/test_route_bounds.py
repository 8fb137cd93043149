"""route against 64 bits where logits lie far apart: each value's bound follows from its own distance to the row's maximum,
so that one far logit widens no other's, and no bound is wider than a hundredth of what it is for."""

import pytest
import torch
from train_ops_reference import E, FLUSH, U, check, tiny

from dtensor_muon_b200.ops import model_ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def bounds(logits, top_k, mask, dgates, dbalance, dz):
    """{output: (value, bound)}.

    An exponential ``exp2((x - m) * log2 e)`` is off by ``(4 + 2 |x - m|) E`` of itself (two roundings of the argument, the
    constant's, two steps of the exponential) and at most 2^-126 where it is flushed; the sum of a row's by theirs, each
    weighted with its share, and 13 additions in a row (eight on a lane, five over a warp). A quotient takes two more
    roundings. ``__log2f`` is off by 4 E for sums up to 2 and by two steps, at most 4 E of itself, above. A sum over tokens
    takes an addition per row that a lane walks over, 13 over the warp and the CTA's warps, and is in 64 bits from there.
    """
    t, e = logits.shape
    u = U[logits.dtype]
    valid = torch.ones(t, dtype=torch.bool, device=logits.device) if mask is None else mask
    full = logits.double()
    experts = torch.sort(torch.where(full.isnan(), torch.inf, full), dim=1, descending=True, stable=True).indices[:, :top_k]
    x = torch.where(valid[:, None], full, 0.0)
    v = valid.double()[:, None]
    n = max(1, int(valid.sum()))
    m = x.amax(1, keepdim=True)
    exp_off = torch.where(x == -torch.inf, 0.0, (4 + 2 * (m - x)) * E)
    hot = torch.zeros_like(x).scatter_(1, experts, 1.0)
    chain = -(-t // (4 * 148 * 8)) + 13  # rows of a lane, on a GPU with 148 multiprocessors; the CPU sums pairwise

    def softmax(z):
        p = torch.softmax(z, 1)
        total = (p * exp_off).sum(1, keepdim=True) + 13 * E
        return p, torch.where(p > 0, p * (exp_off + total + 2 * E) + FLUSH, 0.0), total

    p, p_off, total = softmax(x)
    g, g_off, _ = softmax(torch.where(hot > 0, x, -torch.inf))
    lse = torch.logsumexp(x, 1, keepdim=True)
    log_s = lse - m
    lse_off = total + 4 * E + 6 * E * log_s.abs() + 2 * E * (lse.abs() + m.abs())
    counts = (hot * v).sum(0)
    share = counts / (n * top_k)
    gates, gates_off = (g * v).gather(1, experts), (g_off * v).gather(1, experts)
    balance = e * (share * (p * v).sum(0) / n).sum()
    balance_off = e * (share * (p_off * v).sum(0) / n).sum() + (chain + 1) * E * balance
    z = (lse.square() * v).sum() / n
    z_off = ((2 * lse.abs() * lse_off + lse_off.square()) * v).sum() / n + (chain + 2) * E * z
    dg = torch.zeros_like(x).scatter_(1, experts, dgates.double())
    dot, dot_off = (g * dg).sum(1, keepdim=True), (g_off * dg.abs()).sum(1, keepdim=True)
    size = (g * dg.abs()).sum(1, keepdim=True)
    a, b = dbalance * e / n, dz * 2 / n
    mix, mix_off = (share * p).sum(1, keepdim=True), (share * p_off).sum(1, keepdim=True)
    by = a * (share - mix) + b * lse
    by_size = abs(a) * (share + mix) + abs(b) * lse.abs()
    by_off = abs(a) * mix_off + abs(b) * lse_off + 24 * E * by_size  # 13 additions of the mix, and products
    grad = v * (g * (dg - dot) + p * by)
    grad_off = v * (g_off * (dg - dot).abs() + g * (dot_off + 20 * E * (dg.abs() + size)) + p_off * by.abs() + p * by_off)
    for value, off in ((gates, gates_off), (balance, balance_off), (z, z_off)):
        assert (off <= 1e-2 * value.abs() + 1e-30).all()
    assert (grad_off <= 1e-2 * (g * (dg.abs() + size) + p * by_size) + 1e-30).all()
    z = torch.where(z > torch.finfo(FP32).max, torch.inf, z)  # as fp32 holds it: the square of the lowest logits does not fit
    return dict(gates=(gates, u * gates + gates_off + tiny(logits.dtype)), experts=(experts, None),
                counts=(counts.long(), None), balance=(balance, balance_off + E), z=(z, z_off + E),
                grad=(grad, u * grad.abs() + grad_off + tiny(logits.dtype)))


def _check(x, k, mask=None, dbalance=0.3, dz=0.1):
    g = torch.Generator(device=x.device).manual_seed(3)
    dgates = torch.randn(x.shape[0], k, generator=g, device=x.device).to(x.dtype)
    want = bounds(x, k, mask, dgates, dbalance, dz)
    leaf = x.detach().requires_grad_()
    r = model_ops.route(leaf, k, mask=mask)
    (grad,) = torch.autograd.grad([r.gates, r.balance, r.z], [leaf],
                                  [dgates, torch.tensor(dbalance, device=x.device), torch.tensor(dz, device=x.device)])
    check(dict(r._asdict(), grad=grad), want)


def _normal(device, t, e, dtype, scale=1.5, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(t, e, generator=g, device=device) * scale).to(dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("e,k", [(8, 2), (8, 8), (17, 3), (64, 2), (100, 8), (128, 8), (256, 4), (300, 5), (512, 32)])
def test_far_logits(device, dtype, e, k):
    low = torch.finfo(dtype).min
    x = _normal(device, 96, e, dtype)
    x[:, 5] = -torch.inf  # an expert that is switched off
    x[:, 6] = low
    x[0:8, 3:] = -torch.inf  # fewer left than are chosen
    x[8:16, 1:] = low
    x[16:24] = low  # all alike
    x[24:32] += 300
    x[32:40] *= 20
    x[40:48] -= 300
    _check(x, k)
    mask = torch.rand(96, generator=torch.Generator(device=device).manual_seed(1), device=device) < 0.7
    mask[:3] = True
    _check(x, k, mask)
    y = x.clone()
    y[~mask] = torch.nan  # what does not count may hold anything
    _check(y, k, mask)
    _check(x, k, torch.zeros_like(mask))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (40000, 8, 2), (20011, 64, 2), (30001, 128, 8), (5000, 300, 4)])
def test_many_tokens(device, t, e, k):
    if device == "cpu" and t * e > 1 << 21:
        pytest.skip("as much work as one GPU test")
    for dtype in (BF16, FP32):
        x = _normal(device, t, e, dtype)
        _check(x, k)
        _check(x, k, torch.rand(t, generator=torch.Generator(device=device).manual_seed(1), device=device) < 0.6)
