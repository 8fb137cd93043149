"""The decoder's training operators' kernels against 64-bit formulas, at the sizes, layouts and masks where they could go
wrong."""

import pytest
import torch
import train_ops_reference as ref
from test_train_ops import refusals

from dtensor_muon_b200.models.llama import rope_tables
from dtensor_muon_b200.ops import _ext, model_ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, g, dtype=FP32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    _ext.check_device_errors("cuda")


# --------------------------------------------------------------- qk_norm_rope


def _qk(b, s, h, hk, d, dtype, wdtype=None, seed=0):
    g = _gen(seed)
    q, k = _randn(b, s, h, d, g=g, dtype=dtype, scale=2.0), _randn(b, s, hk, d, g=g, dtype=dtype)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(wdtype or dtype) for _ in range(2))
    cos, sin = rope_tables(d, max(64, s), 10000.0, "cuda")
    return q, k, wq, wk, cos, sin, _randn(b, s, h, d, g=g, dtype=dtype), _randn(b, s, hk, d, g=g, dtype=dtype)


def _check_qk(q, k, wq, wk, cos, sin, dq, dk, pos=None, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = model_ops.qk_norm_rope(*leaves, cos, sin, eps, positions=pos)
    assert yq.is_contiguous() and yk.is_contiguous()
    grads = torch.autograd.grad([yq, yk], leaves, [dq, dk])
    ref.check(dict(q=yq, k=yk, **dict(zip(("dq", "dk", "dwq", "dwk"), grads))),
              ref.qk_norm_rope(q, k, wq, wk, cos, sin, eps, pos, dq, dk))
    return yq, grads


@pytest.mark.parametrize("dtype,wdtype", [(BF16, None), (FP16, None), (FP32, None), (BF16, FP32)])
@pytest.mark.parametrize("b,s,h,hk,d", [
    (1, 1, 1, 1, 8), (3, 1, 32, 8, 128), (2, 33, 9, 3, 96), (1, 257, 4, 4, 64), (2, 5, 7, 1, 256), (1, 130, 40, 40, 128),
    (1, 600, 32, 8, 128), (2, 3, 5, 2, 136),
])
def test_qk_norm_rope(b, s, h, hk, d, dtype, wdtype):
    _check_qk(*_qk(b, s, h, hk, d, dtype, wdtype))


def test_qk_norm_rope_positions_and_strides():
    b, s, h, hk, d = 2, 300, 8, 2, 64
    q, k, wq, wk, cos, sin, dq, dk = _qk(b, s, h, hk, d, BF16)
    for dt in (torch.int64, torch.int32):
        pos = torch.randint(0, cos.shape[0], (b, s), generator=_gen(1), device="cuda").to(dt)
        _check_qk(q, k, wq, wk, cos, sin, dq, dk, pos)
    pos_t = pos.t().contiguous().t()  # not contiguous
    y0, g0 = _check_qk(q, k, wq, wk, cos, sin, dq, dk, pos)
    # slices of a fused projection, gradients with the heads in front, every second token, an odd offset
    fused = torch.cat([q, k, q], dim=2)
    heads_first = dq.transpose(1, 2).contiguous().transpose(1, 2), dk.transpose(1, 2).contiguous().transpose(1, 2)
    y1, g1 = _check_qk(fused[:, :, :h], fused[:, :, h : h + hk], wq, wk, cos, sin, *heads_first, pos_t)
    assert torch.equal(y0, y1) and all(torch.equal(a, c) for a, c in zip(g0, g1))
    _check_qk(q[:, ::2], k[:, ::2], wq, wk, cos, sin, dq[:, ::2], dk[:, ::2])
    flat = torch.empty(q.numel() + 3, device="cuda", dtype=BF16)
    off = flat[3:].view_as(q)
    off.copy_(q)
    _check_qk(off, k, wq, wk, cos, sin, dq.expand(b, s, h, d), dk)
    _check_qk(q, k, torch.cat([wq, wq])[::2], wk, cos, sin, dq, dk)
    one = torch.ones((), device="cuda", dtype=BF16)
    _check_qk(q, k, wq, wk, cos, sin, one.expand(b, s, h, d), dk)  # a broadcast gradient


def test_qk_norm_rope_some_gradients_only():
    q, k, wq, wk, cos, sin, dq, dk = _qk(1, 40, 4, 2, 64, BF16)
    full = _check_qk(q, k, wq, wk, cos, sin, dq, dk)[1]
    q1 = q.clone().requires_grad_()
    yq, yk = model_ops.qk_norm_rope(q1, k, wq, wk, cos, sin)  # frozen weights and keys
    (g,) = torch.autograd.grad([yq, yk], [q1], [dq, dk])
    assert torch.equal(g, full[0])
    w1, k1 = wk.clone().requires_grad_(), k.clone().requires_grad_()
    yq, yk = model_ops.qk_norm_rope(q, k1, wq, w1, cos, sin)
    g = torch.autograd.grad(yk, [k1, w1], dk)  # the queries' output is not used
    assert torch.equal(g[0], full[1]) and torch.equal(g[1], full[3])
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        y = model_ops.qk_norm_rope(q1, k, wq, wk, cos, sin)[0]
        torch.autograd.grad(y, q1, dq, create_graph=True)


def test_qk_norm_rope_zeros_and_large_values():
    q, k, wq, wk, cos, sin, dq, dk = _qk(1, 6, 2, 1, 64, BF16)
    q[:, 0] = 0
    q[:, 1] *= 1e15
    k[:, 2] *= 1e-15
    _check_qk(q, k, wq, wk, cos, sin, dq, dk)


def test_qk_norm_rope_bad_position_is_reported():
    q, k, wq, wk, cos, sin, _, _ = _qk(1, 4, 2, 1, 64, BF16)
    good, _ = model_ops.qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.arange(4, device="cuda")[None])
    for bad in (-1, cos.shape[0], 1 << 40):
        pos = torch.arange(4, device="cuda")[None].clone()
        pos[0, 2] = bad
        yq, yk = model_ops.qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
        assert torch.isnan(yq[0, 2]).all() and torch.isnan(yk[0, 2]).all()
        keep = [0, 1, 3]
        assert torch.equal(yq[0, keep], good[0, keep])
        with pytest.raises(RuntimeError, match="error code 3"):
            _ext.check_device_errors("cuda")


def test_qk_norm_rope_empty():
    q, k, wq, wk, cos, sin, dq, dk = _qk(1, 4, 2, 1, 64, BF16)
    for sl in (slice(0, 0),):
        leaves = [t.detach().requires_grad_() for t in (q[:, sl], k[:, sl], wq, wk)]
        y = model_ops.qk_norm_rope(*leaves, cos, sin)
        g = torch.autograd.grad(list(y), leaves, [dq[:, sl], dk[:, sl]])
        assert g[0].shape == (1, 0, 2, 64) and not g[2].any()
    leaves = [t.detach().requires_grad_() for t in (q, k[:, :, :0], wq, wk)]  # no key heads
    y = model_ops.qk_norm_rope(*leaves, cos, sin)
    g = torch.autograd.grad(list(y), leaves, [dq, dk[:, :, :0]])
    assert torch.equal(g[0], _check_qk(q, k, wq, wk, cos, sin, dq, dk)[1][0]) and not g[3].any()


# ----------------------------------------------------------------------- route


def _check_route(x, k, mask=None, seed=3, db=0.3, dz=0.1):
    x = x.detach().requires_grad_()
    dg = _randn(x.shape[0], k, g=_gen(seed), dtype=x.dtype)
    r = model_ops.route(x, k, mask=mask)
    (grad,) = torch.autograd.grad([r.gates, r.balance, r.z], [x],
                                  [dg, torch.tensor(db, device="cuda"), torch.tensor(dz, device="cuda")])
    ref.check(dict(r._asdict(), grad=grad), ref.route(x.detach(), k, mask, dg, db, dz))
    return r, grad


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,experts,k", [
    (1, 1, 1), (5, 4, 2), (257, 8, 2), (1000, 8, 8), (300, 16, 4), (63, 17, 3), (400, 60, 4), (129, 64, 8), (700, 128, 8),
    (33, 200, 32), (257, 256, 8), (40, 257, 5), (65, 512, 32), (40000, 8, 1), (20011, 64, 2),
])
def test_route(tokens, experts, k, dtype):
    g = _gen(tokens)
    x = _randn(tokens, experts, g=g, dtype=dtype, scale=1.5)
    _check_route(x, k)
    _check_route(x, k, mask=torch.rand(tokens, generator=g, device="cuda") < 0.6)


def test_route_ties_go_to_the_lower_expert():
    for e in (4, 8, 60, 128, 300):
        x = torch.randint(-2, 2, (200, e), generator=_gen(e), device="cuda").float()
        x[x == 0] = torch.where(torch.rand(int((x == 0).sum()), generator=_gen(1), device="cuda") < 0.5, 0.0, -0.0)
        for k in (1, 2, 4):
            r, _ = _check_route(x, k)
            want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(r.experts, want)


def test_route_unusual_logits():
    x = _randn(64, 8, g=_gen(1))
    x[:, 5] = -torch.inf  # an expert that is switched off
    x[:, 6] = torch.finfo(FP32).min
    _check_route(x, 2)
    _check_route(x, 8)
    y = x.clone()
    mask = torch.ones(64, dtype=torch.bool, device="cuda")
    mask[::3] = False
    y[::6] = float("nan")
    y[3::6] = torch.inf
    a, ga = model_ops.route(x, 2, mask=mask), _check_route(y, 2, mask=mask)
    b, grad = ga
    assert torch.equal(a.counts, b.counts) and torch.equal(a.balance, b.balance) and torch.equal(a.z, b.z)
    assert torch.equal(a.gates, b.gates) and not grad[::3].any()
    nan = x.clone()
    nan[7, 3] = float("nan")  # a token that counts: seen in everything that depends on it
    r = model_ops.route(nan, 2)
    assert r.experts[7, 0] == 3 and torch.isnan(r.gates[7]).all() and torch.isnan(r.balance) and torch.isnan(r.z)
    assert torch.equal(r.gates[:7], model_ops.route(x, 2).gates[:7])
    _check_route(x, 2, mask=torch.zeros(64, dtype=torch.bool, device="cuda"))
    empty = model_ops.route(x[:0], 2)
    assert float(empty.balance) == 0 and not empty.counts.any() and empty.experts.shape == (0, 2)


def test_route_strides_and_partial_gradients():
    x = _randn(100, 24, g=_gen(2), dtype=BF16)
    r, grad = _check_route(x[:, :8], 2)
    assert torch.equal(r.gates, model_ops.route(x[:, :8].contiguous(), 2).gates)
    _check_route(x[:, 3:11], 2)
    _check_route(x[::2, :16], 2)
    _check_route(x[:, ::3], 2)
    _check_route(x[:24].t(), 3)
    leaf = x[:, :8].detach().requires_grad_()
    r = model_ops.route(leaf, 2)
    want = ref.route(leaf.detach(), 2, dbalance=1.0)["grad"]
    ref.check(dict(grad=torch.autograd.grad(r.balance, leaf)[0]), dict(grad=want))
    r = model_ops.route(leaf, 2)
    dg = torch.ones((), device="cuda", dtype=BF16).expand(100, 2)
    ref.check(dict(grad=torch.autograd.grad(r.gates, leaf, dg)[0]), dict(grad=ref.route(leaf.detach(), 2, dgates=dg)["grad"]))


def test_route_gives_the_same_bits_each_time():
    x = _randn(30001, 64, g=_gen(5), dtype=BF16)
    a, b = _check_route(x, 4), _check_route(x, 4)
    assert all(torch.equal(p, q) for p, q in zip((*a[0], a[1]), (*b[0], b[1])))


# ----------------------------------------------------- log-probabilities, losses


def _tokens(b, s, v, dtype, seed=0, keep=0.7, scale=3.0):
    g = _gen(seed)
    logits = _randn(b, s, v, g=g, dtype=dtype, scale=scale)
    targets = torch.randint(0, v, (b, s), generator=g, device="cuda")
    mask = torch.rand(b, s, generator=g, device="cuda") < keep
    logp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0].float()
    return (logits, targets, mask, logp + 0.3 * _randn(b, s, g=g), _randn(b, s, g=g), logp + 0.2 * _randn(b, s, g=g))


def _check_losses(logits, targets, mask, old, adv, frozen, what=""):
    x = logits.detach().requires_grad_()
    logp = model_ops.token_logprobs(x, targets, mask=mask)
    dlogp = _randn(*targets.shape, g=_gen(7))
    (grad,) = torch.autograd.grad([logp], [x], [dlogp])
    assert grad.is_contiguous()
    ref.check(dict(logp=logp, grad=grad), ref.token_logprobs(logits, targets, mask, dlogp), what + " logprobs")
    for kl, frozen_ in ((0.1, frozen), (0.0, frozen), (0.0, None)):
        p = model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen_, mask=mask, clip_low=0.1, clip_high=0.3, kl_coef=kl)
        (grad,) = torch.autograd.grad(p.loss * 0.5, x)
        ref.check(dict(p._asdict(), grad=grad),
                  ref.policy_loss(logits, targets, old, adv, frozen_, mask, 0.1, 0.3, kl, scale=0.5), what + " policy")
    if targets.dim() == 2 and targets.shape[0] % 2 == 0 and targets.shape[0]:
        p = model_ops.preference_loss(x, targets, frozen, mask=mask, beta=0.2, label_smoothing=0.1)
        (grad,) = torch.autograd.grad(p.loss * 0.5, x)
        ref.check(dict(p._asdict(), grad=grad), ref.preference_loss(logits, targets, frozen, mask, 0.2, 0.1, scale=0.5),
                  what + " preference")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("b,s,v", [
    (2, 1, 1), (2, 3, 7), (2, 37, 1024), (4, 9, 2048), (4, 9, 2049), (2, 5, 2056), (2, 1, 128256), (2, 7, 32001), (2, 150, 16383),
    (2, 33, 40000), (2, 301, 2500),
])
def test_losses(b, s, v, dtype):
    logits, targets, mask, old, adv, frozen = _tokens(b, s, v, dtype)
    _check_losses(logits, targets, mask, old, adv, frozen)
    _check_losses(logits, targets, None, old, adv, frozen, "no mask")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("v", [5, 1000, 1025, 8192])
def test_losses_of_many_short_rows(v, dtype):
    """Enough rows for a warp each."""
    logits, targets, mask, old, adv, frozen = _tokens(4, 400, v, dtype)
    mask[1] = False
    _check_losses(logits, targets, mask, old, adv, frozen)
    if v == 1025:
        _check_losses(logits[:, :-1, 1:1001], targets[:, :-1] % 1000, *(t[:, :-1] for t in (mask, old, adv, frozen)), "cut")
        bad = logits.clone()
        bad[~mask] = float("nan")
        y = torch.where(mask, targets, -100)
        _check_losses(bad, y, mask, old, adv, frozen, "nothing looked at")
        y[0, int(mask[0].nonzero()[0])] = v
        x = bad.requires_grad_()
        p = model_ops.policy_loss(x, y, old, adv, mask=mask)
        assert torch.isnan(p.loss) and torch.isnan(torch.autograd.grad(p.loss, x)[0][0]).any()
        with pytest.raises(RuntimeError, match="error code 3"):
            _ext.check_device_errors("cuda")


def test_losses_masks():
    logits, targets, mask, old, adv, frozen = _tokens(4, 11, 3001, BF16)
    mask[1] = False  # nothing of one answer counts
    full = [logits, targets, mask, old, adv, frozen]
    _check_losses(*full)
    # what does not count may hold anything
    bad = [t.clone() for t in full]
    bad[0][~mask] = float("nan")
    bad[1][~mask] = -100
    for t in bad[3:]:
        t[~mask] = float("inf")
    _check_losses(bad[0], bad[1], mask, *bad[3:])
    p = model_ops.policy_loss(logits.requires_grad_(), targets, old, adv, ref_logp=frozen, mask=torch.zeros_like(mask), kl_coef=0.1)
    (g,) = torch.autograd.grad(p.loss, logits)
    assert float(p.loss) == 0 and float(p.kl) == 0 and float(p.clipped) == 0 and not g.any()


@pytest.mark.parametrize("b,v", [(2, 1000), (2, 5000), (2, 70000), (260, 1000)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_losses_unusual_logits(b, v, dtype):
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
    _check_losses(logits, targets, None, clean + 0.1, adv, clean - 0.1)
    x = logits.clone()
    x[0, 0] = -torch.inf  # no distribution: NaN, as the softmax of it is, and nothing else is touched
    x[0, 1, 7] = float("nan")
    logp = model_ops.token_logprobs(x, targets)
    assert torch.isnan(logp[0, :2]).all()
    assert torch.equal(logp[0, 2:], model_ops.token_logprobs(logits, targets)[0, 2:])


def test_losses_layouts():
    logits, targets, mask, old, adv, frozen = _tokens(4, 9, 4100, BF16)
    rest = (targets[:, :-1], mask[:, :-1], old[:, :-1], adv[:, :-1], frozen[:, :-1])
    _check_losses(logits[:, :-1], *rest, "without the last")
    _check_losses(logits[:, :-1, 3:4001], targets[:, :-1] % 3998, *rest[1:], "odd offset")
    _check_losses(logits.transpose(0, 1).contiguous().transpose(0, 1), targets, mask, old, adv, frozen, "sequence first")
    _check_losses(logits.transpose(1, 2).contiguous().transpose(1, 2), targets, mask, old, adv, frozen, "vocabulary first")
    flat = [t.reshape(36, *t.shape[2:]) for t in (logits, targets, mask, old, adv, frozen)]
    _check_losses(*flat, "two dims")
    four = [t.reshape(2, 2, *t.shape[1:]) for t in (logits, targets, mask, old, adv, frozen)]
    _check_losses(*four, "four dims")
    wide = torch.zeros(4, 9, 4104, device="cuda", dtype=BF16)[..., :4100]
    wide.copy_(logits)
    _check_losses(wide, targets, mask, old, adv, frozen, "padded rows")
    row = logits[:1, :1].expand(4, 9, 4100)
    _check_losses(row, targets, mask, old, adv, frozen, "one row for all")


def test_losses_of_no_tokens():
    logits, targets, mask, old, adv, frozen = _tokens(2, 3, 500, BF16)
    x = logits[:, :0].detach().requires_grad_()
    cut = [t[:, :0] for t in (targets, mask, old, adv, frozen)]
    assert model_ops.token_logprobs(x, cut[0]).shape == (2, 0)
    p = model_ops.policy_loss(x, cut[0], cut[2], cut[3])
    assert float(p.loss) == 0
    assert torch.autograd.grad(p.loss, x)[0].shape == (2, 0, 500)
    p = model_ops.preference_loss(x, cut[0], cut[4])
    assert float(p.loss) == pytest.approx(0.6931472) and p.rewards.tolist() == [0, 0]


def test_many_pairs_and_long_sequences():
    logits, targets, mask, old, adv, frozen = _tokens(2600, 2, 16, BF16)
    _check_losses(logits, targets, mask, old, adv, frozen, "many")
    logits, targets, mask, old, adv, frozen = _tokens(2, 70001, 24, BF16)
    _check_losses(logits, targets, mask, old, adv, frozen, "long")


def test_bad_targets_are_reported():
    for v in (600, 9000):
        logits, targets, _, old, adv, frozen = _tokens(2, 3, v, BF16)
        good = model_ops.token_logprobs(logits, targets)
        for bad in (-1, v, 1 << 40, -100):
            t = targets.clone()
            t[1, 1] = bad
            x = logits.detach().requires_grad_()
            logp = model_ops.token_logprobs(x, t)
            keep = torch.ones_like(t, dtype=torch.bool)
            keep[1, 1] = False
            assert torch.isnan(logp[1, 1]) and torch.equal(logp[keep], good[keep])
            with pytest.raises(RuntimeError, match="error code 3"):
                _ext.check_device_errors("cuda")
            (g,) = torch.autograd.grad(logp, x, torch.ones_like(logp))
            assert torch.isnan(g[1, 1]).all() and not torch.isnan(g[keep]).any()
            p = model_ops.policy_loss(x, t, old, adv)
            assert torch.isnan(p.loss)
            (g,) = torch.autograd.grad(p.loss, x)
            assert torch.isnan(g[1, 1]).all()
            with pytest.raises(RuntimeError, match="error code 3"):
                _ext.check_device_errors("cuda")


def test_backward_twice_scaled_and_refused_twice():
    logits, targets, mask, old, adv, frozen = _tokens(2, 40, 5000, BF16)
    x = logits.requires_grad_()
    p = model_ops.policy_loss(x, targets, old, adv, mask=mask)
    (a,) = torch.autograd.grad(p.loss, x, retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(p.loss, x, grad_outputs=torch.tensor(0.25, device="cuda"), retain_graph=True)
    (c,) = torch.autograd.grad(p.loss, x)
    assert torch.equal(a, kept) and torch.equal(a, c) and a.data_ptr() != c.data_ptr()
    ref.check(dict(grad=b), ref.policy_loss(logits.detach(), targets, old, adv, None, mask, scale=0.25))
    p = model_ops.policy_loss(x, targets, old, adv, mask=mask)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(p.loss, x, create_graph=True)
    for t in (p.logp, p.kl, p.clipped):
        assert not t.requires_grad
    # the logits may not change between the two directions
    p = model_ops.policy_loss(x, targets, old, adv)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        p.loss.backward()


def test_policy_gradient_under_modes_hooks_and_accumulation():
    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.checkpoint import checkpoint

    logits, targets, mask, old, adv, frozen = _tokens(2, 40, 5000, BF16)

    def loss(x):
        return model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1).loss

    x = logits.detach().requires_grad_()
    (want,) = torch.autograd.grad(loss(x), x)
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Mode():
        out = loss(x)
        (got,) = torch.autograd.grad(out, x)
    assert torch.equal(got, want)
    assert any("policy_loss" in f for f in seen) and any("token_logprobs_backward" in f for f in seen)
    (got,) = torch.autograd.grad(checkpoint(loss, x, use_reentrant=False), x)
    assert torch.equal(got, want)
    with torch.autograd.graph.save_on_cpu():
        out = loss(x)
    assert torch.equal(torch.autograd.grad(out, x)[0], want)
    x.grad = None
    loss(x).backward()
    loss(x).backward()
    ref.check(dict(grad=x.grad), dict(grad=(2 * want.double(), want.double().abs() * 2**-7)))
    # a scaled loss, as in gradient accumulation
    x.grad = None
    (loss(x) / 4).backward()
    ref.check(dict(grad=x.grad), ref.policy_loss(logits, targets, old, adv, frozen, mask, kl_coef=0.1, scale=0.25))


def test_long_rows():
    for dtype in (BF16, FP32):
        _check_losses(*_tokens(2, 2, 300001, dtype))


# ---------------------------------------------------------- offsets past 32 bits


def test_losses_of_more_than_2_31_logits():
    rows, v = 17000, 128256
    logits = torch.zeros(rows, v, device="cuda", dtype=BF16)
    few = _tokens(1, 3, v, BF16)
    logits[-3:] = few[0][0]
    targets = torch.zeros(rows, dtype=torch.int64, device="cuda")
    targets[-3:] = few[1][0]
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[-3:] = True
    x = logits.requires_grad_()
    old, adv = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    old[-3:], adv[-3:] = few[3][0], few[4][0]
    want = ref.policy_loss(few[0][0], few[1][0], few[3][0], few[4][0])
    p = model_ops.policy_loss(x, targets, old, adv, mask=mask)
    (g,) = torch.autograd.grad(p.loss, x)
    ref.check(dict(loss=p.loss, logp=p.logp[-3:], grad=g[-3:]), want)
    assert not g[:-3:1000].any()
    del g
    logp = model_ops.token_logprobs(x, targets, mask=mask)
    (g,) = torch.autograd.grad(logp, x, torch.ones_like(logp))
    ref.check(dict(logp=logp[-3:], grad=g[-3:]), ref.token_logprobs(few[0][0], few[1][0], None, torch.ones(3, device="cuda")))


def test_heads_of_more_than_2_31_values():
    tokens, h, d = 70000, 256, 128
    q = torch.zeros(1, tokens, h, d, device="cuda", dtype=BF16)
    few = _qk(1, 2, h, 1, d, BF16)
    q[:, -2:] = few[0]
    k = torch.zeros(1, tokens, 1, d, device="cuda", dtype=BF16)
    pos = torch.zeros(1, tokens, dtype=torch.int32, device="cuda")
    pos[0, -1] = 5
    x = q.requires_grad_()
    y, _ = model_ops.qk_norm_rope(x, k, few[2], few[3], few[4], few[5], positions=pos)
    one = torch.ones((), device="cuda", dtype=BF16)
    (g,) = torch.autograd.grad(y, x, one.expand_as(y))
    want = ref.qk_norm_rope(few[0], k[:, -2:], few[2], few[3], few[4], few[5], 1e-5, pos[:, -2:],
                            one.expand(1, 2, h, d), k[:, -2:])
    ref.check(dict(q=y[:, -2:], dq=g[:, -2:]), want)


def test_route_of_more_than_2_31_logits():
    tokens, e = 4_200_000, 512
    x = torch.zeros(tokens, e, device="cuda", dtype=BF16)
    few = _randn(3, e, g=_gen(1), dtype=BF16)
    x[-3:] = few
    mask = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    mask[-3:] = True
    x.requires_grad_()
    r = model_ops.route(x, 2, mask=mask)
    dg = _randn(3, 2, g=_gen(2), dtype=BF16)
    wide = torch.zeros(tokens, 2, device="cuda", dtype=BF16)
    wide[-3:] = dg
    (g,) = torch.autograd.grad([r.gates, r.balance], x, [wide, torch.ones((), device="cuda")])
    want = ref.route(few, 2, None, dg, 1.0)
    ref.check(dict(gates=r.gates[-3:], experts=r.experts[-3:], counts=r.counts, balance=r.balance, z=r.z, grad=g[-3:]), want)
    assert not g[: -3 : 10007].any()


# ------------------------------------------------------------------ everywhere


@pytest.mark.parametrize("name,call", refusals(), ids=lambda v: v if isinstance(v, str) else "")
def test_refusals(name, call):
    with pytest.raises(ValueError):
        call("cuda")


def test_tensors_of_two_devices_are_refused():
    logits, targets, mask, old, adv, frozen = _tokens(2, 3, 100, BF16)
    with pytest.raises(ValueError):
        model_ops.token_logprobs(logits, targets.cpu())
    with pytest.raises(ValueError):
        model_ops.policy_loss(logits, targets, old.cpu(), adv)
    with pytest.raises(ValueError):
        model_ops.route(logits[0], 2, mask=torch.ones(3, dtype=torch.bool))
    q, k, wq, wk, cos, sin, _, _ = _qk(1, 4, 2, 1, 64, BF16)
    with pytest.raises(ValueError):
        model_ops.qk_norm_rope(q, k, wq, wk.cpu(), cos, sin)
    with pytest.raises(ValueError):
        model_ops.qk_norm_rope(q, k, wq, wk, cos.cpu(), sin)


def test_fp64_and_other_sizes_take_the_composition():
    logits, targets, mask, old, adv, frozen = _tokens(2, 5, 50, FP32)
    a = model_ops.policy_loss(logits, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1)
    b = model_ops.policy_loss(logits.double(), targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1)
    torch.testing.assert_close(a.loss.double(), b.loss, rtol=1e-5, atol=1e-6)
    q, k, wq, wk, cos, sin, _, _ = _qk(1, 5, 2, 1, 12, FP32)
    n0 = _ext.launch_count
    model_ops.qk_norm_rope(q, k, wq, wk, cos, sin)
    model_ops.route(torch.zeros(4, 600, device="cuda"), 2)
    assert _ext.launch_count == n0


def test_launches_are_counted():
    logits, targets, mask, old, adv, frozen = _tokens(2, 5, 50, FP32)
    x = logits.requires_grad_()
    n0 = _ext.launch_count
    loss = model_ops.policy_loss(x, targets, old, adv).loss
    assert _ext.launch_count - n0 == 2
    loss.backward()
    assert _ext.launch_count - n0 == 3


def _all_directions(seed=0):
    """One call of each operator with its gradient; returns its static inputs and a function that runs it all."""
    q, k, wq, wk, cos, sin, dq, dk = _qk(1, 70, 4, 2, 64, BF16, seed=seed)
    x = _randn(500, 8, g=_gen(seed), dtype=BF16)
    logits, targets, mask, old, adv, frozen = _tokens(2, 35, 5000, BF16, seed=seed)
    data = [q, k, wq, wk, x, logits, old, adv, frozen]
    dg = torch.ones(500, 2, device="cuda", dtype=BF16)

    def run():
        qs = [t.detach().requires_grad_() for t in data[:4]]
        y = model_ops.qk_norm_rope(*qs, cos, sin)
        out = [*y, *torch.autograd.grad(list(y), qs, [dq, dk])]
        xs = data[4].detach().requires_grad_()
        r = model_ops.route(xs, 2)
        out += [*r, *torch.autograd.grad([r.gates, r.balance], xs, [dg, torch.ones((), device="cuda")])]
        ls = data[5].detach().requires_grad_()
        p = model_ops.policy_loss(ls, targets, data[6], data[7], ref_logp=data[8], mask=mask, kl_coef=0.1)
        out += [*p, *torch.autograd.grad(p.loss, ls)]
        p = model_ops.preference_loss(ls, targets, data[8], mask=mask)
        out += [*p, *torch.autograd.grad(p.loss, ls)]
        return [t.detach() for t in out]

    return data, run


def test_captured_and_replayed():
    data, run = _all_directions(0)
    other, run_other = _all_directions(1)
    want, want_other = run(), run_other()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for t, o in zip(data, other):
        t.copy_(o)
    graphs[0][0].replay()
    graphs[1][0].replay()
    graphs[0][0].replay()
    for _, out in graphs:
        # the targets and masks stay the first data's: compare with a fresh eager run
        for got, exp in zip(out, run()):
            assert torch.equal(got, exp)
    del graphs
    assert any(not torch.equal(a, b) for a, b in zip(want, want_other))


def test_on_another_stream():
    data, run = _all_directions(2)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    runs = [_all_directions(s)[1] for s in (3, 4)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = []
    for _ in range(5):
        for r, s in zip(runs, streams):
            with torch.cuda.stream(s):
                got.append(r())
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.multigpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_on_another_device():
    _, run = _all_directions(5)
    want = [t.cpu() for t in run()]
    q, k, wq, wk, cos, sin, _, _ = _qk(1, 70, 4, 2, 64, BF16, seed=5)
    y = model_ops.qk_norm_rope(*(t.to("cuda:1") for t in (q, k, wq, wk, cos, sin)))  # cuda:0 is the current one
    assert torch.equal(y[0].cpu(), want[0])


def test_compiled():
    """The operators trace as one graph, forward and backward."""
    logits, targets, mask, old, adv, frozen = _tokens(2, 9, 3000, BF16)
    q, k, wq, wk, cos, sin, dq, dk = _qk(1, 9, 4, 2, 64, BF16)

    def fn(x, q):
        a = model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1).loss
        b = model_ops.route(x[0, :, :8], 2).balance
        y = model_ops.qk_norm_rope(q, k, wq, wk, cos, sin)[0]
        return a + b + y.float().square().mean()

    want = [t.detach().requires_grad_() for t in (logits, q)]
    got = [t.detach().requires_grad_() for t in (logits, q)]
    fn(*want).backward()
    torch.compile(fn, backend="aot_eager", fullgraph=True)(*got).backward()
    for w, g in zip(want, got):
        torch.testing.assert_close(w.grad, g.grad, rtol=1e-2, atol=1e-6)
