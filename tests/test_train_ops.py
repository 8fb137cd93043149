"""The decoder's training operators on the CPU: values and gradients against 64-bit formulas, differences, refusals,
schemas and fake kernels."""

import pytest
import torch
import train_ops_reference as ref

from dtensor_muon_b200.models.llama import rope_tables
from dtensor_muon_b200.ops import _ext, model_ops

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def qk_inputs(b=2, s=7, h=3, hk=1, d=16, dtype=torch.float32, wdtype=None, seed=0):
    g = _gen(seed)
    q, k = torch.randn(b, s, h, d, generator=g).to(dtype), torch.randn(b, s, hk, d, generator=g).to(dtype)
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g)).to(wdtype or dtype) for _ in range(2))
    cos, sin = rope_tables(d, 4 * max(1, s), 10000.0, "cpu")
    dq, dk = torch.randn(b, s, h, d, generator=g).to(dtype), torch.randn(b, s, hk, d, generator=g).to(dtype)
    return q, k, wq, wk, cos, sin, dq, dk


def token_inputs(b=2, s=5, v=33, dtype=torch.float32, seed=0):
    g = _gen(seed)
    logits = (3 * torch.randn(b, s, v, generator=g)).to(dtype)
    targets = torch.randint(0, v, (b, s), generator=g)
    mask = torch.rand(b, s, generator=g) < 0.7
    logp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0].float()
    old = logp + 0.3 * torch.randn(b, s, generator=g)
    adv = torch.randn(b, s, generator=g)
    frozen = logp + 0.2 * torch.randn(b, s, generator=g)
    return logits, targets, mask, old, adv, frozen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("positions", [False, True])
def test_qk_norm_rope(dtype, positions):
    q, k, wq, wk, cos, sin, dq, dk = qk_inputs(dtype=dtype)
    pos = torch.randint(0, cos.shape[0], q.shape[:2], generator=_gen(1)) if positions else None
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = model_ops.qk_norm_rope(q, k, wq, wk, cos, sin, 1e-5, positions=pos)
    grads = torch.autograd.grad([yq, yk], leaves, [dq, dk])
    want = ref.qk_norm_rope(q.detach(), k.detach(), wq.detach(), wk.detach(), cos, sin, 1e-5, pos, dq, dk)
    ref.check(dict(q=yq, k=yk, **dict(zip(("dq", "dk", "dwq", "dwk"), grads))), want)


def test_qk_norm_rope_is_norm_then_rope():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs(d=8)
    yq, _ = model_ops.qk_norm_rope(q, k, wq, wk, cos, sin, 1e-6)
    plain = model_ops.rope(torch.nn.functional.rms_norm(q, (8,), wq, 1e-6), cos, sin)
    torch.testing.assert_close(yq, plain, rtol=1e-5, atol=1e-6)


def test_gradients_against_differences():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs(b=1, s=3, h=2, d=8)
    leaves = [t.double().requires_grad_() for t in (q, k, wq, wk)]
    assert torch.autograd.gradcheck(
        lambda a, b, c, d: model_ops.qk_norm_rope(a, b, c, d, cos.double(), sin.double(), 1e-5), leaves)
    x = torch.randn(6, 5, generator=_gen(3), dtype=torch.float64, requires_grad=True)
    m = torch.tensor([True, True, False, True, True, True])
    # the counts have no gradient: with them held, the balance loss is what is differentiated
    assert torch.autograd.gradcheck(lambda t: (lambda r: (r.gates, r.balance, r.z))(model_ops.route(t, 2, mask=m)), x)
    logits, targets, mask, old, adv, frozen = token_inputs(b=2, s=4, v=7)
    x = logits.double().requires_grad_()
    assert torch.autograd.gradcheck(lambda t: model_ops.token_logprobs(t, targets, mask=mask), x)
    assert torch.autograd.gradcheck(
        lambda t: model_ops.policy_loss(t, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.3).loss, x)
    assert torch.autograd.gradcheck(
        lambda t: model_ops.preference_loss(t, targets, frozen, mask=mask, beta=0.5, label_smoothing=0.1).loss, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (9, 4, 2), (33, 8, 8), (17, 60, 4)])
@pytest.mark.parametrize("masked", [False, True])
def test_route(dtype, tokens, experts, k, masked):
    g = _gen(tokens)
    x = torch.randn(tokens, experts, generator=g).to(dtype).requires_grad_()
    mask = torch.rand(tokens, generator=g) < 0.6 if masked else None
    dg = torch.randn(tokens, k, generator=g).to(dtype)
    r = model_ops.route(x, k, mask=mask)
    (grad,) = torch.autograd.grad([r.gates, r.balance, r.z], [x], [dg, torch.tensor(0.3), torch.tensor(0.1)])
    ref.check(dict(r._asdict(), grad=grad), ref.route(x.detach(), k, mask, dg, 0.3, 0.1))


def test_route_ties_balance_and_empty():
    x = torch.zeros(4, 6)
    r = model_ops.route(x, 2)
    assert r.experts.tolist() == [[0, 1]] * 4 and r.counts.tolist() == [4, 4, 0, 0, 0, 0]
    assert float(r.balance) == pytest.approx(1.0)
    empty = model_ops.route(x, 2, mask=torch.zeros(4, dtype=torch.bool))
    assert empty.counts.sum() == 0 and float(empty.balance) == 0 and float(empty.z) == 0 and not empty.gates.any()
    none = model_ops.route(torch.zeros(0, 6), 2)
    assert none.gates.shape == (0, 2) and float(none.balance) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 33, 600])
def test_losses(dtype, v):
    logits, targets, mask, old, adv, frozen = token_inputs(b=4, v=v, dtype=dtype)
    mask[1] = False  # a sequence of which nothing counts
    logits[1] = float("nan")
    x = logits.requires_grad_()
    logp = model_ops.token_logprobs(x, targets, mask=mask)
    dlogp = torch.randn(logp.shape, generator=_gen(5))
    (grad,) = torch.autograd.grad([logp], [x], [dlogp])
    ref.check(dict(logp=logp, grad=grad), ref.token_logprobs(x.detach(), targets, mask, dlogp, rounded=True))
    p = model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1)
    (grad,) = torch.autograd.grad(p.loss, x)
    ref.check(dict(p._asdict(), grad=grad),
              ref.policy_loss(x.detach(), targets, old, adv, frozen, mask, kl_coef=0.1, rounded=True))
    p = model_ops.preference_loss(x, targets, frozen, mask=mask, beta=0.2, label_smoothing=0.1)
    (grad,) = torch.autograd.grad(p.loss, x)
    ref.check(dict(p._asdict(), grad=grad),
              ref.preference_loss(x.detach(), targets, frozen, mask, 0.2, 0.1, rounded=True))


def test_policy_of_an_empty_batch_is_zero():
    logits, targets, mask, old, adv, frozen = token_inputs()
    p = model_ops.policy_loss(logits.requires_grad_(), targets, old, adv, ref_logp=frozen,
                              mask=torch.zeros_like(mask), kl_coef=0.1)
    (grad,) = torch.autograd.grad(p.loss, logits)
    assert float(p.loss) == 0 and float(p.kl) == 0 and not grad.any()


def test_first_policy_step_is_the_policy_gradient():
    """Where old and new agree, the gradient is that of -A logp and nothing is clipped."""
    logits, targets, _, _, adv, _ = token_inputs()
    x = logits.requires_grad_()
    old = model_ops.token_logprobs(x, targets).detach()
    p = model_ops.policy_loss(x, targets, old, adv)
    (grad,) = torch.autograd.grad(p.loss, x)
    (want,) = torch.autograd.grad(-(adv * model_ops.token_logprobs(x, targets)).mean(), x)
    torch.testing.assert_close(grad, want, rtol=1e-5, atol=1e-7)
    assert float(p.clipped) == 0


def refusals():
    """(name, call) of calls that are refused, as ``call(device)``."""

    def qk(change):
        def call(dev):
            q, k, wq, wk, cos, sin, _, _ = qk_inputs()
            a = dict(q=q.to(dev), k=k.to(dev), q_weight=wq.to(dev), k_weight=wk.to(dev), cos=cos.to(dev), sin=sin.to(dev))
            a.update(change(a))
            return model_ops.qk_norm_rope(**a)

        return call

    def loss(fn, change):
        def call(dev):
            logits, targets, mask, old, adv, frozen = (t.to(dev) for t in token_inputs())
            a = dict(logits=logits, targets=targets, mask=mask)
            if fn == "policy_loss":
                a.update(old_logp=old, advantages=adv, ref_logp=frozen)
            elif fn == "preference_loss":
                a.update(ref_logp=frozen)
            a.update(change(a))
            return getattr(model_ops, fn)(**a)

        return call

    out = [
        ("qk: three dims", qk(lambda a: dict(q=a["q"][0]))),
        ("qk: other batch", qk(lambda a: dict(k=a["k"][:1]))),
        ("qk: other dtype", qk(lambda a: dict(k=a["k"].bfloat16()))),
        ("qk: weight size", qk(lambda a: dict(q_weight=a["q_weight"][:8]))),
        ("qk: weight dtypes", qk(lambda a: dict(q_weight=a["q_weight"].bfloat16()))),
        ("qk: table width", qk(lambda a: dict(cos=a["cos"][:, :4]))),
        ("qk: table length", qk(lambda a: dict(cos=a["cos"][:3], sin=a["sin"][:3]))),
        ("qk: tables differ", qk(lambda a: dict(cos=a["cos"][:9]))),
        ("qk: positions' shape", qk(lambda a: dict(positions=torch.zeros(7, dtype=torch.int64, device=a["q"].device)))),
        ("qk: positions' dtype", qk(lambda a: dict(positions=torch.zeros(2, 7, device=a["q"].device)))),
        ("route: k = 0", lambda dev: model_ops.route(torch.zeros(3, 4, device=dev), 0)),
        ("route: k > E", lambda dev: model_ops.route(torch.zeros(3, 4, device=dev), 5)),
        ("route: three dims", lambda dev: model_ops.route(torch.zeros(3, 4, 5, device=dev), 2)),
        ("route: no experts", lambda dev: model_ops.route(torch.zeros(3, 0, device=dev), 1)),
        ("route: mask's shape", lambda dev: model_ops.route(torch.zeros(3, 4, device=dev), 2, mask=torch.ones(4, dtype=torch.bool, device=dev))),
        ("route: mask's dtype", lambda dev: model_ops.route(torch.zeros(3, 4, device=dev), 2, mask=torch.ones(3, device=dev))),
    ]
    for fn in ("token_logprobs", "policy_loss", "preference_loss"):
        out += [
            (fn + ": targets' shape", loss(fn, lambda a: dict(targets=a["targets"][:, :2]))),
            (fn + ": targets' dtype", loss(fn, lambda a: dict(targets=a["targets"].int()))),
            (fn + ": mask's dtype", loss(fn, lambda a: dict(mask=a["mask"].float()))),
            (fn + ": mask's shape", loss(fn, lambda a: dict(mask=a["mask"][:1]))),
            (fn + ": no vocabulary", loss(fn, lambda a: dict(logits=a["logits"][..., :0]))),
            (fn + ": integer logits", loss(fn, lambda a: dict(logits=a["logits"].long()))),
        ]
    out += [
        ("policy_loss: old's shape", loss("policy_loss", lambda a: dict(old_logp=a["old_logp"][:1]))),
        ("policy_loss: advantages' dtype", loss("policy_loss", lambda a: dict(advantages=a["advantages"].bfloat16()))),
        ("policy_loss: clip_low", loss("policy_loss", lambda a: dict(clip_low=1.5))),
        ("policy_loss: clip_high", loss("policy_loss", lambda a: dict(clip_high=-0.1))),
        ("policy_loss: kl without ref", loss("policy_loss", lambda a: dict(ref_logp=None, kl_coef=0.1))),
        ("preference_loss: odd", loss("preference_loss", lambda a: {n: a[n][:1] for n in ("logits", "targets", "mask", "ref_logp")})),
        ("preference_loss: one row of tokens", loss("preference_loss", lambda a: {n: a[n][0] for n in ("logits", "targets", "mask", "ref_logp")})),
        ("preference_loss: none", loss("preference_loss", lambda a: {n: a[n][:0] for n in ("logits", "targets", "mask", "ref_logp")})),
        ("preference_loss: beta", loss("preference_loss", lambda a: dict(beta=0.0))),
        ("preference_loss: smoothing", loss("preference_loss", lambda a: dict(label_smoothing=0.5))),
        ("preference_loss: ref's dtype", loss("preference_loss", lambda a: dict(ref_logp=a["ref_logp"].half()))),
    ]
    return out


@pytest.mark.parametrize("name,call", refusals(), ids=lambda v: v if isinstance(v, str) else "")
def test_refusals(name, call):
    with pytest.raises(ValueError):
        call("cpu")


@pytest.mark.skipif(not _ext.available(), reason="needs the built extension")
@pytest.mark.parametrize("name,call", refusals(), ids=lambda v: v if isinstance(v, str) else "")
def test_kernels_refuse_before_they_touch_a_device(name, call, monkeypatch):
    """The CUDA kernels' own checks, seen without a GPU: on tensors that only say that they are on one."""
    from types import SimpleNamespace

    from torch._subclasses.fake_tensor import FakeTensorMode

    cuda = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)

    class Kernels:
        def __getattr__(self, op):
            return lambda *a: getattr(torch.ops.dmb, op).default.redispatch(cuda, *a)

    monkeypatch.setattr(model_ops, "torch", SimpleNamespace(ops=SimpleNamespace(dmb=Kernels())))
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(ValueError):
            call("cuda")


def test_indices_outside_their_tables_are_refused():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs()
    for bad in (-1, cos.shape[0]):
        pos = torch.zeros(2, 7, dtype=torch.int64)
        pos[1, 3] = bad
        with pytest.raises(ValueError):
            model_ops.qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
    logits, targets, mask, *_ = token_inputs()
    mask[0, 0], mask[0, 1] = True, False
    targets[0, 1] = -100  # does not count
    model_ops.token_logprobs(logits, targets, mask=mask)
    for bad in (-1, 33):
        targets[0, 0] = bad
        with pytest.raises(ValueError):
            model_ops.token_logprobs(logits, targets, mask=mask)


def test_schemas_and_fake_kernels():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs()
    logits, targets, mask, old, adv, frozen = token_inputs()
    ops = torch.ops.dmb
    calls = [
        (ops.qk_norm_rope, (q, k, wq, wk, cos, sin, None, 1e-5)),
        (ops.route, (logits[0], 2, None)),
        (ops.token_logprobs, (logits, targets, mask)),
        (ops.policy_loss, (logits, targets, old, adv, frozen, mask, 0.2, 0.2, 0.1)),
        (ops.preference_loss, (logits, targets, frozen, mask, 0.1, 0.0)),
    ]
    for op, args in calls:
        real = op(*args)
        meta = op(*(a.to("meta") if isinstance(a, torch.Tensor) else a for a in args))
        assert [(m.shape, m.dtype) for m in meta] == [(r.shape, r.dtype) for r in real], op


def _all_ops():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs()
    logits, targets, mask, old, adv, frozen = token_inputs()
    ops = torch.ops.dmb
    return [
        (ops.qk_norm_rope.default, (q, k, wq, wk, cos, sin, torch.zeros(2, 7, dtype=torch.int64), 1e-5)),
        (ops.route.default, (logits[0], 2, mask[0])),
        (ops.token_logprobs.default, (logits, targets, mask)),
        (ops.policy_loss.default, (logits, targets, old, adv, frozen, mask, 0.2, 0.2, 0.1)),
        (ops.preference_loss.default, (logits, targets, frozen, mask, 0.1, 0.0)),
    ]


@pytest.mark.parametrize("i", range(5))
def test_opcheck(i):
    op, args = _all_ops()[i]
    args = tuple(a.requires_grad_() if isinstance(a, torch.Tensor) and j == 0 else a for j, a in enumerate(args))
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def test_compiled_on_the_cpu():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs()
    logits, targets, mask, old, adv, frozen = token_inputs()

    def fn(x, q):
        a = model_ops.policy_loss(x, targets, old, adv, ref_logp=frozen, mask=mask, kl_coef=0.1).loss
        b = model_ops.preference_loss(x, targets, frozen, mask=mask).loss
        c = model_ops.route(x[0], 2, mask=mask[0]).balance + model_ops.token_logprobs(x, targets).sum()
        return a + b + c + model_ops.qk_norm_rope(q, k, wq, wk, cos, sin)[0].square().mean()

    want, got = ([t.detach().requires_grad_() for t in (logits, q)] for _ in range(2))
    fn(*want).backward()
    torch.compile(fn, backend="aot_eager", fullgraph=True)(*got).backward()
    for w, g in zip(want, got):
        torch.testing.assert_close(w.grad, g.grad, rtol=1e-5, atol=1e-7)
