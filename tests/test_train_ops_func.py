"""The training operators under torch.func's transforms."""

import pytest
import torch
from test_train_ops import qk_inputs, token_inputs
from torch.func import grad, jvp, vmap

from dtensor_muon_b200.ops import model_ops


def _calls():
    """(name, function of one sample, samples): each sample of a stacked call is a call of its own."""
    q, k, wq, wk, cos, sin, _, _ = qk_inputs(b=3)
    pos = torch.randint(0, cos.shape[0], q.shape[:2], generator=torch.Generator().manual_seed(1))
    logits, targets, mask, old, adv, frozen = token_inputs(b=4)
    bad = targets.clone()
    bad[~mask] = -100  # does not count

    def heads(a, b, p=None):
        return model_ops.qk_norm_rope(a[None], b[None], wq.to(a), wk.to(a), cos.to(a.device), sin.to(a.device),
                                      positions=None if p is None else p[None])

    pairs = [t.reshape(2, 2, *t.shape[1:]) for t in (logits, targets, frozen, mask)]
    return [
        ("heads", heads, (q, k)),
        ("heads, positions", heads, (q, k, pos)),
        ("route", lambda a: tuple(model_ops.route(a, 2)), (logits,)),
        ("route, mask", lambda a, m: tuple(model_ops.route(a, 2, mask=m)), (logits, mask)),
        ("log-probabilities", lambda a, y: model_ops.token_logprobs(a, y), (logits, targets)),
        ("log-probabilities, mask", lambda a, y, m: model_ops.token_logprobs(a, y, mask=m), (logits, bad, mask)),
        ("policy", lambda a, y, o, v, f, m: tuple(model_ops.policy_loss(a, y, o, v, ref_logp=f, mask=m, kl_coef=0.1)),
         (logits, targets, old, adv, frozen, mask)),
        ("preference", lambda a, y, f, m: tuple(model_ops.preference_loss(a, y, f, mask=m)), tuple(pairs)),
    ]


CALLS = pytest.mark.parametrize("i", range(len(_calls())), ids=[c[0] for c in _calls()])


def _same(got, want, rtol=1e-6, atol=1e-6):  # a batched sum may be taken in another order: some steps of fp32
    for g, w in zip(*(t if isinstance(t, tuple) else (t,) for t in (got, want))):
        torch.testing.assert_close(g, w, rtol=rtol, atol=atol)


def _one_by_one(fn, samples):
    outs = [fn(*s) for s in zip(*samples)]
    return tuple(torch.stack(o) for o in zip(*outs)) if isinstance(outs[0], tuple) else torch.stack(outs)


@CALLS
def test_vmap(i):
    _, fn, samples = _calls()[i]
    _same(vmap(fn)(*samples), _one_by_one(fn, samples))


def _scalar(fn):
    def value(*args):
        out = fn(*args)
        return sum(o.square().sum() for o in (out if isinstance(out, tuple) else (out,)) if o.is_floating_point())

    return value


@CALLS
def test_gradient_of_each_sample(i):
    _, fn, samples = _calls()[i]
    f = _scalar(fn)
    want = torch.stack([grad(f)(*s) for s in zip(*samples)])
    _same(vmap(grad(f))(*samples), want, 1e-5, 1e-6)
    x = samples[0].clone().requires_grad_()
    total = sum(f(x[j], *(s[j] for s in samples[1:])) for j in range(len(x)))
    _same(want, torch.autograd.grad(total, x)[0], 1e-5, 1e-6)
    _same(grad(lambda a: vmap(f)(a, *samples[1:]).sum())(samples[0]), want, 1e-5, 1e-6)


@CALLS
def test_jvp(i):
    _, fn, samples = _calls()[i]
    f = _scalar(fn)
    args = [s[0] for s in samples]
    direction = torch.randn(args[0].shape, generator=torch.Generator().manual_seed(4))
    _, got = jvp(lambda a: f(a, *args[1:]), (args[0],), (direction,))
    want = (grad(f)(*args) * direction).sum()
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


def test_every_sample_is_checked():
    q, k, wq, wk, cos, sin, _, _ = qk_inputs()
    logits, targets, mask, *_ = token_inputs(b=4)
    targets[2, 1], mask[2, 1] = 33, True
    with pytest.raises(ValueError, match="vocabulary"):
        vmap(lambda a, y: model_ops.token_logprobs(a, y))(logits, targets)
    with pytest.raises(ValueError, match="vocabulary"):
        vmap(lambda a, y, m: model_ops.token_logprobs(a, y, mask=m))(logits, targets, mask)
    mask[2, 1] = False
    vmap(lambda a, y, m: model_ops.token_logprobs(a, y, mask=m))(logits, targets, mask)
    pos = torch.zeros(2, 7, dtype=torch.int64)
    pos[1, 3] = -1
    with pytest.raises(ValueError, match="positions"):
        vmap(lambda p: model_ops.qk_norm_rope(q[:1], k[:1], wq, wk, cos, sin, positions=p[None]))(pos)


@pytest.mark.gpu
@CALLS
def test_vmap_of_the_kernels(i):
    _, fn, samples = _calls()[i]
    samples = [s.cuda() for s in samples]
    _same(vmap(fn)(*samples), _one_by_one(fn, samples))
    with pytest.raises(RuntimeError):  # their gradients are not torch.func's
        vmap(grad(_scalar(fn)))(*samples)
