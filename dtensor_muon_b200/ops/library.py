"""``torch.library`` registrations of the native kernels (namespace ``dmb``).

Registering the kernels as custom ops makes them visible to ``torch.compile``
and other tracers. A region that calls them traces as one graph: the fake
kernels give output shapes, and the autograd formulas are registered with the
ops. Each op has a CUDA kernel (the sm_100a extension) and a CPU kernel (the
PyTorch composition of the same math). The CPU kernel is the fallback and the
oracle.

Ops:

* ``dmb::rope(x, cos, sin, sign)``: rotates interleaved pairs of the last dim
  of ``x`` [B, S, H, D] by ``sign * angle``.
* ``dmb::swiglu(a, b)`` and ``dmb::swiglu_backward(a, b, g)``.
* ``dmb::cross_entropy(logits, targets) -> (mean loss, lse)`` and
  ``dmb::cross_entropy_backward``.
* ``dmb::qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)``:
  RMS norm of every query and key head with the rotation.
* ``dmb::route(logits, top_k, mask) -> (gates, experts, counts, balance, z)``.
* ``dmb::token_logprobs(logits, targets, mask) -> (logp, stats)``,
  ``dmb::policy_loss`` and ``dmb::preference_loss``; all three share
  ``dmb::token_logprobs_backward``.
* ``dmb::gram(x)``: ``x @ x.mT`` over the last two dims, in bf16.
* ``dmb::zeropower(x, steps, strategy, eps)``: orthogonalises the last two
  dims (Newton-Schulz or Polar Express), in bf16.

The reference compiles its update math with ``torch.compile``
(``src/muonium/optim/optim.py:224-229``). Its Triton Gram kernel
(``src/muonium/kernels/gram.py:109-165``) is the op that ``dmb::gram`` stands
in for.

The CUDA kernels and gradients of ``qk_norm_rope``, ``route``,
``token_logprobs`` and the two losses are registered by the extension itself
(``csrc/train_ops.cpp``), which saves most of a small call's host time. Here
are their schemas, their fake kernels and, for the CPU, the differentiable
composition of the same math.
"""

from __future__ import annotations

import importlib.util

import torch
import torch.nn.functional as F
from torch import Tensor
from torch._subclasses.fake_tensor import FakeTensor

from . import _ext

# ---------------------------------------------------------------- rope


@torch.library.custom_op("dmb::rope", mutates_args=(), device_types="cuda")
def rope(x: Tensor, cos: Tensor, sin: Tensor, sign: float) -> Tensor:
    return _ext.load().rope(x.contiguous(), cos.contiguous(), sin.contiguous(), sign)


@rope.register_kernel("cpu")
def _rope_cpu(x: Tensor, cos: Tensor, sin: Tensor, sign: float) -> Tensor:
    xf = x.float().unflatten(-1, (-1, 2))
    x0, x1 = xf[..., 0], xf[..., 1]
    c = cos[None, : x.shape[1], None, :].float()
    s = sign * sin[None, : x.shape[1], None, :].float()
    return torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2).to(x.dtype)


@rope.register_fake
def _rope_fake(x, cos, sin, sign):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _rope_setup(ctx, inputs, output):
    _, cos, sin, sign = inputs
    ctx.save_for_backward(cos, sin)
    ctx.sign = sign


def _rope_backward(ctx, g):
    cos, sin = ctx.saved_tensors
    # the inverse of a rotation is the rotation by the negated angle
    return rope(g, cos, sin, -ctx.sign), None, None, None


rope.register_autograd(_rope_backward, setup_context=_rope_setup)

# ---------------------------------------------------------------- swiglu


@torch.library.custom_op("dmb::swiglu", mutates_args=(), device_types="cuda")
def swiglu(a: Tensor, b: Tensor) -> Tensor:
    return _ext.load().swiglu_fwd(a.contiguous(), b.contiguous())


@swiglu.register_kernel("cpu")
def _swiglu_cpu(a: Tensor, b: Tensor) -> Tensor:
    return (F.silu(a.float()) * b.float()).to(a.dtype)


@swiglu.register_fake
def _swiglu_fake(a, b):
    return torch.empty_like(a, memory_format=torch.contiguous_format)


@torch.library.custom_op("dmb::swiglu_backward", mutates_args=(), device_types="cuda")
def swiglu_backward(a: Tensor, b: Tensor, g: Tensor) -> tuple[Tensor, Tensor]:
    da, db = _ext.load().swiglu_bwd(a.contiguous(), b.contiguous(), g.contiguous())
    return da, db


@swiglu_backward.register_kernel("cpu")
def _swiglu_backward_cpu(a: Tensor, b: Tensor, g: Tensor) -> tuple[Tensor, Tensor]:
    af, bf, gf = a.float(), b.float(), g.float()
    sig = torch.sigmoid(af)
    da = gf * bf * sig * (1 + af * (1 - sig))
    db = gf * af * sig
    return da.to(a.dtype), db.to(b.dtype)


@swiglu_backward.register_fake
def _swiglu_backward_fake(a, b, g):
    return (torch.empty_like(a, memory_format=torch.contiguous_format),
            torch.empty_like(b, memory_format=torch.contiguous_format))


def _swiglu_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _swiglu_grad(ctx, g):
    a, b = ctx.saved_tensors
    return swiglu_backward(a, b, g)


swiglu.register_autograd(_swiglu_grad, setup_context=_swiglu_setup)

# ---------------------------------------------------------------- cross entropy


@torch.library.custom_op("dmb::cross_entropy", mutates_args=(), device_types="cuda")
def cross_entropy(logits: Tensor, targets: Tensor) -> tuple[Tensor, Tensor]:
    """Mean cross entropy of ``logits`` [T, V] against ``targets`` [T]; also returns the row log-sum-exp."""
    rows, lse = _ext.load().cross_entropy_fwd(logits.contiguous(), targets.contiguous())
    return rows.mean(), lse


@cross_entropy.register_kernel("cpu")
def _cross_entropy_cpu(logits: Tensor, targets: Tensor) -> tuple[Tensor, Tensor]:
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    rows = lse - lf.gather(-1, targets[:, None]).squeeze(-1)
    return rows.mean(), lse


@cross_entropy.register_fake
def _cross_entropy_fake(logits, targets):
    return logits.new_empty((), dtype=torch.float32), logits.new_empty(logits.shape[:1], dtype=torch.float32)


@torch.library.custom_op("dmb::cross_entropy_backward", mutates_args=(), device_types="cuda")
def cross_entropy_backward(logits: Tensor, targets: Tensor, lse: Tensor, g: Tensor) -> Tensor:
    """d(mean loss)/d(logits) times the upstream scalar ``g`` (read on the device: no host sync)."""
    gs = g.reshape(1).to(torch.float32).contiguous()
    return _ext.load().cross_entropy_bwd(logits.contiguous(), targets.contiguous(), lse, 1.0 / logits.shape[0], gs)


@cross_entropy_backward.register_kernel("cpu")
def _cross_entropy_backward_cpu(logits: Tensor, targets: Tensor, lse: Tensor, g: Tensor) -> Tensor:
    p = torch.exp(logits.float() - lse[:, None])
    p[torch.arange(logits.shape[0]), targets] -= 1.0
    return (p * (g.float() / logits.shape[0])).to(logits.dtype)


@cross_entropy_backward.register_fake
def _cross_entropy_backward_fake(logits, targets, lse, g):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _ce_setup(ctx, inputs, output):
    logits, targets = inputs
    ctx.save_for_backward(logits, targets, output[1])


def _ce_grad(ctx, g_loss, g_lse):
    logits, targets, lse = ctx.saved_tensors
    return cross_entropy_backward(logits, targets, lse, g_loss), None


cross_entropy.register_autograd(_ce_grad, setup_context=_ce_setup)

# ---------------------------------------------------------------- operators registered by the extension

_LIB = torch.library.Library("dmb", "FRAGMENT")


def _define(schema: str, fake, cpu=None) -> None:
    name = schema.split("(")[0]
    _LIB.define(schema)
    torch.library.register_fake(f"dmb::{name}", fake, lib=_LIB)
    if cpu is not None:  # one composition serves both keys: autograd follows its torch calls
        _LIB.impl(name, cpu, "CPU")
        _LIB.impl(name, cpu, "AutogradCPU")


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _has_values(x: Tensor) -> bool:
    """Whether ``x``'s values can be looked at: a tracer's tensors have none."""
    return not (torch.compiler.is_compiling() or isinstance(x, FakeTensor) or x.is_meta)


def _require_all(ok: Tensor, message: str) -> None:
    # within torch.func.vmap a value of its own for each sample: all of them are looked at
    while torch._C._functorch.is_functorch_wrapped_tensor(ok):
        ok = torch._C._functorch.get_unwrapped(ok)
    _require(bool(ok.all()), message)


def _wide(x: Tensor) -> Tensor:
    return x if x.dtype == torch.float64 else x.float()


def _like(x: Tensor) -> Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def qk_norm_rope_composition(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor,
                             positions: Tensor | None, eps: float) -> tuple[Tensor, Tensor]:
    _require(q.dim() == 4 and k.dim() == 4 and q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3],
             "q, k: [batch, seq, heads, head_dim] of one batch, seq and head_dim expected")
    _require(q.dtype == k.dtype and q.is_floating_point(), "q, k: one floating dtype expected")
    d = q.shape[3]
    _require(d % 2 == 0 and d > 0, f"head_dim: an even number expected, got {d}")
    for w in (q_weight, k_weight):
        _require(w.shape == (d,) and w.dtype in (q.dtype, torch.float32) and w.dtype == q_weight.dtype,
                 "q_weight, k_weight: [head_dim] in the heads' dtype or both in float32 expected")
    for t in (cos, sin):
        _require(t.dim() == 2 and t.shape == (cos.shape[0], d // 2) and t.is_floating_point()
                 and (positions is not None or t.shape[0] >= q.shape[1]),
                 "cos, sin: float32 [positions, head_dim / 2] with a row for every position expected")
    if positions is None:
        c, s = cos[: q.shape[1]][None, :, None], sin[: q.shape[1]][None, :, None]
    else:
        _require(positions.dtype in (torch.int64, torch.int32) and positions.shape == q.shape[:2],
                 "positions: int64 or int32 [batch, seq] expected")
        if _has_values(positions):
            _require_all((positions >= 0) & (positions < cos.shape[0]), "positions: a row of cos and sin expected")
        c, s = cos[positions.long()][:, :, None], sin[positions.long()][:, :, None]
    c, s = c.detach(), s.detach()

    def one(x, w):
        xf = _wide(x)
        n = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps) * w.to(xf.dtype)
        a, b = n[..., 0::2], n[..., 1::2]
        return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2).to(x.dtype)

    return one(q, q_weight), one(k, k_weight)


_define("qk_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, Tensor sin, Tensor? positions, "
        "float eps) -> (Tensor, Tensor)",
        lambda q, k, qw, kw, cos, sin, positions, eps: (_like(q), _like(k)), qk_norm_rope_composition)
_define("qk_norm_rope_backward(Tensor dq, Tensor dk, Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, "
        "Tensor sin, Tensor? positions, float eps, bool weight_grads) -> (Tensor, Tensor, Tensor, Tensor)",
        lambda dq, dk, q, k, qw, kw, cos, sin, positions, eps, weight_grads: (
            _like(q), _like(k), qw.new_empty(qw.shape if weight_grads else (0,)),
            kw.new_empty(kw.shape if weight_grads else (0,))))


def route_composition(logits: Tensor, top_k: int, mask: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    _require(logits.dim() == 2 and logits.is_floating_point() and logits.shape[1] >= 1,
             "logits: floating [tokens, experts] expected")
    t, e = logits.shape
    _require(1 <= top_k <= e, f"top_k from 1 to {e} expected, got {top_k}")
    if mask is None:
        valid = torch.ones(t, dtype=torch.bool, device=logits.device)
    else:
        _require(mask.dtype == torch.bool and mask.shape == (t,), "mask: bool [tokens] on the logits' device expected")
        valid = mask
    experts = torch.sort(logits.detach(), dim=1, descending=True, stable=True).indices[:, :top_k].contiguous()
    # tokens that do not count keep their choice and give nothing else, whatever their logits are
    x = torch.where(valid[:, None], _wide(logits), torch.zeros((), device=logits.device, dtype=_wide(logits).dtype))
    gates = torch.softmax(x.gather(1, experts), dim=1) * valid[:, None]
    chosen = torch.zeros(t, e, dtype=torch.int64, device=logits.device).scatter(1, experts, 1)
    counts = (chosen * valid[:, None]).sum(0)
    n = valid.sum().clamp(min=1).to(x.dtype)
    share = counts.to(x.dtype) / (n * top_k)
    balance = e * (share * (torch.softmax(x, dim=1) * valid[:, None]).sum(0) / n).sum()
    # not logsumexp, whose gradient is exp(x - lse): of large logits the rounded lse is off by more than the gradient may be
    m = x.detach().amax(1, keepdim=True)
    m = torch.where(m == -torch.inf, torch.zeros_like(m), m)
    lse = m[:, 0] + torch.log(torch.exp(x - m).sum(1))
    z = (lse * lse * valid).sum() / n
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    return gates.to(logits.dtype), experts, counts, balance.to(wide), z.to(wide)


def _route_fake(logits, top_k, mask):
    t, e = logits.shape
    scalar = logits.new_empty((), dtype=torch.float32)
    return (logits.new_empty(t, top_k), logits.new_empty(t, top_k, dtype=torch.int64),
            logits.new_empty(e, dtype=torch.int64), scalar, torch.empty_like(scalar))


_define("route(Tensor logits, int top_k, Tensor? mask) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", _route_fake,
        route_composition)
_define("route_backward(Tensor? dgates, Tensor? dbalance, Tensor? dz, Tensor logits, Tensor experts, Tensor counts, "
        "Tensor? mask) -> Tensor",
        lambda dgates, dbalance, dz, logits, experts, counts, mask: _like(logits))


def _check_tokens(logits: Tensor, targets: Tensor, mask: Tensor | None) -> None:
    _require(logits.dim() >= 2 and logits.is_floating_point() and logits.shape[-1] > 0,
             "logits: floating [..., vocab] with a vocabulary expected")
    _require(targets.dtype == torch.int64 and targets.shape == logits.shape[:-1],
             "targets: int64 tensor of the logits' leading shape on their device expected")
    if mask is not None:
        _require(mask.dtype == torch.bool and mask.shape == targets.shape,
                 "mask: bool tensor of the targets' shape on their device expected")
    if _has_values(targets):
        inside = (targets >= 0) & (targets < logits.shape[-1])
        _require_all(inside if mask is None else inside | ~mask, "targets: a row of the vocabulary expected")


def _row_values(v: Tensor, targets: Tensor, name: str) -> Tensor:
    _require(v.dtype in (torch.float32, torch.float64) and v.shape == targets.shape,
             f"{name}: float32 tensor of the targets' shape on their device expected")
    return v.detach()


def _logprobs(logits: Tensor, targets: Tensor, mask: Tensor | None) -> tuple[Tensor, Tensor]:
    _check_tokens(logits, targets, mask)
    x = _wide(logits)
    if mask is not None:  # rows that do not count are not read
        x = torch.where(mask[..., None], x, torch.zeros((), device=x.device, dtype=x.dtype))
        targets = torch.where(mask, targets, torch.zeros_like(targets))
    m = x.detach().amax(-1) if x.numel() else x.new_zeros(targets.shape)
    m = torch.where(m == -torch.inf, torch.zeros_like(m), m)
    s = torch.exp(x - m[..., None]).sum(-1)
    logp = (x.gather(-1, targets[..., None])[..., 0] - m) - torch.log(s)
    if mask is not None:
        logp = torch.where(mask, logp, torch.zeros_like(logp))
    return logp, torch.stack((m, s.detach()), -1).reshape(-1, 2)


def token_logprobs_composition(logits: Tensor, targets: Tensor, mask: Tensor | None) -> tuple[Tensor, Tensor]:
    return _logprobs(logits, targets, mask)


def policy_loss_composition(logits: Tensor, targets: Tensor, old_logp: Tensor, advantages: Tensor, ref_logp: Tensor | None,
                            mask: Tensor | None, clip_low: float, clip_high: float,
                            kl_coef: float) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    _require(0 <= clip_low <= 1 and clip_high >= 0,
             f"clip_low in [0, 1] and clip_high >= 0 expected, got {clip_low} and {clip_high}")
    _require(kl_coef == 0 or ref_logp is not None, "kl_coef needs ref_logp")
    logp, stats = _logprobs(logits, targets, mask)
    valid = torch.ones_like(targets, dtype=torch.bool) if mask is None else mask
    # 64 bits from here on, as the kernel has it: a ratio of 32 bits is infinite from exp(89) on
    new, t = logp.double(), logp.dtype
    zero = torch.zeros((), device=logp.device, dtype=new.dtype)
    n = valid.sum().clamp(min=1)
    gap = torch.where(valid, new - _row_values(old_logp, targets, "old_logp"), zero)
    adv = torch.where(valid, _row_values(advantages, targets, "advantages").double(), zero)
    ratio = torch.exp(gap.detach())
    held = ratio.clamp(1 - clip_low, 1 + clip_high) * adv
    clipped = ratio * adv > held
    # a clipped token has no gradient, however large its ratio: its exponential is not one that is differentiated
    free = torch.exp(torch.where(clipped, zero, gap)) * adv
    rows = -torch.where(clipped, held, free)
    coef = torch.where(clipped, zero, -free).detach()
    kl = zero
    if ref_logp is not None:
        d = torch.where(valid, _row_values(ref_logp, targets, "ref_logp") - new, zero)
        k3 = torch.expm1(d) - d
        kl = k3.detach().sum() / n
        if kl_coef != 0:
            rows = rows + kl_coef * k3
            coef = coef - kl_coef * torch.expm1(d.detach())
    return ((rows.sum() / n).to(t), logp.detach().clone(), kl.to(t, copy=True), (clipped.sum() / n).to(t), stats,
            (coef / n).to(t))


def preference_loss_composition(logits: Tensor, targets: Tensor, ref_logp: Tensor, mask: Tensor | None, beta: float,
                                label_smoothing: float) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    _require(targets.dim() == 2 and targets.shape[0] > 0 and targets.shape[0] % 2 == 0,
             "targets: [2 * pairs, seq] expected, the chosen sequences in front of the rejected ones")
    _require(beta > 0 and 0 <= label_smoothing < 0.5,
             f"beta > 0 and label_smoothing in [0, 0.5) expected, got {beta} and {label_smoothing}")
    logp, stats = _logprobs(logits, targets, mask)
    diff = logp - _row_values(ref_logp, targets, "ref_logp")
    if mask is not None:
        diff = torch.where(mask, diff, torch.zeros_like(diff))
    ratios = diff.double().sum(-1)
    pairs = ratios.shape[0] // 2
    h = beta * (ratios[:pairs] - ratios[pairs:])
    e = label_smoothing
    loss = -((1 - e) * F.logsigmoid(h) + e * F.logsigmoid(-h)).mean()
    dh = (beta / pairs * (e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h))).detach()
    t = logp.dtype
    return (loss.to(t), logp.detach().clone(), (beta * ratios.detach()).to(t), stats, torch.cat([dh, -dh]).to(t))


def _rows_fake(logits, targets):
    row = logits.new_empty(targets.shape, dtype=torch.float32)
    return row, logits.new_empty((targets.numel(), 2), dtype=torch.float32), logits.new_empty((), dtype=torch.float32)


def _token_logprobs_fake(logits, targets, mask):
    return _rows_fake(logits, targets)[:2]


def _policy_fake(logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef):
    row, stats, scalar = _rows_fake(logits, targets)
    return scalar, row, torch.empty_like(scalar), torch.empty_like(scalar), stats, torch.empty_like(row)


def _preference_fake(logits, targets, ref_logp, mask, beta, label_smoothing):
    row, stats, scalar = _rows_fake(logits, targets)
    seqs = logits.new_empty(targets.shape[:1], dtype=torch.float32)
    return scalar, row, seqs, stats, torch.empty_like(seqs)


_define("token_logprobs(Tensor logits, Tensor targets, Tensor? mask) -> (Tensor, Tensor)", _token_logprobs_fake,
        token_logprobs_composition)
_define("token_logprobs_backward(Tensor coef, Tensor? scale, Tensor logits, Tensor targets, Tensor stats, Tensor? mask) "
        "-> Tensor", lambda coef, scale, logits, targets, stats, mask: _like(logits))
_define("policy_loss(Tensor logits, Tensor targets, Tensor old_logp, Tensor advantages, Tensor? ref_logp, Tensor? mask, "
        "float clip_low, float clip_high, float kl_coef) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        _policy_fake, policy_loss_composition)
_define("preference_loss(Tensor logits, Tensor targets, Tensor ref_logp, Tensor? mask, float beta, float label_smoothing) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)", _preference_fake, preference_loss_composition)

# ---------------------------------------------------------------- orthogonalisation


@torch.library.custom_op("dmb::gram", mutates_args=(), device_types="cuda")
def gram(x: Tensor) -> Tensor:
    from .ortho import gram as native_gram

    return native_gram(x.bfloat16())


@gram.register_kernel("cpu")
def _gram_cpu(x: Tensor) -> Tensor:
    xf = x.float()
    return (xf @ xf.mT).bfloat16()


@gram.register_fake
def _gram_fake(x):
    return x.new_empty((*x.shape[:-1], x.shape[-2]), dtype=torch.bfloat16)


@torch.library.custom_op("dmb::zeropower", mutates_args=(), device_types="cuda")
def zeropower(x: Tensor, steps: int, strategy: str, eps: float) -> Tensor:
    from ..orthogonalize.orthogonalize import orthogonalize_local

    return orthogonalize_local(x, steps, eps, strategy, use_native=True).clone()


@zeropower.register_kernel("cpu")
def _zeropower_cpu(x: Tensor, steps: int, strategy: str, eps: float) -> Tensor:
    from ..orthogonalize.orthogonalize import orthogonalize_local

    return orthogonalize_local(x, steps, eps, strategy, use_native=False).clone()


@zeropower.register_fake
def _zeropower_fake(x, steps, strategy, eps):
    return x.new_empty(x.shape, dtype=torch.bfloat16)


# The extension registers the CUDA kernels of the operators above when it is loaded: torch.ops.dmb has to find them whoever
# calls it first (an exported program, say, which no longer goes through ops.model_ops).
if importlib.util.find_spec("dtensor_muon_b200._C") is not None:
    _ext.available()


__all__ = ["cross_entropy", "cross_entropy_backward", "gram", "rope", "swiglu", "swiglu_backward", "zeropower"]
