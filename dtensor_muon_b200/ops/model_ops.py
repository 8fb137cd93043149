"""Entry points for the fused decoder-block kernels (``ops/csrc/model_ops.cu``).

``rope``, ``swiglu`` and ``cross_entropy`` run the native kernels, registered
as ``torch.library`` ops with their autograd formulas (``ops/library.py``), for
bf16 CUDA inputs and the equivalent PyTorch composition otherwise (CPU, fp32).

``qk_norm_rope``, ``route``, ``token_logprobs``, ``policy_loss`` and
``preference_loss`` run their native kernels for bf16, fp16 and fp32 CUDA
inputs, and the composition otherwise (CPU, fp64, sizes that a kernel does not
take). On a CUDA device they raise where the extension is not built. Wrong
arguments raise ``ValueError``. A target or position outside its table cannot
be seen from the host without waiting for the device: the CPU raises, and a
kernel makes its results NaN and records an error that
``ops._ext.check_device_errors`` raises. Gradients of gradients are refused.

``torch.func``: ``vmap``, ``grad`` and ``jvp`` go through the composition; of a
kernel ``vmap`` takes the forward, sample by sample, and its gradient raises.

CUDA graphs: both directions can be captured. As for any autograd call,
capture a backward pass only while no eager graph of the same leaves lives.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch import Tensor

from . import _ext, library


def _native(*ts: Tensor) -> bool:
    return all(t.is_cuda and t.dtype == torch.bfloat16 for t in ts) and _ext.available()


def rope_reference(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Rotate interleaved pairs of the last dim of x [B, S, H, D] (fp32 math)."""
    xf = x.float().unflatten(-1, (-1, 2))
    x0, x1 = xf[..., 0], xf[..., 1]
    c = cos[None, : x.shape[1], None, :]
    s = sin[None, : x.shape[1], None, :]
    return torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2).to(x.dtype)


def rope(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    if _native(x) and x.shape[-1] % 8 == 0:
        return library.rope(x, cos, sin, 1.0)
    return rope_reference(x, cos, sin)


def swiglu(a: Tensor, b: Tensor) -> Tensor:
    """silu(a) * b."""
    if _native(a, b) and a.numel() % 8 == 0:
        return library.swiglu(a, b)
    return F.silu(a) * b


def cross_entropy(logits: Tensor, targets: Tensor) -> Tensor:
    """Mean next-token cross entropy; fp32 math, bf16 logits read once per pass on CUDA."""
    flat = logits.reshape(-1, logits.shape[-1])
    t = targets.reshape(-1)
    if _native(flat) and flat.shape[-1] % 8 == 0 and t.dtype == torch.int64:
        return library.cross_entropy(flat, t)[0]
    return F.cross_entropy(flat.float(), t)


_NATIVE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _kernel(x: Tensor) -> bool:
    """Whether ``x`` goes to a native kernel of the extension (which then has to be there) or a traced stand-in of one."""
    if not (x.is_cuda and x.dtype in _NATIVE_DTYPES):
        return False
    _ext.load()
    return True


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor, eps: float = 1e-5,
                 positions: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """RMS norm of every query and key head, times its weight, and the rotation of interleaved pairs: one pass.

    ``q`` [B, S, Hq, D], ``k`` [B, S, Hk, D] (any strides; D a multiple of 8 up to 256 for the kernel), weights [D] in
    the same dtype or fp32, ``cos`` / ``sin`` fp32 [positions, D / 2] as ``models.llama.rope_tables`` makes them. A
    token's position is its place in the sequence, or ``positions`` [B, S] (packed documents, one new token of a longer
    sequence). Computed in fp32, rounded once. Gradients reach q, k and the weights; the tables have none.
    """
    if _kernel(q) and q.dim() == 4 and q.shape[3] % 8 == 0 and q.shape[3] <= 256:
        return torch.ops.dmb.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return library.qk_norm_rope_composition(q, k, q_weight, k_weight, cos, sin, positions, eps)


class Routing(NamedTuple):
    """What :func:`route` returns."""

    gates: Tensor  # [T, k] in the logits' dtype, by rank; 0 for tokens that do not count
    experts: Tensor  # int64 [T, k], by rank
    counts: Tensor  # int64 [E]: choices by the tokens that count
    balance: Tensor  # fp32: E / (N^2 k) sum_e counts_e sum_t p_te; 1 where every expert gets the same
    z: Tensor  # fp32: mean over tokens of logsumexp(logits)^2


def route(logits: Tensor, top_k: int, mask: Tensor | None = None) -> Routing:
    """Top-k routing of a sparse layer with its counts, balance loss and z loss, from router logits [T, E].

    Gates are the softmax over a token's ``top_k`` chosen logits; equal logits go to the lower expert, NaN counts as the
    largest. ``mask`` [T] (bool): tokens that do not count still get experts, but gate 0, no place in the counts or the
    losses, and no gradient. The gradient of ``balance`` goes through the probabilities, not through the counts. Up to
    512 experts and top 32 for the kernel.
    """
    if _kernel(logits) and logits.dim() == 2 and logits.shape[1] <= 512 and top_k <= 32:
        return Routing(*torch.ops.dmb.route(logits, top_k, mask))
    return Routing(*library.route_composition(logits, top_k, mask))


def token_logprobs(logits: Tensor, targets: Tensor, mask: Tensor | None = None) -> Tensor:
    """fp32 log-probabilities of ``targets`` [...] under ``logits`` [..., V]; 0 where ``mask`` (bool [...]) is false.

    The logits may be a view with any leading strides (``logits[:, :-1]`` is not copied). Rows that the mask leaves out
    are not read and get no gradient, whatever they and their targets hold.
    """
    if _kernel(logits):
        return torch.ops.dmb.token_logprobs(logits, targets, mask)[0]
    return library.token_logprobs_composition(logits, targets, mask)[0]


class PolicyLoss(NamedTuple):
    """What :func:`policy_loss` returns; only ``loss`` has a gradient."""

    loss: Tensor  # fp32
    logp: Tensor  # fp32, targets' shape
    kl: Tensor  # fp32: mean of the KL estimate, 0 without ref_logp
    clipped: Tensor  # fp32: share of the tokens whose ratio the clipping holds


def policy_loss(logits: Tensor, targets: Tensor, old_logp: Tensor, advantages: Tensor, ref_logp: Tensor | None = None,
                mask: Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0) -> PolicyLoss:
    """Clipped policy loss from logits [..., V], with a KL term towards a frozen model.

    Mean over the tokens that ``mask`` keeps of ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef *
    (exp(d) - 1 - d)`` with ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp``; 0 where it keeps none.
    ``old_logp``, ``advantages`` and ``ref_logp`` are fp32 of the targets' shape, as :func:`token_logprobs` gives them.

    Where the logits need a gradient, the kernel writes it in the same pass, for a loss gradient of 1, and holds it for
    the backward pass; one of another value (a loss that is divided before ``backward``) is computed anew there.
    """
    args = (logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef)
    if _kernel(logits):
        return PolicyLoss(*torch.ops.dmb.policy_loss(*args)[:4])
    return PolicyLoss(*library.policy_loss_composition(*args)[:4])


class PreferenceLoss(NamedTuple):
    """What :func:`preference_loss` returns; only ``loss`` has a gradient."""

    loss: Tensor  # fp32
    logp: Tensor  # fp32 [2P, S]
    rewards: Tensor  # fp32 [2P]: beta times each sequence's log ratio


def preference_loss(logits: Tensor, targets: Tensor, ref_logp: Tensor, mask: Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0) -> PreferenceLoss:
    """Logistic loss of pairs of answers, from logits [2P, S, V]: P chosen sequences, then their P rejected ones.

    A sequence's log ratio is the sum of ``logp - ref_logp`` over the tokens that ``mask`` [2P, S] keeps (0 for none);
    with ``h = beta * (chosen - rejected)`` the loss is the mean over pairs of ``-((1 - label_smoothing) log sigmoid(h)
    + label_smoothing log sigmoid(-h))``. ``ref_logp`` (fp32 [2P, S]) is :func:`token_logprobs` of the frozen model.
    """
    args = (logits, targets, ref_logp, mask, beta, label_smoothing)
    if _kernel(logits):
        return PreferenceLoss(*torch.ops.dmb.preference_loss(*args)[:3])
    return PreferenceLoss(*library.preference_loss_composition(*args)[:3])
