"""Training harness: model construction (optionally FSDP2-sharded), the Muon +
AdamW optimizer split, synthetic data and one training step.

This is the public entry point a user calls to train with the framework:

    model = build_llama(preset("llama3-8b"), device)
    opt = build_optimizer(model)
    trainer = Trainer(model, opt)
    loss = trainer.step(tokens, targets)

``Trainer.policy_step`` and ``Trainer.preference_step`` train on sampled answers
or on pairs of answers instead, with the log-probabilities that
``Trainer.score`` gave of an earlier or a frozen model.
"""

from __future__ import annotations

import torch
import torch.distributed as dist
from torch import Tensor, nn

from .models.llama import Llama, LlamaConfig, aux_layers, detach_aux, lm_loss, muon_and_adam_params
from .ops import model_ops
from .ops.model_ops import PolicyLoss, PreferenceLoss
from .optim import Muon


def build_llama(
    cfg: LlamaConfig,
    device: torch.device,
    dtype: torch.dtype = torch.bfloat16,
    mesh=None,
    seed: int | None = 0,
    block_factory=None,
    reshard_after_forward: bool = False,
    fsdp_comm: str = "p2p",
    fused_gather: bool | str = False,
) -> Llama:
    """Build a randomly initialised Llama on ``device`` without a host copy.

    With ``mesh`` (a 1-D DeviceMesh) every decoder block and the root are
    wrapped with FSDP2 ``fully_shard`` (dim-0 sharding of every parameter).
    ``reshard_after_forward=False`` (default) keeps each block's gathered
    weights until its backward: with 180 GB of HBM per GPU the extra bf16 copy
    of an 8B model (16 GB) is cheap, and it removes the backward re-gather.
    ``fsdp_comm="p2p"`` runs FSDP's all-gather / reduce-scatter on the NVLink
    peer-memory kernels of :mod:`dtensor_muon_b200.parallel.fsdp_comm`;
    ``"nccl"`` keeps FSDP2's NCCL collectives.
    ``fused_gather=True`` (with ``mesh``) takes the q/k/v and gate/up weights out
    of FSDP: they become ``Shard(0)`` DTensors applied by the fused parameter
    all-gather + GEMM kernel (:class:`dtensor_muon_b200.parallel.ag_gemm.GatherLinear`),
    whose gather runs inside the GEMM instead of ahead of it; ``fused_gather="all"``
    does the same for wo and w2 (only the norms stay in FSDP2).
    """
    with torch.device("meta"):
        model = Llama(cfg, block_factory=block_factory).to(dtype)
    if mesh is not None:
        from torch.distributed.fsdp import fully_shard

        ignored: set = set()
        if fused_gather:
            from .parallel.ag_gemm import GatherLinear

            world = mesh.size()

            def make(linears):
                # groups the kernel's layout rules exclude stay on FSDP2
                if not GatherLinear.eligible(linears, world):
                    return None
                g = GatherLinear(linears, mesh)
                ignored.update(g.params)
                return g

            for layer in model.layers:
                att, ffn = layer.attention, layer.feed_forward
                att.gather = make([att.wq, att.wk, att.wv])
                if fused_gather == "all":
                    att.gather_out = make([att.wo])
                if hasattr(ffn, "w1") and hasattr(ffn, "w3"):
                    ffn.gather = make([ffn.w1, ffn.w3])
                    if fused_gather == "all" and ffn.gather is not None:
                        ffn.gather_out = make([ffn.w2])
        kw = dict(ignored_params=ignored) if ignored else {}
        for layer in model.layers:
            fully_shard(layer, mesh=mesh, reshard_after_forward=reshard_after_forward, **kw)
        fully_shard(model, mesh=mesh, reshard_after_forward=reshard_after_forward, **kw)
        # Issue each block's parameter all-gather two blocks ahead of its forward.
        layers = list(model.layers)
        for i, layer in enumerate(layers):
            nxt = layers[i + 1 : i + 3]
            if nxt:
                layer.set_modules_to_forward_prefetch(nxt)
        if fsdp_comm == "p2p" and mesh.size() > 1:
            from .parallel.fsdp_comm import use_p2p_collectives

            use_p2p_collectives(model)
    model.to_empty(device=device)
    if seed is not None:
        torch.manual_seed(seed + (dist.get_rank() if dist.is_initialized() else 0))
    model.init_weights()
    return model


def build_optimizer(model: nn.Module, optimizer_cls=Muon, lr: float = 1e-3, wd: float = 0.1,
                    adam_lr: float | None = None, muon_group: dict | None = None, fuse_momentum: bool = False,
                    **kwargs):
    """Muon on the 2-D / 3-D decoder weights, AdamW on embeddings, norms and head.

    ``fuse_momentum=True`` (FSDP models on the P2P collectives) moves the Muon
    momentum / Nesterov update into FSDP's gradient reduce-scatter, so it runs
    during backward; requires one backward per optimizer step.
    """
    muon, adam = muon_and_adam_params(model)
    groups = [dict(params=muon, **(muon_group or {}))]
    if adam:
        g = {"params": adam, "algorithm": "adamw"}
        if adam_lr is not None:
            g["lr"] = adam_lr
        groups.append(g)
    opt = optimizer_cls(groups, lr=lr, wd=wd, **kwargs)
    if fuse_momentum:
        from .parallel.fsdp_comm import use_p2p_collectives

        use_p2p_collectives(model, opt)
    return opt


def synthetic_batch(batch: int, seq: int, vocab: int, generator: torch.Generator | None = None,
                    pin: bool = False) -> tuple[Tensor, Tensor]:
    """Uniform random token ids; targets are the next token."""
    ids = torch.randint(0, vocab, (batch, seq + 1), generator=generator)
    if pin:
        ids = ids.pin_memory()
    return ids[:, :-1], ids[:, 1:]


class Trainer:
    """forward -> loss -> backward -> optimizer.step -> zero_grad.

    Every kind of step adds the router losses of the model's sparse layers
    (where their config asks for them) to what it differentiates, and returns
    the objective without them. The layers are looked for in the model that is
    trained, also inside a compiled or otherwise wrapped one. After a step they
    are values without a graph. Where a forward leaves none with a gradient (a
    reentrant checkpoint around a sparse layer) the step raises.
    """

    def __init__(self, model: nn.Module, optimizer: torch.optim.Optimizer):
        self.model = model
        self.optimizer = optimizer

    def _module(self) -> nn.Module:
        # a wrapper that is no module itself holds its model in ``module``; a function holds none
        model = self.model if isinstance(self.model, nn.Module) else getattr(self.model, "module", None)
        return model if isinstance(model, nn.Module) else nn.Module()

    def _forward(self, tokens: Tensor) -> Tensor:
        for m in aux_layers(self._module()):
            m.aux = None
        return self.model(tokens)

    def _backward(self, loss: Tensor) -> None:
        model = self._module()
        layers = aux_layers(model)
        aux = [m.aux for m in layers if m.aux is not None]
        asked = [m for m in layers if m.aux_asked and any(p.requires_grad for p in m.parameters())]
        if any(m.aux is not None and not m.aux_graph for m in asked) or (asked and not aux):
            raise RuntimeError("the forward left no router losses with a gradient, which balance_coef and z_coef ask for: "
                               "under activation checkpointing, use_reentrant=False keeps them")
        try:
            (loss + torch.stack(aux).sum() if aux else loss).backward()
        finally:
            detach_aux(model)

    def _update(self) -> None:
        self.optimizer.step()
        self.optimizer.zero_grad(set_to_none=True)

    def forward_backward(self, tokens: Tensor, targets: Tensor) -> Tensor:
        loss = lm_loss(self._forward(tokens), targets)
        self._backward(loss)
        return loss.detach()

    def step(self, tokens: Tensor, targets: Tensor) -> Tensor:
        loss = self.forward_backward(tokens, targets)
        self._update()
        return loss

    @torch.no_grad()
    def score(self, tokens: Tensor, targets: Tensor, mask: Tensor | None = None) -> Tensor:
        """fp32 log-probabilities of ``targets`` [B, S] under the model as it is; 0 where ``mask`` is false."""
        return model_ops.token_logprobs(self.model(tokens), targets, mask=mask)

    def policy_step(self, tokens: Tensor, targets: Tensor, old_logp: Tensor, advantages: Tensor,
                    ref_logp: Tensor | None = None, mask: Tensor | None = None, clip_low: float = 0.2,
                    clip_high: float = 0.2, kl_coef: float = 0.0) -> PolicyLoss:
        """One clipped policy step on sampled tokens; arguments as :func:`ops.model_ops.policy_loss`."""
        out = model_ops.policy_loss(self._forward(tokens), targets, old_logp, advantages, ref_logp=ref_logp, mask=mask,
                                    clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef)
        self._backward(out.loss)
        self._update()
        return out._replace(loss=out.loss.detach())

    def preference_step(self, tokens: Tensor, targets: Tensor, ref_logp: Tensor, mask: Tensor | None = None,
                        beta: float = 0.1, label_smoothing: float = 0.0) -> PreferenceLoss:
        """One step on pairs of answers, the chosen ones in front of the rejected ones; arguments as
        :func:`ops.model_ops.preference_loss`."""
        out = model_ops.preference_loss(self._forward(tokens), targets, ref_logp, mask=mask, beta=beta,
                                        label_smoothing=label_smoothing)
        self._backward(out.loss)
        self._update()
        return out._replace(loss=out.loss.detach())
