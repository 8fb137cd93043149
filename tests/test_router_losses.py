"""The router losses reach the gradient of every step, whatever the trained model is wrapped in."""

import copy
from dataclasses import replace
from functools import partial

import pytest
import torch
from test_train_steps import SMALL, _batch, _near, _sparse
from testkit import run_distributed
from torch import nn
from torch.utils.checkpoint import checkpoint

from dtensor_muon_b200.models.llama import Attention, Block, LlamaConfig, lm_loss
from dtensor_muon_b200.models.mixtral import MixtralConfig, MoEFeedForward, mixtral_preset
from dtensor_muon_b200.train import Trainer, build_llama


def _config(balance_coef=0.5, z_coef=0.1) -> MixtralConfig:
    return mixtral_preset("mixtral-tiny", qk_norm=True, balance_coef=balance_coef, z_coef=z_coef, **SMALL)


def _built(cfg: LlamaConfig, device="cpu", dtype=torch.float32, **kw):
    """A sparse decoder from the builder that also shards: a ``Llama`` with sparse blocks."""
    return build_llama(cfg, torch.device(device), dtype, block_factory=lambda: Block(cfg, ffn=MoEFeedForward(cfg)), **kw)


@pytest.fixture(autouse=True)
def _compiled_anew():
    torch._dynamo.reset()


class _Held(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, tokens):
        return self.inner(tokens)


class _Plain:
    """No module itself, as a data-parallel wrapper of another library may be."""

    def __init__(self, module):
        self.module = module

    def __call__(self, tokens):
        return self.module(tokens)


WRAPPED = {
    "bare": lambda m: m,
    "held": _Held,
    "plain": _Plain,
    "compiled": lambda m: torch.compile(m, backend="eager"),
    "compiled and held": lambda m: _Held(torch.compile(m, backend="eager")),
}


def _seen(model):
    """What each parameter's gradient is at the end of a step's backward pass."""
    seen = {}
    for n, p in model.named_parameters():
        p.register_post_accumulate_grad_hook(lambda q, n=n: seen.__setitem__(n, q.grad.clone()))
    return seen


def _router_gradients(model, tokens):
    """Of the router losses alone, from the layers' own."""
    model(tokens)
    loss = sum(layer.feed_forward.aux for layer in model.layers)
    params = {n: p for n, p in model.named_parameters()}
    grads = torch.autograd.grad(loss, list(params.values()), allow_unused=True)
    return {n: g for n, g in zip(params, grads) if g is not None}


def _take(trainer, step, tokens, targets, mask):
    zero = torch.zeros(tokens.shape, device=tokens.device)
    if step == "policy_step":  # without advantages the objective has no gradient
        return trainer.policy_step(tokens, targets, zero, zero, mask=mask).loss
    if step == "preference_step":  # nor has it where nothing counts
        return trainer.preference_step(tokens, targets, zero, mask=torch.zeros_like(mask)).loss
    return trainer.step(tokens, targets)


@pytest.mark.parametrize("made", ["mixtral", "build_llama"])
@pytest.mark.parametrize("wrapped", WRAPPED)
@pytest.mark.parametrize("step", ["policy_step", "preference_step"])
def test_every_step_adds_them(made, wrapped, step):
    model = _sparse() if made == "mixtral" else _built(_config())
    tokens, targets, mask, _ = _batch()
    want = _router_gradients(model, tokens)
    assert any("router" in n and float(g.norm()) > 1e-3 for n, g in want.items())
    seen = _seen(model)
    _take(Trainer(WRAPPED[wrapped](model), torch.optim.SGD(model.parameters(), lr=0.0)), step, tokens, targets, mask)
    # fp32, the same operations: the objective's zeros are all that differs
    _near({n: seen[n] for n in want}, want, 1e-5)


@pytest.mark.parametrize("wrapped", WRAPPED)
def test_the_language_model_step_adds_them(wrapped):
    model = _built(_config())
    tokens, targets, _, _ = _batch()
    loss = lm_loss(model(tokens), targets) + sum(layer.feed_forward.aux for layer in model.layers)
    loss.backward()
    want = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    out = Trainer(WRAPPED[wrapped](model), None).forward_backward(tokens, targets)
    _near({n: p.grad for n, p in model.named_parameters()}, want, 1e-5)
    assert float(out) < float(loss.detach())  # the objective alone


def test_the_model_says_them():
    model, tokens = _built(_config()), _batch()[0]
    assert model.aux_loss() is None
    model(tokens)
    torch.testing.assert_close(model.aux_loss(), sum(layer.feed_forward.aux for layer in model.layers))
    silent = _built(_config(0.0, 0.0))
    silent(tokens)
    assert silent.aux_loss() is None


@pytest.mark.parametrize("step", ["step", "policy_step", "preference_step"])
def test_no_graph_is_left_after_a_step(step):
    model = _sparse()
    tokens, targets, mask, _ = _batch()
    model(tokens)
    want = model.aux_loss().detach()
    trainer = Trainer(model, torch.optim.SGD(model.parameters(), lr=0.0))
    _take(trainer, step, tokens, targets, mask)
    aux = [layer.feed_forward.aux for layer in model.layers]
    assert all(a is not None and a.grad_fn is None and not a.requires_grad for a in aux)
    torch.testing.assert_close(model.aux_loss(), want)  # the value can be logged
    model(tokens)
    with pytest.raises(ZeroDivisionError):  # nor after one that fails
        trainer._backward(_Broken.apply(torch.zeros((), requires_grad=True)))
    assert all(layer.feed_forward.aux.grad_fn is None for layer in model.layers)


def _checkpointed(model, reentrant):
    for layer in model.layers:
        layer.forward = partial(checkpoint, layer.forward, use_reentrant=reentrant)
    return model


@pytest.mark.parametrize("step", ["step", "policy_step", "preference_step"])
def test_checkpointed_layers(step):
    model = _sparse()
    tokens, targets, mask, _ = _batch()
    want = _router_gradients(model, tokens)
    trainer = Trainer(_checkpointed(model, False), torch.optim.SGD(model.parameters(), lr=0.0))
    if step != "step":
        seen = _seen(model)
        _take(trainer, step, tokens, targets, mask)
        _near({n: seen[n] for n in want}, want, 1e-5)
    else:
        trainer.step(tokens, targets)
    assert all(layer.feed_forward.aux.grad_fn is None for layer in model.layers)
    # a reentrant one's forward has no gradients: the losses would be lost
    model = _sparse()
    trainer = Trainer(_checkpointed(model, True), torch.optim.SGD(model.parameters(), lr=0.0))
    with pytest.raises(RuntimeError, match="use_reentrant=False"):
        _take(trainer, step, tokens, targets, mask)
    assert all(p.grad is None for p in model.parameters())
    # nothing is lost where nothing is asked for, or where the layers are frozen
    model = _built(_config(0.0, 0.0))
    _take(Trainer(_checkpointed(model, True), torch.optim.SGD(model.parameters(), lr=0.0)), step, tokens, targets, mask)
    model = _sparse()
    for layer in model.layers:
        layer.feed_forward.requires_grad_(False)
    _take(Trainer(_checkpointed(model, True), torch.optim.SGD(model.parameters(), lr=0.0)), step, tokens, targets, mask)


def test_a_model_whose_layers_never_ran_is_refused():
    """As a wrapper that trains a copy: the trained model's layers leave nothing."""
    model = _sparse()
    wrapper = _Held(copy.deepcopy(model))
    wrapper.forward = copy.deepcopy(model).forward
    tokens, targets, _, _ = _batch()
    with pytest.raises(RuntimeError, match="router losses"):
        Trainer(wrapper, None).forward_backward(tokens, targets)


def test_a_coefficient_may_change():
    model = _sparse()
    tokens, targets, mask, _ = _batch()
    trainer = Trainer(model, torch.optim.SGD(model.parameters(), lr=0.0))
    trainer.step(tokens, targets)
    for layer in model.layers:
        layer.feed_forward.balance_coef = layer.feed_forward.z_coef = 0.0
    seen = _seen(model)
    _take(trainer, "preference_step", tokens, targets, mask)
    assert model.aux_loss() is None and not any(g.any() for g in seen.values())


def test_modules_saved_whole_before_the_options():
    """Their state has no head norms and no coefficients."""
    model = _built(_config(0.0, 0.0))
    plain = _built(replace(_config(0.0, 0.0), qk_norm=False))
    plain.load_state_dict(model.state_dict(), strict=False)
    tokens, targets, _, _ = _batch()
    want = plain(tokens)
    for layer in plain.layers:
        state = dict(layer.attention.__dict__)
        for name in ("q_norm", "k_norm"):
            del state[name]
        layer.attention = Attention.__new__(Attention)
        layer.attention.__setstate__(state)
        state = dict(layer.feed_forward.__dict__)
        for name in ("balance_coef", "z_coef", "aux"):
            state.pop(name, None)
        layer.feed_forward = MoEFeedForward.__new__(MoEFeedForward)
        layer.feed_forward.__setstate__(state)
    assert torch.equal(plain(tokens), want) and plain.aux_loss() is None
    Trainer(copy.deepcopy(plain), None).forward_backward(tokens, targets)


class _Broken(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        raise ZeroDivisionError


@pytest.mark.gpu
def test_a_step_is_captured_after_an_eager_one():
    model = _sparse("cuda", torch.bfloat16)
    tokens, targets, _, _ = _batch("cuda")
    trainer = Trainer(model, None)
    eager = trainer.forward_backward(tokens, targets)
    want = {n: p.grad for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = trainer.forward_backward(tokens, targets)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, eager)
    # the same kernels on the same numbers; sums of rows of one token or expert may come in another order
    _near({n: p.grad.float() for n, p in model.named_parameters()}, {n: g.float() for n, g in want.items()}, 2**-8)


@pytest.mark.gpu
@pytest.mark.parametrize("step", ["policy_step", "preference_step"])
def test_a_compiled_model_gpu(step):
    model = _built(_config(), "cuda")
    tokens, targets, mask, _ = _batch("cuda")
    want = _router_gradients(model, tokens)
    seen = _seen(model)
    trainer = Trainer(torch.compile(model, backend="aot_eager"), torch.optim.SGD(model.parameters(), lr=0.0))
    for _ in range(2):
        _take(trainer, step, tokens, targets, mask)
        # fp32; sums over tokens may come in another order
        _near({n: seen[n] for n in want}, want, 1e-5)


def test_other_callables_are_trained_as_they_are():
    """A function has no layers to look through, and a foreign model's own ``aux_loss`` is not ours to call."""
    model = nn.Sequential(nn.Embedding(512, 8), nn.Linear(8, 512))
    model.aux_loss = lambda: pytest.fail("called")
    tokens, targets, _, _ = _batch()
    for m in (model, lambda t: model(t)):
        model.zero_grad()
        Trainer(m, None).forward_backward(tokens, targets)
        assert all(p.grad.any() for p in model.parameters())


def _sharded(rank, world, reshard):
    from torch.distributed.device_mesh import init_device_mesh

    cfg = _config()
    mesh = init_device_mesh("cpu", (world,))
    model = _built(cfg, mesh=mesh, fsdp_comm="nccl", reshard_after_forward=reshard)
    whole = _built(cfg)
    with torch.no_grad():
        for p, q in zip(whole.parameters(), model.parameters()):
            p.copy_(q.full_tensor())
    batches = [torch.randint(0, 512, (2, 18), generator=torch.Generator().manual_seed(r)) for r in range(world)]
    each = [_router_gradients(whole, b[:, :-1]) for b in batches]
    seen = _seen(model)
    tokens, targets = batches[rank][:, :-1], batches[rank][:, 1:]
    _take(Trainer(model, torch.optim.SGD(model.parameters(), lr=0.0)), "policy_step", tokens, targets, None)
    # the ranks' gradients are averaged
    _near({n: seen[n].full_tensor() for n in each[0]}, {n: sum(e[n] for e in each) / world for n in each[0]}, 1e-5)


@pytest.mark.parametrize("reshard", [False, True])
def test_a_sharded_decoder(reshard):
    run_distributed(_sharded, 2, args=(reshard,), backend="gloo", device_type="cpu", timeout_s=120)
