"""The training operators where they are used: normed heads, router losses, and policy and preference steps of a small
sparse decoder, all of it in one run."""

import copy

import pytest
import torch
import torch.nn.functional as F

from dtensor_muon_b200.models.llama import Llama, preset
from dtensor_muon_b200.models.mixtral import Mixtral, MixtralConfig, mixtral_preset
from dtensor_muon_b200.ops import _ext, model_ops
from dtensor_muon_b200.train import Trainer, build_optimizer

SMALL = dict(vocab_size=512, dim=128, n_layers=2, ffn_dim=128)


def _sparse(device="cpu", dtype=torch.float32, **over):
    cfg = mixtral_preset("mixtral-tiny", qk_norm=True, balance_coef=0.02, z_coef=0.003, **SMALL, **over)
    model = Mixtral(cfg)
    model.init_weights(seed=0)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "q_norm" in name or "k_norm" in name:  # their gradient is then not the same for all
                p.copy_(1 + 0.2 * torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))))
    return model.to(device=device, dtype=dtype)


def _batch(device="cpu", b=4, s=17, vocab=512):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, vocab, (b, s + 1), generator=g)
    mask = torch.rand(b, s, generator=g) < 0.7
    adv = torch.randn(b, s, generator=g)
    return [t.to(device) for t in (ids[:, :-1], ids[:, 1:], mask, adv)]


def _by_hand(model, tokens):
    """Logits and router losses from plain torch operations, next to the model's own forward."""
    cfg = model.cfg
    b, s = tokens.shape
    h = model.tok_embeddings(tokens)
    cos, sin = model.rope(s, tokens.device)
    aux = 0.0

    def rotate(x):
        x0, x1 = x[..., 0::2], x[..., 1::2]
        c, sn = cos[:s, None], sin[:s, None]
        return torch.stack((x0 * c - x1 * sn, x0 * sn + x1 * c), -1).flatten(-2)

    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + cfg.norm_eps) * w

    for layer in model.layers:
        a = layer.attention
        x = norm(h, layer.attention_norm.weight)
        q = rotate(norm(a.wq(x).view(b, s, cfg.n_heads, -1), a.q_norm.weight)).transpose(1, 2)
        k = rotate(norm(a.wk(x).view(b, s, cfg.n_kv_heads, -1), a.k_norm.weight)).transpose(1, 2)
        v = a.wv(x).view(b, s, cfg.n_kv_heads, -1).transpose(1, 2)
        h = h + a.wo(F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(b, s, -1))
        m = layer.feed_forward
        x = norm(h, layer.ffn_norm.weight).reshape(b * s, -1)
        logits = m.router(x)
        top, idx = torch.topk(logits, cfg.top_k, dim=-1)
        gate = torch.softmax(top, -1)
        out = torch.zeros_like(x)
        for e in range(cfg.n_experts):
            y = (F.silu(x @ m.w1[e].t()) * (x @ m.w3[e].t())) @ m.w2[e].t()
            out = out + y * (gate * (idx == e)).sum(-1, keepdim=True)
        h = h + out.view(b, s, -1)
        share = F.one_hot(idx, cfg.n_experts).sum((0, 1)).float() / idx.numel()
        balance = cfg.n_experts * (share * torch.softmax(logits, -1).mean(0)).sum()
        aux = aux + cfg.balance_coef * balance + cfg.z_coef * torch.logsumexp(logits, -1).square().mean()
    return model.output(norm(h, model.norm.weight)), aux


def _grads(model, loss):
    model.zero_grad()
    loss.backward()
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


def _near(got, want, rel):
    for n in want:
        scale = want[n].norm()
        assert (got[n].cpu() - want[n].cpu()).norm() <= rel * scale + 1e-9, (n, float((got[n].cpu() - want[n].cpu()).norm() / scale))


def _policy_by_hand(logits, targets, old, adv, frozen, mask):
    logp = torch.log_softmax(logits, -1).gather(-1, targets[..., None])[..., 0]
    ratio = torch.exp(logp - old)
    loss = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.1 * (torch.exp(frozen - logp) - 1 - (frozen - logp))
    return loss[mask].mean()


def _preference_by_hand(logits, targets, frozen, mask):
    logp = torch.log_softmax(logits, -1).gather(-1, targets[..., None])[..., 0]
    s = ((logp - frozen) * mask).sum(-1)
    p = s.shape[0] // 2
    return -F.logsigmoid(0.1 * (s[:p] - s[p:])).mean()


def _run(device):
    """Gradients of both objectives through the whole model: the framework's operators against plain torch on the CPU."""
    model = _sparse(device)
    plain = copy.deepcopy(model).cpu()
    tokens, targets, mask, adv = _batch(device)
    cpu = [t.cpu() for t in (tokens, targets, mask, adv)]
    frozen = Trainer(model, None).score(tokens, targets)
    want = torch.log_softmax(_by_hand(plain, cpu[0])[0], -1).gather(-1, cpu[1][..., None])[..., 0].detach()
    torch.testing.assert_close(frozen.cpu(), want, rtol=1e-4, atol=1e-4)
    g = torch.Generator().manual_seed(5)
    old = want + 0.3 * torch.randn(want.shape, generator=g)
    ref = want + 0.2 * torch.randn(want.shape, generator=g)
    # fp32 throughout: what differs is the order of sums, some hundred roundings of 6e-8 through two layers
    logits, aux = _by_hand(plain, cpu[0])
    expect = _grads(plain, _policy_by_hand(logits, cpu[1], old, cpu[3], ref, cpu[2]) + aux)
    out = model_ops.policy_loss(model(tokens), targets, old.to(device), adv, ref_logp=ref.to(device), mask=mask, kl_coef=0.1)
    _near(_grads(model, out.loss + model.aux_loss()), expect, 1e-4)
    logits, aux = _by_hand(plain, cpu[0])
    expect = _grads(plain, _preference_by_hand(logits, cpu[1], ref, cpu[2]) + aux)
    out = model_ops.preference_loss(model(tokens), targets, ref.to(device), mask=mask)
    _near(_grads(model, out.loss + model.aux_loss()), expect, 1e-4)


def test_gradients_of_a_sparse_decoder():
    _run("cpu")


@pytest.mark.gpu
def test_gradients_of_a_sparse_decoder_gpu():
    n0 = _ext.launch_count
    _run("cuda")
    assert _ext.launch_count > n0
    _ext.check_device_errors("cuda")


def _steps(device, dtype):
    model = _sparse(device, dtype)
    opt = build_optimizer(model, lr=1e-3)
    trainer = Trainer(model, opt)
    tokens, targets, mask, adv = _batch(device)
    frozen = trainer.score(tokens, targets)
    assert frozen.dtype == torch.float32 and not frozen.requires_grad
    before = [p.detach().clone() for p in opt.param_groups[0]["params"]]
    p = trainer.policy_step(tokens, targets, frozen, adv, ref_logp=frozen, mask=mask, kl_coef=0.1)
    assert torch.isfinite(p.loss) and not p.loss.requires_grad
    # scores and step take the same logits: the first step's ratios are all but 1
    assert float(p.clipped) == 0 and float(p.kl) < 1e-4
    torch.testing.assert_close(p.logp[mask], frozen[mask], rtol=1e-5, atol=1e-5)
    q = trainer.preference_step(tokens, targets, frozen, mask=mask)
    assert torch.isfinite(q.loss) and q.rewards.shape == (4,)
    assert torch.isfinite(trainer.step(tokens, targets))
    assert all(not torch.equal(a, b) for a, b in zip(before, opt.param_groups[0]["params"]))
    assert all(p.grad is None for p in model.parameters())


def test_every_step_adds_the_router_losses():
    """With an objective that has no gradient, what is left is theirs."""
    model = _sparse()
    trainer = Trainer(model, torch.optim.SGD(model.parameters(), lr=0.0))
    tokens, targets, mask, adv = _batch()
    model(tokens)
    want = _grads(model, model.aux_loss())
    model.zero_grad()
    seen = {}
    for n, p in model.named_parameters():
        p.register_post_accumulate_grad_hook(lambda q, n=n: seen.__setitem__(n, q.grad.clone()))
    out = trainer.policy_step(tokens, targets, torch.zeros_like(adv), torch.zeros_like(adv), mask=mask)
    assert float(out.loss) == 0
    _near({n: seen[n] for n in want}, want, 1e-5)


def test_trainer_steps():
    _steps("cpu", torch.float32)


@pytest.mark.gpu
def test_trainer_steps_gpu():
    _steps("cuda", torch.bfloat16)
    _ext.check_device_errors("cuda")


def test_models_without_the_options_are_as_they_were():
    cfg = preset("tiny", vocab_size=64, n_layers=1)
    assert not cfg.qk_norm
    by_place = MixtralConfig(512, 128, 2, 4, 4, 128, 1e-5, 1e4, 512, 0.02, 4, 1)
    assert (by_place.n_experts, by_place.top_k) == (4, 1)
    names = {n for n, _ in Llama(cfg).named_parameters()}
    assert not any("q_norm" in n for n in names)
    plain = Mixtral(mixtral_preset("mixtral-tiny", **SMALL))
    plain.init_weights(seed=0)
    asked = Mixtral(mixtral_preset("mixtral-tiny", balance_coef=0.02, **SMALL))
    asked.load_state_dict(plain.state_dict())
    tokens = _batch()[0]
    torch.testing.assert_close(plain(tokens), asked(tokens), rtol=1e-5, atol=1e-6)
    assert plain.aux_loss() is None and asked.aux_loss().requires_grad


def test_a_model_can_be_copied_after_a_step():
    """As for a frozen model to stay near."""
    model = _sparse()
    tokens = _batch()[0]
    out = model(tokens)
    frozen = copy.deepcopy(model)
    assert frozen.aux_loss() is None and model.aux_loss().requires_grad
    assert torch.equal(frozen(tokens), out)


def test_parameter_groups_and_initialisation():
    model = _sparse()
    model.init_weights(seed=1)
    opt = build_optimizer(model)
    adam = {id(p) for p in opt.param_groups[1]["params"]}
    for n, p in model.named_parameters():
        if "q_norm" in n or "k_norm" in n:
            assert id(p) in adam and torch.equal(p, torch.ones_like(p))


def test_normed_heads_refuse_tensor_parallelism():
    from dtensor_muon_b200.parallel.tensor_parallel import apply_tensor_parallel

    class Two:
        def size(self):
            return 2

    with pytest.raises(ValueError, match="qk_norm"):
        apply_tensor_parallel(_sparse(), Two())
