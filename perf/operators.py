"""Cases of the decoder's training operators: their plain forms in elementary torch operations, and the framework's calls.

Operators (``dtensor_muon_b200.ops.model_ops``):

* ``qk_norm_rope``: RMS norm of every query and key head and the position rotation, in one pass, with its gradient.
* ``route``: top-k gates of a sparse layer's router with the per-expert counts, the balance loss and the z loss, with its gradient.
* ``token_logprobs``: log-probabilities of the target tokens (scoring), with its gradient.
* ``policy_loss``: clipped policy loss with a KL term, with its gradient.
* ``preference_loss``: logistic loss of paired log ratios, with its gradient.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one new token of each of 8 sequences, heads of the 8B preset: latency alone
        dict(name="qk_token", op="qk", batch=8, seq=1, heads=32, kv_heads=8, dim=128, dtype="bf16", theta=500000.0,
             table=4096, positions=True, layout="plain", train=False),
        # one training sequence of the 8B preset
        dict(name="qk_train_8b", op="qk", batch=1, seq=4096, heads=32, kv_heads=8, dim=128, dtype="bf16",
             theta=500000.0, table=4096, positions=False, layout="plain", train=True),
        # packed documents of odd lengths in a fused projection, heads of the 13B preset
        dict(name="qk_packed_fp16", op="qk", batch=3, seq=1363, heads=40, kv_heads=40, dim=128, dtype="fp16",
             theta=10000.0, table=4096, positions=True, layout="fused", train=True),
        # the small sparse preset: 4 experts, two chosen, one short sequence
        dict(name="route_tiny", op="route", tokens=509, experts=4, top_k=2, dtype="bf16", mask=False),
        # four training sequences of the 8-expert preset
        dict(name="route_8", op="route", tokens=16384, experts=8, top_k=2, dtype="bf16", mask=False),
        # many small experts, fp32 router, padded batch
        dict(name="route_many_fp32", op="route", tokens=65535, experts=128, top_k=8, dtype="fp32", mask=True),
        # scoring a batch of answers with a frozen model
        dict(name="logprobs_score", op="logprobs", batch=4, seq=1024, vocab=32000, dtype="bf16", keep=1.0, train=False),
        # a few tokens of the small preset, with the gradient: latency alone
        dict(name="logprobs_tiny", op="logprobs", batch=2, seq=37, vocab=1024, dtype="bf16", keep=0.8, train=True),
        # policy step on one sequence of the 8B preset, the prompt masked
        dict(name="policy_8b", op="policy", batch=1, seq=4096, vocab=128256, dtype="bf16", keep=0.75, kl=0.05),
        # fp32 logits, a vocabulary of odd size, no reference model
        dict(name="policy_odd_fp32", op="policy", batch=5, seq=211, vocab=32001, dtype="fp32", keep=0.6, kl=0.0),
        # two pairs of answers
        dict(name="preference_13b", op="preference", batch=4, seq=1024, vocab=32000, dtype="bf16", keep=0.6,
             smoothing=0.0),
        # one pair of short answers of the small preset
        dict(name="preference_tiny", op="preference", batch=2, seq=129, vocab=1024, dtype="bf16", keep=0.7,
             smoothing=0.1),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("qk", "route", "logprobs", "policy", "preference"))
    if op == "qk":
        heads, kv_heads = rng.choice(((32, 8), (40, 40), (4, 4), (16, 1), (9, 3)))
        batch = spread(1, 16)
        seq = max(1, spread(1, 8192) // batch)
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=rng.choice((64, 96, 128, 256)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), theta=rng.choice((10000.0, 500000.0)),
                    table=max(4096, seq), positions=rng.random() < 0.5, layout=rng.choice(("plain", "fused")),
                    train=rng.random() < 0.7)
    if op == "route":
        experts = rng.choice((4, 8, 8, 16, 60, 64, 128, 256))
        return dict(op=op, tokens=spread(1, 65536), experts=experts, top_k=rng.choice((1, 2, 2, 4, 8)[:3 if experts < 8 else 5]),
                    dtype=rng.choice(("bf16", "bf16", "fp32")), mask=rng.random() < 0.5)
    vocab = rng.choice((1024, 32000, 32001, 128256, spread(1000, 128000)))
    rows = spread(2, min(8192, 400_000_000 // vocab))
    batch = 2 * rng.randint(1, 4) if op == "preference" else rng.randint(1, 8)
    case = dict(op=op, batch=batch, seq=max(1, rows // batch), vocab=vocab, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                keep=round(rng.uniform(0.3, 1.0), 3))
    if op == "logprobs":
        case["train"] = rng.random() < 0.6
    elif op == "policy":
        case["kl"] = rng.choice((0.0, 0.01, 0.1))
    else:
        case["smoothing"] = rng.choice((0.0, 0.0, 0.2))
    return case


# ------------------------------------------------------------------ inputs


def _prepare_qk(c, g):
    t = DTYPES[c["dtype"]]
    b, s, h, hk, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEVICE) * scale

    if c["layout"] == "fused":  # queries, keys and values are slices of one projection
        qkv = normal(b, s, h + 2 * hk, d, scale=1.5).to(t)
        q, k = qkv[:, :, :h], qkv[:, :, h : h + hk]
    else:
        q, k = normal(b, s, h, d, scale=1.5).to(t), normal(b, s, hk, d, scale=1.5).to(t)
    freq = c["theta"] ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
    angle = torch.arange(c["table"], device=DEVICE, dtype=torch.float64)[:, None] * freq
    pos = None
    if c["positions"]:
        if s == 1:  # each sequence is somewhere in its own context
            pos = torch.randint(0, c["table"], (b, 1), generator=g, device=DEVICE)
        else:  # documents packed one behind the other: positions start again at each
            first = torch.rand(b, s, generator=g, device=DEVICE) < 5.0 / s
            at = torch.arange(s, device=DEVICE).expand(b, s)
            pos = at - torch.cummax(torch.where(first, at, torch.zeros_like(at)), dim=1).values
    x = dict(q=q, k=k, wq=(1 + 0.1 * normal(d)).to(t), wk=(1 + 0.1 * normal(d)).to(t))
    state = dict(x, cos=angle.cos().float(), sin=angle.sin().float(), pos=pos, eps=1e-5)
    if c["train"]:
        state.update({n: v.detach().requires_grad_() for n, v in x.items()})
        # attention hands its gradients back with the heads in front of the sequence
        state["dq"], state["dk"] = normal(b, h, s, d).to(t).transpose(1, 2), normal(b, hk, s, d).to(t).transpose(1, 2)
    return state


def _prepare_route(c, g):
    n, e = c["tokens"], c["experts"]
    # router outputs: some experts are liked more than others
    logits = torch.randn(n, e, generator=g, device=DEVICE) + 0.5 * torch.randn(e, generator=g, device=DEVICE)
    logits = logits.to(DTYPES[c["dtype"]]).requires_grad_()
    mask = torch.rand(n, generator=g, device=DEVICE) < 0.8 if c["mask"] else None
    if mask is not None:
        mask[0] = True
    return dict(logits=logits, mask=mask, k=c["top_k"],
                dgates=torch.randn(n, c["top_k"], generator=g, device=DEVICE).to(logits.dtype) * 1e-2,
                dbalance=torch.tensor(0.01, device=DEVICE), dz=torch.tensor(0.001, device=DEVICE))


def _prepare_tokens(c, g):
    b, s, v = c["batch"], c["seq"], c["vocab"]
    logits = torch.randn(b, s, v, generator=g, device=DEVICE) * 2
    targets = torch.randint(0, v, (b, s), generator=g, device=DEVICE)
    # the tokens were drawn from a model much like this one: they are likely ones
    likely = math.log(v) + 2 * torch.randn(b, s, generator=g, device=DEVICE)
    logits.scatter_(2, targets[..., None], likely[..., None])
    logits = logits.to(DTYPES[c["dtype"]])
    # a prompt in front and padding behind do not count
    keep = max(1, round(c["keep"] * s))
    first = torch.randint(0, s - keep + 1, (b, 1), generator=g, device=DEVICE)
    at = torch.arange(s, device=DEVICE)
    mask = (at >= first) & (at < first + keep) if keep < s else None
    state = dict(logits=logits, targets=targets, mask=mask)
    if c["op"] == "logprobs":
        if c["train"]:
            logits.requires_grad_()
            state["dlogp"] = torch.randn(b, s, generator=g, device=DEVICE) / (b * s)
        return state
    x = logits.float()
    logp = x.gather(2, targets[..., None])[..., 0] - torch.logsumexp(x, -1)
    del x
    noise = 0.15 * torch.randn(b, s, generator=g, device=DEVICE)
    # the KL estimate has a double zero where both models agree: no token is left all but on it
    apart = 0.1 * torch.randn(b, s, generator=g, device=DEVICE)
    state["ref"] = logp - apart - torch.where(apart < 0, -0.03, 0.03)
    if c["op"] == "policy":
        # ratios next to a clipping border are moved off it: which side of it a token is on must not hang on rounding
        border = torch.tensor([math.log(0.8), math.log(1.2)], device=DEVICE)
        near = (noise[..., None] - border).abs().amin(-1) < 1e-3
        state["old"] = logp - torch.where(near, torch.zeros_like(noise), noise)
        state["adv"] = 0.3 + torch.randn(b, s, generator=g, device=DEVICE)
        state["kl"] = c["kl"]
        if not c["kl"]:
            state["ref"] = None
    else:
        state["beta"], state["smoothing"] = 0.1, c["smoothing"]
    logits.requires_grad_()
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"qk": _prepare_qk, "route": _prepare_route}.get(case["op"], _prepare_tokens)(case, g)
    state["op"] = case["op"]
    state["train"] = case.get("train", True)
    return state


# ------------------------------------------------------------- plain forms


def _head_norm_rope(x, w, cos, sin, eps):
    xf = x.float()
    n = xf / (xf.square().mean(-1, keepdim=True) + eps).sqrt() * w.float()
    a, b = n[..., 0::2], n[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2).to(x.dtype)


def _plain_qk(s):
    if s["pos"] is None:
        cos, sin = s["cos"][: s["q"].shape[1], None], s["sin"][: s["q"].shape[1], None]
    else:
        cos, sin = s["cos"][s["pos"]][:, :, None], s["sin"][s["pos"]][:, :, None]
    return _head_norm_rope(s["q"], s["wq"], cos, sin, s["eps"]), _head_norm_rope(s["k"], s["wk"], cos, sin, s["eps"])


def _plain_route(s):
    x, k = s["logits"].float(), s["k"]
    e = x.shape[1]
    experts = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :k]
    top = x.gather(1, experts)
    gates = torch.exp(top - top.detach().amax(1, keepdim=True))
    gates = gates / gates.sum(1, keepdim=True)
    m = x.detach().amax(1, keepdim=True)
    ex = torch.exp(x - m)
    total = ex.sum(1, keepdim=True)
    prob, lse = ex / total, (m + total.log())[:, 0]
    valid = torch.ones_like(lse, dtype=torch.bool) if s["mask"] is None else s["mask"]
    w = valid.float()
    n = w.sum()
    counts = ((experts[:, :, None] == torch.arange(e, device=x.device)) & valid[:, None, None]).sum((0, 1))
    balance = e * (counts.float() / (n * k) * ((prob * w[:, None]).sum(0) / n)).sum()
    z = (lse.square() * w).sum() / n
    return (gates * w[:, None]).to(s["logits"].dtype), experts, counts, balance, z


def _plain_logprobs(logits, targets, mask):
    """The rows are summed in 32 bits; the last step is in 64, as differences of log-probabilities nearly cancel."""
    x = logits.float()
    m = x.detach().amax(-1, keepdim=True)
    total = torch.exp(x - m).sum(-1)
    logp = (x.gather(-1, targets[..., None]) - m)[..., 0].double() - total.double().log()
    return logp if mask is None else torch.where(mask, logp, torch.zeros_like(logp))


def _plain_policy(s):
    logp = _plain_logprobs(s["logits"], s["targets"], s["mask"])
    w = torch.ones_like(logp) if s["mask"] is None else s["mask"].double()
    n = w.sum()
    ratio = torch.exp(logp - s["old"])
    free, held = ratio * s["adv"], ratio.clamp(0.8, 1.2) * s["adv"]
    loss = -torch.minimum(free, held)
    kl = torch.zeros_like(n)
    if s["ref"] is not None:
        d = (s["ref"] - logp) * w
        k3 = torch.expm1(d) - d
        loss = loss + s["kl"] * k3
        kl = (k3.detach() * w).sum() / n
    clipped = ((free > held) * w).sum() / n
    return ((loss * w).sum() / n).float(), logp.detach().float(), kl.float(), clipped.float()


def _plain_preference(s):
    logp = _plain_logprobs(s["logits"], s["targets"], s["mask"])
    diff = logp - s["ref"]
    if s["mask"] is not None:
        diff = torch.where(s["mask"], diff, torch.zeros_like(diff))
    ratios = diff.sum(-1)
    half = ratios.shape[0] // 2
    h = s["beta"] * (ratios[:half] - ratios[half:])
    log_sigmoid = h.clamp(max=0) - torch.log1p(torch.exp(-h.abs()))
    loss = -((1 - s["smoothing"]) * log_sigmoid + s["smoothing"] * (log_sigmoid - h)).mean()
    return loss.float(), logp.detach().float(), (s["beta"] * ratios.detach()).float()


# --------------------------------------------------------------------- run


def _run_qk(s):
    if own:
        from dtensor_muon_b200.ops import model_ops

        q, k = model_ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["eps"], positions=s["pos"])
    else:
        q, k = _plain_qk(s)
    out = dict(q=q.detach(), k=k.detach())
    if s["train"]:
        grads = torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]], [s["dq"], s["dk"]])
        out.update(zip(("dq", "dk", "dwq", "dwk"), grads))
    return out


def _run_route(s):
    if own:
        from dtensor_muon_b200.ops import model_ops

        gates, experts, counts, balance, z = model_ops.route(s["logits"], s["k"], mask=s["mask"])
    else:
        gates, experts, counts, balance, z = _plain_route(s)
    (grad,) = torch.autograd.grad([gates, balance, z], [s["logits"]], [s["dgates"], s["dbalance"], s["dz"]])
    return dict(gates=gates.detach(), experts=experts, counts=counts, balance=balance.detach(), z=z.detach(), grad=grad)


def _run_logprobs(s):
    if own:
        from dtensor_muon_b200.ops import model_ops

        logp = model_ops.token_logprobs(s["logits"], s["targets"], mask=s["mask"])
    else:
        logp = _plain_logprobs(s["logits"], s["targets"], s["mask"]).float()
    out = dict(logp=logp.detach())
    if s["train"]:
        (out["grad"],) = torch.autograd.grad([logp], [s["logits"]], [s["dlogp"]])
    return out


def _run_policy(s):
    if own:
        from dtensor_muon_b200.ops import model_ops

        loss, logp, kl, clipped = model_ops.policy_loss(
            s["logits"], s["targets"], s["old"], s["adv"], ref_logp=s["ref"], mask=s["mask"], kl_coef=s["kl"])
    else:
        loss, logp, kl, clipped = _plain_policy(s)
    (grad,) = torch.autograd.grad([loss], [s["logits"]])
    return dict(loss=loss.detach(), logp=logp, kl=kl, clipped=clipped, grad=grad)


def _run_preference(s):
    if own:
        from dtensor_muon_b200.ops import model_ops

        loss, logp, rewards = model_ops.preference_loss(
            s["logits"], s["targets"], s["ref"], mask=s["mask"], beta=s["beta"], label_smoothing=s["smoothing"])
    else:
        loss, logp, rewards = _plain_preference(s)
    (grad,) = torch.autograd.grad([loss], [s["logits"]])
    return dict(loss=loss.detach(), logp=logp, rewards=rewards, grad=grad)


RUN = {"qk": _run_qk, "route": _run_route, "logprobs": _run_logprobs, "policy": _run_policy, "preference": _run_preference}


def run(state):
    return RUN[state["op"]](state)


# -------------------------------------------------------------------- work


def work(case):
    c = case
    size = BYTES[c["dtype"]]
    if c["op"] == "qk":
        rows = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"])
        values = rows * c["dim"]
        table = min(c["table"], c["batch"] * c["seq"]) * c["dim"] * 4
        # forward: in and out; backward: in, its gradient, out
        return {"bytes": values * size * (5 if c["train"] else 2) + table, "flops": values * (20 if c["train"] else 7)}
    if c["op"] == "route":
        values, chosen = c["tokens"] * c["experts"], c["tokens"] * c["top_k"]
        # logits once and their gradient; gates, experts and the gates' gradient
        return {"bytes": 2 * values * size + chosen * (2 * size + 8), "flops": 12 * values}
    rows = c["batch"] * c["seq"]
    train = c["op"] != "logprobs" or c["train"]
    read = max(1, round(c["keep"] * c["seq"])) * c["batch"] * c["vocab"]
    # the rows that count once; every row of the gradient
    return {"bytes": (read + (rows * c["vocab"] if train else 0)) * size + rows * 12, "flops": read * (8 if train else 4)}


# ------------------------------------------------------------------- exact


def _exact_head(x, w, cos, sin, eps, dy):
    """Output, and the gradients of the input and the weight, of one set of heads by their formulas."""
    x, w = x.double(), w.double()
    r = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + eps).rsqrt()
    turn = torch.complex(cos.double(), sin.double())
    pairs = torch.view_as_complex((x * r * w).unflatten(-1, (-1, 2)).contiguous())
    y = torch.view_as_real(pairs * turn).flatten(-2)
    if dy is None:
        return y, None, None
    dn = torch.view_as_real(torch.view_as_complex(dy.double().unflatten(-1, (-1, 2)).contiguous()) * turn.conj()).flatten(-2)
    dw = (dn * x * r).sum((0, 1, 2))
    u = dn * w
    return y, r * u - r.pow(3) * x * (u * x).mean(-1, keepdim=True), dw


def _exact_qk(s):
    at = torch.arange(s["q"].shape[1], device=DEVICE) if s["pos"] is None else s["pos"]
    cos, sin = s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2)
    q, dq, dwq = _exact_head(s["q"], s["wq"], cos, sin, s["eps"], s.get("dq"))
    k, dk, dwk = _exact_head(s["k"], s["wk"], cos, sin, s["eps"], s.get("dk"))
    out = dict(q=q, k=k)
    if s["train"]:
        out.update(dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    return out


def _exact_route(s):
    x = s["logits"].double()
    n_tokens, e = x.shape
    k = s["k"]
    # rank of each expert: how many are greater, or equal and in front of it
    order = torch.argsort(-x, dim=1, stable=True)[:, :k]
    chosen = torch.zeros_like(x).scatter_(1, order, 1.0)
    valid = torch.ones(n_tokens, dtype=torch.float64, device=x.device) if s["mask"] is None else s["mask"].double()
    n = valid.sum()
    gates = torch.softmax(x.gather(1, order), 1) * valid[:, None]
    p = torch.softmax(x, 1)
    lse = torch.logsumexp(x, 1)
    counts = (chosen * valid[:, None]).sum(0)
    share = counts / (n * k)
    balance = e * (share * (p * valid[:, None]).sum(0) / n).sum()
    z = (lse.pow(2) * valid).sum() / n
    dg = s["dgates"].double()
    dtop = gates * (dg - (gates * dg).sum(1, keepdim=True))
    grad = torch.zeros_like(x).scatter_(1, order, dtop)
    db, dz = s["dbalance"].double(), s["dz"].double()
    grad += valid[:, None] * p * (db * e / n * (share - (share * p).sum(1, keepdim=True)) + 2 * dz / n * lse[:, None])
    return dict(gates=gates, experts=None, counts=None, balance=balance, z=z, grad=grad)


def _exact_logprobs(s):
    x = s["logits"].detach().double()
    all_logp = torch.log_softmax(x, -1)
    logp = all_logp.gather(-1, s["targets"][..., None])[..., 0]
    valid = torch.ones_like(logp) if s["mask"] is None else s["mask"].double()
    return all_logp, logp * valid, valid


def _exact_grad(all_logp, targets, coef):
    """Gradient of sum(coef * logp) with respect to the logits."""
    grad = all_logp.exp_().mul_(-coef[..., None])
    return grad.scatter_add_(-1, targets[..., None], coef[..., None])


def _exact_policy(s):
    all_logp, logp, valid = _exact_logprobs(s)
    n = valid.sum()
    adv, ratio = s["adv"].double(), (logp - s["old"].double()).exp()
    low, high = ratio * adv, torch.clamp(ratio, 0.8, 1.2) * adv
    value = -torch.where(low <= high, low, high)
    coef = torch.where(low <= high, -low, torch.zeros_like(low))
    kl = torch.zeros_like(n)
    if s["ref"] is not None:
        d = s["ref"].double() - logp
        k3 = d.exp() - 1 - d
        value = value + s["kl"] * k3
        coef = coef + s["kl"] * (1 - d.exp())
        kl = (k3 * valid).sum() / n
    clipped = ((low > high) * valid).sum() / n
    grad = _exact_grad(all_logp, s["targets"], coef * valid / n)
    return dict(loss=(value * valid).sum() / n, logp=logp, kl=kl, clipped=clipped, grad=grad)


def _exact_preference(s):
    all_logp, logp, valid = _exact_logprobs(s)
    ratios = ((logp - s["ref"].double()) * valid).sum(-1)
    pairs = ratios.shape[0] // 2
    h = s["beta"] * (ratios[:pairs] - ratios[pairs:])
    e = s["smoothing"]
    loss = -((1 - e) * torch.nn.functional.logsigmoid(h) + e * torch.nn.functional.logsigmoid(-h)).mean()
    dh = -((1 - e) * torch.sigmoid(-h) - e * torch.sigmoid(h)) / pairs
    coef = s["beta"] * torch.cat([dh, -dh])[:, None] * valid
    return dict(loss=loss, logp=logp, rewards=s["beta"] * ratios, grad=_exact_grad(all_logp, s["targets"], coef))


def _exact_scores(s):
    all_logp, logp, valid = _exact_logprobs(s)
    out = dict(logp=logp)
    if s["train"]:
        out["grad"] = _exact_grad(all_logp, s["targets"], s["dlogp"].double() * valid)
    return out


EXACT = {"qk": _exact_qk, "route": _exact_route, "logprobs": _exact_scores, "policy": _exact_policy,
         "preference": _exact_preference}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return EXACT[state["op"]](state)
