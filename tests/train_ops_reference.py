"""64-bit values of the decoder's training operators with the error each output may have.

Every function returns ``{output: (value, bound)}``. The bounds follow from the arithmetic the operators promise: inputs
as they are, sums and statistics in 32 bits, one rounding (half a step, ``U[dtype]``) at the end. ``E`` is half a step
of fp32. A sum of n terms in 32 bits is off by at most ``n * E`` times the sum of their absolute values, and
``exp2((x - m) * log2 e)`` by ``(4 + 2 |x - m|) * E`` of itself: two roundings of the argument, and two steps of the
exponential.
"""

import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32, torch.float64)}
E = 2.0**-24
# Exponentials are taken against the row's maximum, and one below 2^-126 (the smallest normal fp32) may come out as 0:
# what it is multiplied with is then off by at most that much of itself.
FLUSH = 2.0**-126


def tiny(dtype):
    """Half the spacing of the smallest numbers of a type, below which its rounding is no longer relative."""
    return torch.finfo(dtype).smallest_normal * U[dtype]


def check(got, want, what=""):
    assert set(got) <= set(want), (set(got), set(want))
    for name, g in got.items():
        value, bound = want[name]
        assert tuple(g.shape) == tuple(value.shape), (what, name, g.shape, value.shape)
        if not g.is_floating_point():
            assert torch.equal(g, value), (what, name)
            continue
        g = g.double()
        nan = torch.isnan(value)
        assert torch.equal(torch.isnan(g), nan), (what, name, "NaN where none belongs, or none where one does")
        off = torch.where(nan, 0.0, (g - value).abs() - bound)
        same = g == value  # infinities
        off = torch.where(same, torch.zeros_like(off), off)
        if off.numel():
            i = int(off.argmax())
            assert not (off > 0).any(), (
                f"{what} {name}: {int((off > 0).sum())} of {off.numel()} values outside their bounds; at {i}: "
                f"{g.flatten()[i]} for {value.flatten()[i]}, bound {bound.expand_as(value).flatten()[i]}")


# --------------------------------------------------------------- qk_norm_rope


def _heads(x, w, cos, sin, eps, dy):
    t, d = x.dtype, x.shape[-1]
    u = U[t]
    x, wd = x.double(), w.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * wd
    c, s = cos.double(), sin.double()

    def turn(v, sign):
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack((a * c - sign * b * s, sign * a * s + b * c), -1).flatten(-2)

    def turned_size(v):
        a, b = v[..., 0::2].abs(), v[..., 1::2].abs()
        return torch.stack((a * c.abs() + b * s.abs(), a * s.abs() + b * c.abs()), -1).flatten(-2)

    # the sum of squares is off by (8 + 5) E, its root by half of that and the root's own 2 steps; 4 products
    rel = (d / 2 + 32) * E
    y = turn(n, 1)
    out = dict(y=(y, u * y.abs() + rel * turned_size(n) + tiny(t)))
    if dy is not None:
        g = dy.double()
        dn, dn_size = turn(g, -1), turned_size(g)
        uw, uw_size = dn * wd, dn_size * wd.abs()
        dx = r * uw - r**3 * x * (uw * x).mean(-1, keepdim=True)
        size = r * uw_size + r**3 * x.abs() * (uw_size * x.abs()).mean(-1, keepdim=True)
        out["dx"] = (dx, u * dx.abs() + 2 * rel * size + tiny(t))
        dw = (dn * x * r).sum((0, 1, 2))
        rows = x.numel() // max(1, d)
        out["dw"] = (dw, U[w.dtype] * dw.abs() + (rel + rows * E) * (dn_size * x.abs() * r).sum((0, 1, 2)) + tiny(w.dtype))
    return out


def qk_norm_rope(q, k, wq, wk, cos, sin, eps, positions=None, dq=None, dk=None):
    at = torch.arange(q.shape[1], device=q.device) if positions is None else positions.long()
    c, s = cos[at].unsqueeze(-2), sin[at].unsqueeze(-2)
    a, b = _heads(q, wq, c, s, eps, dq), _heads(k, wk, c, s, eps, dk)
    out = dict(q=a["y"], k=b["y"])
    if dq is not None:
        out.update(dq=a["dx"], dk=b["dx"], dwq=a["dw"], dwk=b["dw"])
    return out


# ----------------------------------------------------------------------- route


def route(logits, top_k, mask=None, dgates=None, dbalance=None, dz=None):
    t, e = logits.shape
    u = U[logits.dtype]
    x = logits.double()
    valid = torch.ones(t, dtype=torch.bool, device=x.device) if mask is None else mask
    experts = torch.sort(torch.where(x.isnan(), torch.inf, x), dim=1, descending=True, stable=True).indices[:, :top_k]
    x = torch.where(valid[:, None], x, 0.0)
    v = valid.double()[:, None]
    counts = torch.zeros(t, e, dtype=torch.int64, device=x.device).scatter_(1, experts, 1)[valid].sum(0)
    n = max(1, int(valid.sum()))
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    gap = torch.where(x == -torch.inf, 0.0, m - x)
    wide = gap.amax(1, keepdim=True)
    rel = (2 * (4 + 2 * wide) + e + 8) * E  # of a quotient of an exponential by a sum of them
    p = torch.softmax(x, 1)
    gates = torch.softmax(x.gather(1, experts), 1) * v
    lse = torch.logsumexp(x, 1, keepdim=True)
    lse_off = rel + 4 * E * (1 + m.abs() + lse.abs())
    share = counts.double() / (n * top_k)
    balance = e * (share * (p * v).sum(0) / n).sum()
    z = (lse.square() * v).sum() / n
    out = dict(gates=(gates, (u + rel) * gates + tiny(logits.dtype)), experts=(experts, None), counts=(counts, None),
               balance=(balance, (float(rel.max() if t else 0) + t * E) * balance + E),
               z=(z, (2 * lse.abs() * lse_off * v).sum() / n + t * E * z + E))
    if dgates is not None or dbalance is not None or dz is not None:
        dg = torch.zeros_like(gates) if dgates is None else dgates.double()
        a = float(dbalance or 0) * e / n
        b = float(dz or 0) * 2 / n
        mean = (gates * dg).sum(1, keepdim=True)
        top = torch.zeros_like(x).scatter_(1, experts, gates * (dg - mean))
        size = torch.zeros_like(x).scatter_(1, experts, gates * (dg.abs() + (gates * dg.abs()).sum(1, keepdim=True)))
        mix = (share * p).sum(1, keepdim=True)
        grad = top + v * p * (a * (share - mix) + b * lse)
        size = size + v * p * (abs(a) * (share + mix) + abs(b) * (lse.abs() + lse_off / rel))
        out["grad"] = (grad, u * grad.abs() + 3 * rel * size + tiny(logits.dtype))
    return out


# ----------------------------------------------------- log-probabilities, losses


def _rows(logits, targets, mask, rounded):
    """logp, its error before and after rounding to fp32, all log-probabilities and their exponentials' relative error."""
    x = logits.double()
    valid = torch.ones(targets.shape, dtype=torch.bool, device=x.device) if mask is None else mask
    x = torch.where(valid[..., None], x, 0.0)
    y = torch.where(valid, targets, 0)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    logs = torch.log_softmax(x, -1)
    p = logs.exp()
    gap = torch.where(x == -torch.inf, 0.0, m - x)
    # sum: each exponential's own error weighted with its share, and an addition per 512-th value, 32 at a time, and joins
    s_rel = ((4 + 2 * gap) * p).sum(-1) * E + (x.shape[-1] / 512 + 64) * E
    logp = logs.gather(-1, y[..., None])[..., 0]
    off = s_rel
    if rounded:  # the logarithm and the difference are rounded to fp32 before they are used
        off = off + 2 * E * (logp.abs() + gap.gather(-1, y[..., None])[..., 0] + (logs.amax(-1)).abs() + 1)
    p_rel = s_rel[..., None] + (4 + 2 * gap) * E
    v = valid.double()
    return torch.where(valid, logp, 0.0), off * v, p, p_rel, y, v


def _grad(dtype, p, p_rel, y, coef, coef_off):
    hot = torch.zeros_like(p).scatter_(-1, y[..., None], 1.0)
    grad = coef[..., None] * (hot - p)
    u = U[dtype]
    bound = u * grad.abs() + coef.abs()[..., None] * (p * (p_rel + 6 * E) + hot * 4 * E + FLUSH) + coef_off[..., None] * (hot - p).abs()
    rows = (coef != 0)[..., None]
    return torch.where(rows, grad, 0.0), bound + tiny(dtype)


def token_logprobs(logits, targets, mask=None, dlogp=None, rounded=False):
    logp, off, p, p_rel, y, v = _rows(logits, targets, mask, rounded)
    out = dict(logp=(logp, off + E * logp.abs()))
    if dlogp is not None:
        out["grad"] = _grad(logits.dtype, p, p_rel, y, dlogp.double() * v, torch.zeros_like(v))
    return out


def policy_loss(logits, targets, old_logp, advantages, ref_logp=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                scale=1.0, rounded=False):
    logp, off, p, p_rel, y, v = _rows(logits, targets, mask, rounded)
    valid = v > 0
    n = max(1.0, float(v.sum()))
    zero = torch.zeros_like(logp)
    ratio = torch.where(valid, logp - old_logp.double(), 0.0).exp()
    adv = torch.where(valid, advantages.double(), 0.0)
    low, high = ratio * adv, ratio.clamp(1 - clip_low, 1 + clip_high) * adv
    clipped = low > high
    value = -torch.where(clipped, high, low)
    coef = torch.where(clipped, 0.0, -low)
    slope = torch.where(clipped, 0.0, low.abs())  # of the coefficient by logp
    off = off + 4 * E  # the ratio's own exponential
    value_off = slope * off + E * value.abs()
    kl, kl_off = zero, zero
    if ref_logp is not None:
        d = torch.where(valid, ref_logp.double() - logp, 0.0)
        kl = torch.expm1(d) - d
        kl_off = torch.expm1(d).abs() * off + 2 * E * (d.abs() if rounded else kl)
        value, coef = value + kl_coef * kl, coef - kl_coef * torch.expm1(d)
        value_off, slope = value_off + kl_coef * kl_off + E * value.abs(), slope + kl_coef * d.exp()
    coef_off = (slope * off + 4 * E * coef.abs()) * v * abs(scale) / n
    loss = (value * v).sum() / n
    loss_off = (value_off * v).sum() / n + E * loss.abs()
    if rounded:
        loss_off = loss_off + v.numel() * E * (value.abs() * v).sum() / n
    kl_mean = (kl * v).sum() / n
    share = (clipped & valid).double().sum() / n
    out = dict(loss=(loss, loss_off), logp=(logp, off + E * logp.abs()),
               kl=(kl_mean, (kl_off * v).sum() / n + v.numel() * E * kl_mean), clipped=(share, 2 * E * share))
    out["grad"] = _grad(logits.dtype, p, p_rel, y, scale * coef * v / n, coef_off)
    return out


def preference_loss(logits, targets, ref_logp, mask=None, beta=0.1, label_smoothing=0.0, scale=1.0, rounded=False):
    logp, off, p, p_rel, y, v = _rows(logits, targets, mask, rounded)
    diff = torch.where(v > 0, logp - ref_logp.double(), 0.0)
    ratios = diff.sum(-1)
    ratio_off = off.sum(-1) + (2 * E * diff.abs().sum(-1) if rounded else 0)
    pairs = ratios.shape[0] // 2
    beta32 = float(torch.tensor(beta, dtype=torch.float32))
    h = beta * (ratios[:pairs] - ratios[pairs:])
    h_off = beta * (ratio_off[:pairs] + ratio_off[pairs:]) + 2 * abs(beta32 - beta) / beta * h.abs() + E * h.abs()
    e = label_smoothing
    up, down = torch.nn.functional.logsigmoid(h), torch.nn.functional.logsigmoid(-h)
    loss = -((1 - e) * up + e * down).mean()
    dh = e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h)
    c = scale * beta * dh / pairs
    # the sigmoid's slope is at most itself; beta and the smoothing are rounded to fp32
    c_off = abs(scale) * beta / pairs * (torch.sigmoid(h) * torch.sigmoid(-h) * h_off + 6 * E)
    loss_off = (dh.abs() * h_off).mean() + h_off.square().mean() + 4 * E * (up.abs() + down.abs()).mean()
    rewards = beta * ratios
    coef = torch.cat([c, -c])[:, None] * v
    return dict(loss=(loss, loss_off), logp=(logp, off + E * logp.abs()),
                rewards=(rewards, beta * ratio_off + 4 * E * rewards.abs()),
                grad=_grad(logits.dtype, p, p_rel, y, coef, torch.cat([c_off, c_off])[:, None] * v))
