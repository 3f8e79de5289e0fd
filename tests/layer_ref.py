"""Plain 64-bit forms of routing, the weighted sum, shared projections and the gradients' norm, with the bounds their tests
use.  grouped_ref has the bounds of sums (F32: a whole fp32 step per addition) and of the last rounding."""
import math

import torch

from grouped_ref import F32, half_step  # noqa: F401

INF = math.inf


def scores(logits, score):
    """softmax or sigmoid in 64 bits, infinite logits at their limits; zeros where every logit is -inf."""
    l = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(l)
    finite = torch.where(l.isnan(), -INF, l)
    top = finite.amax(1, keepdim=True)
    e = torch.where(finite == -INF, 0.0, torch.where(finite == top, 1.0, torch.exp(finite - top)))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def route(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0):
    """(ids int64, weights float64) by the definition; ids -1 and weight 0 where no expert is left."""
    l = logits.double()
    s = scores(logits, score)
    c = l if bias is None else s + bias.double()
    c = torch.where(l.isnan() | (l == -INF) | c.isnan(), -INF, c)
    n_tok, n_exp = l.shape
    if n_group > 1:
        of = c if bias is not None or group_best == 1 else torch.where(c == -INF, -INF, s)
        best = of.reshape(n_tok, n_group, -1).sort(2, descending=True).values[:, :, :group_best]
        value = torch.where(best[:, :, 0] == -INF, -INF, torch.where(best == -INF, 0.0, best).sum(2))
        kept = torch.argsort(value, dim=1, descending=True, stable=True)[:, :topk_group]
        keep = torch.zeros((n_tok, n_group), dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        c = torch.where(keep.repeat_interleave(n_exp // n_group, 1), c, -INF)
    ids = torch.argsort(c, dim=1, descending=True, stable=True)[:, :k]
    has = c.gather(1, ids) > -INF
    w = chosen_weights(l, ids, has, score, renorm, scale)
    w = torch.where(l.isnan().any(1, keepdim=True), math.nan, w)
    return torch.where(has, ids, -1), w


def chosen_weights(l, ids, has, score, renorm, scale):
    """The weights of the places that have an id (differentiable in l where it is finite)."""
    u = l.gather(1, ids.clamp(min=0))
    if not renorm:
        return scale * torch.where(has, scores(l, score).gather(1, ids.clamp(min=0)), 0.0)
    # s / sum(s), in logarithms: scores of any magnitude
    log_s = torch.nn.functional.logsigmoid(u) if score == "sigmoid" else u
    log_s = torch.where(has, log_s, -INF)
    top = log_s.amax(1, keepdim=True)
    e = torch.where(log_s == -INF, 0.0, torch.where(log_s == top, 1.0, torch.exp(log_s - top)))
    total = e.sum(1, keepdim=True)
    return scale * torch.where(total > 0, e / total, 0.0)


def weight_slack(logits, k, want):
    """Relative: an exponential's argument is rounded, which its value shows |argument| times (up to 110, where fp32 ends; in
    both the score and the sum), then 8 steps for the function and the quotient, one per addition of the sum's longest chain.
    Absolute: what fp32 does not hold."""
    l = logits.double()
    spread = torch.where(l.abs() < INF, l, 0.0)
    spread = (spread.amax(1, keepdim=True) - spread.amin(1, keepdim=True)).clamp(max=110) + spread.abs().amax(1, keepdim=True).clamp(max=110)
    return want.abs() * (2 * spread + 32 + k + logits.shape[1] / 64) * F32 + 2.0 ** -126


def route_grad(dweights, logits, ids, score, renorm, scale):
    """(gradient, bound before rounding) by autograd in 64 bits."""
    l = logits.double().clone().requires_grad_()
    has = (ids >= 0) & (ids < l.shape[1])
    at = torch.where(has, ids, 0).long()
    u = torch.where(has, l.gather(1, at), -INF)
    if renorm:
        log_s = torch.nn.functional.logsigmoid(u) if score == "sigmoid" else u
        w = torch.softmax(torch.where(has, log_s, -INF), 1)
        w = torch.where(has.any(1, keepdim=True), w, 0.0)
    else:
        s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, 1)
        w = torch.where(has, s.gather(1, at), 0.0)
    g = torch.where(has, scale * dweights.double(), 0.0)
    d = torch.autograd.grad((w * g).sum(), l)[0].nan_to_num(0.0) if has.any() else torch.zeros_like(l)
    # every term p (g - sum p g), with its own error and the difference's
    p = w.detach().abs()
    mag = torch.zeros_like(d)
    terms = p * (g.abs() + (p * g.abs()).sum(1, keepdim=True))
    mag.scatter_add_(1, at, torch.where(has, terms, 0.0))
    if score == "softmax" and not renorm:
        mag += torch.softmax(logits.double(), 1) * (p * g.abs()).sum(1, keepdim=True)
    return d.detach(), 4 * weight_slack(logits, ids.shape[1], mag)


def combine(y, weights, residual=None):
    """y [n_tok, k, hidden]: (sum, bound before rounding)."""
    n_tok, k = weights.shape
    yd = y.double().reshape(n_tok, k, -1)
    w = weights.double().unsqueeze(2)
    terms = torch.where(w == 0, 0.0, w * yd)
    out, mag = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        out, mag = out + residual.double(), mag + residual.double().abs()
    return out, (k + 2) * F32 * mag


def combine_grad(dout, y, weights):
    n_tok, k = weights.shape
    d, yd = dout.double().unsqueeze(1), y.double().reshape(n_tok, k, -1)
    dy = weights.double().unsqueeze(2) * d
    return dy, dy.abs() * F32, (d * yd).sum(2), (yd.shape[2] + 2) * F32 * (d * yd).abs().sum(2)


def activation(z, act):
    if act is None:
        return z
    f = torch.nn.functional
    return f.silu(z) if act == "silu" else f.gelu(z) if act == "gelu" else f.relu(z).square()


def slope(z, act):
    if act is None:
        return torch.ones_like(z)
    z = z.clone().requires_grad_()
    return torch.autograd.grad(activation(z, act).sum(), z)[0]


def activation_slack(z, act):
    """The function's own error in fp32 at z.  silu: exponential and quotient, (|z| + 8) steps of 2^-22 of its value.  gelu: the
    integral to 2^-20, whatever method gives it.  relu2: one product."""
    if act is None:
        return torch.zeros_like(z)
    if act == "gelu":
        return z.abs() * 2.0 ** -20
    return activation(z, act).abs() * (2.0 ** -23 if act == "relu2" else (z.abs().clamp(max=200) + 8) * 2.0 ** -22)


def slope_slack(z, act):
    if act is None:
        return torch.zeros_like(z)
    if act == "relu2":
        return 2 * z.abs() * F32
    if act == "gelu":
        return (1 + z.abs() * torch.exp(-0.5 * z * z) * (z * z / 2 + 8)) * 2.0 ** -20
    sig = torch.sigmoid(z)
    return sig * (1 + z.abs() * (1 - sig)) * 2 * (z.abs().clamp(max=200) + 8) * 2.0 ** -22


def linear(x, w, bias=None, act=None, residual=None):
    """(y, bound, z, bound) of act(x w^T + bias) + residual."""
    xd, wd = x.double(), w.double()
    z, mag = xd @ wd.T.contiguous(), xd.abs() @ wd.abs().T.contiguous()
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    sz = (x.shape[1] + 3) * F32 * mag
    y = activation(z, act)
    steep = 2 * (z.abs() + sz) if act == "relu2" else 1.13
    sy = sz * steep + activation_slack(z.abs() + sz if act == "gelu" else z, act)
    if residual is not None:
        y = y + residual.double()
        sy = sy + F32 * (y.abs() + residual.double().abs())
    return y, sy, z, sz


def linear_grad(dy, x, w, z, act):
    """((dx, bound), (dw, bound), (db, bound)); dz is rounded to x's type unless it is dy as it came."""
    d = dy.double()
    sd = torch.zeros_like(d)
    if act is not None:
        s = slope(z.double(), act)
        sd = d.abs() * slope_slack(z.double(), act) + (d * s).abs() * F32
        d = d * s
    sz = sd + half_step(d.abs() + sd, x.dtype) if act is not None or dy.dtype == torch.float32 else sd
    wd, xd, dT, sT = w.double(), x.double(), d.T.contiguous(), sz.T.contiguous()
    n_tok, n_out = d.shape
    dx = (d @ wd, sz @ wd.abs() + (n_out + 2) * F32 * ((d.abs() + sz) @ wd.abs()))
    dw = (dT @ xd, sT @ xd.abs() + (n_tok + 2) * F32 * ((dT.abs() + sT) @ xd.abs()))
    db = (d.sum(0), sd.sum(0) + (n_tok + 2) * F32 * (d.abs() + sd).sum(0))
    return dx, dw, db
