"""Plain 64-bit forms of the grouped products, their gradients and the adapters, with the bounds their tests use; on the
device of the sorted rows they are given (the CPU but for the largest sizes).

Bounds.  Inputs are fp16 or bf16, so a product of two is exact in fp32 (at most 22 significand bits).  A sum of
c of them in fp32, in any order and with either rounding or truncation per addition, is off by at most
c * 2^-23 * sum |p_i q_i| (truncation is off by a whole step, 2^-23, of the running sum).  The result is then
rounded once: eps / 2 of the value, or half the smallest subnormal step where that is more.
"""
import torch

F32 = 2.0 ** -23


def half_step(want, dtype):
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return want.abs() * (torch.finfo(dtype).eps / 2) + tiny


def check(got, want, slack, what=""):
    """|got - want| <= half a step of got's type + slack, where slack bounds the error before rounding."""
    got_d, want_d = got.detach().to(want.device).double(), want.double()
    assert got_d.shape == want_d.shape, (what, got_d.shape, want_d.shape)
    # the value that is rounded may be `slack` larger than want, and its step with it
    room = half_step(want_d.abs() + slack, got.dtype) + slack
    off = (got_d - want_d).abs()
    bad = ~(off <= room)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off - room).max()):.3e} over"


def segments(seg_start, seg_slot, n_slots, n_rows):
    """[(r0, r1, slot)] of the segments whose slot exists."""
    s = [min(max(int(v), 0), n_rows) for v in seg_start]
    out = []
    for u in range(len(s) - 1):
        slot = u if seg_slot is None else int(seg_slot[u])
        if 0 <= slot < n_slots and s[u + 1] > s[u]:
            out.append((s[u], s[u + 1], slot))
    return out


def gather(x, rows):
    """x[rows] in 64 bits, zeros for a row that x does not have."""
    x = x.double().cpu()
    rows = torch.as_tensor(rows, dtype=torch.int64)
    ok = (rows >= 0) & (rows < x.shape[0])
    out = torch.zeros((rows.numel(), x.shape[1]), dtype=torch.float64)
    out[ok] = x[rows[ok]]
    return out


def product(xr, seg_start, w, seg_slot=None, scale=None, transposed=False):
    """(values, bound before rounding, rows that a segment covers) of the sorted rows' products."""
    w = w.to(xr.device).double()
    n_out = w.shape[2] if transposed else w.shape[1]
    y = torch.zeros((xr.shape[0], n_out), dtype=torch.float64, device=xr.device)
    mag, has = y.clone(), torch.zeros(xr.shape[0], dtype=torch.bool, device=xr.device)
    for r0, r1, slot in segments(seg_start, seg_slot, w.shape[0], xr.shape[0]):
        m = w[slot] if transposed else w[slot].T
        s = 1.0 if scale is None else float(scale[slot])
        y[r0:r1] = s * (xr[r0:r1] @ m)
        mag[r0:r1] = abs(s) * (xr[r0:r1].abs() @ m.abs())
        has[r0:r1] = True
    c = w.shape[1] if transposed else w.shape[2]
    return y, (c + 2) * F32 * mag, has


def glu(g, u, slack_g, slack_u):
    """silu(g) * u and its bound: |silu'| < 1.1; the exponential and the quotient in fp32 are off by (|g| + 8)
    steps of 2^-22 (the argument of exp is rounded, which its value shows |g| times)."""
    sig = torch.sigmoid(g)
    h = g * sig * u
    slack = 1.1 * slack_g * (u.abs() + slack_u) + (g * sig).abs() * slack_u + h.abs() * (g.abs() + 8) * 2.0 ** -22
    return h, slack


def glu_grad(dh, slack_dh, gu):
    g, u = gu.to(dh.device).double().chunk(2, 1)
    sig = torch.sigmoid(g)
    fg, fu = u * sig * (1 + g * (1 - sig)), g * sig
    # 1 + g (1 - sig) may cancel: its parts' roundings count with their magnitude
    mg = u.abs() * sig * (1 + g.abs() * (1 - sig))
    rel = (g.abs() + 8) * 2.0 ** -22
    want = torch.cat([dh * fg, dh * fu], 1)
    slack = torch.cat([slack_dh * mg + dh.abs() * mg * 2 * rel, slack_dh * fu.abs() + (dh * fu).abs() * rel], 1)
    return want, slack


def weight_grad(dyr, xr, seg_start, n_seg, scale=None):
    n_rows = dyr.shape[0]
    dw = torch.zeros((n_seg, dyr.shape[1], xr.shape[1]), dtype=torch.float64, device=xr.device)
    slack = dw.clone()
    for r0, r1, u in segments(seg_start, None, n_seg, n_rows):
        s = 1.0 if scale is None else float(scale[u])
        dw[u] = s * (dyr[r0:r1].T @ xr[r0:r1])
        slack[u] = (r1 - r0 + 2) * F32 * abs(s) * (dyr[r0:r1].abs().T @ xr[r0:r1].abs())
    return dw, slack


def lora(base, x, a, b, ids, scale=None):
    """(base + scale b (a x), bound): both sums in fp32, the second over scale v with v's own error and, where v is
    taken apart into 16-bit parts, a rest of 2^-22 of each value and 2^-39 of the token's largest."""
    out, xd = base.double().cpu().clone(), x.double().cpu()
    slack = torch.zeros_like(out)
    for j in range(a.shape[0]):
        rows = (ids.cpu() == j).nonzero()[:, 0]
        if not rows.numel():
            continue
        aj, bj, s = a[j].double().cpu(), b[j].double().cpu(), 1.0 if scale is None else float(scale[j])
        v = xd[rows] @ aj.T
        dv = (aj.shape[1] + 3) * F32 * (xd[rows].abs() @ aj.abs().T)
        dv = dv + 2.0 ** -22 * (v.abs() + dv) + 2.0 ** -39 * (v.abs() + dv).amax(1, keepdim=True)
        delta = s * (v @ bj.T)
        out[rows] += delta
        mag = abs(s) * ((v.abs() + dv) @ bj.abs().T)
        # every value comes in up to three parts, each a term of its own in the sum
        slack[rows] = (3 * aj.shape[0] + 3) * F32 * mag + abs(s) * (dv @ bj.abs().T) + F32 * (out[rows].abs() + mag)
    return out, slack
