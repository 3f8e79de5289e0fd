"""The operators of the unquantised expert layer and of the adapters beside it, as cases to time and compare.

A case is a dict of plain values with a "kind":

  plan       the (token, k) expert ids of a batch -> its rows sorted by expert (the row plan that every
             grouped product takes)
  gate_up    the sorted rows through their experts' gate and up projections: silu(G x) * (U x)
  down       the sorted rows through their experts' down projections, each written at its (token, k) place
  grad_up    the gradients of a grouped product y[r] = W x[token of r]: one row of dx per (token, k) and
             the weights' gradient
  grad_down  the gradients of the down product behind a SwiGLU: of the gate and up pre-activations, and of
             the weights
  lora       a shared projection's output plus each token's own request's low-rank adapter
  lora_grad  the gradients of that: of the tokens and of both factors of every adapter

Sizes are those of the repository's workloads (512 experts, top-10, 2048 x 512; the checkpoint's
2560 x 640; the odd 1152 x 320 over 100 experts), or generic ones with few experts and long segments.
"""
import math
import os
import sys

import torch

own = False


def listed():
    work = {"k": 10, "n_exp": 512, "hidden": 2048, "inter": 512}
    real = {"k": 10, "n_exp": 512, "hidden": 2560, "inter": 640}
    few = {"k": 4, "n_exp": 16, "hidden": 4096, "inter": 1024}
    return [
        # a batch of decoding requests, one token each: the smallest call, all latency
        {"name": "plan_64", "kind": "plan", "tokens": 64, "k": 10, "n_exp": 512},
        # a long prompt's rows
        {"name": "plan_16384", "kind": "plan", "tokens": 16384, "k": 10, "n_exp": 512},
        # one decoded token: ten experts with one row each, every weight read once
        {"name": "up_decode", "kind": "gate_up", "tokens": 1, "dtype": "bf16", **work},
        # the ordinary prompt chunk: about ten rows per expert
        {"name": "up_chunk", "kind": "gate_up", "tokens": 512, "dtype": "fp16", **real},
        # a ragged prompt over few experts, sizes that are no power of two
        {"name": "down_odd", "kind": "down", "tokens": 777, "dtype": "fp16", "k": 6, "n_exp": 100, "hidden": 1152,
         "inter": 320},
        # a training batch over few large experts: about 2048 rows each
        {"name": "down_few", "kind": "down", "tokens": 8192, "dtype": "bf16", **few},
        # backward of the gate and up projections of a training batch, many experts: about 40 rows each
        {"name": "grad_up_many", "kind": "grad_up", "tokens": 2048, "dtype": "bf16", **work},
        # backward through down and SwiGLU, few experts
        {"name": "grad_down_few", "kind": "grad_down", "tokens": 4096, "dtype": "bf16", **few},
        # eight requests decoding, each with its own adapter
        {"name": "lora_decode", "kind": "lora", "tokens": 8, "requests": 8, "n_ad": 32, "rank": 16, "n_in": 2048,
         "n_out": 2048, "dtype": "bf16"},
        # the prompts of a dozen requests in one batch, some of them without an adapter
        {"name": "lora_prompts", "kind": "lora", "tokens": 4096, "requests": 12, "n_ad": 16, "rank": 64, "n_in": 2560,
         "n_out": 2560, "dtype": "fp16"},
        # training adapters: a small odd batch, and a long one
        {"name": "lora_grad_odd", "kind": "lora_grad", "tokens": 333, "requests": 5, "n_ad": 5, "rank": 8, "n_in": 640,
         "n_out": 2560, "dtype": "bf16"},
        {"name": "lora_grad_long", "kind": "lora_grad", "tokens": 4096, "requests": 8, "n_ad": 8, "rank": 64,
         "n_in": 2560, "n_out": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of step between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, step * round(v / step))))


def draw(rng):
    kind = rng.choice(["plan", "gate_up", "gate_up", "down", "down", "grad_up", "grad_down", "lora", "lora_grad"])
    if kind == "plan":
        n_exp = _log(rng, 1, 1024)
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "k": rng.randint(1, min(10, n_exp)), "n_exp": n_exp}
    dtype = rng.choice(["bf16", "fp16"])
    if kind in ("lora", "lora_grad"):
        n_ad = _log(rng, 1, 64)
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "requests": rng.randint(1, 16), "n_ad": n_ad,
                "rank": rng.choice([8, 16, 24, 32, 48, 64, 96, 128]), "n_in": _log(rng, 256, 2560, 8),
                "n_out": _log(rng, 256, 2560, 8), "dtype": dtype}
    while True:
        c = {"kind": kind, "tokens": _log(rng, 1, 8192), "dtype": dtype, "k": 0, "n_exp": _log(rng, 1, 512),
             "hidden": _log(rng, 256, 4096, 8), "inter": _log(rng, 64, 2048, 8)}
        c["k"] = rng.randint(1, min(10, c["n_exp"]))
        m = c["tokens"] * c["k"]
        if c["n_exp"] * c["hidden"] * c["inter"] <= 512 * 2048 * 512 and m * c["hidden"] * c["inter"] <= 2 ** 37 and m <= 40960:
            return c


# ---- inputs -------------------------------------------------------------------------------------

def _routing(case, g):
    """int32 [tokens, k] distinct expert ids per token, some experts more popular than others."""
    T, k, E = case["tokens"], case["k"], case["n_exp"]
    pop = torch.randn(E, device="cuda", generator=g) * 0.5
    u = torch.rand((T, E), device="cuda", generator=g).clamp_(1e-7, 1 - 1e-7)
    return (pop - torch.log(-torch.log(u))).topk(k, dim=1).indices.to(torch.int32)


def _rand(shape, dtype, g, scale=1.0):
    t = torch.randn(shape, dtype=dtype, device="cuda", generator=g)
    return t.mul_(scale) if scale != 1.0 else t


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    kind, s = case["kind"], {"case": case}
    if kind == "plan":
        s["ids"] = _routing(case, g)
        return s
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    if kind in ("lora", "lora_grad"):
        T, R, K, N, n_ad = case["tokens"], case["rank"], case["n_in"], case["n_out"], case["n_ad"]
        s["x"] = _rand((T, K), dt, g)
        s["a"] = _rand((n_ad, R, K), dt, g, K ** -0.5)
        s["b"] = _rand((n_ad, N, R), dt, g, R ** -0.5)
        s["scale"] = 0.5 + torch.rand(n_ad, device="cuda", generator=g)
        # requests take turns along the batch in runs of their own length; a request may have no adapter (-1)
        q = min(case["requests"], T)
        cut = torch.sort(torch.randperm(T - 1, device="cuda", generator=g)[:q - 1] + 1).values
        run = torch.searchsorted(cut, torch.arange(T, device="cuda"), right=True)
        ad = torch.randint(0 if q < 10 else -1, n_ad, (q,), device="cuda", generator=g)
        s["ids"] = ad[run].to(torch.int32)
        s["base" if kind == "lora" else "dy"] = _rand((T, N), dt, g)
        return s
    T, k, E, H, I = case["tokens"], case["k"], case["n_exp"], case["hidden"], case["inter"]
    M = T * k
    ids = _routing(case, g).reshape(-1).long()
    order = torch.argsort(ids, stable=True)
    seg = torch.searchsorted(ids[order], torch.arange(E + 1, device="cuda"))
    s["row_token"], s["row_out"] = (order // k).to(torch.int32), order.to(torch.int32)
    s["seg_start"] = seg.to(torch.int32)
    s["longest"] = int((seg[1:] - seg[:-1]).max())
    if kind == "gate_up":
        s["x"] = _rand((T, H), dt, g)
        s["w"] = _rand((E, 2 * I, H), dt, g, H ** -0.5)
    elif kind == "down":
        s["x"] = _rand((M, I), dt, g)
        s["w"] = _rand((E, H, I), dt, g, I ** -0.5)
    elif kind == "grad_up":
        s["x"] = _rand((T, H), dt, g)
        s["dy"] = _rand((M, 2 * I), dt, g)
        s["w"] = _rand((E, 2 * I, H), dt, g, H ** -0.5)
    else:
        s["gu"] = _rand((M, 2 * I), dt, g)
        gate, up = s["gu"].float().chunk(2, 1)
        s["x"] = (gate * torch.sigmoid(gate) * up).to(dt)      # the activations that the forward pass kept
        s["dy"] = _rand((M, H), dt, g)
        s["w"] = _rand((E, H, I), dt, g, I ** -0.5)
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    if os.path.join(os.getcwd(), "moe-offload_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "moe-offload_amd"))
    from moe_offload import ops
    kind = s["case"]["kind"]
    if kind == "plan":
        return ops.expert_plan(s["ids"], s["case"]["n_exp"])
    if kind == "gate_up":
        return ops.grouped_gate_up(s["x"], s["row_token"], s["seg_start"], s["w"])
    if kind == "down":
        return ops.grouped_mm(s["x"], s["seg_start"], s["w"], row_out=s["row_out"])
    if kind == "grad_up":
        return (ops.grouped_mm_dx(s["dy"], s["seg_start"], s["w"], row_out=s["row_out"]),
                ops.grouped_mm_dw(s["dy"], s["x"], s["seg_start"], row_x=s["row_token"]))
    if kind == "grad_down":
        return (ops.grouped_mm_dx(s["dy"], s["seg_start"], s["w"], row_in=s["row_out"], gu=s["gu"]),
                ops.grouped_mm_dw(s["dy"], s["x"], s["seg_start"], row_dy=s["row_out"]))
    if kind == "lora":
        return ops.lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"])
    return ops.lora_grad(s["dy"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"])


class _Padded:
    """Sorted rows laid out as [expert, place in its segment], with zeros where a segment is shorter."""

    def __init__(self, s):
        seg, rows = s["seg_start"].long(), s["row_out"].numel()
        r = torch.arange(rows, device="cuda")
        self.e = torch.searchsorted(seg, r, right=True) - 1
        self.p = r - seg[self.e]
        self.shape = (seg.numel() - 1, s["longest"])

    def spread(self, rows):
        out = torch.zeros((*self.shape, rows.shape[1]), dtype=torch.float32, device="cuda")
        out[self.e, self.p] = rows.float()
        return out

    def gather(self, padded):
        return padded[self.e, self.p]


def _product(s, rows, transposed=False):
    """W rows (or W^T rows) of every sorted row's expert, in 32 bits: with fewer rows than experts each row
    fetches its own matrix, otherwise one batched product over the padded segments."""
    if rows.shape[0] < s["seg_start"].numel() - 1:
        e = torch.searchsorted(s["seg_start"].long(), torch.arange(rows.shape[0], device="cuda"), right=True) - 1
        w = s["w"][e].float()
        w = w.transpose(1, 2).contiguous() if transposed else w
        return torch.bmm(w, rows.float().unsqueeze(2)).squeeze(2)
    pad = _Padded(s)
    if transposed:
        return pad.gather(torch.bmm(pad.spread(rows), s["w"].float()))
    return pad.gather(torch.bmm(s["w"].float(), pad.spread(rows).transpose(1, 2).contiguous()).transpose(1, 2))


def _weight_grad(s, dy, x):
    pad = _Padded(s)
    return torch.bmm(pad.spread(dy).transpose(1, 2).contiguous(), pad.spread(x))


def _scatter(s, rows):
    out = torch.empty_like(rows)
    out[s["row_out"].long()] = rows
    return out


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "plan":
        ids = s["ids"].reshape(-1).long()
        order = torch.argsort(ids, stable=True)
        seg = torch.searchsorted(ids[order], torch.arange(case["n_exp"] + 1, device="cuda"))
        return (order // case["k"]).to(torch.int32), order.to(torch.int32), seg.to(torch.int32)
    dt = s["x"].dtype
    if kind == "gate_up":
        gate, up = _product(s, s["x"][s["row_token"].long()]).chunk(2, 1)
        return (gate / (1 + torch.exp(-gate)) * up).to(dt)
    if kind == "down":
        return _scatter(s, _product(s, s["x"]).to(dt))
    if kind == "grad_up":
        dx = _product(s, s["dy"], transposed=True)
        dw = _weight_grad(s, s["dy"], s["x"][s["row_token"].long()])
        return _scatter(s, dx.to(dt)), dw.to(dt)
    if kind == "grad_down":
        dy = s["dy"][s["row_out"].long()]
        dh = _product(s, dy, transposed=True)
        gate, up = s["gu"].float().chunk(2, 1)
        sig = 1 / (1 + torch.exp(-gate))
        dgu = torch.cat([dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig], 1)
        return dgu.to(dt), _weight_grad(s, dy, s["x"]).to(dt)
    # the factors of all adapters side by side: one product with each, the other adapters' places masked to zero
    ids, R = s["ids"].long(), case["rank"]
    mine = torch.arange(case["n_ad"], device="cuda").repeat_interleave(R) == ids.unsqueeze(1)
    scale = torch.where(mine, s["scale"].repeat_interleave(R), 0.0)
    a = s["a"].float().reshape(-1, case["n_in"])
    b = s["b"].float().transpose(1, 2).reshape(-1, case["n_out"])
    x = s["x"].float()
    v = scale * (x @ a.T)
    if kind == "lora":
        return (s["base"].float() + v @ b).to(dt)
    dy = s["dy"].float()
    dv = scale * (dy @ b.T)
    da = (dv.T @ x).reshape(s["a"].shape)
    db = (v.T @ dy).reshape(case["n_ad"], R, -1).transpose(1, 2)
    return (dv @ a).to(dt), da.to(dt), db.to(dt).contiguous()


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        m = case["tokens"] * case["k"]
        return {"bytes": 12 * m + 4 * (case["n_exp"] + 1), "flops": m}
    if kind in ("lora", "lora_grad"):
        T, R, K, N = case["tokens"], case["rank"], case["n_in"], case["n_out"]
        used = min(case["requests"], case["n_ad"], T)
        if kind == "lora":
            return {"bytes": 2 * T * (K + 2 * N) + 4 * T + 2 * used * R * (K + N), "flops": 2 * T * R * (K + N)}
        return {"bytes": 2 * T * (2 * K + N) + 4 * T + 2 * (used + case["n_ad"]) * R * (K + N), "flops": 6 * T * R * (K + N)}
    T, k, E, H, I = case["tokens"], case["k"], case["n_exp"], case["hidden"], case["inter"]
    m = T * k
    touched = E * (1.0 - (1.0 - k / E) ** T)
    if kind == "gate_up":
        return {"bytes": 2 * (touched * 2 * I * H + T * H + m * I), "flops": 4 * m * H * I}
    if kind == "down":
        return {"bytes": 2 * (touched * I * H + m * (H + I)), "flops": 2 * m * H * I}
    if kind == "grad_up":
        return {"bytes": 2 * ((touched + E) * 2 * I * H + T * H + m * (2 * I + H)), "flops": 8 * m * H * I}
    return {"bytes": 2 * ((touched + E) * I * H + m * (H + 5 * I)), "flops": 4 * m * H * I}


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None
    x = s["x"].double()
    if kind in ("lora", "lora_grad"):
        out = s["base"].double() if kind == "lora" else torch.zeros_like(x)
        da, db = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
        for j in range(case["n_ad"]):
            rows = (s["ids"] == j).nonzero()[:, 0]
            a, b, c = s["a"][j].double(), s["b"][j].double(), s["scale"][j].double()
            v = x[rows] @ a.T
            if kind == "lora":
                out[rows] += c * (v @ b.T)
            else:
                dy = s["dy"][rows].double()
                dv = c * (dy @ b)
                out[rows] = dv @ a
                da[j] = dv.T @ x[rows]
                db[j] = c * (dy.T @ v)
        return out if kind == "lora" else (out, da, db)
    starts = s["seg_start"].tolist()
    m = s["row_out"].numel()
    tok, place = s["row_token"].long(), s["row_out"].long()
    w = s["w"]
    if kind == "gate_up":
        out = torch.empty((m, case["inter"]), dtype=torch.float64, device="cuda")
    elif kind == "grad_down":
        out = torch.empty((m, 2 * case["inter"]), dtype=torch.float64, device="cuda")
    else:
        out = torch.empty((m, case["hidden"]), dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda") if kind.startswith("grad") else None
    for e in range(case["n_exp"]):
        r0, r1 = starts[e], starts[e + 1]
        if r0 == r1:
            continue
        we, at = w[e].double(), place[r0:r1]
        if kind == "gate_up":
            y = x[tok[r0:r1]] @ we.T
            gate, up = y[:, :case["inter"]], y[:, case["inter"]:]
            out[r0:r1] = gate * torch.sigmoid(gate) * up
        elif kind == "down":
            out[at] = x[r0:r1] @ we.T
        elif kind == "grad_up":
            dy = s["dy"][r0:r1].double()
            out[at] = dy @ we
            dw[e] = dy.T @ x[tok[r0:r1]]
        else:
            dy = s["dy"][at].double()
            dh = dy @ we
            gate, up = s["gu"][r0:r1].double().chunk(2, 1)
            sg = torch.sigmoid(gate)
            out[r0:r1] = torch.cat([dh * up * (sg + gate * sg * (1 - sg)), dh * gate * sg], 1)
            dw[e] = dy.T @ x[r0:r1]
    return out if dw is None else (out, dw)
