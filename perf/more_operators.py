"""The operators around the unquantised experts of a layer in training and serving, as cases to time and compare.

A case is a dict of plain values with a "kind":

  route         router logits of a batch -> each token's experts and their weights: softmax or sigmoid scores, a bias for
                balance that only the choice sees, groups of experts of which a few are kept, renormalised weights
  route_grad    the gradient of those weights in the logits
  combine       the weighted sum of a token's per-expert rows, plus a residual
  combine_grad  its gradients: a row per (token, k), and the weights'
  linear        a projection that all tokens share (router, shared expert): act(x W^T + bias) + residual
  linear_grad   its gradients in x, W and the bias, from the pre-activations that the forward pass kept
  clip          the norm of all gradients of a step, and the gradients scaled to at most a given norm

Sizes are those of the repository's workloads (512 experts, top-10, 2048 x 512; 240 experts, top-9; the checkpoint's
2560 x 640; 48 layers of adapters; 16 experts of 4096 x 1024), or generic ones.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a batch of decoding requests, one token each: the smallest call, all latency
        {"name": "route_decode", "kind": "route", "tokens": 8, "n_exp": 512, "k": 10, "dtype": "fp32", "score": "softmax",
         "renorm": True, "bias": False, "n_group": 1, "topk_group": 1, "group_best": 1, "scale": 1.0},
        # a long prompt
        {"name": "route_prompt", "kind": "route", "tokens": 16384, "n_exp": 512, "k": 10, "dtype": "fp32", "score": "softmax",
         "renorm": True, "bias": False, "n_group": 1, "topk_group": 1, "group_best": 1, "scale": 1.0},
        # a ragged training batch with a balancing bias and groups of 30 experts, logits in 16 bits
        {"name": "route_groups", "kind": "route", "tokens": 5001, "n_exp": 240, "k": 9, "dtype": "bf16", "score": "sigmoid",
         "renorm": True, "bias": True, "n_group": 8, "topk_group": 4, "group_best": 2, "scale": 2.5},
        # backward of the router of a training batch whose weights are plain softmax values: every logit has a gradient
        {"name": "route_grad_long", "kind": "route_grad", "tokens": 8192, "n_exp": 512, "k": 10, "dtype": "fp32",
         "score": "softmax", "renorm": False, "scale": 1.0},
        # the ordinary prompt chunk of the checkpoint's shape
        {"name": "combine_chunk", "kind": "combine", "tokens": 512, "k": 10, "hidden": 2560, "dtype": "fp16", "residual": True},
        # backward of a training batch over few large experts
        {"name": "combine_grad_few", "kind": "combine_grad", "tokens": 8192, "k": 4, "hidden": 4096, "dtype": "bf16"},
        # eight requests decoding: a shared expert's output projection onto the residual stream, all weight bytes
        {"name": "linear_decode", "kind": "linear", "tokens": 8, "n_in": 2048, "n_out": 2048, "dtype": "bf16", "out": "bf16",
         "bias": True, "act": "none", "residual": True, "keep": False},
        # the router of a training batch: logits in 32 bits
        {"name": "linear_router", "kind": "linear", "tokens": 4096, "n_in": 2048, "n_out": 512, "dtype": "bf16", "out": "fp32",
         "bias": False, "act": "none", "residual": False, "keep": False},
        # a shared expert's first projection in a long training batch, its pre-activations kept
        {"name": "linear_large", "kind": "linear", "tokens": 8192, "n_in": 4096, "n_out": 4096, "dtype": "bf16", "out": "bf16",
         "bias": True, "act": "gelu", "residual": False, "keep": True},
        # backward of an odd batch through silu, the checkpoint's shape
        {"name": "linear_grad_odd", "kind": "linear_grad", "tokens": 1999, "n_in": 2560, "n_out": 640, "dtype": "fp16",
         "bias": True, "act": "silu"},
        # adapters of 48 layers, two factors of four projections each: many small gradients, norm within the limit
        {"name": "clip_adapters", "kind": "clip", "sizes": "96x32768 192x40960 96x10240", "dtype": "bf16", "clipped": False},
        # two layers of 16 experts of 4096 x 1024, their routers and norms: few large gradients, scaled into the optimizer's
        # buffers
        {"name": "clip_experts", "kind": "clip", "sizes": "2x134217728 2x67108864 2x65536 2x4096", "dtype": "bf16", "clipped": True},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of step between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, step * round(v / step))))


def draw(rng):
    kind = rng.choice(["route", "route", "route_grad", "combine", "combine_grad", "linear", "linear", "linear_grad", "clip"])
    half = rng.choice(["bf16", "fp16"])
    if kind in ("route", "route_grad"):
        n_group = rng.choice([1, 1, 2, 4, 8, 16]) if kind == "route" else 1
        per = _log(rng, 2, 1024 // n_group)
        n_exp = n_group * per
        c = {"kind": kind, "tokens": _log(rng, 1, 16384), "n_exp": n_exp, "k": 1, "dtype": rng.choice(["fp32", "fp32", half]),
             "score": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
        if kind == "route":
            c.update(bias=rng.random() < 0.5, n_group=n_group, topk_group=rng.randint(1, n_group),
                     group_best=rng.choice([1, 2]) if n_group > 1 else 1)
            n_exp = c["topk_group"] * per
        c["k"] = rng.randint(1, min(16, n_exp))
        while c["tokens"] * c["n_exp"] > 16384 * 512 or (kind == "route_grad" and c["tokens"] * c["n_exp"] > 8192 * 512):
            c["tokens"] //= 2
        return c
    if kind in ("combine", "combine_grad"):
        c = {"kind": kind, "tokens": _log(rng, 1, 8192), "k": rng.randint(1, 10), "hidden": _log(rng, 64, 4096, 8), "dtype": half}
        if kind == "combine":
            c["residual"] = rng.random() < 0.5
        while c["tokens"] * c["k"] * c["hidden"] > (8192 * 4 * 4096 if kind == "combine_grad" else 4096 * 10 * 2560):
            c["tokens"] //= 2
        return c
    if kind in ("linear", "linear_grad"):
        c = {"kind": kind, "tokens": _log(rng, 1, 8192), "n_in": _log(rng, 64, 4096, 8), "n_out": _log(rng, 64, 4096, 8),
             "dtype": half, "bias": rng.random() < 0.5, "act": rng.choice(["none", "silu", "gelu", "relu2"])}
        if kind == "linear":
            c.update(out=rng.choice([half, half, "fp32"]), residual=rng.random() < 0.5, keep=rng.random() < 0.3)
        return c
    largest, left, sizes = _log(rng, 8, 1 << 26), 1 << 28, []
    for _ in range(_log(rng, 1, 400)):
        sizes.append(max(1, min(_log(rng, max(1, largest // 1000), largest), left // 8)))
        left -= sizes[-1]
    return {"kind": kind, "sizes": " ".join("1x%d" % n for n in sizes), "dtype": rng.choice(["bf16", "fp16", "fp32", "mixed"]),
            "clipped": rng.random() < 0.5}


# ---- inputs -------------------------------------------------------------------------------------

def _rand(shape, dtype, g, scale=1.0):
    t = torch.randn(shape, dtype=dtype, device="cuda", generator=g)
    return t.mul_(scale) if scale != 1.0 else t


def _logits(case, g):
    """Router logits: some experts are more popular than others."""
    popular = torch.randn(case["n_exp"], device="cuda", generator=g) * 0.5
    return (popular + 1.2 * torch.randn((case["tokens"], case["n_exp"]), device="cuda", generator=g)).to(_TYPES[case["dtype"]])


def _sizes(case):
    """Elements of each gradient, from "2x4096 1x7": two of 4096, one of 7."""
    return [int(n) for run in case["sizes"].split() for n in [run.split("x")[1]] * int(run.split("x")[0])]


def _grad_types(case):
    return ["bf16", "fp32", "fp16"] if case["dtype"] == "mixed" else [case["dtype"]]


def _views(flat, sizes):
    """The gradients: those of each type, in turn, next to each other in that type's buffer."""
    parts = [list(buf.split(sizes[i::len(flat)])) for i, buf in enumerate(flat)]
    return [parts[i % len(flat)][i // len(flat)] for i in range(len(sizes))]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    kind, s = case["kind"], {"case": case}
    if kind == "route":
        s["logits"] = _logits(case, g)
        s["bias"] = 0.05 * torch.randn(case["n_exp"], device="cuda", generator=g) if case["bias"] else None
    elif kind == "route_grad":
        s["logits"] = _logits(case, g)
        s["ids"] = s["logits"].float().topk(case["k"], dim=1).indices.to(torch.int32)
        s["dweights"] = torch.randn((case["tokens"], case["k"]), device="cuda", generator=g)
    elif kind in ("combine", "combine_grad"):
        dt = _TYPES[case["dtype"]]
        s["y"] = _rand((case["tokens"], case["k"], case["hidden"]), dt, g)
        s["weights"] = torch.softmax(torch.randn((case["tokens"], case["k"]), device="cuda", generator=g), 1)
        if kind == "combine":
            s["residual"] = _rand((case["tokens"], case["hidden"]), dt, g) if case["residual"] else None
        else:
            s["dout"] = _rand((case["tokens"], case["hidden"]), dt, g)
    elif kind in ("linear", "linear_grad"):
        T, K, N, dt = case["tokens"], case["n_in"], case["n_out"], _TYPES[case["dtype"]]
        s["x"] = _rand((T, K), dt, g)
        s["w"] = _rand((N, K), dt, g, K ** -0.5)
        if kind == "linear":
            s["bias"] = _rand((N,), dt, g, 0.5) if case["bias"] else None
            s["residual"] = _rand((T, N), dt, g) if case["residual"] else None
        else:
            s["dy"] = _rand((T, N), dt, g)
            s["z"] = _rand((T, N), dt, g) if case["act"] != "none" else None     # what the forward pass kept
    else:
        # the gradients are views of one buffer of each type, side by side, as data-parallel training keeps them
        types, sizes = _grad_types(case), _sizes(case)
        s["flat"] = [_rand((sum(sizes[i::len(types)]),), _TYPES[t], g, 0.01) for i, t in enumerate(types)]
        s["grads"] = _views(s["flat"], sizes)
        # A limit in reach leaves smaller gradients in place, which the next pass would find: those go to the optimizer's
        # own buffers.  Within the limit the gradients stay what they are.
        norm = 0.01 * math.sqrt(sum(sizes))
        s["max_norm"] = 0.37 * norm if case["clipped"] else 4 * norm + 1.0
        s["flat_out"] = [torch.empty_like(t) for t in s["flat"]] if case["clipped"] else None
        s["out"] = _views(s["flat_out"], sizes) if case["clipped"] else None
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _act(case):
    return None if case["act"] == "none" else case["act"]


def _own(s):
    if os.path.join(os.getcwd(), "moe-offload_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "moe-offload_amd"))
    from moe_offload import ops
    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        return ops.route(s["logits"], case["k"], score=case["score"], bias=s["bias"], n_group=case["n_group"],
                         topk_group=case["topk_group"], group_best=case["group_best"], renorm=case["renorm"], scale=case["scale"])
    if kind == "route_grad":
        return ops.route_grad(s["dweights"], s["logits"], s["ids"], score=case["score"], renorm=case["renorm"], scale=case["scale"])
    if kind == "combine":
        return ops.combine(s["y"], s["weights"], residual=s["residual"])
    if kind == "combine_grad":
        return ops.combine_grad(s["dout"], s["y"], s["weights"])
    if kind == "linear":
        z = torch.empty((case["tokens"], case["n_out"]), dtype=s["x"].dtype, device="cuda") if case["keep"] else None
        y = ops.linear(s["x"], s["w"], bias=s["bias"], act=_act(case), residual=s["residual"], z_out=z, dtype=_TYPES[case["out"]])
        return (y, z) if case["keep"] else y
    if kind == "linear_grad":
        dx, dw, db = ops.linear_grad(s["dy"], s["x"], s["w"], z=s["z"], act=_act(case), bias=case["bias"])
        return (dx, dw, db) if case["bias"] else (dx, dw)
    norm = ops.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
    return (norm, *(s["flat"] if s["out"] is None else s["flat_out"]))


def _scores(logits, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _activation(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return torch.where(z > 0, z * z, 0.0) if act == "relu2" else z


def _slope(z, act):
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    return torch.where(z > 0, 2 * z, 0.0)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        T, E, k, groups = case["tokens"], case["n_exp"], case["k"], case["n_group"]
        # scores next to each other decide who is chosen: 64 bits where a bias or a sum of them makes the order
        logits = s["logits"].double()
        scores = _scores(logits, case["score"])
        choice = logits if s["bias"] is None else scores + s["bias"].double()
        if groups > 1:
            of = choice if s["bias"] is not None or case["group_best"] == 1 else scores
            best = torch.sort(of.reshape(T, groups, E // groups), dim=2, descending=True).values[:, :, :case["group_best"]].sum(2)
            kept = torch.argsort(best, dim=1, descending=True, stable=True)[:, :case["topk_group"]]
            keep = torch.zeros((T, groups), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
            choice = torch.where(keep.repeat_interleave(E // groups, 1), choice, -math.inf)
        ids = torch.argsort(choice, dim=1, descending=True, stable=True)[:, :k]
        w = torch.gather(scores, 1, ids).float()
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return ids.to(torch.int32), w * case["scale"]
    if kind == "route_grad":
        logits, ids = s["logits"].float(), s["ids"].long()
        scores = _scores(logits, case["score"])
        w = torch.gather(scores, 1, ids)
        dw = s["dweights"] * case["scale"]
        if case["renorm"]:
            total = w.sum(1, keepdim=True)
            dw = (dw - (dw * w).sum(1, keepdim=True) / total) / total
        ds = torch.zeros_like(scores).scatter_(1, ids, dw)
        if case["score"] == "sigmoid":
            d = ds * scores * (1 - scores)
        else:
            d = scores * (ds - (ds * scores).sum(1, keepdim=True))
        return d.to(s["logits"].dtype)
    if kind == "combine":
        out = (s["weights"].unsqueeze(2) * s["y"].float()).sum(1)
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return out.to(s["y"].dtype)
    if kind == "combine_grad":
        dout = s["dout"].float().unsqueeze(1)
        return (s["weights"].unsqueeze(2) * dout).to(s["y"].dtype), (s["y"].float() * dout).sum(2)
    if kind == "linear":
        z = s["x"].float() @ s["w"].float().T
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _activation(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        y = y.to(_TYPES[case["out"]])
        return (y, z.to(s["x"].dtype)) if case["keep"] else y
    if kind == "linear_grad":
        dt = s["x"].dtype
        dz = s["dy"].float()
        if s["z"] is not None:
            dz = dz * _slope(s["z"].float(), case["act"])
        dx, dw = dz @ s["w"].float(), dz.T @ s["x"].float()
        return (dx.to(dt), dw.to(dt), dz.sum(0).to(dt)) if case["bias"] else (dx.to(dt), dw.to(dt))
    # the norm of hundreds of millions of values: squares in 32 bits, their sum in 64
    squares = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]])
    norm = torch.sqrt(squares.sum()).float()
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    out = s["grads"] if s["out"] is None else s["out"]
    for t, o in zip(s["grads"], out):
        o.copy_(t.float() * factor)
    return (norm, *(s["flat"] if s["out"] is None else s["flat_out"]))


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind in ("route", "route_grad"):
        T, E, k = case["tokens"], case["n_exp"], case["k"]
        if kind == "route":
            return {"bytes": T * (E * size + 8 * k) + (4 * E if case["bias"] else 0), "flops": 2 * T * E}
        read = k if case["renorm"] or case["score"] == "sigmoid" else E
        return {"bytes": T * ((E + read) * size + 8 * k), "flops": 2 * T * E}
    if kind in ("combine", "combine_grad"):
        T, k, H = case["tokens"], case["k"], case["hidden"]
        if kind == "combine":
            return {"bytes": T * (2 * H * (k + 1 + case["residual"]) + 4 * k), "flops": 2 * T * k * H}
        return {"bytes": T * (2 * H * (2 * k + 1) + 8 * k), "flops": 3 * T * k * H}
    if kind in ("linear", "linear_grad"):
        T, K, N = case["tokens"], case["n_in"], case["n_out"]
        if kind == "linear":
            out = (4 if case["out"] == "fp32" else 2) + 2 * case["residual"] + 2 * case["keep"]
            return {"bytes": 2 * (T * K + N * K + N * case["bias"]) + T * N * out, "flops": 2 * T * K * N}
        return {"bytes": 2 * (2 * T * K + 2 * N * K + T * N * (1 + (case["act"] != "none")) + N * case["bias"]), "flops": 4 * T * K * N}
    types, sizes = _grad_types(case), _sizes(case)
    total = sum(n * (4 if types[i % len(types)] == "fp32" else 2) for i, n in enumerate(sizes))
    return {"bytes": total * (2 if case["clipped"] else 1), "flops": 2 * sum(sizes)}


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        logits, E = s["logits"].double(), case["n_exp"]
        scores = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
        choice = logits if s["bias"] is None else scores + s["bias"].double()
        if case["n_group"] > 1:
            per = E // case["n_group"]
            of = (choice if s["bias"] is not None or case["group_best"] == 1 else scores).reshape(-1, case["n_group"], per)
            first, second = (of.topk(min(2, per), dim=2).values[:, :, i] for i in (0, min(1, per - 1)))
            ranks = first + second if case["group_best"] == 2 else first
            member = torch.arange(E, device="cuda") // per
            kept = torch.zeros_like(choice, dtype=torch.bool)
            for _ in range(case["topk_group"]):
                at = _first_largest(ranks)
                kept |= member == at
                ranks = ranks.scatter(1, at, -math.inf)
            choice = choice.masked_fill(~kept, -math.inf)
        ids = []
        for _ in range(case["k"]):
            ids.append(_first_largest(choice))
            choice = choice.scatter(1, ids[-1], -math.inf)
        ids = torch.cat(ids, 1)
        w = scores.gather(1, ids)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return ids.to(torch.int32), w * case["scale"]
    if kind == "route_grad":
        logits = s["logits"].double().requires_grad_()
        scores = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, 1)
        w = scores.gather(1, s["ids"].long())
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return torch.autograd.grad((w * case["scale"] * s["dweights"].double()).sum(), logits)[0]
    if kind == "combine":
        out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")
        if s["residual"] is not None:
            out += s["residual"]
        for j in range(case["k"]):
            out.addcmul_(s["weights"][:, j:j + 1].double(), s["y"][:, j].double())
        return out
    if kind == "combine_grad":
        dout = s["dout"].double()
        dy = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda")
        dw = torch.empty(s["weights"].shape, dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            torch.mul(dout, s["weights"][:, j:j + 1], out=dy[:, j])
            dw[:, j] = torch.linalg.vecdot(dout, s["y"][:, j].double())
        return dy, dw
    if kind == "linear":
        z = torch.nn.functional.linear(s["x"].double(), s["w"].double(), None if s["bias"] is None else s["bias"].double())
        y = _exact_activation(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"]
        return (y, z) if case["keep"] else y
    if kind == "linear_grad":
        dz = s["dy"].double()
        if s["z"] is not None:
            z = s["z"].double().requires_grad_()
            dz = torch.autograd.grad(_exact_activation(z, case["act"]), z, dz)[0]
        dx, dw = torch.mm(dz, s["w"].double()), torch.mm(dz.T.contiguous(), s["x"].double())
        return (dx, dw, dz.sum(0)) if case["bias"] else (dx, dw)
    norm = sum(float(torch.linalg.vector_norm(t, dtype=torch.float64)) ** 2 for t in s["flat"]) ** 0.5
    factor = min(1.0, s["max_norm"] / (norm + 1e-6))
    return (torch.tensor(norm, dtype=torch.float64, device="cuda"), *(t.double() * factor for t in s["flat"]))


def _first_largest(v):
    """The lowest index of each row's largest value, [rows, 1]."""
    at = torch.arange(v.shape[1], device="cuda")
    return torch.where(v == v.amax(1, keepdim=True), at, v.shape[1]).amin(1, keepdim=True)


def _exact_activation(z, act):
    f = torch.nn.functional
    if act == "silu":
        return f.silu(z)
    if act == "gelu":
        return f.gelu(z)
    return f.relu(z).square() if act == "relu2" else z
