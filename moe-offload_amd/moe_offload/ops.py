"""torch-facing wrappers of the HIP compute entry points (tensors in, tensors out).

Every function calls straight into libmoe_offload.so on torch's current HIP stream; there is
no PyTorch fallback for any of them.
"""
from __future__ import annotations

import torch

from . import _lib

_ROUTER_WS: dict[tuple[int, int], torch.Tensor] = {}


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream)


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def router_workspace(n_exp: int, device=None) -> torch.Tensor:
    """Zeroed scratch for one router launch site (logits + the block-done counter)."""
    dev = torch.device(device or "cuda")
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), n_exp)
    ws = _ROUTER_WS.get(key)
    if ws is None:
        nb = _lib.lib().moe_router_workspace_bytes(n_exp)
        ws = torch.zeros(int(nb), dtype=torch.uint8, device=dev)
        _ROUTER_WS[key] = ws
    return ws


def router(w: torch.Tensor, k: int, *, x: torch.Tensor | None = None, h: torch.Tensor | None = None,
           norm_w: torch.Tensor | None = None, eps: float = 1e-6, w_next: torch.Tensor | None = None,
           m: int = 12, x_out: torch.Tensor | None = None, ids: torch.Tensor | None = None,
           scores: torch.Tensor | None = None, pred: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None):
    """Fused router for one token.

    x: fp16 [hidden] input, or h: fp32 [hidden] residual to RMSNorm first (written to x_out).
    w: fp16 [n_exp, hidden].  Returns (ids int32 [k] ascending-gate order, scores fp16 [k],
    pred int32 [m] (next-layer prediction, descending) or None).
    """
    n_exp, hidden = w.shape
    assert w.dtype == torch.float16 and w.is_contiguous()
    assert (x is None) != (h is None)
    if x is not None:
        assert x.dtype == torch.float16 and x.numel() == hidden and x.is_contiguous()
    if h is not None:
        assert h.dtype == torch.float32 and h.numel() == hidden and h.is_contiguous()
    if w_next is not None:
        assert w_next.shape == w.shape and w_next.dtype == torch.float16 and w_next.is_contiguous()
    dev = w.device
    ids = ids if ids is not None else torch.empty(k, dtype=torch.int32, device=dev)
    scores = scores if scores is not None else torch.empty(k, dtype=torch.float16, device=dev)
    if w_next is not None and pred is None:
        pred = torch.empty(m, dtype=torch.int32, device=dev)
    ws = workspace if workspace is not None else router_workspace(n_exp, dev)
    rc = _lib.lib().moe_router(_p(h), _p(norm_w), eps, _p(x), _p(x_out), _p(w), _p(w_next), hidden, n_exp, k,
                               m if w_next is not None else 0, _p(ws), _p(ids), _p(scores), _p(pred), _stream())
    _lib.check(rc, "moe_router")
    return ids, scores, (pred if w_next is not None else None)


def rmsnorm(h: torch.Tensor, norm_w: torch.Tensor | None, eps: float = 1e-6, out: torch.Tensor | None = None):
    """fp16 RMSNorm of an fp32 vector (fp64 math, one rounding)."""
    assert h.dtype == torch.float32 and h.is_contiguous()
    out = out if out is not None else torch.empty(h.numel(), dtype=torch.float16, device=h.device)
    rc = _lib.lib().moe_rmsnorm(_p(h), _p(norm_w), eps, h.numel(), _p(out), _stream())
    _lib.check(rc, "moe_rmsnorm")
    return out


def q2_switch_glu(x: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor, hidden: int, inter: int,
                  group: int = 64, scores: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                  per_expert: bool = False, h_ws: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """SwitchGLU over the Q2 blobs pool[slots[j]] for one token.

    Returns fp32 [hidden] = residual + sum_j scores[j] * expert_j(x), or fp32 [k, hidden] of
    per-expert outputs when per_expert.
    """
    k = slots.numel()
    assert x.dtype == torch.float16 and x.numel() == hidden and x.is_contiguous()
    assert pool.dtype == torch.uint8 and pool.dim() == 2 and pool.is_contiguous()
    assert slots.dtype == torch.int32 and slots.is_contiguous()
    dev = x.device
    if h_ws is None:
        h_ws = torch.empty(k * inter, dtype=torch.float16, device=dev)
    if out is None:
        out = torch.empty((k, hidden) if per_expert else (hidden,), dtype=torch.float32, device=dev)
    rc = _lib.lib().moe_q2_switch_glu(_p(x), _p(pool), pool.shape[1], pool.shape[0], _p(slots), _p(scores), k,
                                      hidden, inter,
                                      group, _p(residual), _p(h_ws), _p(out), int(per_expert), _stream())
    _lib.check(rc, "moe_q2_switch_glu")
    return out


def q2_gate_up(x, pool, slots, hidden, inter, group=64, h_out=None):
    k = slots.numel()
    h_out = h_out if h_out is not None else torch.empty(k * inter, dtype=torch.float16, device=x.device)
    rc = _lib.lib().moe_q2_gate_up(_p(x), _p(pool), pool.shape[1], pool.shape[0], _p(slots), k, hidden, inter,
                                   group, _p(h_out), _stream())
    _lib.check(rc, "moe_q2_gate_up")
    return h_out


def q2_down(h, pool, slots, hidden, inter, group=64, scores=None, residual=None, per_expert=False, out=None):
    k = slots.numel()
    if out is None:
        out = torch.empty((k, hidden) if per_expert else (hidden,), dtype=torch.float32, device=h.device)
    rc = _lib.lib().moe_q2_down(_p(h), _p(pool), pool.shape[1], pool.shape[0], _p(slots), _p(scores), k, hidden,
                                inter, group,
                                _p(residual), _p(out), int(per_expert), _stream())
    _lib.check(rc, "moe_q2_down")
    return out


def q2_grouped_gate_up(x, row_token, seg_start, pool, hidden, inter, group=64, seg_slot=None, h_out=None):
    """h[r] = silu(G x[row_token[r]]) * (U x[row_token[r]]) for rows sorted by expert.

    x: fp16 [n_tok, hidden]; row_token int32 [M]; seg_start int32 [n_seg + 1] (segment u = rows
    seg_start[u]:seg_start[u+1], weights pool[seg_slot[u]], or pool[u] when seg_slot is None).
    Returns fp16 [M, inter].
    """
    n_tok, M, n_seg = x.shape[0], row_token.numel(), seg_start.numel() - 1
    h_out = h_out if h_out is not None else torch.empty((M, inter), dtype=torch.float16, device=x.device)
    rc = _lib.lib().moe_q2_grouped_gate_up(_p(x), n_tok, _p(row_token), M, _p(seg_start), _p(seg_slot), n_seg,
                                           _p(pool), pool.shape[1], pool.shape[0], hidden, inter, group, _p(h_out),
                                           _stream())
    _lib.check(rc, "moe_q2_grouped_gate_up")
    return h_out


def q2_grouped_down(h, seg_start, pool, hidden, inter, group=64, row_out=None, n_out_rows=None, seg_slot=None,
                    out=None):
    """y[row_out[r]] = D h[r] (fp16) for rows sorted by expert; row_out None writes row r."""
    M, n_seg = h.shape[0], seg_start.numel() - 1
    n_out = n_out_rows if n_out_rows is not None else M
    out = out if out is not None else torch.empty((n_out, hidden), dtype=torch.float16, device=h.device)
    rc = _lib.lib().moe_q2_grouped_down(_p(h), M, _p(row_out), n_out, _p(seg_start), _p(seg_slot), n_seg, _p(pool),
                                        pool.shape[1], pool.shape[0], hidden, inter, group, _p(out), _stream())
    _lib.check(rc, "moe_q2_grouped_down")
    return out


def q2_grouped_switch_glu(x, row_token, seg_start, pool, hidden, inter, group=64, row_out=None, n_out_rows=None,
                          seg_slot=None, h_ws=None, out=None):
    """Both grouped projections: fp16 [n_out_rows, hidden] per-(token, k) SwitchGLU outputs."""
    n_tok, M, n_seg = x.shape[0], row_token.numel(), seg_start.numel() - 1
    n_out = n_out_rows if n_out_rows is not None else M
    h_ws = h_ws if h_ws is not None else torch.empty((M, inter), dtype=torch.float16, device=x.device)
    out = out if out is not None else torch.empty((n_out, hidden), dtype=torch.float16, device=x.device)
    rc = _lib.lib().moe_q2_grouped_switch_glu(_p(x), n_tok, _p(row_token), _p(row_out), M, n_out, _p(seg_start),
                                              _p(seg_slot), n_seg, _p(pool), pool.shape[1], pool.shape[0], hidden,
                                              inter, group, _p(h_ws), _p(out), _stream())
    _lib.check(rc, "moe_q2_grouped_switch_glu")
    return out


def pair_combine(y, scores, residual=None, out=None):
    """out fp32 [n_tok, hidden] = residual + sum_j scores[t, j] * y[t*k + j].

    y (a row per (token, k)), scores [n_tok, k] and residual [n_tok, hidden] are fp16 and contiguous; no gradient.
    """
    n_tok, k = scores.shape
    hidden = y.shape[-1]
    for name, t, dtype, n in (("y", y, torch.float16, n_tok * k * hidden), ("scores", scores, torch.float16, n_tok * k),
                              ("residual", residual, torch.float16, n_tok * hidden), ("out", out, torch.float32, n_tok * hidden)):
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"pair_combine: {name} is {t.dtype}, not {dtype}")
        if not t.is_contiguous() or t.numel() < n:
            raise ValueError(f"pair_combine: {name} of shape {tuple(t.shape)} must be contiguous with {n} values for {n_tok} tokens")
    out = out if out is not None else torch.empty((n_tok, hidden), dtype=torch.float32, device=y.device)
    rc = _lib.lib().moe_pair_combine(_p(y), _p(scores), _p(residual), n_tok, k, hidden, _p(out), _stream())
    _lib.check(rc, "moe_pair_combine")
    return out


# ---- 2-bit codebook experts (non-gated: up -> squared ReLU -> down) ---------------------------

def cb_moe(x: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor, grid: torch.Tensor, hidden: int, inter: int,
           scores: torch.Tensor | None = None, residual: torch.Tensor | None = None, per_expert: bool = False,
           h_ws: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """Codebook experts pool[slots[j]] (format of moe_offload.cbformat) for one token.

    Returns fp32 [hidden] = residual + sum_j scores[j] * down_j(relu(up_j x)^2), or fp32
    [k, hidden] per-expert outputs when per_expert.  grid: device uint8 [256, 8]."""
    k = slots.numel()
    assert x.dtype == torch.float16 and x.numel() == hidden and x.is_contiguous()
    assert pool.dtype == torch.uint8 and pool.dim() == 2 and pool.is_contiguous()
    assert slots.dtype == torch.int32 and slots.is_contiguous()
    assert grid.dtype == torch.uint8 and grid.numel() == 256 * 8 and grid.is_cuda
    dev = x.device
    if h_ws is None:
        h_ws = torch.empty(k * inter, dtype=torch.bfloat16, device=dev)
    if out is None:
        out = torch.empty((k, hidden) if per_expert else (hidden,), dtype=torch.float32, device=dev)
    rc = _lib.lib().moe_cb_moe(_p(x), _p(pool), pool.shape[1], pool.shape[0], _p(slots), _p(scores), k, hidden, inter,
                               _p(grid), _p(residual), _p(h_ws), _p(out), int(per_expert), _stream())
    _lib.check(rc, "moe_cb_moe")
    return out


def cb_up(x, pool, slots, grid, hidden, inter, h_out=None):
    """bf16 [k, inter] = relu(up_j x)^2."""
    k = slots.numel()
    h_out = h_out if h_out is not None else torch.empty((k, inter), dtype=torch.bfloat16, device=x.device)
    rc = _lib.lib().moe_cb_up(_p(x), _p(pool), pool.shape[1], pool.shape[0], _p(slots), k, hidden, inter, _p(grid),
                              _p(h_out), _stream())
    _lib.check(rc, "moe_cb_up")
    return h_out


# ---- unquantised experts (fp16 / bf16): sorted rows, their products and gradients ---------------

_HALF = {torch.float16: 0, torch.bfloat16: 1}


def _one_gpu(who: str, names: str, *tensors) -> int:
    """The index of the one GPU that every given tensor is on (names: theirs, in order)."""
    dev = None
    for i, t in enumerate(tensors):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{who}: {names.split()[i]} must be a tensor, not {type(t).__name__}")
        at = t.get_device()
        if at == dev:
            continue
        if at < 0:
            raise ValueError(f"{who}: {names.split()[i]} is on {t.device}, not on a GPU")
        if dev is not None:
            raise ValueError(f"{who}: {names.split()[i]} is on GPU {at}, others on GPU {dev}")
        dev = at
    return dev


# sizes go to the library as 32-bit integers, which ctypes would cut without a word
_MAX_SIDE = 2 ** 30


def _rows(who: str, name: str, t: torch.Tensor, dtype: torch.dtype, rows: int | None, width: int | None) -> int:
    """Checks a matrix with contiguous rows; returns the elements from row to row."""
    shape = t.shape
    if t.dtype != dtype:
        raise TypeError(f"{who}: {name} is {t.dtype}, not {dtype}")
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (width is not None and shape[1] != width):
        raise ValueError(f"{who}: {name} has shape {tuple(shape)}, not ({'*' if rows is None else rows}, "
                         f"{'*' if width is None else width})")
    n, w = shape
    if n > _MAX_SIDE or w > _MAX_SIDE:
        raise ValueError(f"{who}: {name}: {n} rows of {w} elements (up to 2^30)")
    step, inner = t.stride()
    if w % 8 or w == 0:
        raise ValueError(f"{who}: {name}: rows of {w} elements (a multiple of 8 wanted)")
    if n == 0 or (n == 1 and inner == 1):
        return w
    if inner != 1 or step < w or step % 8:
        raise ValueError(f"{who}: {name}: rows must be contiguous and a multiple of 8 elements apart, not {t.stride()}")
    return step


def _mats(who: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> int:
    """Checks a stack of contiguous matrices; returns the elements from one to the next."""
    have = t.shape
    if t.dtype != dtype:
        raise TypeError(f"{who}: {name} is {t.dtype}, not {dtype}")
    if len(have) != 3 or any(s is not None and s != d for s, d in zip(shape, have)):
        raise ValueError(f"{who}: {name} has shape {tuple(have)}, not {tuple('*' if s is None else s for s in shape)}")
    m, n, k = have
    if m > _MAX_SIDE or n > _MAX_SIDE or k > _MAX_SIDE:
        raise ValueError(f"{who}: {name}: {m} matrices of {n} x {k} (up to 2^30)")
    if n % 8 or n == 0 or k % 8 or k == 0:
        raise ValueError(f"{who}: {name}: matrices of {n} x {k} (multiples of 8 wanted)")
    if m == 0:
        return n * k
    step, row, inner = t.stride()
    if inner != 1 or row != k or (m > 1 and (step < n * k or step % 8)):
        raise ValueError(f"{who}: {name}: matrices must be contiguous and a multiple of 8 elements apart, not {t.stride()}")
    return step if m > 1 else n * k


def _index(who: str, name: str, t: torch.Tensor | None, n: int | None = None) -> None:
    if t is None:
        return
    if t.dtype != torch.int32:
        raise TypeError(f"{who}: {name} is {t.dtype}, not torch.int32")
    if t.numel() > _MAX_SIDE:
        raise ValueError(f"{who}: {name} has {t.numel()} entries (up to 2^30)")
    if not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{who}: {name} must be contiguous" + ("" if n is None else f" with {n} entries, not {t.numel()}"))


def _scale(who: str, t: torch.Tensor | None, n: int) -> None:
    if t is None:
        return
    if t.dtype != torch.float32:
        raise TypeError(f"{who}: scale is {t.dtype}, not torch.float32")
    if not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{who}: scale must be contiguous with {n} entries")


def _half(who: str, t: torch.Tensor) -> int:
    dt = _HALF.get(t.dtype)
    if dt is None:
        raise TypeError(f"{who}: {t.dtype} (torch.float16 and torch.bfloat16 are supported)")
    return dt


# the current stream's handle without a Stream object around it, where torch has that (a microsecond per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(name: str, dev: int, *args) -> None:
    """Calls an entry point on the tensors' own GPU and that GPU's current stream."""
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    _lib.check(rc, name)


def _scratch(nbytes: int, like: torch.Tensor, given: torch.Tensor | None, who: str) -> torch.Tensor:
    """A call's own scratch: given, or new from torch's allocator (which keeps it for the stream, or the graph)."""
    if given is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    have = given.numel() * given.element_size()
    if not given.is_contiguous() or have < nbytes:
        raise ValueError(f"{who}: a contiguous workspace of {nbytes} bytes is wanted, not {have}")
    return given


def _fresh_rows(n_out_rows: int | None, n_rows: int, width: int, like: torch.Tensor) -> torch.Tensor:
    """A new output.  With a row for each sorted row the kernels write all of them themselves."""
    make = torch.empty if n_out_rows is None else torch.zeros
    return make((n_rows if n_out_rows is None else n_out_rows, width), dtype=like.dtype, device=like.device)


def expert_plan(ids: torch.Tensor, n_exp: int, row_token: torch.Tensor | None = None, row_out: torch.Tensor | None = None,
                seg_start: torch.Tensor | None = None):
    """The row plan of prefill.resident_plan, made on the GPU: the (token, k) pairs sorted by expert.

    ids: int32 [n_tok, k] (or [n_tok]: k = 1).  Returns int32 (row_token [M], row_out [M], seg_start
    [n_exp + 1]): sorted row r is pair row_out[r] (= token * k + j) of token row_token[r]; expert e has
    rows seg_start[e]:seg_start[e + 1], in pair order.  One segment per expert, empty ones too, so the
    slot is the expert id and no seg_slot is needed.  Pairs with an id outside 0 .. n_exp - 1 come
    behind the last segment.  n_exp up to 1024.
    """
    who = "expert_plan"
    dev = _one_gpu(who, "ids row_token row_out seg_start", ids, row_token, row_out, seg_start)
    _index(who, "ids", ids)
    if ids.dim() not in (1, 2) or not 1 <= n_exp <= 1024:
        raise ValueError(f"{who}: ids of shape {tuple(ids.shape)}, n_exp={n_exp} (ids [n_tok, k] or [n_tok], n_exp 1..1024)")
    k = ids.shape[1] if ids.dim() == 2 else 1
    m = ids.numel()
    if row_token is None and row_out is None and seg_start is None:
        row_token, row_out, seg_start = torch.empty(2 * m + n_exp + 1, dtype=torch.int32, device=ids.device).split((m, m, n_exp + 1))
    if row_token is None:
        row_token = torch.empty(m, dtype=torch.int32, device=ids.device)
    if row_out is None:
        row_out = torch.empty(m, dtype=torch.int32, device=ids.device)
    if seg_start is None:
        seg_start = torch.empty(n_exp + 1, dtype=torch.int32, device=ids.device)
    for name, t, n in (("row_token", row_token, m), ("row_out", row_out, m), ("seg_start", seg_start, n_exp + 1)):
        _index(who, name, t, n)
    nb = _lib.lib().moe_expert_plan_workspace_bytes(m, n_exp)
    ws = _scratch(nb, ids, None, who) if nb else None
    _call("moe_expert_plan", dev, _p(ids), m, max(k, 1), n_exp, _p(ws), _p(row_token), _p(row_out), _p(seg_start))
    return row_token, row_out, seg_start


def _segments(who, seg_start, seg_slot):
    _index(who, "seg_start", seg_start)
    n_seg = seg_start.numel() - 1
    if not 0 <= n_seg <= 1024:
        raise ValueError(f"{who}: seg_start has {n_seg + 1} entries (1..1025)")
    _index(who, "seg_slot", seg_slot, n_seg)
    return n_seg


def grouped_mm(x, seg_start, w, row_in=None, row_out=None, n_out_rows=None, seg_slot=None, scale=None, out=None):
    """y[row_out[r]] = scale[s] * (w[s] @ x[row_in[r]]) for rows r sorted into segments, s the segment's slot.

    x: fp16 or bf16 [*, K]; w: same type [n_slots, N, K]; segment u is rows seg_start[u]:seg_start[u + 1]
    with slot seg_slot[u] (u when None).  row_in / row_out None: row r.  The number of sorted rows is
    row_in's or row_out's, else x's.  A new output has n_out_rows rows, or as many as there are sorted rows
    (row_out must then name each of its rows once, as expert_plan's does); rows of no segment, or of one whose slot is
    outside w, are zeros in it and left as they are in a given `out`.  A row_in outside x gives a row of
    zeros, a row_out outside the output is dropped.  Outputs, here and below, must not overlap inputs.
    """
    who = "grouped_mm"
    dev = _one_gpu(who, "x seg_start w row_in row_out seg_slot scale out", x, seg_start, w, row_in, row_out, seg_slot, scale, out)
    dt = _half(who, x)
    n_seg = _segments(who, seg_start, seg_slot)
    w_stride = _mats(who, "w", w, x.dtype, (None, None, None))
    n_slots, N, K = w.shape
    ldx = _rows(who, "x", x, x.dtype, None, K)
    n_rows = row_in.numel() if row_in is not None else row_out.numel() if row_out is not None else x.shape[0]
    _index(who, "row_in", row_in, n_rows)
    _index(who, "row_out", row_out, n_rows)
    _scale(who, scale, n_slots)
    fill = out is None
    if fill:
        out = _fresh_rows(n_out_rows, n_rows, N, x)
    ldy = _rows(who, "out", out, x.dtype, n_out_rows, N)
    if (row_in is None and n_rows > x.shape[0]) or (row_out is None and n_rows > out.shape[0]):
        raise ValueError(f"{who}: {n_rows} sorted rows, x has {x.shape[0]} and out {out.shape[0]}")
    _call("moe_grouped_mm", dev, _p(x), ldx, x.shape[0], _p(row_in), _p(seg_start), _p(seg_slot), n_seg, n_rows, _p(w),
          w_stride, n_slots, N, K, _p(scale), _p(out), ldy, out.shape[0], _p(row_out), dt, int(fill))
    return out


def grouped_gate_up(x, row_token, seg_start, w, seg_slot=None, h_out=None, gu_out=None):
    """h[r] = silu(g) * u, (g, u) = w[slot] @ x[row_token[r]], for rows sorted by expert (row_token None: row r).

    x: fp16 or bf16 [n_tok, hidden]; w: same type [n_slots, 2 * inter, hidden], a slot's inter gate rows
    before its inter up rows; seg_start, seg_slot as grouped_mm.  gu_out ([M, 2 * inter], optional)
    receives (g, u) for grouped_mm_dx.  Returns [M, inter]; rows of no valid segment are zeros, in gu_out
    too, if h_out is None, and left as they are in both if it is given.
    """
    who = "grouped_gate_up"
    dev = _one_gpu(who, "x row_token seg_start w seg_slot h_out gu_out", x, row_token, seg_start, w, seg_slot, h_out, gu_out)
    dt = _half(who, x)
    n_seg = _segments(who, seg_start, seg_slot)
    w_stride = _mats(who, "w", w, x.dtype, (None, None, None))
    n_slots, N, K = w.shape
    if N % 16:
        raise ValueError(f"{who}: w has {N} rows per slot: twice a multiple of 8 wanted")
    ldx = _rows(who, "x", x, x.dtype, None, K)
    M = row_token.numel() if row_token is not None else x.shape[0]
    _index(who, "row_token", row_token, M)
    fill = h_out is None
    if fill:
        h_out = torch.empty((M, N // 2), dtype=x.dtype, device=x.device)
    ldh = _rows(who, "h_out", h_out, x.dtype, M, N // 2)
    ldgu = _rows(who, "gu_out", gu_out, x.dtype, M, N) if gu_out is not None else 0
    _call("moe_grouped_gate_up", dev, _p(x), ldx, x.shape[0], _p(row_token), _p(seg_start), _p(seg_slot), n_seg, M, _p(w),
          w_stride, n_slots, N // 2, K, _p(h_out), ldh, _p(gu_out), ldgu, dt, int(fill))
    return h_out


def grouped_switch_glu(x, row_token, seg_start, w_gate_up, w_down, row_out=None, n_out_rows=None, seg_slot=None, h_ws=None,
                       out=None):
    """Both projections of unquantised experts, as q2_grouped_switch_glu has them for 2-bit ones:
    [n_out_rows, hidden] per-(token, k) SwitchGLU outputs, sorted row r written at row_out[r]."""
    h = grouped_gate_up(x, row_token, seg_start, w_gate_up, seg_slot=seg_slot, h_out=h_ws)
    return grouped_mm(h, seg_start, w_down, row_out=row_out, n_out_rows=n_out_rows, seg_slot=seg_slot, out=out)


def grouped_mm_dx(dy, seg_start, w, row_in=None, row_out=None, n_out_rows=None, seg_slot=None, scale=None, gu=None, out=None):
    """dx[row_out[r]] = scale[s] * (w[s]^T @ dy[row_in[r]]): grouped_mm's gradient in x, one row per sorted row.

    Where grouped_mm read x[a[r]] and wrote y[b[r]], this takes row_in=b and writes one row per sorted
    row; rows of x read several times get the sum of theirs from the caller (row_out = the pairs' order,
    then a sum over k).  gu: w's input was grouped_gate_up's h, and gu the (g, u) it kept, [M, 2 * K] in
    sorted order; the result is then the gradient of (g, u), [*, 2 * K] (an infinite g, past the type's range,
    has its limit's).  Other arguments as grouped_mm.
    """
    who = "grouped_mm_dx"
    dev = _one_gpu(who, "dy seg_start w row_in row_out seg_slot scale gu out", dy, seg_start, w, row_in, row_out, seg_slot, scale, gu, out)
    dt = _half(who, dy)
    n_seg = _segments(who, seg_start, seg_slot)
    w_stride = _mats(who, "w", w, dy.dtype, (None, None, None))
    n_slots, N, K = w.shape
    width = K if gu is None else 2 * K
    lddy = _rows(who, "dy", dy, dy.dtype, None, N)
    n_rows = row_in.numel() if row_in is not None else row_out.numel() if row_out is not None else dy.shape[0]
    _index(who, "row_in", row_in, n_rows)
    _index(who, "row_out", row_out, n_rows)
    _scale(who, scale, n_slots)
    ldgu = _rows(who, "gu", gu, dy.dtype, n_rows, width) if gu is not None else 0
    fill = out is None
    if fill:
        out = _fresh_rows(n_out_rows, n_rows, width, dy)
    lddx = _rows(who, "out", out, dy.dtype, n_out_rows, width)
    if (row_in is None and n_rows > dy.shape[0]) or (row_out is None and n_rows > out.shape[0]):
        raise ValueError(f"{who}: {n_rows} sorted rows, dy has {dy.shape[0]} and out {out.shape[0]}")
    _call("moe_grouped_mm_dx", dev, _p(dy), lddy, dy.shape[0], _p(row_in), _p(seg_start), _p(seg_slot), n_seg, n_rows,
          _p(w), w_stride, n_slots, N, K, _p(scale), _p(gu), ldgu, _p(out), lddx, out.shape[0], _p(row_out), dt, int(fill))
    return out


def grouped_mm_dw(dy, x, seg_start, row_dy=None, row_x=None, scale=None, dtype=None, out=None):
    """dw[u] = scale[u] * sum over the rows r of segment u of dy[row_dy[r]] (outer) x[row_x[r]]: [n_seg, N, K].

    grouped_mm's gradient in the weights, one matrix per segment (zeros for an empty one; segments that
    shared a slot are summed by the caller).  dtype: the inputs' (default) or torch.float32.  Where
    grouped_mm took row_in and row_out, this takes row_x=row_in and row_dy=row_out.
    """
    who = "grouped_mm_dw"
    dev = _one_gpu(who, "dy x seg_start row_dy row_x scale out", dy, x, seg_start, row_dy, row_x, scale, out)
    dt = _half(who, dy)
    n_seg = _segments(who, seg_start, None)
    lddy, ldx = _rows(who, "dy", dy, dy.dtype, None, None), _rows(who, "x", x, dy.dtype, None, None)
    N, K = dy.shape[1], x.shape[1]
    n_rows = row_dy.numel() if row_dy is not None else row_x.numel() if row_x is not None else dy.shape[0]
    _index(who, "row_dy", row_dy, n_rows)
    _index(who, "row_x", row_x, n_rows)
    if (row_dy is None and n_rows > dy.shape[0]) or (row_x is None and n_rows > x.shape[0]):
        raise ValueError(f"{who}: {n_rows} sorted rows, dy has {dy.shape[0]} and x {x.shape[0]}")
    _scale(who, scale, n_seg)
    dtype = dtype if dtype is not None else out.dtype if out is not None else dy.dtype
    if dtype not in (dy.dtype, torch.float32):
        raise TypeError(f"{who}: gradients of {dy.dtype} come as {dy.dtype} or torch.float32, not {dtype}")
    if out is None:
        out = torch.empty((n_seg, N, K), dtype=dtype, device=dy.device)
    stride = _mats(who, "out", out, dtype, (n_seg, N, K))
    _call("moe_grouped_mm_dw", dev, _p(dy), lddy, dy.shape[0], _p(row_dy), _p(x), ldx, x.shape[0], _p(row_x), _p(seg_start),
          n_seg, n_rows, N, K, _p(scale), _p(out), stride, int(dtype == torch.float32), dt)
    return out


# ---- low-rank adapters -------------------------------------------------------------------------

def _lora_args(who, x, a, b, ids, scale):
    dt = _half(who, x)
    if x.dim() != 2:
        raise ValueError(f"{who}: x has {x.dim()} dimensions")
    a_stride = _mats(who, "a", a, x.dtype, (None, None, x.shape[1]))
    n_ad, rank, n_in = a.shape
    if rank > 256:
        raise ValueError(f"{who}: rank {rank} (up to 256)")
    b_stride = _mats(who, "b", b, x.dtype, (n_ad, None, rank))
    _index(who, "ids", ids, x.shape[0])
    _scale(who, scale, n_ad)
    return dt, n_ad, rank, n_in, b.shape[1], a_stride, b_stride


def lora_add(base, x, a, b, ids, scale=None, out=None, workspace=None):
    """out[t] = base[t] + scale[i] * (b[i] @ (a[i] @ x[t])), i = ids[t]: each token's own request's adapter
    beside a projection that all share.

    base: fp16 or bf16 [n_tok, n_out], the shared projection's output; x: same type [n_tok, n_in]; a [n_ad,
    rank, n_in], b [n_ad, n_out, rank] (rank a multiple of 8 up to 256); ids: int32 [n_tok], an id outside
    the adapters leaves base[t]; scale: fp32 [n_ad] or None.  out=base adds in place.  workspace: scratch of
    moe_lora_workspace_bytes, for callers that keep one per call in flight.
    """
    who = "lora_add"
    dev = _one_gpu(who, "base x a b ids scale out workspace", base, x, a, b, ids, scale, out, workspace)
    dt, n_ad, rank, n_in, n_out, a_stride, b_stride = _lora_args(who, x, a, b, ids, scale)
    n_tok = x.shape[0]
    ldx = _rows(who, "x", x, x.dtype, n_tok, n_in)
    ld_base = _rows(who, "base", base, x.dtype, n_tok, n_out)
    if out is None:
        out = torch.empty((n_tok, n_out), dtype=x.dtype, device=x.device)
    ld_out = _rows(who, "out", out, x.dtype, n_tok, n_out)
    workspace = _scratch(4 * n_tok * rank, x, workspace, who)
    _call("moe_lora_add", dev, _p(base), ld_base, _p(x), ldx, _p(a), a_stride, _p(b), b_stride, _p(ids), _p(scale), n_tok,
          n_ad, n_in, n_out, rank, dt, _p(workspace), _p(out), ld_out)
    return out


def lora_grad(dy, x, a, b, ids, scale=None, workspace=None):
    """The gradients of lora_add in x (the adapter's part; base's is dy itself), a and b: (dx, da, db).

    With the tokens sorted by adapter: v = a x, dv = scale b^T dy, dx = a^T dv, da = sum dv x^T, db = scale
    sum dy v^T.  v and dv are fp32 between the products.  Tokens without an adapter get dx = 0, adapters
    without tokens da = db = 0.  At most 1024 adapters.  workspace: scratch of moe_lora_grad_workspace_bytes.
    """
    who = "lora_grad"
    dev = _one_gpu(who, "dy x a b ids scale workspace", dy, x, a, b, ids, scale, workspace)
    dt, n_ad, rank, n_in, n_out, a_stride, b_stride = _lora_args(who, x, a, b, ids, scale)
    n_tok = x.shape[0]
    ldx = _rows(who, "x", x, x.dtype, n_tok, n_in)
    lddy = _rows(who, "dy", dy, x.dtype, n_tok, n_out)
    if not 1 <= n_ad <= 1024:
        raise ValueError(f"{who}: {n_ad} adapters (1..1024)")
    dx = torch.empty((n_tok, n_in), dtype=x.dtype, device=x.device)
    da = torch.empty((n_ad, rank, n_in), dtype=x.dtype, device=x.device)
    db = torch.empty((n_ad, n_out, rank), dtype=x.dtype, device=x.device)
    workspace = _scratch(_lib.lib().moe_lora_grad_workspace_bytes(n_tok, n_ad, rank), x, workspace, who)
    _call("moe_lora_grad", dev, _p(dy), lddy, _p(x), ldx, _p(a), a_stride, _p(b), b_stride, _p(ids), _p(scale), n_tok, n_ad,
          n_in, n_out, rank, dt, _p(workspace), _p(dx), n_in, _p(da), _p(db))
    return dx, da, db
