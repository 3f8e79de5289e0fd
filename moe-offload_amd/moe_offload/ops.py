"""torch-facing wrappers of the HIP compute entry points (tensors in, tensors out).

Every function calls straight into libmoe_offload.so on torch's current HIP stream; there is
no PyTorch fallback for any of them.
"""
from __future__ import annotations

from array import array
from operator import attrgetter

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
_current_gpu = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name: str, dev: int, *args) -> None:
    """Calls an entry point on the tensors' own GPU and that GPU's current stream."""
    fn = getattr(_lib.lib(), name)
    if _current_gpu() == dev:
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


# ---- around the unquantised experts: routing, the weighted sum, shared projections, the gradients' norm ----------

_REAL = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_ACTS = {None: 0, "silu": 1, "gelu": 2, "relu2": 3}


def _choice(who: str, name: str, value, of: dict) -> int:
    if value not in of:
        raise ValueError(f"{who}: {name}={value!r} (one of {', '.join(repr(v) for v in of)})")
    return of[value]


def _scored_rows(who: str, name: str, t: torch.Tensor, shape: tuple | None = None) -> int:
    """Checks logits or their gradient (any real type, rows contiguous at any step); returns the step."""
    if t.dtype not in _REAL:
        raise TypeError(f"{who}: {name} is {t.dtype} (torch.float16, torch.bfloat16 and torch.float32 are supported)")
    if t.dim() != 2 or (shape is not None and t.shape != shape):
        raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}" + ("" if shape is None else f", not {tuple(shape)}"))
    n, w = t.shape
    if n > _MAX_SIDE or not 1 <= w <= 1024:
        raise ValueError(f"{who}: {name}: {n} tokens (up to 2^30), {w} experts (1..1024)")
    step, inner = t.stride()
    if (w > 1 and inner != 1) or (n > 1 and step < w):
        raise ValueError(f"{who}: {name}: rows must be contiguous and apart, not {t.stride()}")
    return step if n > 1 else w


def _per_place(who: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{who}: {name} is {t.dtype}, not {dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be contiguous of shape {tuple(shape)}, not {tuple(t.shape)}")


def _route_k(who: str, k: int, n_exp: int) -> None:
    if not 1 <= k <= min(32, n_exp):
        raise ValueError(f"{who}: k={k} of {n_exp} experts (1..32)")


def route(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0, ids=None,
          weights=None):
    """Each token's k experts and their weights: int32 ids [n_tok, k] and fp32 weights [n_tok, k], the best first.

    logits: fp16, bf16 or fp32 [n_tok, n_exp], up to 1024 experts.  s = softmax(logits) or sigmoid(logits); experts compare by
    c = s + bias (fp32 [n_exp]), without a bias by their logits.  n_group > 1: of the n_group groups of adjacent experts only
    the topk_group stay whose group_best (1 or 2) largest c have the largest sum (without a bias, and for 2, of s).  Equals go
    to the lowest index.  weights = scale * s[ids], renorm: divided by the sum of the chosen s first.

    An expert whose logit or bias is -inf or NaN is never chosen (mask with -inf: any other value may be chosen where
    there is too little else); places left over get id -1 and weight 0, which expert_plan, the grouped products and combine take.
    A NaN among a token's logits makes all its weights NaN.  Several logits of +inf share a softmax evenly.
    """
    who = "route"
    dev = _one_gpu(who, "logits bias ids weights", logits, bias, ids, weights)
    score = _choice(who, "score", score, _SCORES)
    ld = _scored_rows(who, "logits", logits)
    n_tok, n_exp = logits.shape
    _route_k(who, k, n_exp)
    if bias is not None:
        _per_place(who, "bias", bias, (n_exp,), torch.float32)
    if not 1 <= n_group <= 64 or n_exp % n_group or not 1 <= topk_group <= n_group or group_best not in (1, 2):
        raise ValueError(f"{who}: n_group={n_group} (1..64, a divisor of {n_exp}), topk_group={topk_group} (1..n_group), "
                         f"group_best={group_best} (1 or 2)")
    if ids is None:
        ids = logits.new_empty((n_tok, k), dtype=torch.int32)
    else:
        _per_place(who, "ids", ids, (n_tok, k), torch.int32)
    if weights is None:
        weights = logits.new_empty((n_tok, k), dtype=torch.float32)
    else:
        _per_place(who, "weights", weights, (n_tok, k), torch.float32)
    _call("moe_route", dev, _p(logits), ld, n_tok, n_exp, k, score, int(bool(renorm)), _p(bias), n_group, topk_group, group_best,
          scale, _REAL[logits.dtype], _p(ids), _p(weights))
    return ids, weights


def route_grad(dweights, logits, ids, score="softmax", renorm=True, scale=1.0, out=None):
    """The gradient in the logits, [n_tok, n_exp] of their type, of the weights that route gave with these ids.

    dweights: fp32 [n_tok, k].  The choice has no gradient, so neither has the bias.  Places whose id is outside the experts
    add nothing.
    """
    who = "route_grad"
    dev = _one_gpu(who, "dweights logits ids out", dweights, logits, ids, out)
    score = _choice(who, "score", score, _SCORES)
    ld = _scored_rows(who, "logits", logits)
    n_tok, n_exp = logits.shape
    if ids.dim() != 2:
        raise ValueError(f"{who}: ids has shape {tuple(ids.shape)}, not (n_tok, k)")
    k = ids.shape[1]
    _route_k(who, k, n_exp)
    _per_place(who, "ids", ids, (n_tok, k), torch.int32)
    _per_place(who, "dweights", dweights, (n_tok, k), torch.float32)
    if out is None:
        out, ldd = logits.new_empty((n_tok, n_exp)), n_exp
    elif out.dtype != logits.dtype:
        raise TypeError(f"{who}: out is {out.dtype}, not {logits.dtype}")
    else:
        ldd = _scored_rows(who, "out", out, logits.shape)
    _call("moe_route_grad", dev, _p(dweights), _p(logits), ld, _p(ids), n_tok, n_exp, k, score, int(bool(renorm)), scale,
          _REAL[logits.dtype], _p(out), ldd)
    return out


def _pair_rows(who: str, name: str, t: torch.Tensor, n_tok: int, k: int) -> tuple[int, int]:
    """Checks a row per (token, place), given as [n_tok, k, hidden] or [n_tok * k, hidden]; returns hidden and the step."""
    if t.dim() == 3:
        if t.shape[0] != n_tok or t.shape[1] != k:
            raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, not ({n_tok}, {k}, *)")
        far, near, inner = t.stride()
        if n_tok > 1 and k > 1 and far != k * near:
            raise ValueError(f"{who}: {name}: a token's rows must follow the token's before it, not {t.stride()}")
        hidden, step = t.shape[2], near if k > 1 else far
        if inner != 1 or hidden % 8 or hidden == 0 or (n_tok * k > 1 and (step < hidden or step % 8)):
            raise ValueError(f"{who}: {name}: rows of {hidden} elements at {t.stride()} (contiguous, multiples of 8 wanted)")
        return hidden, step if n_tok * k > 1 else hidden
    return t.shape[-1], _rows(who, name, t, t.dtype, n_tok * k, None)


def _any_rows(who: str, name: str, t: torch.Tensor, dtypes: tuple, rows: int, width: int) -> int:
    """_rows for outputs of one of two types."""
    if t.dtype not in dtypes:
        raise TypeError(f"{who}: {name} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    return _rows(who, name, t, t.dtype, rows, width)


def _result(who: str, like: torch.Tensor, out: torch.Tensor | None, dtype: torch.dtype | None, rows: int, width: int):
    """The output and its step: new, of like's type or fp32 as dtype says, or checked."""
    if out is not None:
        if dtype not in (None, out.dtype):
            raise TypeError(f"{who}: out is {out.dtype}, not {dtype}")
        return out, _any_rows(who, "out", out, (like.dtype, torch.float32), rows, width)
    if dtype not in (None, like.dtype, torch.float32):
        raise TypeError(f"{who}: results of {like.dtype} come as {like.dtype} or torch.float32, not {dtype}")
    return like.new_empty((rows, width), dtype=dtype), width


def combine(y, weights, residual=None, dtype=None, out=None):
    """out[t] = residual[t] + sum over j of weights[t, j] * y[t * k + j]: a layer's output from its experts' rows.

    y: fp16 or bf16 [n_tok, k, hidden] (or [n_tok * k, hidden]), as grouped_mm and dense.switch_glu give them; weights: fp32
    [n_tok, k]; residual: of y's type or None; out: of y's type, or fp32 with dtype=torch.float32.  A weight of 0 adds
    nothing, whatever its row holds.  out=residual adds in place.
    """
    who = "combine"
    dev = _one_gpu(who, "y weights residual out", y, weights, residual, out)
    dt = _half(who, y)
    if weights.dim() != 2 or weights.shape[1] < 1:
        raise ValueError(f"{who}: weights has shape {tuple(weights.shape)}, not (n_tok, k)")
    n_tok, k = weights.shape
    _per_place(who, "weights", weights, (n_tok, k), torch.float32)
    hidden, ldy = _pair_rows(who, "y", y, n_tok, k)
    ldr = _rows(who, "residual", residual, y.dtype, n_tok, hidden) if residual is not None else 0
    out, ldo = _result(who, y, out, dtype, n_tok, hidden)
    _call("moe_combine", dev, _p(y), ldy, _p(weights), _p(residual), ldr, n_tok, k, hidden, dt, int(out.dtype == torch.float32),
          _p(out), ldo)
    return out


def combine_grad(dout, y, weights):
    """combine's gradients: dy, of y's shape and type, and fp32 dweights [n_tok, k] (the residual's is dout, of y's type).

    Of a weight of 0 dy is 0 whatever dout holds, and dweights is 0 where it would be infinite or NaN.
    """
    who = "combine_grad"
    dev = _one_gpu(who, "dout y weights", dout, y, weights)
    dt = _half(who, y)
    if weights.dim() != 2 or weights.shape[1] < 1:
        raise ValueError(f"{who}: weights has shape {tuple(weights.shape)}, not (n_tok, k)")
    n_tok, k = weights.shape
    _per_place(who, "weights", weights, (n_tok, k), torch.float32)
    hidden, ldy = _pair_rows(who, "y", y, n_tok, k)
    ldd = _rows(who, "dout", dout, y.dtype, n_tok, hidden)
    dy, dw = torch.empty_like(y, memory_format=torch.contiguous_format), torch.empty_like(weights)
    _call("moe_combine_grad", dev, _p(dout), ldd, _p(y), ldy, _p(weights), n_tok, k, hidden, dt, _p(dy), hidden, _p(dw))
    return dy, dw


def _shared_weight(who: str, w: torch.Tensor, dtype: torch.dtype, n_in: int) -> None:
    if _rows(who, "w", w, dtype, None, n_in) != n_in or w.shape[0] % 8 or w.shape[0] == 0:
        raise ValueError(f"{who}: w must be contiguous with a multiple of 8 rows, not {tuple(w.shape)} at {w.stride()}")


def linear(x, w, bias=None, act=None, residual=None, z_out=None, dtype=None, out=None, workspace=None):
    """act(x @ w.T + bias) + residual: a projection that all tokens share (the router, a shared expert), in one launch.

    x: fp16 or bf16 [n_tok, n_in]; w: same type [n_out, n_in], contiguous; bias: same type [n_out] or None; act: None, "silu",
    "gelu" (z times the normal distribution's integral, within z^2 / 2 + 10 steps of 2^-23 of its value) or "relu2" (the squared
    relu); residual: same type [n_tok, n_out] or None.  The result has the inputs' type, or fp32 with dtype=torch.float32 (router logits).  z_out, [n_tok, n_out] of the inputs'
    type, receives x @ w.T + bias for linear_grad.  out=residual adds in place.  workspace: scratch of
    moe_linear_workspace_bytes.
    """
    who = "linear"
    dev = _one_gpu(who, "x w bias residual z_out out workspace", x, w, bias, residual, z_out, out, workspace)
    dt = _half(who, x)
    act = _choice(who, "act", act, _ACTS)
    ldx = _rows(who, "x", x, x.dtype, None, None)
    n_tok, n_in = x.shape
    _shared_weight(who, w, x.dtype, n_in)
    n_out = w.shape[0]
    if bias is not None:
        _per_place(who, "bias", bias, (n_out,), x.dtype)
    ldr = _rows(who, "residual", residual, x.dtype, n_tok, n_out) if residual is not None else 0
    ldz = _rows(who, "z_out", z_out, x.dtype, n_tok, n_out) if z_out is not None else 0
    out, ldy = _result(who, x, out, dtype, n_tok, n_out)
    nb = _lib.lib().moe_linear_workspace_bytes(n_tok, n_in, n_out)
    ws = _scratch(nb, x, workspace, who) if nb else None
    _call("moe_linear", dev, _p(x), ldx, _p(w), _p(bias), _p(residual), ldr, n_tok, n_in, n_out, act, dt,
          int(out.dtype == torch.float32), _p(ws), _p(z_out), ldz, _p(out), ldy)
    return out


def linear_grad(dy, x, w, z=None, act=None, bias=False, want_dx=True, want_dw=True, dw_dtype=None, workspace=None):
    """linear's gradients (dx, dw, dbias), None for those that are not wanted; the residual's is dy.

    dy: x's type, or fp32, [n_tok, n_out]; z: what linear wrote to z_out, where act is not None; bias: whether the bias's
    gradient is wanted.  dw in x's type, or fp32 with dw_dtype=torch.float32.  dz = dy act'(z) (dy alone too, where it is fp32) goes
    through the products in parts, with more bits than 16-bit results show, for an fp32 dw with all of its own.  workspace:
    scratch of moe_linear_grad_workspace_bytes.
    """
    who = "linear_grad"
    dev = _one_gpu(who, "dy x w z workspace", dy, x, w, z, workspace)
    dt = _half(who, x)
    act_id = _choice(who, "act", act, _ACTS)
    ldx = _rows(who, "x", x, x.dtype, None, None)
    n_tok, n_in = x.shape
    _shared_weight(who, w, x.dtype, n_in)
    n_out = w.shape[0]
    lddy = _any_rows(who, "dy", dy, (x.dtype, torch.float32), n_tok, n_out)
    if (z is None) != (act is None):
        raise ValueError(f"{who}: z goes with an activation (act={act!r})")
    ldz = _rows(who, "z", z, x.dtype, n_tok, n_out) if z is not None else 0
    dw_dtype = dw_dtype or x.dtype
    if dw_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{who}: gradients of {x.dtype} come as {x.dtype} or torch.float32, not {dw_dtype}")
    dx = x.new_empty((n_tok, n_in)) if want_dx else None
    dw = x.new_empty((n_out, n_in), dtype=dw_dtype) if want_dw else None
    db = x.new_empty(n_out) if bias else None
    dy_f32 = int(dy.dtype == torch.float32)
    nb = _lib.lib().moe_linear_grad_workspace_bytes(n_tok, n_in, n_out, act_id, dy_f32, int(want_dw), int(bool(bias)))
    ws = _scratch(nb, x, workspace, who) if nb else None
    _call("moe_linear_grad", dev, _p(dy), lddy, dy_f32, _p(x), ldx, _p(w), _p(z), ldz, n_tok, n_in, n_out, act_id, dt, _p(ws), _p(dx),
          _p(dw), int(dw_dtype == torch.float32), _p(db))
    return dx, dw, db


def _dense_layout(t: torch.Tensor) -> bool:
    """Whether a tensor's elements fill one piece of memory, in whatever order of its dimensions."""
    if t.layout != torch.strided:
        return False
    if t.is_contiguous() or t.numel() == 0:
        return True
    want = 1
    for step, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if step != want:
            return False
        want *= n
    return True


_dtype_of = attrgetter("dtype")
_Tensor = torch.Tensor


def _tensor_list(who: str, name: str, tensors) -> tuple[list, array]:
    """The tensors of a list and their types' numbers.  (Lists are long: whole passes in C, no code per tensor.)"""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for kind in set(map(type, tensors)):
        if not issubclass(kind, torch.Tensor):
            raise TypeError(f"{who}: {name} must be tensors, not {kind.__name__}")
    types = list(map(_REAL.get, map(_dtype_of, tensors)))
    if None in types:
        raise TypeError(f"{who}: {name}: {tensors[types.index(None)].dtype} (torch.float16, torch.bfloat16 and torch.float32 are supported)")
    if not all(map(_Tensor.is_contiguous, tensors)):
        for t in tensors:
            if not _dense_layout(t):
                raise ValueError(f"{who}: {name}: a tensor of shape {tuple(t.shape)} does not fill its memory")
    return tensors, array("i", types)


def _clip(who, grads, types, outs, max_norm):
    gpus = set(map(_Tensor.get_device, grads))
    if outs is not None and outs is not grads:
        gpus.update(map(_Tensor.get_device, outs))
    if len(gpus) != 1 or min(gpus) < 0:
        raise ValueError(f"{who}: the tensors must be on one GPU" + (" (there are none)" if not gpus else f", not {sorted(gpus)}"))
    dev = gpus.pop()
    # (an array takes a list faster than a map)
    sizes, ptrs = array("q", list(map(_Tensor.numel, grads))), array("Q", list(map(_Tensor.data_ptr, grads)))
    out_ptrs = None if outs is None else ptrs if outs is grads else array("Q", list(map(_Tensor.data_ptr, outs)))
    ws = grads[0].new_empty(_lib.lib().moe_clip_workspace_bytes(len(grads), sum(sizes)), dtype=torch.uint8)
    norm = grads[0].new_empty((), dtype=torch.float32)
    _call("moe_clip_grads", dev, len(grads), ptrs.buffer_info()[0], None if out_ptrs is None else out_ptrs.buffer_info()[0],
          sizes.buffer_info()[0], types.buffer_info()[0], max_norm, _p(ws), _p(norm))
    return norm


def grad_norm(grads):
    """The norm of all tensors together, sqrt(sum of squares), fp32 on their GPU.  Any mixture of fp16, bf16 and fp32 tensors of
    any shape whose elements fill their memory; the squares are summed in 64 bits."""
    return _clip("grad_norm", *_tensor_list("grad_norm", "grads", grads), None, 0.0)


def clip_grad_norm(grads, max_norm, out=None):
    """grad_norm, and every tensor times min(1, max_norm / (norm + 1e-6)), as torch.nn.utils.clip_grad_norm_: in place, or into
    the tensors of `out` (their shapes, types and strides).  Returns the norm before.  Nothing that is written may overlap
    another tensor (the same one twice in the list, say).  An infinite norm leaves zeros and NaN, a NaN leaves NaN."""
    who = "clip_grad_norm"
    grads, types = _tensor_list(who, "grads", grads)
    if not max_norm >= 0:
        raise ValueError(f"{who}: max_norm={max_norm}")
    outs = grads
    if out is not None:
        outs, _ = _tensor_list(who, "out", out)
        if len(outs) != len(grads):
            raise ValueError(f"{who}: {len(outs)} tensors in out for {len(grads)}")
        for g, o in zip(grads, outs):
            if o.shape != g.shape or o.dtype != g.dtype or (o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous())):
                raise ValueError(f"{who}: out has {o.dtype} {tuple(o.shape)} at {o.stride()} for {g.dtype} {tuple(g.shape)} at {g.stride()}")
    return _clip(who, grads, types, outs, float(max_norm))
