"""The grouped products of unquantised experts and their gradients against 64-bit forms (grouped_ref.py, which
derives the bounds): ragged, empty and single-row segments, sizes that end inside every tile, gathered and
scattered rows, strides, rows that nothing covers, indexes outside, offsets past 32 bits, other streams, replayed
graphs, and a layer's whole forward and backward pass."""
import numpy as np
import pytest

import grouped_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def i32(v):
    return torch.as_tensor(np.asarray(v), dtype=torch.int32).to(DEV)


# segment lengths: empty, one row, and both sides of the tiles' edges
LENGTHS = {
    "one": [1],
    "ones": [1, 1, 0, 1, 1, 0, 0, 1],
    "few": [3, 0, 17, 1, 16, 15],
    "edges": [63, 64, 65, 0, 31, 33, 1, 128],
    "long": [257, 0, 130],
    "longer": [1000, 5, 0, 300],
    "many": [2, 0, 1, 5] * 60,
}
SHAPES = [(8, 8), (64, 64), (16, 264), (136, 40), (264, 72), (128, 512), (320, 1152), (520, 8)]


def case(name):
    lens = LENGTHS[name]
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LENGTHS))
def test_mm_every_length(name, dtype):
    from moe_offload import ops
    seg = case(name)
    m, e = int(seg[-1]), len(seg) - 1
    for n, k in SHAPES:
        x, w = rnd((m, k), dtype, 1), rnd((e, n, k), dtype, 2, k ** -0.5)
        y = ops.grouped_mm(x, i32(seg), w)
        want, slack, _ = ref.product(x.double().cpu(), seg, w)
        ref.check(y, want, slack, f"mm {name} n={n} k={k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LENGTHS))
def test_gate_up_every_length(name, dtype):
    from moe_offload import ops
    seg = case(name)
    m, e = int(seg[-1]), len(seg) - 1
    for inter, k in SHAPES:
        x, w = rnd((m, k), dtype, 3), rnd((e, 2 * inter, k), dtype, 4, k ** -0.5)
        gu = torch.empty((m, 2 * inter), dtype=dtype, device=DEV)
        h = ops.grouped_gate_up(x, None, i32(seg), w, gu_out=gu)
        want, slack, _ = ref.product(x.double().cpu(), seg, w)
        ref.check(gu, want, slack, f"gu {name} inter={inter} k={k}")
        hw, hs = ref.glu(*want.chunk(2, 1), *slack.chunk(2, 1))
        ref.check(h, hw, hs, f"h {name} inter={inter} k={k}")
        assert torch.equal(h, ops.grouped_gate_up(x, None, i32(seg), w)), "h without gu_out"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LENGTHS))
def test_dx_every_length(name, dtype):
    from moe_offload import ops
    seg = case(name)
    m, e = int(seg[-1]), len(seg) - 1
    for n, k in SHAPES:
        dy, w = rnd((m, n), dtype, 5), rnd((e, n, k), dtype, 6, n ** -0.5)
        dx = ops.grouped_mm_dx(dy, i32(seg), w)
        want, slack, _ = ref.product(dy.double().cpu(), seg, w, transposed=True)
        ref.check(dx, want, slack, f"dx {name} n={n} k={k}")
        gu = rnd((m, 2 * k), dtype, 7)
        dgu = ops.grouped_mm_dx(dy, i32(seg), w, gu=gu)
        ref.check(dgu, *ref.glu_grad(want, slack, gu), f"dgu {name} n={n} k={k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LENGTHS))
def test_dw_every_length(name, dtype):
    from moe_offload import ops
    seg = case(name)
    m, e = int(seg[-1]), len(seg) - 1
    for n, k in SHAPES:
        dy, x = rnd((m, n), dtype, 8), rnd((m, k), dtype, 9)
        want, slack = ref.weight_grad(dy.double().cpu(), x.double().cpu(), seg, e)
        for out in (dtype, torch.float32):
            dw = ops.grouped_mm_dw(dy, x, i32(seg), dtype=out)
            assert dw.dtype == out
            ref.check(dw, want, slack, f"dw {name} n={n} k={k} {out}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gathered_scattered_strided_scaled(dtype):
    """Every optional argument at once: rows read by index (some outside x), written by index (some outside the
    output), slots out of order, repeated and outside, scales, row strides, matrix strides."""
    from moe_offload import ops
    rng = np.random.default_rng(1)
    seg = np.array([2, 40, 40, 47, 120, 121, 150], np.int32)       # rows 0-1 and 150-159 belong to no segment
    slot = np.array([3, 1, -1, 0, 3, 9], np.int32)                 # 4 slots: -1 and 9 do not exist
    m, nx, ny, n, k = 160, 50, 170, 72, 136
    row_in = rng.integers(0, nx, m).astype(np.int32)
    row_in[[5, 50, 121]] = [-1, nx, 2 ** 31 - 1]
    row_out = rng.permutation(ny)[:m].astype(np.int32)
    row_out[[6, 60]] = [-5, ny]
    scale = torch.tensor([0.5, -2.0, 1.0, 1.5], device=DEV)
    big = rnd((nx, k + 24), dtype, 10)
    x = big[:, 8:8 + k]
    w = rnd((4 * (n * k + 64),), dtype, 11, k ** -0.5).as_strided((4, n, k), (n * k + 64, k, 1))
    xr = ref.gather(x, row_in)
    want, slack, has = ref.product(xr, seg, w, slot, scale)

    full = torch.full((ny, n + 16), 7.0, dtype=dtype, device=DEV)
    out = full[:, 8:8 + n]
    ops.grouped_mm(x, i32(seg), w, row_in=i32(row_in), row_out=i32(row_out), seg_slot=i32(slot), scale=scale, out=out)
    expect, room = torch.full((ny, n), 7.0, dtype=torch.float64), torch.zeros((ny, n), dtype=torch.float64)
    for r in range(m):
        if has[r] and 0 <= row_out[r] < ny:
            expect[row_out[r]], room[row_out[r]] = want[r], slack[r]
    ref.check(out, expect, room, "given output")
    assert bool((full[:, :8] == 7).all()) and bool((full[:, 8 + n:] == 7).all())

    new = ops.grouped_mm(x, i32(seg), w, row_in=i32(row_in), row_out=i32(row_out), n_out_rows=ny, seg_slot=i32(slot), scale=scale)
    zeroed = expect.clone()
    zeroed[room.sum(1) == 0] = 0
    ref.check(new, zeroed, room, "new output")
    same = ops.grouped_mm(x, i32(seg), w, row_in=i32(row_in), seg_slot=i32(slot), scale=scale)
    ref.check(same, want, slack, "new output, a row for each")        # the rows of no segment are zeros in want

    h = torch.full((m, n // 2 - 4), 7.0, dtype=dtype, device=DEV)     # inter 32 of the 72 rows' first 64
    w2 = w[:, :64].contiguous()
    gu = torch.full((m, 64 + 8), 7.0, dtype=dtype, device=DEV)
    ops.grouped_gate_up(x, i32(row_in), i32(seg), w2, seg_slot=i32(slot), h_out=h, gu_out=gu[:, :64])
    gw, gs, _ = ref.product(xr, seg, w2, slot)
    hw, hs = ref.glu(*gw.chunk(2, 1), *gs.chunk(2, 1))
    gw[~has], gs[~has], hw[~has], hs[~has] = 7.0, 0.0, 7.0, 0.0
    ref.check(h, hw, hs, "h")
    ref.check(gu[:, :64], gw, gs, "gu")
    assert bool((gu[:, 64:] == 7).all())

    # gradients: dy at the places that the product wrote, dx one row per sorted row
    dy = rnd((ny, n + 8), dtype, 12)[:, :n]
    dyr = ref.gather(dy, row_out)
    dwant, dslack, _ = ref.product(dyr, seg, w, slot, scale, transposed=True)
    dx = ops.grouped_mm_dx(dy, i32(seg), w, row_in=i32(row_out), seg_slot=i32(slot), scale=scale)
    ref.check(dx, dwant, dslack, "dx")
    g2 = rnd((m, 2 * k), dtype, 13)
    g2[~has.to(DEV)] = float("inf")                                   # rows of no segment: zeros whatever they hold
    dgu = ops.grouped_mm_dx(dy, i32(seg), w, row_in=i32(row_out), seg_slot=i32(slot), scale=scale, gu=g2)
    fine = g2.clone()
    fine[~has.to(DEV)] = 0
    ref.check(dgu, *ref.glu_grad(dwant, dslack, fine), "dgu")
    s6 = torch.tensor([1.0, 0.5, 2.0, -1.0, 0.25, 3.0], device=DEV)
    both = torch.tensor((row_in >= 0) & (row_in < nx) & (row_out >= 0) & (row_out < ny)).unsqueeze(1)
    ww, ws = ref.weight_grad(dyr * both, xr * both, seg, 6, s6)
    buf = torch.full((6 * (n * k + 8),), 7.0, device=DEV)
    dw = buf.as_strided((6, n, k), (n * k + 8, k, 1))
    ops.grouped_mm_dw(dy, x, i32(seg), row_dy=i32(row_out), row_x=i32(row_in), scale=s6, out=dw)
    ref.check(dw, ww, ws, "dw")
    assert bool((buf.view(6, -1)[:, n * k:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_do(dtype):
    from moe_offload import ops
    w = rnd((3, 16, 24), dtype, 1)
    z = torch.zeros((0, 24), dtype=dtype, device=DEV)
    seg0 = i32([0, 0, 0, 0])
    assert ops.grouped_mm(z, seg0, w).shape == (0, 16)
    assert ops.grouped_gate_up(z, None, seg0, w).shape == (0, 8)
    assert ops.grouped_mm_dx(torch.zeros((0, 16), dtype=dtype, device=DEV), seg0, w).shape == (0, 24)
    dw = ops.grouped_mm_dw(torch.zeros((0, 16), dtype=dtype, device=DEV), z, seg0)
    assert dw.shape == (3, 16, 24) and not bool(dw.any())
    # rows, but no segments and no weights: zeros in a new output, nothing in a given one
    x = rnd((70, 24), dtype, 2)
    assert not bool(ops.grouped_mm(x, i32([0]), w[:0]).any())
    out = torch.full((70, 16), 3.0, dtype=dtype, device=DEV)
    ops.grouped_mm(x, i32([0]), w[:0], out=out)
    assert bool((out == 3).all())
    # rows by index from an x without rows
    y = ops.grouped_mm(z, i32([0, 2, 2, 4]), w, row_in=i32([0, 1, 2, 3]))
    assert not bool(y.any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_segments_in_disorder_stay_in_bounds(dtype):
    """Starts outside the rows or out of order: rows outside are never touched, the rest is unspecified."""
    from moe_offload import ops
    w = rnd((4, 64, 64), dtype, 1)
    buf = torch.full((100 + 64, 64), 5.0, dtype=dtype, device=DEV)
    for starts in ([-5, 30, 20, 500, 90], [2 ** 31 - 1, -2 ** 31, 0, 100, 101], [90, 60, 30, 0, -1]):
        ops.grouped_mm(rnd((100, 64), dtype, 2), i32(starts), w, out=buf[:100])
        ops.grouped_mm(rnd((100, 64), dtype, 2), i32(starts), w)
        ops.grouped_mm_dx(rnd((100, 64), dtype, 2), i32(starts), w, out=buf[:100])
        ops.grouped_mm_dw(rnd((100, 64), dtype, 2), rnd((100, 64), dtype, 3), i32(starts))
        torch.cuda.synchronize()
        assert bool((buf[100:] == 5).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_stay_in_their_rows(dtype):
    """A row that holds inf or NaN changes its own outputs alone, and so does a slot's weight; a NaN in a row that
    no segment covers, or behind a segment's end, reaches nothing."""
    from moe_offload import ops
    seg, n, k = i32([0, 20, 33, 90]), 72, 136
    x, w = rnd((100, k), dtype, 1), rnd((3, n, k), dtype, 2, k ** -0.5)
    clean, cdx = ops.grouped_mm(x, seg, w), ops.grouped_mm_dx(rnd((100, n), dtype, 4), seg, w)
    cdw = ops.grouped_mm_dw(rnd((100, n), dtype, 4), x, seg)
    x2, dy2 = x.clone(), rnd((100, n), dtype, 4)
    x2[20, 3], x2[95] = float("nan"), float("inf")
    dy2[20, 3], dy2[91] = float("inf"), float("nan")
    y, dx, dw = ops.grouped_mm(x2, seg, w), ops.grouped_mm_dx(dy2, seg, w), ops.grouped_mm_dw(dy2, x, seg)
    keep = torch.ones(100, dtype=torch.bool, device=DEV)
    keep[20] = False
    assert torch.equal(y[keep], clean[keep]) and bool(y[20].isnan().all())
    assert torch.equal(dx[keep], cdx[keep]) and not bool(dx[20].isfinite().any())
    assert torch.equal(dw[0], cdw[0]) and torch.equal(dw[2], cdw[2])
    rows = torch.ones(n, dtype=torch.bool, device=DEV)
    rows[3] = False
    assert torch.equal(dw[1][rows], cdw[1][rows]) and not bool(dw[1][3].isfinite().any())
    # a row left out of the weights' gradient on one side does not meet the other side's infinity
    out = list(range(100))
    out[40], out[41] = -1, 100
    x2, dy2 = x.clone(), rnd((100, n), dtype, 4)
    x2[40:42], dy2[50] = float("inf"), float("nan")
    xin = list(range(100))
    xin[50] = 200
    assert bool(ops.grouped_mm_dw(dy2, x2, seg, row_dy=i32(out), row_x=i32(xin)).isfinite().all())
    w2 = w.clone()
    w2[1, 7, 9] = float("nan")
    y = ops.grouped_mm(x, seg, w2)
    assert bool(y[20:33, 7].isnan().all())
    y[20:33, 7] = clean[20:33, 7]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_has_the_same_bits_in_every_call(dtype):
    """Alone, among few, among many, among thousands: the products and their gradients in x add in one order."""
    from moe_offload import ops
    n, k, e = 136, 1096, 3
    w, wu = rnd((e, n, k), dtype, 1, k ** -0.5), rnd((e, 2 * n, k), dtype, 2, k ** -0.5)
    first = None
    for lens in ([1, 1, 1], [5, 16, 2], [40, 33, 17], [130, 200, 300], [2100, 1500, 2000]):
        seg = np.concatenate([[0], np.cumsum(lens)])
        m = int(seg[-1])
        x, dy = rnd((m, k), dtype, 3), rnd((m, n), dtype, 4)
        for i in range(3):                              # the first row of each segment is the same in every call
            x[seg[i]], dy[seg[i]] = rnd((k,), dtype, 10 + i), rnd((n,), dtype, 20 + i)
        at = torch.as_tensor(seg[:3], device=DEV)
        got = [ops.grouped_mm(x, i32(seg), w)[at], ops.grouped_gate_up(x, None, i32(seg), wu)[at], ops.grouped_mm_dx(dy, i32(seg), w)[at]]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got)), lens


def test_values_out_of_fp16_range_become_infinite():
    from moe_offload import ops
    x = torch.full((3, 64), 100.0, dtype=torch.float16, device=DEV)
    w = torch.full((1, 8, 64), 100.0, dtype=torch.float16, device=DEV)
    y = ops.grouped_mm(x, i32([0, 3]), w)
    assert bool((y == float("inf")).all())


@pytest.mark.parametrize("op", ["mm", "dx", "dw"])
def test_offsets_past_32_bits(op):
    """Matrices and rows that lie further than 2^32 bytes, and 2^31 elements, from the first."""
    from moe_offload import ops
    dt, n, k = torch.bfloat16, 40, 72
    step = 2 ** 31 + 64
    buf = torch.empty(2 * step + 64 * 2 ** 10, dtype=dt, device=DEV)
    far = buf.as_strided((3, n, k), (step, k, 1))
    w, x, dy, seg = rnd((3, n, k), dt, 1, 0.1), rnd((30, k), dt, 2), rnd((30, n), dt, 3), i32([0, 11, 12, 30])
    if op == "dw":
        far.fill_(9.0)
        ops.grouped_mm_dw(dy, x, seg, out=far)
        ref.check(far, *ref.weight_grad(dy.double().cpu(), x.double().cpu(), seg.tolist(), 3))
        return
    far.copy_(w)
    if op == "mm":
        ref.check(ops.grouped_mm(x, seg, far), *ref.product(x.double().cpu(), seg.tolist(), w)[:2])
        rows = buf.as_strided((3, k), (step, 1))
        rows.copy_(x[:3])
        out = buf.as_strided((3, n), (step, 1), 2 ** 14)
        ops.grouped_mm(rows, i32([0, 1, 2, 3]), w, out=out)
        ref.check(out, *ref.product(x[:3].double().cpu(), [0, 1, 2, 3], w)[:2])
    else:
        ref.check(ops.grouped_mm_dx(dy, seg, far), *ref.product(dy.double().cpu(), seg.tolist(), w, transposed=True)[:2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_products(dtype):
    """Long segments and wide outputs, where the largest tiles run; sizes that end inside them."""
    from moe_offload import ops
    seg = np.array([0, 2100, 2100, 3601, 5602], np.int32)
    m, e, n, k = 5602, 4, 2056, 200
    x, w, wu = rnd((m, k), dtype, 1), rnd((e, n, k), dtype, 2, k ** -0.5), rnd((e, 2 * 1048, k), dtype, 3, k ** -0.5)
    rng = np.random.default_rng(0)
    order = i32(rng.permutation(m))
    xr, at = x[order.long()].double(), order.long()
    y = ops.grouped_mm(x, i32(seg), w, row_in=order, row_out=order)
    want, slack, _ = ref.product(xr, seg, w)
    ref.check(y[at], want, slack, "mm")
    gu = torch.empty((m, 2096), dtype=dtype, device=DEV)
    h = ops.grouped_gate_up(x, order, i32(seg), wu, gu_out=gu)
    want, slack, _ = ref.product(xr, seg, wu)
    ref.check(gu, want, slack, "gu")
    ref.check(h, *ref.glu(*want.chunk(2, 1), *slack.chunk(2, 1)), "h")
    dy, wd = rnd((m, k), dtype, 4), rnd((e, k, n), dtype, 5, k ** -0.5)
    dyr = dy[at].double()
    want, slack, _ = ref.product(dyr, seg, wd, transposed=True)
    ref.check(ops.grouped_mm_dx(dy, i32(seg), wd, row_in=order, row_out=order)[at], want, slack, "dx")
    g2 = rnd((m, 2 * n), dtype, 6)
    ref.check(ops.grouped_mm_dx(dy, i32(seg), wd, row_in=order, gu=g2), *ref.glu_grad(want, slack, g2), "dgu")


@pytest.mark.parametrize("dtype", DTYPES)
def test_middle_products(dtype):
    """Segments of a few hundred rows, wide outputs: tiles of 128 rows, ends inside them."""
    from moe_offload import ops
    seg = np.array([0, 300, 300, 633, 890], np.int32)
    m, e, n, k = 890, 4, 3728, 72
    x, w, wu = rnd((m, k), dtype, 1), rnd((e, n, k), dtype, 2, k ** -0.5), rnd((e, n, k), dtype, 3, k ** -0.5)
    order = i32(np.random.default_rng(0).permutation(m))
    at, xr = order.long(), x[order.long()].double()
    want, slack, _ = ref.product(xr, seg, w)
    ref.check(ops.grouped_mm(x, i32(seg), w, row_in=order, row_out=order)[at], want, slack, "mm")
    gu = torch.empty((m, n), dtype=dtype, device=DEV)
    h = ops.grouped_gate_up(x, order, i32(seg), wu, gu_out=gu)
    want, slack, _ = ref.product(xr, seg, wu)
    ref.check(gu, want, slack, "gu")
    ref.check(h, *ref.glu(*want.chunk(2, 1), *slack.chunk(2, 1)), "h")
    wd = rnd((e, k, n), dtype, 5, k ** -0.5)
    want, slack, _ = ref.product(xr, seg, wd, transposed=True)
    ref.check(ops.grouped_mm_dx(x, i32(seg), wd, row_in=order, row_out=order)[at], want, slack, "dx")
    g2 = rnd((m, 2 * n), dtype, 6)
    ref.check(ops.grouped_mm_dx(x, i32(seg), wd, row_in=order, gu=g2), *ref.glu_grad(want, slack, g2), "dgu")


@pytest.mark.parametrize("lens", [[16400], [90] * 40, [40] * 40], ids=["long", "middle", "short"])
def test_several_tiles_of_a_block(lens):
    """More columns than blocks: each has several tiles of columns.  Rows have the bits that they have in a call of their own."""
    from moe_offload import ops
    dtype, n, k, e = torch.bfloat16, 8208, 72, len(lens)
    seg = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    m = int(seg[-1])
    x, w, wd = rnd((m, k), dtype, 1), rnd((e, n, k), dtype, 2, k ** -0.5), rnd((e, k, n), dtype, 3, k ** -0.5)
    gu = torch.empty((m, n), dtype=dtype, device=DEV)
    g2 = rnd((m, 16), dtype, 4).repeat(1, n // 8)
    y, h = ops.grouped_mm(x, i32(seg), w), ops.grouped_gate_up(x, None, i32(seg), w, gu_out=gu)
    dx, dgu = ops.grouped_mm_dx(x, i32(seg), wd), ops.grouped_mm_dx(x, i32(seg), wd, gu=g2)
    for u, r0 in ((0, 0), (0, lens[0] // 2), (e - 1, m - min(lens[-1], 150))):
        r1 = min(r0 + 150, int(seg[u + 1]))
        s, part = i32([0, r1 - r0]), slice(r0, r1)
        assert torch.equal(y[part], ops.grouped_mm(x[part], s, w[u:u + 1])), (u, "mm")
        g1 = torch.empty((r1 - r0, n), dtype=dtype, device=DEV)
        assert torch.equal(h[part], ops.grouped_gate_up(x[part], None, s, w[u:u + 1], gu_out=g1)) and torch.equal(gu[part], g1), (u, "gate_up")
        assert torch.equal(dx[part], ops.grouped_mm_dx(x[part], s, wd[u:u + 1])), (u, "dx")
        assert torch.equal(dgu[part], ops.grouped_mm_dx(x[part], s, wd[u:u + 1], gu=g2[part])), (u, "dgu")


@pytest.mark.parametrize("dtype", DTYPES)
def test_most_segments(dtype):
    """1024 segments, most of them empty or of one row."""
    from moe_offload import ops
    lens = np.random.default_rng(5).integers(0, 3, 1024)
    lens[700] = 130
    seg = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    m, n, k = int(seg[-1]), 24, 72
    x, w = rnd((m, k), dtype, 1), rnd((1024, n, k), dtype, 2, k ** -0.5)
    ref.check(ops.grouped_mm(x, i32(seg), w), *ref.product(x.double().cpu(), seg, w)[:2], "mm")
    dy = rnd((m, n), dtype, 3)
    ref.check(ops.grouped_mm_dx(dy, i32(seg), w), *ref.product(dy.double().cpu(), seg, w, transposed=True)[:2], "dx")
    ref.check(ops.grouped_mm_dw(dy, x, i32(seg)), *ref.weight_grad(dy.double().cpu(), x.double().cpu(), seg, 1024), "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,lens", [(64, 264, [1024, 0, 1025, 2500]), (200, 40, [3000, 1]), (264, 392, [1100, 2049, 64]),
                                      (1032, 1000, [512] * 10 + [0, 1030, 2600, 511, 700, 3]),
                                      (2056, 2088, [600, 0, 1500])])
def test_dw_of_long_segments(dtype, n, k, lens):
    """More rows than a block holds the numbers of, in each of the tile sizes, some rows missing."""
    from moe_offload import ops
    seg = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    m, e = int(seg[-1]), len(lens)
    rng = np.random.default_rng(n)
    rows_dy, rows_x = rng.integers(-2, 900, m), rng.integers(0, 1002, m)
    dy, x = rnd((900, n), dtype, 1), rnd((1000, k), dtype, 2)
    both = torch.tensor((rows_dy >= 0) & (rows_x < 1000)).unsqueeze(1)
    dyr, xr = ref.gather(dy, rows_dy) * both, ref.gather(x, rows_x) * both
    want, slack = ref.weight_grad(dyr.to(DEV), xr.to(DEV), seg, e)
    ref.check(ops.grouped_mm_dw(dy, x, i32(seg), row_dy=i32(rows_dy), row_x=i32(rows_x)), want, slack, "by index")
    ref.check(ops.grouped_mm_dw(dy, x, i32(seg), row_dy=i32(rows_dy), row_x=i32(rows_x), dtype=torch.float32), want, slack, "fp32")
    dy, x = rnd((m, n), dtype, 3), rnd((m, k), dtype, 4)
    ref.check(ops.grouped_mm_dw(dy, x, i32(seg)), *ref.weight_grad(dy.double(), x.double(), seg, e), "in order")


def _layer(dtype, tokens, k, n_exp, hidden, inter, seed=0, drop=False):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(n_exp, generator=g)[:k] for _ in range(tokens)]).to(torch.int32)
    if drop:
        ids[::3, 0] = -1
        ids[1] = -1
    return (rnd((tokens, hidden), dtype, seed + 1), ids.to(DEV), rnd((n_exp, 2 * inter, hidden), dtype, seed + 2, hidden ** -0.5),
            rnd((n_exp, hidden, inter), dtype, seed + 3, inter ** -0.5))


def _layer64(x, ids, wgu, wd):
    rows = []
    for t in range(ids.shape[0]):
        for e in ids[t].tolist():
            if e < 0 or e >= wgu.shape[0]:
                rows.append(torch.zeros_like(x[0]) + 0 * x[t])
                continue
            g, u = (wgu[e] @ x[t]).chunk(2)
            rows.append(wd[e] @ (g * torch.sigmoid(g) * u))
    return torch.stack(rows).view(*ids.shape, -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("drop", [False, True])
def test_layer_forward_and_backward(dtype, drop):
    """plan -> gate_up -> down and back under autograd, against the same layer in 64 bits.  Four roundings to the
    inputs' type lie on the longest way (h or (g, u), dgu, a pair's row, the result): each moves a value by at most
    half a step, a sum of independently rounded terms by less than their norm's share, so 4 * eps / 2 of the
    outputs' norm bounds the whole."""
    from moe_offload import dense
    x, ids, wgu, wd = _layer(dtype, 29, 3, 7, 72, 40, seed=5, drop=drop)
    leaves = [t.clone().requires_grad_() for t in (x, wgu, wd)]
    scores = torch.rand((29, 3), device=DEV).requires_grad_()
    y = dense.switch_glu(leaves[0], ids, leaves[1], leaves[2])
    out = (y.float() * scores.unsqueeze(2)).sum(1)
    c = torch.randn(out.shape, generator=torch.Generator().manual_seed(9)).to(DEV)
    (out * c).sum().backward()
    l64 = [t.double().cpu().requires_grad_() for t in (x, wgu, wd)]
    s64 = scores.detach().double().cpu().requires_grad_()
    y64 = _layer64(l64[0], ids.cpu(), l64[1], l64[2])
    ((y64 * s64.unsqueeze(2)).sum(1) * c.double().cpu()).sum().backward()
    tol = 4 * torch.finfo(dtype).eps / 2
    for name, a, b in [("y", y, y64)] + [(n, p.grad, q.grad) for n, p, q in zip(("dx", "dw_gate_up", "dw_down"), leaves, l64)] \
            + [("dscores", scores.grad, s64.grad)]:
        err = (a.detach().double().cpu() - b.detach()).norm() / b.detach().norm()
        assert err <= tol, f"{name}: {err:.2e}"
    if drop:
        assert not bool(y[1].any()) and not bool(leaves[0].grad[1].any())


def test_layer_gradient_against_differences():
    """The gradient along a direction against a central difference of the 64-bit layer."""
    from moe_offload import dense
    dtype = torch.float16
    x, ids, wgu, wd = _layer(dtype, 12, 2, 4, 40, 24, seed=8)
    leaves = [t.clone().requires_grad_() for t in (x, wgu, wd)]
    c = torch.randn((12, 2, 40), generator=torch.Generator().manual_seed(3))
    (dense.switch_glu(leaves[0], ids, leaves[1], leaves[2]).float() * c.to(DEV)).sum().backward()
    base = [t.double().cpu() for t in (x, wgu, wd)]
    f = lambda v: float((_layer64(v[0], ids.cpu(), v[1], v[2]) * c.double()).sum())  # noqa: E731
    for i, leaf in enumerate(leaves):
        d = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)
        e = 1e-4
        up, dn = [b.clone() for b in base], [b.clone() for b in base]
        up[i] += e * d
        dn[i] -= e * d
        want = (f(up) - f(dn)) / (2 * e)
        got = leaf.grad.double().cpu()
        # the difference's own error is O(e^2); the gradient's is 4 half steps of its norm, seen along d
        room = 4 * torch.finfo(dtype).eps / 2 * float(got.norm() * d.norm()) + 1e-5 * abs(want) + 1e-5
        assert abs(float((got * d).sum()) - want) <= room, i


def test_gradients_only_where_wanted_and_broadcast_inputs():
    from moe_offload import dense
    x, ids, wgu, wd = _layer(torch.bfloat16, 16, 2, 4, 64, 32)
    wd2 = wd.clone().requires_grad_()
    dense.switch_glu(x, ids, wgu, wd2).sum().backward()               # dy is an expanded scalar
    full = wd2.grad.clone()
    leaves = [t.clone().requires_grad_() for t in (x, wgu, wd)]
    dense.switch_glu(leaves[0], ids, leaves[1], leaves[2]).sum().backward()
    assert torch.equal(full, leaves[2].grad)
    # one token's row for all: the gradient is the sum over them
    one = x[:1].clone().requires_grad_()
    dense.switch_glu(one.expand(16, -1).contiguous(), ids, wgu, wd).float().sum().backward()
    many = x[:1].repeat(16, 1).requires_grad_()
    dense.switch_glu(many, ids, wgu, wd).float().sum().backward()
    assert torch.equal(one.grad, many.grad.sum(0, keepdim=True))


def test_autograd_refuses_capture():
    from moe_offload import dense
    x, ids, wgu, wd = _layer(torch.bfloat16, 16, 2, 4, 64, 32)
    leaves = [t.clone().requires_grad_() for t in (x, wgu, wd)]
    y = dense.switch_glu(leaves[0], ids, leaves[1], leaves[2])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="not captured"):
            dense.switch_glu(leaves[0], ids, leaves[1], leaves[2])
    y.float().sum().backward()
    assert bool(leaves[0].grad.isfinite().all())


@pytest.mark.parametrize("tokens", [1, 300])
def test_captured_step_replays(tokens):
    """A whole step (plan, both products, both gradients) captured twice and replayed with other data between."""
    from moe_offload import ops
    dt = torch.bfloat16
    x, ids, wgu, wd = _layer(dt, tokens, 3, 8, 72, 40)
    dy = rnd((tokens * 3, 72), dt, 30)

    def step():
        tok, order, seg = ops.expert_plan(ids, 8)
        gu = torch.empty((tokens * 3, 80), dtype=dt, device=DEV)
        h = ops.grouped_gate_up(x, tok, seg, wgu, gu_out=gu)
        y = ops.grouped_mm(h, seg, wd, row_out=order)
        dgu = ops.grouped_mm_dx(dy, seg, wd, row_in=order, gu=gu)
        return (h, y, dgu, ops.grouped_mm_dx(dgu, seg, wgu, row_out=order), ops.grouped_mm_dw(dy, h, seg, row_dy=order),
                ops.grouped_mm_dw(dgu, x, seg, row_x=tok, dtype=torch.float32))
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for n in range(3):
        x.copy_(rnd(x.shape, dt, 40 + n))
        dy.copy_(rnd(dy.shape, dt, 50 + n))
        ids.copy_(_layer(dt, tokens, 3, 8, 72, 40, seed=60 + n)[1])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_two_streams_at_once():
    from moe_offload import ops
    dt = torch.float16
    seg = i32(case("edges"))
    m, e = int(seg[-1]), seg.numel() - 1
    a = [(rnd((m, 264), dt, i), rnd((e, 136, 264), dt, 10 + i)) for i in range(2)]
    want = [ops.grouped_mm(x, seg, w) for x, w in a]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [[], []]
    for _ in range(10):
        with torch.cuda.stream(side):
            got[0].append(ops.grouped_mm(a[0][0], seg, a[0][1]))
        got[1].append(ops.grouped_mm(a[1][0], seg, a[1][1]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_again_and_alone(dtype):
    """No result depends on the order of blocks: calls repeat bit for bit."""
    from moe_offload import ops
    x, ids, wgu, wd = _layer(dtype, 200, 4, 12, 264, 136)
    tok, order, seg = ops.expert_plan(ids, 12)
    dy = rnd((800, 264), dtype, 3)
    f = lambda: (ops.grouped_switch_glu(x, tok, seg, wgu, wd, row_out=order),  # noqa: E731
                 ops.grouped_mm_dx(dy, seg, wd, row_in=order), ops.grouped_mm_dw(dy, x, seg, row_dy=order, row_x=tok))
    first = f()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, f()))
