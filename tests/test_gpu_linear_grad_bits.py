"""Gradients of shared projections whose dz = dy act'(z) is computed: it keeps its bits and its range on the way through the
products, whatever type the results have."""
import math

import pytest

import layer_ref as ref
from grouped_ref import F32, check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "relu2"]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def exact(dy, x, w, z, act, part, floor=2.0 ** -126):
    """((dx, bound), (dw, bound)).  The products take dz in parts, the rest behind them is lost: `part` of a value, or `floor`.  The
    function's own error and the sums' as ref.linear_grad has them."""
    d = dy.double()
    sd = torch.zeros_like(d)
    if act is not None:
        s = ref.slope(z.double(), act)
        sd = d.abs() * ref.slope_slack(z.double(), act) + (d * s).abs() * F32
        d = d * s
    sz = sd + (d.abs() + sd) * part + floor
    xd, wd = x.double(), w.double()
    n_tok, n_out = d.shape
    mag = d.abs() + sz
    dx = d @ wd, sz @ wd.abs() + (3 * n_out + 2) * F32 * (mag @ wd.abs())
    dT, sT, mT = (t.T.contiguous() for t in (d, sz, mag))
    dw = dT @ xd, sT @ xd.abs() + (3 * n_tok + 2) * F32 * (mT @ xd.abs())
    return dx, dw


# two parts: the first is cut at 8 bits (a step is 2^-7 of a value at most), the rest is rounded to 8 bits, off by half a step of its
# own, 2^-8; three: 24 bits, all there are
TWO, THREE = 2.0 ** -15, 0.0
# two fp16 values: half of dz cut at 11 bits, the rest times 2^10 rounded to 11 (or to 2^-25, or 2^-24 in the place of nothing)
HALVES = 2.0 ** -21, 2.0 ** -33


def lost(dtype, dy_type, act):
    """What 16-bit results' parts lose."""
    return HALVES if dtype == dy_type == torch.float16 and act in ("silu", "gelu") else (TWO,)

# few terms to a sum, so that what a term loses shows behind the result's own rounding; then every kind of tile, parts of the tokens,
# contractions that end inside a step
SMALL = [(16, 8, 8), (9, 64, 16), (24, 136, 8), (300, 16, 16)]
LARGE = [(100, 2560, 640), (777, 72, 520), (2500, 264, 1544), (777, 2056, 1032), (513, 2056, 520), (2049, 2056, 2056), (4097, 2056, 4104),
         (8200, 520, 72), (6001, 72, 264), (1500, 4104, 1544), (1999, 2560, 640)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", SMALL + LARGE)
def test_computed_dz_keeps_its_bits(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    x, w, z = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_out ** -0.5), rnd((n_tok, n_out), dtype, 3)
    for act, dy_type in (("silu", dtype), (None, torch.float32), ("gelu", torch.float32)) if n_tok * n_out < 1 << 21 else (("silu", dtype),):
        dy = rnd((n_tok, n_out), dy_type, 4)
        zz = None if act is None else z
        two = exact(dy, x, w, zz, act, *lost(dtype, dy_type, act))
        got = ops.linear_grad(dy, x, w, z=zz, act=act)
        check(got[0], *two[0], f"{act} {dy_type} dx")
        check(got[1], *two[1], f"{act} {dy_type} dw")
        got = ops.linear_grad(dy, x, w, z=zz, act=act, dw_dtype=torch.float32)
        check(got[0], *exact(dy, x, w, zz, act, TWO)[0], f"{act} {dy_type} dx beside fp32 dw")
        check(got[1], *exact(dy, x, w, zz, act, THREE)[1], f"{act} {dy_type} fp32 dw")


@pytest.mark.parametrize("act", [None] + ACTS)
def test_no_further_from_64_bits_than_one_rounding(act):
    """The norm of the error against that of one rounding of the exact values.  What two parts leave of a dz is at most 2^-15 of it, either
    way: a norm of 2^-15 / sqrt(3), next to 2.1e-4 for the rounding: 0.4% more, and the functions in fp32 less.  A dz in 16 bits
    adds as much as the rounding again (40% more)."""
    from moe_offload import ops
    n_tok, n_in, n_out = 1999, 640, 320
    dy = rnd((n_tok, n_out), torch.float32 if act is None else torch.float16, 1)
    x, w, z = rnd((n_tok, n_in), torch.float16, 2), rnd((n_out, n_in), torch.float16, 3, n_out ** -0.5), rnd((n_tok, n_out), torch.float16, 4)
    zz = None if act is None else z
    got = ops.linear_grad(dy, x, w, z=zz, act=act)
    for g, (want, _) in zip(got, exact(dy, x, w, zz, act, 0.0)):
        assert float((g.double() - want).norm()) < 1.05 * float((want.half().double() - want).norm())


@pytest.mark.parametrize("n_tok,n_in,n_out", [(8, 16, 16), (1500, 72, 264)])
def test_values_past_fp16_and_below_it(n_tok, n_in, n_out):
    """An fp32 dy whose values fp16 does not hold, with results that are held."""
    from moe_offload import ops
    x, w = rnd((n_tok, n_in), torch.float16, 1), rnd((n_out, n_in), torch.float16, 2)
    for scale, wide in ((1e-9, 1.0), (3e6, 2.0 ** -12), (1e-20, 1.0), (1e25, 1.0)):
        dy = rnd((n_tok, n_out), torch.float32, 3) * scale
        ww = (w.float() * wide).half()
        (want_dx, sx), _ = exact(dy, x, ww, None, None, TWO)
        dx, dw, _ = ops.linear_grad(dy, x, ww, dw_dtype=torch.float32)
        check(dw, *exact(dy, x, ww, None, None, THREE)[1], f"dw {scale}")
        if scale < 1e10:
            check(dx, want_dx, sx, f"dx {scale}")
    z, dy = rnd((n_tok, n_out), torch.float16, 4, 400.0), rnd((n_tok, n_out), torch.float16, 5, 400.0)
    ww = (w.float() * 2.0 ** -10).half()
    dx, dw, _ = ops.linear_grad(dy, x, ww, z=z, act="relu2", dw_dtype=torch.float32)
    (want_dx, sx), _ = exact(dy, x, ww, z, "relu2", TWO)
    check(dx, want_dx, sx, "relu2 dx")
    check(dw, *exact(dy, x, ww, z, "relu2", THREE)[1], "relu2 dw")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_fp16_gradients_from_the_smallest_to_the_largest(act):
    """dy at fp16's ends: its largest through slopes above 1, its subnormals."""
    from moe_offload import ops
    n_tok, n_in, n_out = 200, 72, 16
    x, z = rnd((n_tok, n_in), torch.float16, 1), torch.linspace(-8, 8, n_tok * n_out, device=DEV).reshape(n_tok, n_out).half()
    for scale, wide in ((2.0 ** -20, 2.0 ** 8), (2.0 ** -12, 16.0), (65504.0, 2.0 ** -9)):
        dy = torch.full((n_tok, n_out), scale, device=DEV).half() * rnd((n_tok, n_out), torch.float16, 2).sign()
        w = rnd((n_out, n_in), torch.float16, 3, wide)
        xx = (x.float() * wide).half()
        got = ops.linear_grad(dy, xx, w, z=z, act=act)
        for g, (want, slack), name in zip(got, exact(dy, xx, w, z, act, *HALVES), ("dx", "dw")):
            check(g, want, slack, f"{scale} {name}")


def kinds(t):
    """-1, 1 for infinities, 2 for NaN, 0 for numbers."""
    return torch.where(t.isnan(), 2, torch.where(t == math.inf, 1, torch.where(t == -math.inf, -1, 0)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dy_type,act", [(torch.float32, None), (None, "silu")])
def test_infinities_and_nan_go_where_the_formulas_put_them(dtype, dy_type, act):
    """One in dy, x or w at a time (two could cancel): an infinity meets all parts of a value with the same sign."""
    from moe_offload import ops
    for n_tok, n_in, n_out in ((12, 16, 16), (300, 72, 136)):
        for bad in (math.inf, -math.inf, math.nan):
            for where in ("dy", "x", "w"):
                t = {"dy": rnd((n_tok, n_out), dy_type or dtype, 1), "x": rnd((n_tok, n_in), dtype, 2), "w": rnd((n_out, n_in), dtype, 3)}
                t["dy"][2], t["dy"][3, ::2], t["x"][4], t["w"][5] = 1.0, 0.0, 1.0, -2.0      # values that one part holds whole
                t[where][2, 5] = bad
                z = None if act is None else torch.full((n_tok, n_out), 0.5, dtype=dtype, device=DEV)
                d = t["dy"].double() * (1 if z is None else ref.slope(z.double(), act))
                # (products one by one: a library's own may take a shorter way to an infinity)
                want_dx = (d.unsqueeze(2) * t["w"].double()).sum(1)
                want_dw = (d.unsqueeze(2) * t["x"].double().unsqueeze(1)).sum(0)
                for dw_type in (None, torch.float32):
                    dx, dw, _ = ops.linear_grad(t["dy"], t["x"], t["w"], z=z, act=act, dw_dtype=dw_type)
                    assert torch.equal(kinds(dx), kinds(want_dx)), (where, bad, "dx")
                    assert torch.equal(kinds(dw), kinds(want_dw)), (where, bad, "dw")


def test_the_router_of_a_layer_gets_its_logits_gradient_whole():
    """fp32 logits of an fp16 layer, a gradient below fp16's smallest value: the router's weights still move."""
    from moe_offload import dense
    x, w = rnd((64, 128), torch.float16, 1, 100.0).requires_grad_(), rnd((16, 128), torch.float16, 2, 0.1).requires_grad_()
    logits = dense.linear(x, w, dtype=torch.float32)
    dy = rnd(logits.shape, torch.float32, 3, 1e-8)
    logits.backward(dy)
    (want_dx, sx), (want_dw, sw) = exact(dy, x.detach(), w.detach(), None, None, TWO)
    check(x.grad, want_dx, sx)
    check(w.grad, want_dw, sw)
    assert bool(w.grad.any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_images_past_32_bits(dtype):
    """Images of dz of 2^30 elements and more, the rows that count at their end."""
    from moe_offload import ops
    n_tok, n_in, n_out = (1 << 20) + 24, 64, 1032
    x, w = torch.zeros((n_tok, n_in), dtype=dtype, device=DEV), rnd((n_out, n_in), dtype, 1, n_out ** -0.5)
    dy, z = torch.zeros((n_tok, n_out), dtype=dtype, device=DEV), torch.zeros((n_tok, n_out), dtype=dtype, device=DEV)
    x[-40:], dy[-40:], z[-40:] = rnd((40, n_in), dtype, 2), rnd((40, n_out), dtype, 3), rnd((40, n_out), dtype, 4)
    for dw_type, lose in ((None, lost(dtype, dtype, "silu")), (torch.float32, (THREE,))):
        dx, dw, _ = ops.linear_grad(dy, x, w, z=z, act="silu", dw_dtype=dw_type)
        want_dx = exact(dy[-40:], x[-40:], w, z[-40:], "silu", *(lose if dw_type is None else (TWO,)))[0]
        check(dx[-40:], *want_dx, "dx")
        check(dw, *exact(dy[-40:], x[-40:], w, z[-40:], "silu", *lose)[1], "dw")
        assert not bool(dx[:-40].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_replayed_and_side_by_side(dtype):
    """Every form of dz in a graph, replayed with other inputs between eager calls, and on two streams at once."""
    from moe_offload import ops
    x, w = rnd((300, 136), dtype, 1), rnd((72, 136), dtype, 2)
    z, dy, wide = rnd((300, 72), dtype, 3), rnd((300, 72), dtype, 4), rnd((300, 72), torch.float32, 5)
    forms = [lambda: ops.linear_grad(dy, x, w, z=z, act="silu", bias=True), lambda: ops.linear_grad(dy, x, w, z=z, act="relu2"),
             lambda: ops.linear_grad(wide, x, w, dw_dtype=torch.float32), lambda: ops.linear_grad(wide, x, w, z=z, act="gelu")]
    graphs, held = [], []
    for form in forms:
        form()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(form())
    for seed in (1, 2, 3):
        dy.copy_(rnd(dy.shape, dtype, seed + 10))
        wide.copy_(rnd(wide.shape, torch.float32, seed + 20))
        for i in (0, 1, 2, 3, 3, 1, 2, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for h, form in zip(held, forms):
            assert all(torch.equal(a, b) for a, b in zip(h, form()) if a is not None)
    want = [form() for form in forms]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append([form() for form in forms])
    torch.cuda.synchronize()
    for runs in got:
        for run in runs:
            for r, v in zip(run, want):
                assert all(torch.equal(a, b) for a, b in zip(r, v) if a is not None)
