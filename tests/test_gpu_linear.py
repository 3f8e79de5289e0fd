"""Shared projections with bias, activation and residual, and their gradients, against the formulas in 64 bits."""
import math

import pytest

import layer_ref as ref
from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
ACTS = [None, "silu", "gelu", "relu2"]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def make(n_tok, n_in, n_out, dtype, seed=0):
    """x, w, bias, residual"""
    return (rnd((n_tok, n_in), dtype, seed), rnd((n_out, n_in), dtype, seed + 1, n_in ** -0.5), rnd((n_out,), dtype, seed + 2, 0.5),
            rnd((n_tok, n_out), dtype, seed + 3))


# one token to several tiles of every kind, sides that end inside a tile and a step, contractions of one step and of a part of one
SIZES = [(1, 8, 8), (1, 2048, 2048), (2, 520, 24), (7, 64, 1000), (8, 2048, 512), (16, 4096, 256), (17, 136, 72), (33, 1000, 264),
         (64, 64, 64), (100, 2560, 640), (129, 256, 2056), (300, 72, 4096), (513, 640, 520), (777, 1152, 320), (1111, 512, 1032),
         (2500, 264, 1544), (4100, 128, 2048)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", SIZES)
def test_product(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    x, w, b, res = make(n_tok, n_in, n_out, dtype, n_tok)
    want, slack, *_ = ref.linear(x, w)
    got = ops.linear(x, w)
    assert got.dtype == dtype
    check(got, want, slack, "plain")
    got = ops.linear(x, w, dtype=torch.float32)
    assert got.dtype == torch.float32
    check(got, want, slack, "fp32")
    z = torch.full((n_tok, n_out), math.nan, dtype=dtype, device=DEV)
    act = ACTS[1 + (n_tok + n_in) % 3]
    got = ops.linear(x, w, bias=b, act=act, residual=res, z_out=z)
    want, slack, wz, sz = ref.linear(x, w, b, act, res)
    check(got, want, slack, act)
    check(z, wz, sz, "z")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n_tok", [5, 40, 1500])
def test_epilogue(dtype, act, n_tok):
    from moe_offload import ops
    x, w, b, res = make(n_tok, 200, 328, dtype, 50)
    x = x * 3
    for bias in (None, b):
        for r in (None, res):
            want, slack, wz, sz = ref.linear(x, w, bias, act, r)
            z = torch.empty((n_tok, 328), dtype=dtype, device=DEV)
            check(ops.linear(x, w, bias=bias, act=act, residual=r, z_out=z), want, slack, f"{bias is not None} {r is not None}")
            check(z, wz, sz, "z")
            check(ops.linear(x, w, bias=bias, act=act, residual=r, dtype=torch.float32), want, slack, "fp32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok", [3, 90, 1300])
def test_steps_given_outputs_and_in_place(dtype, n_tok):
    from moe_offload import ops
    xs, w, b, _ = make(n_tok, 320, 136, dtype, 60)
    x, wide = xs[:, 24:152], w[:, :128].contiguous()
    out = torch.full((n_tok, 160), 7.0, dtype=dtype, device=DEV)
    z = torch.full((n_tok, 176), 7.0, dtype=dtype, device=DEV)
    res = rnd((n_tok, 200), dtype, 61)
    ops.linear(x, wide, bias=b, act="silu", residual=res[:, 8:144], z_out=z[:, 16:152], out=out[:, 8:144])
    want, slack, wz, sz = ref.linear(x, wide, b, "silu", res[:, 8:144])
    check(out[:, 8:144], want, slack)
    check(z[:, 16:152], wz, sz)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 144:] == 7).all()) and bool((z[:, :16] == 7).all()) and bool((z[:, 152:] == 7).all())
    stream = res[:, 8:144].clone()
    assert ops.linear(x, wide, bias=b, act="silu", residual=stream, out=stream) is stream
    check(stream, want, slack)
    assert ops.linear(x[:0], wide).shape == (0, 136)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n_tok", [4, 200])
def test_infinities_and_nan_stay_in_their_rows(act, n_tok):
    from moe_offload import ops
    x, w, b, _ = make(n_tok, 64, 64, torch.float16, 70)
    w = w.abs() + 0.01
    x[1, 3], x[2, 5], x[3, 7] = math.nan, math.inf, -math.inf
    x[0] = 60000.0                                 # past fp16's range
    got, z = torch.empty((n_tok, 64), device=DEV), torch.empty((n_tok, 64), dtype=torch.float16, device=DEV)
    ops.linear(x, w, bias=b, act=act, z_out=z, out=got)
    assert bool(got[1].isnan().all()) and bool(got[2].eq(math.inf).all())
    if act in ("silu", "gelu", "relu2"):
        assert not bool(got[3].any())              # their limits
    else:
        assert bool(got[3].eq(-math.inf).all())
    want, slack, *_ = ref.linear(x[4:], w, b, act)
    check(got[4:], want, slack)
    assert bool(got[0].isfinite().all())


def grads(dtype, n_tok, n_in, n_out, act, dy_type=None, seed=0):
    x, w, _, z = make(n_tok, n_in, n_out, dtype, seed)
    return rnd((n_tok, n_out), dy_type or dtype, seed + 9), x, w, None if act is None else z


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", [(1, 8, 8), (3, 64, 1000), (17, 136, 72), (64, 64, 64), (100, 2560, 640), (300, 72, 4096), (513, 640, 520),
                                              (777, 1152, 320), (2500, 264, 1544), (4100, 512, 128)])
def test_gradients(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    for act in (None, ACTS[1 + (n_tok + n_in) % 3]):
        dy, x, w, z = grads(dtype, n_tok, n_in, n_out, act, seed=n_tok)
        got = ops.linear_grad(dy, x, w, z=z, act=act, bias=True)
        for g, (want, slack), name in zip(got, ref.linear_grad(dy, x, w, z, act), ("dx", "dw", "db")):
            assert g.dtype == dtype
            check(g, want, slack, f"{act} {name}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gradients_of_every_activation_and_of_fp32(dtype, act):
    from moe_offload import ops
    for dy_type in (dtype, torch.float32):
        dy, x, w, z = grads(dtype, 200, 192, 264, act, dy_type, seed=80)
        if z is not None:
            z = z * 4
        want = ref.linear_grad(dy, x, w, z, act)
        got = ops.linear_grad(dy, x, w, z=z, act=act, bias=True, dw_dtype=torch.float32)
        assert got[1].dtype == torch.float32
        for g, (v, slack), name in zip(got, want, ("dx", "dw", "db")):
            check(g, v, slack, f"{dy_type} {name}")
        for which in ("dx", "dw", "db"):
            one = ops.linear_grad(dy, x, w, z=z, act=act, bias=which == "db", want_dx=which == "dx", want_dw=which == "dw")
            assert [g is not None for g in one] == [which == n for n in ("dx", "dw", "db")]
            i = ("dx", "dw", "db").index(which)
            check(one[i], *want[i], f"only {which}")


@pytest.mark.parametrize("act", ["silu", "gelu", "relu2"])
def test_gradients_against_differences(act):
    """In z of 64 bits: (act(z + h) - act(z - h)) / 2h, h = 2^-10, off by h^2 / 6 of a third derivative below 2 (relu2: where the
    parabola starts, by h at most)."""
    from moe_offload import ops
    z = torch.linspace(-8, 8, 64, device=DEV).half().reshape(1, 64)
    eye = torch.eye(64, device=DEV).half()
    dx, _, db = ops.linear_grad(torch.ones((1, 64), device=DEV, dtype=torch.float16), eye[:1], eye, z=z, act=act, bias=True)
    h = 2.0 ** -10
    diff = (ref.activation(z.double() + h, act) - ref.activation(z.double() - h, act)) / (2 * h)
    room = h * h / 3 + (h if act == "relu2" else 0) + diff.abs() * 2.0 ** -11 + 2.0 ** -19 + 2.0 ** -25
    assert bool(((dx.double() - diff).abs() <= room).all()) and bool(((db.double() - diff[0]).abs() <= room[0]).all())


@pytest.mark.parametrize("act", ["silu", "gelu", "relu2"])
def test_gradients_where_z_left_the_range(act):
    """z = +-inf (fp16's range) and its lowest and highest values: the slope's limits."""
    from moe_offload import ops
    z = torch.tensor([[math.inf, -math.inf, 65504.0, -65504.0, 0.0, -0.0, 200.0, -200.0]], device=DEV).half()
    dy = torch.ones((1, 8), dtype=torch.float16, device=DEV)
    eye = torch.eye(8, device=DEV).half()
    dz = ops.linear_grad(dy, eye[:1], eye, z=z, act=act, bias=True)[2]
    if act == "relu2":
        want = [math.inf, 0, math.inf, 0, 0, 0, 400, 0]
    else:
        want = [1, 0, 1, 0, 0.5, 0.5, 1, 0]
    assert dz.tolist() == want
    z[0, 3] = math.nan
    assert bool(ops.linear_grad(dy, eye[:1], eye, z=z, act=act, bias=True)[2][3].isnan())


def test_gradients_without_tokens_and_with_steps():
    from moe_offload import ops
    dy, x, w, z = grads(torch.bfloat16, 0, 64, 128, "silu")
    dx, dw, db = ops.linear_grad(dy, x, w, z=z, act="silu", bias=True)
    assert dx.shape == (0, 64) and not bool(dw.any()) and not bool(db.any())
    xs, dys, zs = rnd((70, 96), torch.bfloat16, 1), rnd((70, 160), torch.bfloat16, 2), rnd((70, 144), torch.bfloat16, 3)
    w = rnd((128, 64), torch.bfloat16, 4, 0.1)
    args = dys[:, 16:144], xs[:, 8:72], w, zs[:, 8:136]
    for act in (None, "gelu"):
        zz = None if act is None else args[3]
        for g, (want, slack) in zip(ops.linear_grad(*args[:3], z=zz, act=act, bias=True), ref.linear_grad(*args[:3], zz, act)):
            check(g, want, slack)


def test_captured_and_replayed():
    from moe_offload import ops
    x, w, b, res = make(150, 256, 512, torch.bfloat16, 90)

    def both():
        z = torch.empty_like(res)
        y = ops.linear(x, w, bias=b, act="gelu", residual=res, z_out=z)
        return (y, z, *ops.linear_grad(y, x, w, z=z, act="gelu", bias=True))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (1, 2, 3):
        x.copy_(rnd(x.shape, x.dtype, seed))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, both()):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_does_not_depend_on_its_neighbours(dtype):
    """A token's result in a batch of one kind of tile: rows that are not its own do not reach it."""
    from moe_offload import ops
    x, w, b, _ = make(300, 512, 384, dtype, 91)
    a = ops.linear(x, w, bias=b, act="silu")
    other = x.clone()
    other[1::2] = math.nan
    assert torch.equal(ops.linear(other, w, bias=b, act="silu")[::2], a[::2])
