"""Routing, weighted sums, shared projections and clipping where sizes, streams and graphs are at their edges: every tile that a
call's sizes select, offsets past 32 bits, several launches, calls side by side."""
import math

import pytest

import layer_ref as ref
from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


# (tokens, n_in, n_out), one size at least for every kind of tile, with sides that end inside one
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", [(40, 200, 72), (600, 264, 520), (1030, 72, 1856), (513, 72, 2056), (513, 72, 4104), (2049, 136, 2056),
                                              (2049, 72, 4104), (8192, 328, 4104), (70, 4104, 1032), (100, 2600, 328), (520, 4000, 200)])
def test_every_tile_forward(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    x, w, b, res = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_in ** -0.5), rnd((n_out,), dtype, 3), rnd((n_tok, n_out), dtype, 4)
    want, slack, wz, sz = ref.linear(x, w, b, "gelu", res)
    z = torch.empty((n_tok, n_out), dtype=dtype, device=DEV)
    check(ops.linear(x, w, bias=b, act="gelu", residual=res, z_out=z), want, slack)
    check(z, wz, sz, "z")
    check(ops.linear(x, w, bias=b, act="gelu", residual=res, dtype=torch.float32), want, slack, "fp32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", [(40, 200, 72), (777, 72, 520), (2500, 264, 1544), (513, 2056, 520), (777, 2056, 1032), (2049, 2056, 2056),
                                              (4097, 2056, 4104), (8200, 520, 72), (6000, 72, 264)])
def test_every_tile_backward(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    dy, x, w, z = rnd((n_tok, n_out), dtype, 1), rnd((n_tok, n_in), dtype, 2), rnd((n_out, n_in), dtype, 3, n_out ** -0.5), rnd((n_tok, n_out), dtype, 4)
    want = ref.linear_grad(dy, x, w, z, "silu")
    got = ops.linear_grad(dy, x, w, z=z, act="silu", bias=True)
    for g, (v, slack), name in zip(got, want, ("dx", "dw", "db")):
        check(g, v, slack, name)
    # alone, of either type
    check(ops.linear_grad(dy, x, w, z=z, act="silu", want_dw=False)[0], *want[0], "dx alone")
    check(ops.linear_grad(dy, x, w, z=z, act="silu", want_dx=False, dw_dtype=torch.float32)[1], *want[1], "dw alone")


# large tiles over contractions of a part of a step, of one, and of few more than are under way at once; the kinds that the sizes above
# leave out
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", [(3000, 8, 4104), (3000, 72, 4104), (2900, 328, 4104), (5000, 64, 776), (5000, 200, 776), (2049, 8, 4104),
                                              (2100, 264, 4104), (777, 8, 2568), (777, 392, 2568), (564, 8, 10904), (564, 136, 10904), (12000, 72, 264),
                                              (131, 72, 8264)])
def test_large_tiles_short_contractions(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    x, w, b, res = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_in ** -0.5), rnd((n_out,), dtype, 3), rnd((n_tok, n_out), dtype, 4)
    want, slack, wz, sz = ref.linear(x, w, b, "silu", res)
    z = torch.empty((n_tok, n_out), dtype=dtype, device=DEV)
    check(ops.linear(x, w, bias=b, act="silu", residual=res, z_out=z), want, slack)
    check(z, wz, sz, "z")
    check(ops.linear(x, w, bias=b, act="silu", residual=res, dtype=torch.float32), want, slack, "fp32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,n_in,n_out", [(1500, 4104, 1544), (2049, 4104, 1544), (300, 4104, 264), (777, 4104, 776), (513, 4104, 520), (8192, 72, 1032),
                                              (40, 4104, 4104), (8200, 4104, 8)])
def test_large_tiles_backward(dtype, n_tok, n_in, n_out):
    from moe_offload import ops
    dy, x, w, z = rnd((n_tok, n_out), dtype, 1), rnd((n_tok, n_in), dtype, 2), rnd((n_out, n_in), dtype, 3, n_out ** -0.5), rnd((n_tok, n_out), dtype, 4)
    want = ref.linear_grad(dy, x, w, z, "gelu")
    got = ops.linear_grad(dy, x, w, z=z, act="gelu", bias=True)
    for g, (v, slack), name in zip(got, want, ("dx", "dw", "db")):
        check(g, v, slack, name)
    check(ops.linear_grad(dy, x, w, z=z, act="gelu", want_dw=False)[0], *want[0], "dx alone")
    check(ops.linear_grad(dy, x, w, z=z, act="gelu", want_dx=False, dw_dtype=torch.float32)[1], *want[1], "dw alone")


def test_offsets_past_32_bits():
    """x and y of more than 2^32 bytes, the rows that count at their end."""
    from moe_offload import ops
    n_tok, n_in, n_out = (1 << 20) + 24, 2056, 64
    x = torch.zeros((n_tok, n_in), dtype=torch.bfloat16, device=DEV)
    tail = rnd((40, n_in), torch.bfloat16, 1)
    x[-40:] = tail
    w, b = rnd((n_out, n_in), torch.bfloat16, 2, n_in ** -0.5), rnd((n_out,), torch.bfloat16, 3)
    got = ops.linear(x, w, bias=b)
    want, slack, *_ = ref.linear(tail, w, b)
    check(got[-40:], want, slack)
    assert torch.equal(got[:-40], b.expand(n_tok - 40, n_out))
    dy = torch.zeros((n_tok, n_out), dtype=torch.bfloat16, device=DEV)
    dy[-40:] = rnd((40, n_out), torch.bfloat16, 4)
    dx, dw, db = ops.linear_grad(dy, x, w, bias=True)
    (wx, sx), (ww, sw), (wb, sb) = ref.linear_grad(dy[-40:], tail, w, None, None)
    check(dx[-40:], wx, sx, "dx")
    check(dw, ww, sw, "dw")
    check(db, wb, sb, "db")
    assert not bool(dx[:-40].any())
    # the transposed case: many columns
    wide = torch.zeros((n_tok, 8), dtype=torch.bfloat16, device=DEV)
    wide[-40:] = rnd((40, 8), torch.bfloat16, 5)
    x8 = rnd((2056, 8), torch.bfloat16, 6)
    out = ops.linear(x8, wide[:(1 << 20)])
    assert out.numel() > 1 << 31 and not bool(out[:, :-24].any())
    want, slack, *_ = ref.linear(x8, wide[(1 << 20) - 16:(1 << 20)])
    check(out[:, -16:], want, slack)


def test_more_tokens_than_one_launch_routes():
    from moe_offload import ops
    n_tok = (1 << 24) + 5
    logits = torch.zeros((n_tok, 2), dtype=torch.bfloat16, device=DEV)
    logits[:, 1] = torch.arange(n_tok, device=DEV).remainder(3).sub(1)           # -1, 0, 1 in turn
    ids, w = ops.route(logits, 1, renorm=False)
    assert torch.equal(ids[:, 0], (logits[:, 1] > 0).int())
    p = torch.tensor([1 / (1 + math.exp(-1)), 0.5], dtype=torch.float64, device=DEV)
    want = torch.where(logits[:, 1] == 0, p[1], p[0])
    check(w[:, 0], want, want * 40 * ref.F32)
    dw = torch.ones((n_tok, 1), device=DEV)
    d = ops.route_grad(dw, logits, ids, renorm=False)
    g = want * (1 - want)
    sign = torch.where(ids[:, 0] == 0, 1.0, -1.0)
    check(d[:, 0], g * sign, g * 100 * ref.F32)
    check(d[:, 1], -g * sign, g * 100 * ref.F32)


def test_calls_side_by_side_on_two_streams():
    """Gradients with a workspace of their own each: neither call sees the other's."""
    from moe_offload import ops
    cases = [[rnd(s, torch.bfloat16, 10 * i + j) for j, s in enumerate([(3000, 264), (3000, 520), (264, 520), (3000, 264)])] for i in range(2)]
    want = [ops.linear_grad(dy, x, w, z=z, act="gelu", bias=True) for dy, x, w, z in cases]
    norms = [ops.clip_grad_norm([t for t in w], 1.0, out=[torch.empty_like(t) for t in w]) for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got, gn = [[], []], [[], []]
    for _ in range(10):
        for i, (s, (dy, x, w, z)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_grad(dy, x, w, z=z, act="gelu", bias=True))
                gn[i].append(ops.clip_grad_norm(list(got[i][-1]), 1.0, out=[torch.empty_like(t) for t in got[i][-1]]))
    torch.cuda.synchronize()
    for i in range(2):
        for g, n in zip(got[i], gn[i]):
            assert all(torch.equal(a, b) for a, b in zip(g, want[i])) and torch.equal(n, norms[i])


def test_two_graphs_replayed_in_turn():
    from moe_offload import ops
    data = [[rnd(s, torch.bfloat16, 100 + 10 * i + j) for j, s in enumerate([(2200, 72), (2200, 264), (72, 264), (2200, 72)])] for i in range(2)]

    def step(dy, x, w, z):
        grads = ops.linear_grad(dy, x, w, z=z, act="silu", bias=True)
        return (*grads, ops.clip_grad_norm(list(grads), 0.5))

    step(*data[0])
    torch.cuda.synchronize()
    graphs, held = [], []
    for d in data:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(*d))
    for seed in (1, 2, 3):
        for i, d in enumerate(data):
            d[0].copy_(rnd(d[0].shape, torch.bfloat16, seed + 7 * i))
        for i in (0, 1, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for h, d in zip(held, data):
            for a, b in zip(h, step(*d)):
                assert torch.equal(a, b)


def test_a_given_workspace_may_be_larger_and_hold_anything():
    from moe_offload import ops
    dy, x, w, z = (rnd(s, torch.float16, j) for j, s in enumerate([(1500, 72), (1500, 264), (72, 264), (1500, 72)]))
    want = ops.linear_grad(dy, x, w, z=z, act="relu2", bias=True)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device=DEV)
    got = ops.linear_grad(dy, x, w, z=z, act="relu2", bias=True, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="workspace"):
        ops.linear_grad(dy, x, w, z=z, act="relu2", bias=True, workspace=ws[:100])
    # a long contraction over few tiles; with 512 columns it needs none
    for n_out in (512, 1032):
        a, b = rnd((70, 4096), torch.float16, 5), rnd((n_out, 4096), torch.float16, 6, 1 / 64)
        out = torch.full((90, n_out + 8), 7.0, dtype=torch.float16, device=DEV)
        want = ops.linear(a, b, act="gelu")
        assert torch.equal(ops.linear(a, b, act="gelu", workspace=ws), want)
        ops.linear(a, b, act="gelu", workspace=ws, out=out[:70, 8:])
        assert torch.equal(out[:70, 8:], want) and bool((out[70:] == 7).all()) and bool((out[:, :8] == 7).all())
    with pytest.raises(ValueError, match="workspace"):
        ops.linear(a, b, workspace=ws[:100])


def test_refusals_on_the_gpu():
    from moe_offload import ops
    x, w = rnd((4, 64), torch.bfloat16, 1), rnd((16, 64), torch.bfloat16, 2)
    y, s, l = rnd((4, 2, 64), torch.bfloat16, 3), torch.ones((4, 2), device=DEV), rnd((4, 16), torch.float32, 4)
    ids = torch.zeros((4, 2), dtype=torch.int32, device=DEV)
    value = [lambda: ops.linear(x, w, act="tanh"), lambda: ops.linear(x, w[:, :56]), lambda: ops.linear(x, w[:12]), lambda: ops.linear(x, w, bias=x[0]),
             lambda: ops.linear(x, w, residual=x), lambda: ops.linear(x, w.T), lambda: ops.linear_grad(x[:, :16], x, w, act="silu"),
             lambda: ops.linear_grad(x[:, :16], x, w, z=x[:, :16]), lambda: ops.combine(y, s[:3]), lambda: ops.combine(y[:, :1], s),
             lambda: ops.combine(y, s.T.contiguous()), lambda: ops.combine_grad(x[:3], y, s), lambda: ops.route(l, 17), lambda: ops.route(l, 0),
             lambda: ops.route(l, 2, score="tanh"), lambda: ops.route(l, 2, n_group=3), lambda: ops.route(l, 2, n_group=4, topk_group=5),
             lambda: ops.route(l, 2, group_best=3), lambda: ops.route(l, 2, bias=l[0, :8].contiguous()), lambda: ops.route(l.T, 2),
             lambda: ops.route_grad(s[:3], l, ids), lambda: ops.route_grad(s, l, ids[0])]
    kind = [lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w, dtype=torch.float16),
            lambda: ops.combine(y, s.half()), lambda: ops.combine(y, s, out=x.half()), lambda: ops.route(l.double(), 2), lambda: ops.route(l, 2, bias=l[0].half()),
            lambda: ops.route_grad(s, l, ids.long()), lambda: ops.route_grad(s.half(), l, ids), lambda: ops.linear_grad(x[:, :16].half(), x, w),
            lambda: ops.linear_grad(x[:, :16], x, w, dw_dtype=torch.float16)]
    for call in value:
        with pytest.raises(ValueError):
            call()
    for call in kind:
        with pytest.raises(TypeError):
            call()
    for bad in (x[:, 4:12], torch.empty((4, 68), dtype=torch.bfloat16, device=DEV)[:, 4:]):
        with pytest.raises(Exception):
            ops.linear(bad, w)
