"""Long contractions in parts: lengths that leave whole parts nothing when rounded, sums in place, two calls at a time."""
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


# 121 steps in 15 parts of 9, 14 of which have something; 1563 in 97 parts of 17 (92)
@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_that_rounding_would_leave_empty(dtype):
    from moe_offload import ops
    n_tok, n_in, n_out = 64, 7744, 1040
    x, w, b, res = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_in ** -0.5), rnd((n_out,), dtype, 3), rnd((n_tok, n_out), dtype, 4)
    want, slack, wz, sz = ref.linear(x, w, b, "silu", res)
    z = torch.empty_like(res)
    check(ops.linear(x, w, bias=b, act="silu", residual=res, z_out=z), want, slack)
    check(z, wz, sz, "z")
    n_tok = 100000
    dy, x, w = rnd((n_tok, 64), dtype, 5), rnd((n_tok, 64), dtype, 6), rnd((64, 64), dtype, 7)
    for dw_type in (None, torch.float32):
        got = ops.linear_grad(dy, x, w, bias=True, dw_dtype=dw_type)
        for g, (v, s), name in zip(got, ref.linear_grad(dy, x, w, None, None), ("dx", "dw", "db")):
            check(g, v, s, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_on_the_residual(dtype):
    from moe_offload import ops
    lib_bytes = ops._lib.lib().moe_linear_workspace_bytes
    for n_tok, n_in, n_out in ((32, 4096, 4096), (100, 2560, 640)):
        assert lib_bytes(n_tok, n_in, n_out) > 0
        x, w, b, wide = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_in ** -0.5), rnd((n_out,), dtype, 3), rnd((n_tok, n_out + 16), dtype, 4)
        stream = wide[:, 8:-8]
        want, slack, *_ = ref.linear(x, w, b, "gelu", stream)
        kept = wide.clone()
        assert ops.linear(x, w, bias=b, act="gelu", residual=stream, out=stream) is stream
        check(stream, want, slack)
        assert torch.equal(wide[:, :8], kept[:, :8]) and torch.equal(wide[:, -8:], kept[:, -8:])


def test_two_calls_at_a_time_and_replayed():
    from moe_offload import ops
    cases = [(rnd((32, 4096), torch.bfloat16, 10 * i), rnd((4096, 4096), torch.bfloat16, 10 * i + 1, 1 / 64)) for i in range(2)]
    want = [ops.linear(x, w, act="silu") for x, w in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, (s, (x, w)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(ops.linear(x, w, act="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    graphs, held = [], []
    for x, w in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(ops.linear(x, w, act="silu"))
    for seed in (1, 2, 3):
        for i, (x, w) in enumerate(cases):
            x.copy_(rnd(x.shape, torch.bfloat16, seed + 7 * i))
        for i in (0, 1, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for h, (x, w) in zip(held, cases):
            assert torch.equal(h, ops.linear(x, w, act="silu"))
