"""The norm of many tensors and their scaling against 64 bits."""
import math

import pytest

from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# the norm is a sum in 64 bits, rounded once: half a step of it, and the square root's and sum's own rounding far below that;
# the factor one more, and a product
NORM, SCALED = 2.0 ** -30, 3 * 2.0 ** -24


def make(sizes, dtype, seed=0, scale=0.01):
    g = torch.Generator(device=DEV).manual_seed(seed)
    types = TYPES if dtype is None else [dtype]
    return [(torch.randn(n, device=DEV, generator=g) * scale).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def norm_of(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def verify(ts, max_norm, before, norm, outs):
    want = norm_of(before)
    check(norm, torch.tensor(want, dtype=torch.float64, device=DEV), want * NORM, "norm")
    f = min(1.0, max_norm / (want + 1e-6))
    for i, (b, o) in enumerate(zip(before, outs)):
        v = b.double() * f
        check(o, v, v.abs() * SCALED, f"tensor {i}")
        if f == 1.0:
            assert torch.equal(o, b)


SIZES = [[1], [7], [8], [16384], [16385], [65537, 0, 3], [1000] * 7, [5, 1, 4, 1, 3, 1, 2], [1 << 20, 12345, 1], list(range(0, 300)), [33] * 100]


@pytest.mark.parametrize("dtype", TYPES + [None])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_scaling(dtype, sizes):
    from moe_offload import ops
    ts = make(sizes, dtype)
    before = [t.clone() for t in ts]
    norm = norm_of(ts)
    check(ops.grad_norm(ts), torch.tensor(norm, dtype=torch.float64, device=DEV), norm * NORM)
    for limit in (0.3 * norm, 2 * norm + 1):
        outs = [torch.full_like(t, 7) for t in ts]
        verify(ts, limit, before, ops.clip_grad_norm(ts, limit, out=outs), outs)
        assert all(torch.equal(t, b) for t, b in zip(ts, before))
    verify(ts, 0.3 * norm, before, ops.clip_grad_norm(ts, 0.3 * norm), ts)


@pytest.mark.parametrize("dtype", TYPES)
def test_starts_anywhere_and_borders_kept(dtype):
    """Views that start at any element, neighbours in one buffer, outputs that start elsewhere in their line."""
    from moe_offload import ops
    for shift in (0, 1, 3, 5):
        flat = make([50000], dtype, shift)[0]
        cuts = [shift, shift + 1, shift + 18, shift + 9000, shift + 9003, shift + 40000, 49999]
        ts = [flat[a:b] for a, b in zip(cuts[:-1], cuts[1:])]
        before, whole = [t.clone() for t in ts], flat.clone()
        norm = norm_of(ts)
        for other in (0, 1, 4):
            space = torch.full((50008,), 7.0, dtype=dtype, device=DEV)
            outs = [space[a + other:b + other] for a, b in zip(cuts[:-1], cuts[1:])]
            verify(ts, norm / 2, before, ops.clip_grad_norm(ts, norm / 2, out=outs), outs)
            assert bool((space[:cuts[0] + other] == 7).all()) and bool((space[cuts[-1] + other:] == 7).all())
        apart = ts[::2]
        verify(apart, norm / 9, before[::2], ops.clip_grad_norm(apart, norm / 9), apart)
        for i in (1, 3, 5):
            assert torch.equal(ts[i], before[i])
        assert torch.equal(flat[:shift], whole[:shift]) and torch.equal(flat[49999:], whole[49999:])


def test_large_and_small_magnitudes():
    from moe_offload import ops
    for scale in (1e30, 1e-30):
        ts = make([5000, 77], torch.float32, 3, scale)
        before = [t.clone() for t in ts]
        want = norm_of(ts)
        check(ops.grad_norm(ts), torch.tensor(want, dtype=torch.float64, device=DEV), want * NORM)
        verify(ts, scale, before, ops.clip_grad_norm(ts, scale), ts)


def test_infinities_nan_and_zeros():
    from moe_offload import ops
    ts = make([100, 50], torch.bfloat16, 4)
    ts[0][3] = math.inf
    assert float(ops.clip_grad_norm(ts, 1.0)) == math.inf
    assert bool(ts[0][3].isnan()) and int(ts[0].isnan().sum()) == 1 and not bool(ts[1].any())
    ts = make([100, 50], torch.bfloat16, 5)
    ts[1][3] = math.nan
    assert math.isnan(float(ops.clip_grad_norm(ts, 1.0)))
    assert all(bool(t.isnan().all()) for t in ts)
    ts = [torch.zeros(10, device=DEV), torch.zeros(0, device=DEV)]
    assert float(ops.clip_grad_norm(ts, 0.0)) == 0.0 and not bool(ts[0].any())
    ts = make([10], torch.float32, 6)
    ops.clip_grad_norm(ts, 0.0)
    assert not bool(ts[0].any())
    ts = make([10], torch.float32, 7)
    keep = ts[0].clone()
    ops.clip_grad_norm(ts, math.inf)
    assert torch.equal(ts[0], keep)


def test_shapes_orders_and_refusals():
    from moe_offload import ops
    a = torch.randn((6, 5, 4), device=DEV).permute(2, 0, 1)
    keep, want = a.clone(), norm_of([a])
    check(ops.clip_grad_norm(a, want / 2), torch.tensor(want, dtype=torch.float64, device=DEV), want * NORM)
    check(a, keep.double() / 2, keep.double().abs() * 2e-6)
    whole = torch.randn(64, device=DEV)
    for bad in (whole[::2], torch.zeros(1, device=DEV).expand(5)):
        with pytest.raises(ValueError):
            ops.grad_norm([bad])
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm([whole, whole], 1.0)
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm([whole[:40], whole[32:]], 1.0)
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm([whole[:32]], 1.0, out=[whole[16:48]])
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm([whole[:32], whole[32:]], 1.0, out=[whole[32:], whole[:32]])
    # reading the same tensor twice is fine
    two = ops.clip_grad_norm([whole, whole], 1.0, out=[torch.empty_like(whole), torch.empty_like(whole)])
    want = norm_of([whole, whole])
    check(two, torch.tensor(want, dtype=torch.float64, device=DEV), want * NORM)
    with pytest.raises(ValueError):
        ops.clip_grad_norm([whole], 1.0, out=[whole.half()])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([whole], -1.0)
    with pytest.raises(ValueError):
        ops.clip_grad_norm([whole], math.nan)
    with pytest.raises(ValueError):
        ops.grad_norm([])
    with pytest.raises(TypeError):
        ops.grad_norm([whole.double()])


def test_the_same_bits_every_time_and_captured():
    from moe_offload import ops
    ts = make([300000, 5, 70000], None, 8)
    outs = [torch.empty_like(t) for t in ts]
    first = ops.clip_grad_norm(ts, 1.0, out=outs)
    keep = [o.clone() for o in outs]
    for _ in range(3):
        assert torch.equal(ops.clip_grad_norm(ts, 1.0, out=outs), first) and all(torch.equal(o, k) for o, k in zip(outs, keep))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm(ts, 1.0, out=outs)
    for seed in (1, 2, 3):
        for t, v in zip(ts, make([300000, 5, 70000], None, seed, 0.1 * seed)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        eager = ops.clip_grad_norm(ts, 1.0, out=outs)
        assert torch.equal(norm, eager) and all(torch.equal(o, k) for o, k in zip(outs, got))


def test_past_32_bits_of_bytes():
    from moe_offload import ops
    t = torch.zeros((1 << 31) + 40, dtype=torch.bfloat16, device=DEV)
    t[-3:] = 2
    norm = ops.clip_grad_norm(t, 1.0)
    assert abs(float(norm) - math.sqrt(12)) < 1e-6
    check(t[-3:], torch.full((3,), 2 / math.sqrt(12), dtype=torch.float64, device=DEV), torch.tensor(1e-6, device=DEV))
    assert not bool(t[:-3].any())
