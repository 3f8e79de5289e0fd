"""The adapters' gradients against the formula in 64 bits where the values between the products leave the inputs' type, on
every tile that a call's sizes select, and over segments that end anywhere in a step.

Bounds.  v = A x and dv = s B^T dy are fp32 sums of exact products; between the products they keep their fp32 bits, in three
parts of one sign.  In a product with fp16 values those are two parts of one sign each, so c products are at most 6 c terms
whose magnitudes add up to the products' own."""
import pytest

import grouped_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def make(dtype, tokens, n_ad, rank, n_in, n_out, scales=None, seed=0):
    """(dy, x, a, b, ids, scale); ids from -1 to n_ad, some of them no adapter's."""
    sx, sa, sb, sdy = scales or (1.0, n_in ** -0.5, rank ** -0.5, 1.0)
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-1, n_ad + 1, (tokens,), generator=g).to(torch.int32).to(DEV)
    return (rnd((tokens, n_out), dtype, seed + 1, sdy), rnd((tokens, n_in), dtype, seed + 2, sx), rnd((n_ad, rank, n_in), dtype, seed + 3, sa),
            rnd((n_ad, n_out, rank), dtype, seed + 4, sb), ids, (torch.rand(n_ad, generator=g) + 0.5).to(DEV))


def close(got, want, slack, what):
    """ref.check, and where the exact value itself rounds to infinity (fp16: from 65504 + half its step, 65520) that infinity."""
    if got.dtype == torch.float16:
        over = want.abs() - slack >= 65520
        assert torch.equal(got[over], want[over].sign().half() * float("inf")), what
        got, want = got.masked_fill(over, 0), want.masked_fill(over, 0)
    ref.check(got, want, slack, what)


def check(got, dy, x, a, b, ids, scale):
    dx, da, db = got
    wx, sx = torch.zeros(x.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    n_ad, rank, n_in = a.shape
    n_out = b.shape[1]
    for j in range(n_ad):
        rows = (ids == j).nonzero()[:, 0]
        xd, dyd, aj, bj, s = x.double()[rows], dy.double()[rows], a[j].double(), b[j].double(), 1.0 if scale is None else float(scale[j])
        m = rows.numel()
        v, dv = xd @ aj.T.contiguous(), s * (dyd @ bj)
        ev = (n_in + 2) * ref.F32 * (xd.abs() @ aj.abs().T.contiguous())
        edv = (n_out + 3) * ref.F32 * abs(s) * (dyd.abs() @ bj.abs())
        av, adv = v.abs() + ev, dv.abs() + edv
        wx[rows] = dv @ aj
        sx[rows] = edv @ aj.abs() + (6 * rank + 2) * ref.F32 * (adv @ aj.abs())
        close(da[j], dv.T.contiguous() @ xd, edv.T.contiguous() @ xd.abs() + (6 * m + 2) * ref.F32 * (adv.T.contiguous() @ xd.abs()), f"da {j}")
        close(db[j], s * (dyd.T.contiguous() @ v), abs(s) * (dyd.abs().T.contiguous() @ ev + (6 * m + 3) * ref.F32 * (dyd.abs().T.contiguous() @ av)),
                  f"db {j}")
    close(dx, wx, sx, "dx")


# standard deviations of x, a, b and dy
RANGES = {
    "v past 65504": (64.0, 64.0, 2.0 ** -12, 2.0 ** -10),
    "dv past 65504": (2.0 ** -10, 2.0 ** -10, 64.0, 256.0),
    "small dv": (1.0, 2.0 ** -4, 2.0 ** -7, 2.0 ** -13),
    "dv below the least step": (64.0, 2.0 ** -4, 2.0 ** -12, 2.0 ** -16),
    "v below the least step": (2.0 ** -14, 2.0 ** -16, 64.0, 256.0),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(RANGES))
@pytest.mark.parametrize("tokens", [30, 700])
def test_values_between_the_products_keep_their_bits(dtype, name, tokens):
    from moe_offload import ops
    dy, *rest = make(dtype, tokens, 3, 24, 512, 264, RANGES[name])
    dy[::3] = 0                                                                # what is multiplied by zero stays out
    got = ops.lora_grad(dy, *rest[:-1], scale=rest[-1])
    assert all(bool(t.isfinite().all()) for t in got)
    check(got, dy, *rest)


def test_one_large_token_beside_small_ones():
    """A token whose v and dv are 2^40 times the others' does not cost them bits, nor does it reach where dy or x is zero."""
    from moe_offload import ops
    dy, x, a, b, ids, scale = make(torch.float16, 200, 2, 16, 128, 64, (2.0 ** -10, 1.0, 1.0, 2.0 ** -12))
    ids[7] = 1
    x[7], dy[7] = 0, 0
    x[7, 0], dy[7, 0] = 60000.0, 2.0
    a[1, :, 0], b[1, 0, :] = 2.0 ** -9, 2.0 ** -9
    a[1, 3, 0], b[1, 0, 5] = 30000.0, 0.5
    check(ops.lora_grad(dy, x, a, b, ids, scale=scale), dy, x, a, b, ids, scale)


# dx's tiles are chosen by the call's sizes: few tokens 64 x 64 and 64 x 128, then 128 x 128, then 256 x 256
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,n_ad,rank,n_in,n_out", [
    (900, 20, 40, 2568, 136), (1200, 30, 24, 2568, 72), (4096, 8, 64, 2560, 520), (4096, 32, 136, 2568, 264), (6000, 3, 256, 1288, 72), (5000, 300, 24, 328, 2056)])
def test_larger_batches(dtype, tokens, n_ad, rank, n_in, n_out):
    from moe_offload import ops
    args = make(dtype, tokens, n_ad, rank, n_in, n_out)
    check(ops.lora_grad(*args[:-1], scale=args[-1]), *args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 15, 31, 32, 33, 63, 64, 65, 96, 97, 257, 1024, 1025, 2200])
def test_every_length(dtype, tokens):
    """One adapter's tokens end anywhere in a step of 64; another's are none; ranks and widths end inside the tiles."""
    from moe_offload import ops
    for rank, n_in, n_out in ((8, 8, 72), (72, 136, 8), (64, 64, 64)):
        dy, x, a, b, ids, scale = make(dtype, tokens + 3, 3, rank, n_in, n_out, seed=tokens)
        ids[:] = 1
        ids[0], ids[1], ids[tokens + 1] = -1, 2, 3
        check(ops.lora_grad(dy, x, a, b, ids, scale=scale), dy, x, a, b, ids, scale)
        check(ops.lora_grad(dy, x, a, b, ids), dy, x, a, b, ids, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_several_tiles_of_a_block(dtype):
    """Many adapters of few tokens each: a block has several tiles along the wide operand, of one step and of two."""
    from moe_offload import ops
    for tokens, n_ad in ((600, 200), (4000, 100)):
        args = make(dtype, tokens, n_ad, 16, 1608, 904)
        check(ops.lora_grad(*args[:-1], scale=args[-1]), *args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_an_idle_adapter_s_scale_is_not_used(dtype, bad):
    from moe_offload import ops
    dy, x, a, b, ids, scale = make(dtype, 70, 4, 16, 72, 136)
    ids[ids == 2] = 1
    scale[2] = bad
    dx, da, db = ops.lora_grad(dy, x, a, b, ids, scale=scale)
    assert not bool(da[2].any()) and not bool(db[2].any())
    scale[2] = 1.0
    check((dx, da, db), dy, x, a, b, ids, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_without_adapters_and_with_many(dtype):
    from moe_offload import dense
    base, x = rnd((5, 24), dtype, 1).requires_grad_(), rnd((5, 16), dtype, 2).requires_grad_()
    a, b = rnd((0, 8, 16), dtype, 3).requires_grad_(), rnd((0, 24, 8), dtype, 4).requires_grad_()
    ids = torch.zeros(5, dtype=torch.int32, device=DEV)
    out = dense.lora_add(base, x, a, b, ids)
    dy = rnd((5, 24), dtype, 5)
    out.backward(dy)
    assert torch.equal(out, base) and torch.equal(base.grad, dy) and not bool(x.grad.any()) and a.grad.shape == a.shape and b.grad.shape == b.shape
    a, b = rnd((1025, 8, 16), dtype, 3), rnd((1025, 24, 8), dtype, 4)
    base.grad = None
    dense.lora_add(base, x.detach(), a, b, ids + 1024).backward(dy)               # base's own gradient has no such limit
    assert torch.equal(base.grad, dy)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_long_adapter_among_many(dtype):
    """The sizes promise short segments, so a block has many tiles; one segment is longer than the row numbers it holds."""
    from moe_offload import ops
    dy, x, a, b, ids, scale = make(dtype, 3000, 500, 16, 1608, 904)
    ids[torch.arange(3000, device=DEV) % 5 != 0] = 123
    check(ops.lora_grad(dy, x, a, b, ids, scale=scale), dy, x, a, b, ids, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [40, 1500])
def test_infinities_and_nan_stay_in_their_token_and_adapter(dtype, tokens):
    from moe_offload import ops
    dy, x, a, b, ids, scale = make(dtype, tokens, 4, 16, 136, 72)
    clean = ops.lora_grad(dy, x, a, b, ids, scale=scale)
    t = int((ids == 1).nonzero()[0])
    for bad in (float("nan"), float("inf")):
        x2, dy2 = x.clone(), dy.clone()
        x2[(ids < 0) | (ids >= 4)] = bad                                       # not read: these tokens have no adapter
        dy2[(ids < 0) | (ids >= 4)] = bad
        assert all(torch.equal(p, q) for p, q in zip(ops.lora_grad(dy2, x2, a, b, ids, scale=scale), clean))
        x2[t, 5] = bad                                                         # v, so db; and da's column 5
        dx, da, db = ops.lora_grad(dy2, x2, a, b, ids, scale=scale)
        keep = [0, 2, 3]
        assert torch.equal(dx, clean[0]) and torch.equal(da[keep], clean[1][keep]) and torch.equal(db[keep], clean[2][keep])
        assert not bool(da[1, :, 5].isfinite().any()) and not bool(db[1].isfinite().any())
        cols = torch.arange(136, device=DEV) != 5
        assert torch.equal(da[1][:, cols], clean[1][1][:, cols])
        dy2[t, 3] = bad                                                        # dv, so dx of the token and da of its adapter
        dx, da, db = ops.lora_grad(dy2, x, a, b, ids, scale=scale)
        others = torch.arange(tokens, device=DEV) != t
        assert torch.equal(dx[others], clean[0][others]) and not bool(dx[t].isfinite().any())
        assert torch.equal(da[keep], clean[1][keep]) and not bool(da[1].isfinite().any())
        rows = torch.arange(72, device=DEV) != 3
        assert torch.equal(db[keep], clean[2][keep]) and torch.equal(db[1][rows], clean[2][1][rows]) and not bool(db[1, 3].isfinite().any())
