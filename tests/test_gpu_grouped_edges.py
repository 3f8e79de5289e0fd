"""The grouped products and the layer under autograd where a batch leaves something empty, unaligned or out of range."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n,k,rows", [(64, 72, 40), (136, 264, 90), (1032, 1032, 4000)])
def test_weights_gradient_of_no_rows_is_zero_whatever_the_scale(dtype, bad, n, k, rows):
    from moe_offload import ops
    dy, x = rnd((rows, n), dtype, 1), rnd((rows, k), dtype, 2)
    seg, good = i32([0, 0, rows, rows]), torch.tensor([1.0, 0.5, 1.0], device=DEV)
    scale = torch.tensor([bad, 0.5, bad], device=DEV)
    for out in (dtype, torch.float32):
        dw = ops.grouped_mm_dw(dy, x, seg, scale=scale, dtype=out)
        assert not bool(dw[0].any()) and not bool(dw[2].any())
        assert torch.equal(dw, ops.grouped_mm_dw(dy, x, seg, scale=good, dtype=out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k", [(0, 2), (0, 1), (5, 0)])
def test_layer_without_tokens(dtype, tokens, k):
    """A step whose batch routes nothing here runs back too: no rows of dx (or zeros without experts), zero weights' gradients."""
    from moe_offload import dense
    x, ids = rnd((tokens, 64), dtype, 1).requires_grad_(), torch.zeros((tokens, k), dtype=torch.int32, device=DEV)
    wgu, wd = rnd((3, 48, 64), dtype, 2).requires_grad_(), rnd((3, 64, 24), dtype, 3).requires_grad_()
    y = dense.switch_glu(x, ids, wgu, wd)
    assert y.shape == (tokens, k, 64) and y.dtype == dtype
    y.sum().backward()
    assert x.grad.shape == (tokens, 64) and not bool(x.grad.any())
    assert wgu.grad.shape == wgu.shape and not bool(wgu.grad.any()) and wd.grad.shape == wd.shape and not bool(wd.grad.any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wanted", range(1, 8))
def test_each_subset_of_the_layer_s_gradients(dtype, wanted):
    from moe_offload import dense
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-1, 4, (37, 3), generator=g, dtype=torch.int32).to(DEV)
    data = rnd((37, 72), dtype, 1), rnd((4, 80, 72), dtype, 2, 0.1), rnd((4, 72, 40), dtype, 3, 0.1)
    dy = rnd((37, 3, 72), dtype, 4)

    def grads(mask):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(data)]
        dense.switch_glu(leaves[0], ids, leaves[1], leaves[2]).backward(dy)
        return [t.grad for t in leaves]
    for i, (got, full) in enumerate(zip(grads(wanted), grads(7))):
        assert (got is None) if not wanted >> i & 1 else torch.equal(got, full)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ahead", [3, 8])
def test_incoming_gradients_that_start_anywhere(dtype, ahead):
    """Behind a concatenation autograd hands down a view of the whole gradient, contiguous and aligned to an element only."""
    from moe_offload import dense
    ids = i32([[0, 2], [1, 0], [2, 2], [-1, 1], [0, 1]])
    leaves = [t.requires_grad_() for t in (rnd((5, 72), dtype, 1), rnd((3, 48, 72), dtype, 2), rnd((3, 72, 24), dtype, 3), rnd((5, 40), dtype, 4),
                                           rnd((2, 8, 72), dtype, 5), rnd((2, 40, 8), dtype, 6))]
    x, wgu, wd, base, a, b = leaves
    w = rnd((ahead + 5 * 2 * 72 + 5 * 40,), dtype, 7)

    def grads(shift):
        y, z = dense.switch_glu(x, ids, wgu, wd), dense.lora_add(base, x, a, b, ids[:, 0].contiguous())
        if shift:
            out = torch.cat([torch.zeros(ahead, dtype=dtype, device=DEV), y.reshape(-1), z.reshape(-1)])
            return torch.autograd.grad((out * w).sum(), leaves)
        n = ahead + y.numel()
        return torch.autograd.grad([y, z], leaves, [w[ahead:n].view(y.shape).clone(), w[n:].view(z.shape).clone()])
    for got, want in zip(grads(True), grads(False)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [3, 200, 700])
def test_gradient_of_gates_past_fp16(rows):
    """g = -70000 or 70000 is finite in the forward pass' fp32 and infinite in the (g, u) it keeps: silu' is 0 or 1 there."""
    from moe_offload import ops
    dt = torch.float16
    x = torch.zeros((rows, 8), dtype=dt, device=DEV)
    x[:, 0], x[:, 1] = 700.0, 1.0
    x[1::3, 0] = -700.0
    x[2::3, 0] = 0.5
    w = torch.zeros((1, 128, 8), dtype=dt, device=DEV)
    w[0, :64, 0], w[0, 64:, 1] = 100.0, 2.0 ** -7
    seg = i32([0, rows])
    gu = torch.empty((rows, 128), dtype=dt, device=DEV)
    h = ops.grouped_gate_up(x, None, seg, w, gu_out=gu)
    assert bool(h.isfinite().all()) and bool(gu[0::3, :64].isposinf().all()) and bool(gu[1::3, :64].isneginf().all())
    wd = torch.zeros((1, 8, 64), dtype=dt, device=DEV)
    wd[0, 0] = 1.0
    dy = torch.zeros((rows, 8), dtype=dt, device=DEV)
    dy[:, 0] = 0.25
    d = ops.grouped_mm_dx(dy, seg, wd, gu=gu).float()
    assert bool((d[0::3, :64] == 2.0 ** -9).all()) and bool(d[0::3, 64:].isposinf().all())          # dh u, dh g
    assert not bool(d[1::3].any())
    sg = torch.sigmoid(torch.tensor(50.0))
    assert torch.equal(d[2::3, :64], torch.full_like(d[2::3, :64], 2.0 ** -9)) and bool((d[2::3, 64:] == 12.5).all()) and float(sg) == 1.0
