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
