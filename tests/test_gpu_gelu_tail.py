"""gelu and its slope where they are small: against 64 bits, relative to their own value."""
import pytest

from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"
STEP = 2.0 ** -23


def values(dtype, n):
    """n values between -12 and 12, dense near 0 and in the tail, and a few of both ends of the type."""
    z = torch.cat([torch.linspace(-12, 12, n - 64, device=DEV), torch.logspace(-7, 0, 30, device=DEV), -torch.logspace(-7, 0, 30, device=DEV),
                   torch.tensor([0.0, -0.0, 100.0, -100.0], device=DEV)])
    return z.to(dtype)


def gelu64(z):
    """(gelu, its slope) by the normal distribution's integral in 64 bits."""
    z = z.double()
    below = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    density = torch.exp(-0.5 * z * z) * 0.3989422804014327
    return z * below, below + z * density


def room(z):
    """fp32 steps.  The exponential's argument is rounded twice, half a step of it each: z^2 / 2 steps of its value.  The polynomial's
    coefficients and terms 4, the reciprocal and its argument 2, the exponential 1, the products and the sum 3."""
    return (0.5 * z.double() ** 2 + 10) * STEP


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_gelu_relative_to_its_own_value(dtype, rows):
    """One token goes through the kernel of few results, 40 through a tile's: z = x W^T with a unit W is x."""
    from moe_offload import ops
    n = 1024
    z = values(dtype, n)
    w = torch.eye(n, device=DEV).to(dtype)
    x = z.expand(rows, n).contiguous()
    want, _ = gelu64(x)
    slack = want.abs() * room(x) + 2.0 ** -126
    got = ops.linear(x, w, act="gelu", dtype=torch.float32)
    check(got, want, slack, "fp32")
    check(ops.linear(x, w, act="gelu"), want, slack, "16 bits")
    zero = x.float() == 0
    assert not bool(got[zero].any()) and bool((got[x.float() == 100] == 100).all()) and not bool(got[x.float() == -100].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_slope_in_the_tail(dtype):
    """Through the weights' gradient in fp32, which takes all bits of dz.  Below -1 the two terms differ by 0.242 / 0.159 at least, above
    0 they add up, in between the bound is the terms' own."""
    from moe_offload import ops
    n = 1024
    z = values(dtype, n).reshape(1, n)
    x = torch.zeros((1, 8), dtype=dtype, device=DEV)
    x[0, 0] = 1
    w = torch.zeros((n, 8), dtype=dtype, device=DEV)
    dw = ops.linear_grad(torch.ones_like(z), x, w, z=z, act="gelu", dw_dtype=torch.float32)[1][:, 0]
    _, want = gelu64(z[0])
    zd = z[0].double()
    below = 0.5 * torch.special.erfc(-zd * 0.5 ** 0.5)
    terms = below + zd.abs() * torch.exp(-0.5 * zd * zd) * 0.3989422804014327
    # above 0 one term is 1 - tail, rounded to a step of 1 at most
    check(dw, want, terms * room(zd) + 2.0 ** -126, "slope")
