"""The weighted sum of a token's expert rows and its gradients against the formulas in 64 bits."""
import math

import pytest

import layer_ref as ref
from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def make(n_tok, k, hidden, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    y = torch.randn((n_tok, k, hidden), device=DEV, generator=g).to(dtype)
    w = torch.rand((n_tok, k), device=DEV, generator=g) - 0.3
    return y, w, torch.randn((n_tok, hidden), device=DEV, generator=g).to(dtype)


SIZES = [(1, 1, 8), (3, 10, 64), (17, 3, 520), (65, 6, 2048), (9, 33, 264), (40, 2, 4104), (2, 5, 16392), (513, 10, 640), (700, 4, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,k,hidden", SIZES)
def test_sum(dtype, n_tok, k, hidden):
    from moe_offload import ops
    y, w, res = make(n_tok, k, hidden, dtype, hidden)
    for r in (None, res):
        for out_type in (None, torch.float32):
            got = ops.combine(y, w, residual=r, dtype=out_type)
            assert got.dtype == (out_type or dtype)
            want, slack = ref.combine(y, w, r)
            check(got, want, slack, f"{r is not None} {out_type}")
    assert torch.equal(ops.combine(y.reshape(n_tok * k, hidden), w), ops.combine(y, w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok,k,hidden", SIZES)
def test_gradients(dtype, n_tok, k, hidden):
    from moe_offload import ops
    y, w, dout = make(n_tok, k, hidden, dtype, hidden + 1)
    dy, dw = ops.combine_grad(dout, y, w)
    assert dy.shape == y.shape and dy.dtype == dtype and dw.dtype == torch.float32
    want_dy, slack_dy, want_dw, slack_dw = ref.combine_grad(dout, y, w)
    check(dy, want_dy, slack_dy, "dy")
    check(dw, want_dw, slack_dw, "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_against_differences(dtype):
    """The sum is linear in each: <combine(y + v) - combine(y), dout> = <v, dy>, taken by the reference in 64 bits."""
    from moe_offload import ops
    y, w, dout = make(12, 4, 256, dtype, 2)
    dy, dw = ops.combine_grad(dout, y, w)
    v, u, _ = make(12, 4, 256, dtype, 3)
    along = ((ref.combine(y.double() + v.double(), w)[0] - ref.combine(y, w)[0]) * dout.double()).sum()
    # dy's rounding: half a step of each of 12 x 4 x 256 products
    room = float((dy.double().abs() * v.double().abs()).sum()) * torch.finfo(dtype).eps / 2 * 1.01 + 1e-9
    assert abs(float(along - (dy.double() * v.double()).sum())) <= room
    along = ((ref.combine(y, (w + u).double())[0] - ref.combine(y, w)[0]) * dout.double()).sum()
    mag = float((u.double().abs() * (y.double() * dout.double().unsqueeze(1)).abs().sum(2)).sum())
    # (w + u is rounded to fp32 before it is widened)
    room = mag * 260 * 2.0 ** -23 + float(((w.abs() + u.abs()).double() * (y.double() * dout.double().unsqueeze(1)).abs().sum(2)).sum()) * 2.0 ** -23
    assert abs(float(along - (dw.double() * u.double()).sum())) <= room


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_weight_of_zero_adds_nothing(dtype):
    from moe_offload import ops
    y, w, res = make(20, 4, 128, dtype, 4)
    w[::2, 1] = 0
    w[3] = 0                                       # a token without experts
    w[5, 0] = -0.0
    y[w == 0] = math.nan
    y[0, 1, :5] = math.inf
    want, slack = ref.combine(y, w, res)
    assert bool(want.isfinite().all())
    check(ops.combine(y, w, residual=res), want, slack)
    assert torch.equal(ops.combine(y, w, residual=res)[3], res[3])
    assert not bool(ops.combine(y, w)[3].any())
    dy, _ = ops.combine_grad(res, y, w)
    assert not bool(dy[w == 0].any())


def test_nan_and_infinities_of_places_that_count():
    from moe_offload import ops
    y, w, _ = make(4, 2, 64, torch.bfloat16, 5)
    y[1, 0, 7], y[2, 1, 9] = math.nan, math.inf
    w[3, 0] = math.nan
    w[:3] = w[:3].abs() + 0.1
    got = ops.combine(y, w)
    assert bool(got[1, 7].isnan()) and int(got[1].isnan().sum()) == 1
    assert float(got[2, 9]) == math.inf and bool(got[3].isnan().all()) and bool(got[0].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_given_outputs_and_in_place(dtype):
    from moe_offload import ops
    wide = make(30, 3, 96, dtype, 6)[0].reshape(90, 96)
    y, (_, w, res) = wide[:, 8:72], make(30, 3, 64, dtype, 7)
    out = torch.full((30, 80), 7.0, dtype=dtype, device=DEV)
    got = ops.combine(y, w, residual=res, out=out[:, 8:72])
    want, slack = ref.combine(y, w, res)
    check(got, want, slack)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 72:] == 7).all())
    stream = res.clone()
    assert ops.combine(y, w, residual=stream, out=stream) is stream
    check(stream, want, slack)
    wide_dout = make(30, 1, 96, dtype, 8)[2]
    dy, dw = ops.combine_grad(wide_dout[:, 16:80], y, w)
    want_dy, s1, want_dw, s2 = ref.combine_grad(wide_dout[:, 16:80], y, w)
    check(dy.reshape(30, 3, 64), want_dy, s1)
    check(dw, want_dw, s2)
    assert ops.combine(y[:0], w[:0]).shape == (0, 64) and ops.combine_grad(res[:0], y[:0], w[:0])[1].shape == (0, 3)


def test_offsets_past_32_bits():
    """Rows behind element 2^31: 2^20 + 8 rows of 2056."""
    from moe_offload import ops
    n_tok, k, hidden = (2 ** 20 + 8) // 4, 4, 2056
    y = torch.empty((n_tok, k, hidden), dtype=torch.bfloat16, device=DEV)
    y.view(-1)[:8] = 1
    g = torch.Generator(device=DEV).manual_seed(9)
    tail = torch.randn((5, k, hidden), device=DEV, generator=g).bfloat16()
    y.zero_()
    y[-5:] = tail
    w = torch.rand((n_tok, k), device=DEV, generator=g) + 0.1
    got = ops.combine(y, w)
    want, slack = ref.combine(tail, w[-5:])
    check(got[-5:], want, slack)
    assert not bool(got[:-5].any())
    dout = torch.zeros((n_tok, hidden), dtype=torch.bfloat16, device=DEV)
    dout[-5:] = tail[:, 0]
    dy, dw = ops.combine_grad(dout, y, w)
    want_dy, s1, want_dw, s2 = ref.combine_grad(dout[-5:], tail, w[-5:])
    check(dy[-5:], want_dy, s1)
    check(dw[-5:], want_dw, s2)
    assert not bool(dy[:-5].any()) and not bool(dw[:-5].any())
