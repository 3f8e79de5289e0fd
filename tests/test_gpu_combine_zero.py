"""The weighted sum's gradients where a place has weight 0: as in the sum, nothing that its row holds gets through."""
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
    return y, torch.rand((n_tok, k), device=DEV, generator=g) + 0.1, torch.randn((n_tok, hidden), device=DEV, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden", [8, 264, 2048])
def test_rows_without_weight_leave_no_trace_in_the_gradients(dtype, hidden):
    from moe_offload import ops
    y, w, dout = make(20, 4, hidden, dtype, 1)
    clean = y.clone()
    w[::2, 1], w[3], w[5, 0] = 0, 0, -0.0
    y[0, 1] = math.nan
    y[2, 1, 3], y[3, 2, -1], y[5, 0, 7] = math.inf, -math.inf, math.nan
    y[4, 1, 0], y[4, 1, 1] = math.inf, -math.inf
    dirty = torch.zeros((20, 4), dtype=torch.bool, device=DEV)
    for t, j in ((0, 1), (2, 1), (3, 2), (5, 0), (4, 1)):
        dirty[t, j] = True
    want_dy, s1, want_dw, s2 = ref.combine_grad(dout, clean, w)
    dy, dw = ops.combine_grad(dout, y, w)
    check(dy, want_dy, s1, "dy")
    # a weight that is 0 over a finite row has its gradient all the same
    check(dw[~dirty], want_dw[~dirty], s2[~dirty], "dw")
    assert not bool(dw[dirty].any())
    # and a dout that is not finite leaves dy 0 there
    dout[0, 0], dout[3, 1], dout[5, 2] = math.inf, math.nan, -math.inf
    dy, dw = ops.combine_grad(dout, y, w)
    assert not bool(dy[w == 0].any()) and not bool(dw[dirty].any())
    assert not bool(dw[0, 1].any()) and not bool(dw[3].any()) and not bool(dw[5, 0].any())
    assert bool(dy[0, 0, 0].isinf()) and bool(dw[0, 0].isinf()) and bool(dy[5, 1, 2].isinf())


def test_nan_where_there_is_a_weight_stays_one():
    from moe_offload import ops
    y, w, dout = make(6, 3, 64, torch.bfloat16, 2)
    y[1, 2, 5], y[2, 0, 6] = math.nan, math.inf
    w[4, 1] = math.nan
    dy, dw = ops.combine_grad(dout, y, w)
    assert bool(dw[1, 2].isnan()) and bool(dw[2, 0].isinf()) and bool(dy[4, 1].isnan().all())
    assert int(dw.isfinite().sum()) == 16 and int(dy.isnan().sum()) == 64


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_a_place_of_weight_zero_does_not_reach_the_logits(score, renorm):
    """Through autograd: a place that the caller drops by a weight of 0, its row NaN, next to places that count.  The ids are all valid."""
    from moe_offload import dense
    n_tok, n_exp, k, hidden = 10, 16, 4, 128
    g = torch.Generator(device=DEV).manual_seed(3)
    start = torch.randn((n_tok, n_exp), device=DEV, generator=g)
    y, _, dout = make(n_tok, k, hidden, torch.bfloat16, 4)
    drop = torch.ones((n_tok, k), device=DEV)
    drop[2, 1] = drop[7, 3] = 0
    grads = []
    for bad in (0.0, math.nan, math.inf):
        yy = y.clone()
        yy[drop == 0] = bad
        yy.requires_grad_()
        logits = start.clone().requires_grad_()
        ids, w = dense.route(logits, k, score=score, renorm=renorm)
        assert bool((ids >= 0).all())
        out = dense.combine(yy, w * drop)
        assert bool(out.isfinite().all())
        out.backward(dout)
        assert bool(logits.grad.isfinite().all()) and not bool(yy.grad[drop == 0].any())
        grads.append(logits.grad)
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
