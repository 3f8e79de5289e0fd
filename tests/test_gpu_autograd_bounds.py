"""The weighted sum and shared projections under autograd, each input alone and all together, whatever gradient autograd hands down,
against 64 bits within the operators' own bounds."""
import itertools

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


def handed_down(shape, dtype):
    """Gradients as autograd has them: whole, one value for all, transposed, starting anywhere."""
    rows, cols = shape
    odd = rnd((rows * cols + 3,), dtype, 12)
    return {"whole": rnd(shape, dtype, 11), "expanded": rnd((1, 1), dtype, 13).expand(shape), "transposed": rnd((cols, rows), dtype, 14).T,
            "odd": odd[3:].view(shape), "columns": rnd((rows, cols + 8), dtype, 15)[:, 5:5 + cols]}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_combine(dtype, with_residual):
    from moe_offload import dense
    n_tok, k, hidden = 33, 3, 72
    y, w, res = rnd((n_tok, k, hidden), dtype, 1), rnd((n_tok, k), torch.float32, 2), rnd((n_tok, hidden), dtype, 3)
    for wanted in itertools.product((False, True), repeat=3 if with_residual else 2):
        for name, dout in handed_down((n_tok, hidden), dtype).items():
            leaves = [t.clone().requires_grad_(want) for t, want in zip((y, w, res), wanted)]
            out = dense.combine(*leaves)
            check(out, *ref.combine(y, w, res if with_residual else None), "out")
            if not any(wanted):
                assert not out.requires_grad
                continue
            out.backward(dout)
            want_dy, s1, want_dw, s2 = ref.combine_grad(dout, y, w)
            assert [t.grad is not None for t in leaves] == list(wanted)
            if wanted[0]:
                check(leaves[0].grad, want_dy, s1, f"{name} dy")
            if wanted[1]:
                check(leaves[1].grad, want_dw, s2, f"{name} dw")
            if with_residual and wanted[2]:
                assert torch.equal(leaves[2].grad, dout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu2"])
@pytest.mark.parametrize("out_type", [None, torch.float32])
def test_linear(dtype, act, out_type):
    """z, where there is an activation, is what the forward kernel gives: the bound of the gradients from a given z holds."""
    from moe_offload import dense, ops
    n_tok, n_in, n_out = 37, 72, 136
    x, w, b, res = rnd((n_tok, n_in), dtype, 1), rnd((n_out, n_in), dtype, 2, n_in ** -0.5), rnd((n_out,), dtype, 3), rnd((n_tok, n_out), dtype, 4)
    z = torch.empty((n_tok, n_out), dtype=dtype, device=DEV)
    ops.linear(x, w, bias=b, act=act, z_out=z)
    zz = None if act is None else z
    for wanted in [w for w in itertools.product((False, True), repeat=4) if any(w)]:
        for name, dy in handed_down((n_tok, n_out), out_type or dtype).items():
            leaves = [t.clone().requires_grad_(want) for t, want in zip((x, w, b, res), wanted)]
            out = dense.linear(*leaves[:3], act=act, residual=leaves[3], dtype=out_type)
            want, slack, *_ = ref.linear(x, w, b, act, res)
            check(out, want, slack, "out")
            out.backward(dy)
            assert [t.grad is not None for t in leaves] == list(wanted)
            for t, (v, s), n in zip(leaves, ref.linear_grad(dy, x, w, zz, act), ("dx", "dw", "db")):
                if t.grad is not None:
                    check(t.grad, v, s, f"{name} {n}")
            if wanted[3]:
                assert torch.equal(leaves[3].grad, dy.to(dtype))
