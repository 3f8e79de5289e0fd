"""A layer of unquantised experts under autograd from its tokens to the clipped gradients: router, choice, experts, weighted
sum, against the same layer in 64 bits with the choice held."""
import pytest

import layer_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def layer64(x, wr, wg, wd, ids, k, score, renorm, scale, res):
    """The layer in 64 bits with the ids given."""
    logits = x @ wr.T
    w = ref.chosen_weights(logits, ids.long(), ids >= 0, score, renorm, scale)
    out = res
    inter = wd.shape[2]
    for j in range(k):
        e = ids[:, j].long()
        gu = torch.einsum("tnk,tk->tn", wg[e], x)
        h = torch.nn.functional.silu(gu[:, :inter]) * gu[:, inter:]
        out = out + w[:, j:j + 1] * torch.einsum("tnk,tk->tn", wd[e], h)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n_tok,score,renorm,groups", [(1, "softmax", True, False), (37, "softmax", False, False), (64, "sigmoid", True, True)])
def test_layer_forward_and_backward(dtype, n_tok, score, renorm, groups):
    """Relative to a tensor's largest value: each of the chain's six roundings to 16 bits (h, y, (g, u) and back: dy, dgu, rows
    of dx) is half a step of a value of its own magnitude, and a value is made of at least 64 of them: their sum stays
    within 8 half steps of the largest."""
    from moe_offload import dense, ops
    n_exp, hidden, inter, k = 16, 64, 64, 4
    rule = {"score": score, "renorm": renorm, "scale": 1.5}
    if groups:
        rule.update(bias=rnd((n_exp,), torch.float32, 9, 0.1), n_group=4, topk_group=2, group_best=2)
    leaves = [rnd((n_tok, hidden), dtype, 1), rnd((n_exp, hidden), dtype, 2, hidden ** -0.5), rnd((n_exp, 2 * inter, hidden), dtype, 3, hidden ** -0.5),
              rnd((n_exp, hidden, inter), dtype, 4, inter ** -0.5), rnd((n_tok, hidden), dtype, 5)]
    dout = rnd((n_tok, hidden), dtype, 6)
    for t in leaves:
        t.requires_grad_()
    x, wr, wg, wd, res = leaves
    out = dense.moe_layer(x, wr, wg, wd, k, residual=res, **rule)
    out.backward(dout)
    ids, _ = ops.route(ops.linear(x.detach(), wr.detach(), dtype=torch.float32), k, **rule)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = layer64(*wide[:4], ids, k, score, renorm, 1.5, wide[4])
    want.backward(dout.double())
    room = 8 * torch.finfo(dtype).eps / 2
    pairs = [("out", out.detach(), want.detach())] + [(n, t.grad, w.grad) for n, t, w in zip(("x", "router", "gate_up", "down", "res"), leaves, wide)]
    for name, got, exact in pairs:
        off = float((got.double() - exact).abs().max())
        assert off <= room * float(exact.abs().max()) + 1e-6, (name, off, float(exact.abs().max()))

    # and the step's end: all gradients together
    before = [t.grad.clone() for t in leaves]
    norm = dense.clip_grad_norm(leaves, 0.5)
    total = sum(float(g.double().square().sum()) for g in before) ** 0.5
    assert abs(float(norm) - total) <= 1e-6 * total
    after = sum(float(t.grad.double().square().sum()) for t in leaves) ** 0.5
    assert after <= 0.5 * (1 + torch.finfo(dtype).eps) and after >= 0.5 * (1 - torch.finfo(dtype).eps) - 1e-3


def test_layer_without_tokens():
    from moe_offload import dense
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    wr, wg, wd = (rnd(s, torch.bfloat16, 1).requires_grad_() for s in ((8, 64), (8, 128, 64), (8, 64, 64)))
    out = dense.moe_layer(x, wr, wg, wd, 2)
    out.sum().backward()
    assert out.shape == (0, 64) and all(not bool(t.grad.any()) for t in (x, wr, wg, wd))


def test_tokens_whose_logits_are_masked_keep_their_residual():
    from moe_offload import dense, ops
    n_tok, n_exp = 12, 8
    x = rnd((n_tok, 64), torch.bfloat16, 1)
    logits = rnd((n_tok, n_exp), torch.float32, 2)
    logits[3] = -float("inf")
    logits[4, 1:] = -float("inf")
    logits.requires_grad_()
    wg, wd = rnd((n_exp, 128, 64), torch.bfloat16, 3, 0.1), rnd((n_exp, 64, 64), torch.bfloat16, 4, 0.1)
    ids, w = dense.route(logits, 2)
    y = dense.switch_glu(x, ids, wg, wd)
    out = dense.combine(y, w, x)
    assert torch.equal(out[3], x[3]) and ids[4].tolist()[1] == -1
    out.float().sum().backward()
    assert bool(logits.grad.isfinite().all()) and not bool(logits.grad[3].any())
    assert ids.requires_grad is False and ops.route(logits.detach(), 2)[0].equal(ids)


def test_linear_and_combine_under_autograd():
    from moe_offload import dense
    x, w, b, r = (rnd(s, torch.bfloat16, i, 0.3).requires_grad_() for i, s in enumerate([(20, 64), (96, 64), (96,), (20, 96)]))
    for act in (None, "silu", "gelu", "relu2"):
        for dtype in (None, torch.float32):
            for t in (x, w, b, r):
                t.grad = None
            y = dense.linear(x, w, bias=b, act=act, residual=r, dtype=dtype)
            dy = rnd(y.shape, y.dtype, 9)
            y.backward(dy)
            assert torch.equal(r.grad, dy.bfloat16())
            z = ref.linear(x.detach(), w.detach(), b.detach())[2].bfloat16()
            for t, (want, slack) in zip((x, w, b), ref.linear_grad(dy, x.detach(), w.detach(), None if act is None else z, act)):
                # z, rounded to bf16, may be a step off next to a border between two: the slope moves by at most 2 steps of z
                room = slack + 2 * want.abs() * 2.0 ** -8 + 0.02 * float(want.abs().max())
                assert bool(((t.grad.double() - want).abs() <= room).all()), act
    frozen = dense.linear(x.detach(), w.detach(), residual=r)
    frozen.backward(torch.ones_like(frozen))


def test_capture_is_refused():
    from moe_offload import dense
    x, w = rnd((4, 64), torch.bfloat16, 1), rnd((64, 64), torch.bfloat16, 2)
    y, s = rnd((4, 2, 64), torch.bfloat16, 3), torch.ones((4, 2), device=DEV)
    logits = rnd((4, 8), torch.float32, 4)
    keep = torch.zeros(1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep.add_(1)
        for call in (lambda: dense.linear(x, w), lambda: dense.combine(y, s), lambda: dense.route(logits, 2)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
