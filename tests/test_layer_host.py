"""Refusals of routing, the weighted sum, shared projections and the gradients' norm, without a GPU: the tensor checks of
moe_offload.ops and the argument checks of the C entry points, none of which launches anything."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from moe_offload import _lib, dense, ops  # noqa: E402

P = 64                                             # stands for some aligned device address, which is never read here
BF = torch.bfloat16


def refused(name, *args):
    lib = _lib.lib()
    lib.c_clear_error()
    rc = getattr(lib, name)(*args)
    msg = _lib.last_error()
    lib.c_clear_error()
    assert rc == -1 and msg, (name, args)
    return msg


def taken(name, *args):
    lib = _lib.lib()
    lib.c_clear_error()
    assert getattr(lib, name)(*args) == 0 and not _lib.last_error(), (name, args)


def swapped(good, i, value):
    return good[:i] + (value,) + good[i + 1:]


def test_tensors_off_the_gpu_are_refused():
    x, w, l = torch.zeros((4, 16), dtype=BF), torch.zeros((8, 16), dtype=BF), torch.zeros((4, 8))
    ids, s = torch.zeros((4, 2), dtype=torch.int32), torch.zeros((4, 2))
    y = torch.zeros((4, 2, 16), dtype=BF)
    for call in (lambda: ops.route(l, 2), lambda: ops.route_grad(s, l, ids), lambda: ops.combine(y, s), lambda: ops.combine_grad(x, y, s),
                 lambda: ops.linear(x, w), lambda: ops.linear_grad(x[:, :8], x, w), lambda: dense.route(l, 2), lambda: dense.combine(y, s),
                 lambda: dense.linear(x, w), lambda: dense.moe_layer(x, w, torch.zeros((8, 16, 16), dtype=BF), torch.zeros((8, 16, 8), dtype=BF), 2)):
        with pytest.raises(ValueError, match="not on a GPU"):
            call()
    for call in (lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm([x], 1.0)):
        with pytest.raises(ValueError, match="on one GPU"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        ops.route([1.0], 1)
    with pytest.raises(TypeError, match="must be tensors"):
        ops.grad_norm([1.0])
    for sparse in (torch.eye(4).to_sparse(), torch.eye(4).to_sparse_csr()):
        with pytest.raises((ValueError, RuntimeError)):
            ops.grad_norm([sparse])


def test_row_checks():
    rows = lambda t, *a: ops._scored_rows("op", "logits", t, *a)  # noqa: E731
    assert rows(torch.zeros((4, 7))) == 7
    assert rows(torch.zeros((4, 9), dtype=BF)[:, 2:]) == 9
    assert rows(torch.zeros((1, 9))[:, :5]) == 5
    assert rows(torch.zeros((0, 9))) == 9
    for bad in (torch.zeros(4), torch.zeros((4, 0)), torch.zeros((4, 1025)), torch.zeros((7, 4)).T, torch.zeros((1, 5)).expand(4, 5),
                torch.zeros(64).as_strided((4, 8), (4, 1))):
        with pytest.raises(ValueError):
            rows(bad)
    with pytest.raises(TypeError):
        rows(torch.zeros((4, 4), dtype=torch.float64))
    with pytest.raises(ValueError):
        rows(torch.zeros((4, 4)), (4, 5))
    y = torch.zeros((6, 2, 16), dtype=BF)
    pairs = lambda t: ops._pair_rows("op", "y", t, 6, 2)  # noqa: E731
    assert pairs(y) == (16, 16) and pairs(y.reshape(12, 16)) == (16, 16) and pairs(torch.zeros((6, 2, 32), dtype=BF)[:, :, 8:24]) == (16, 32)
    assert ops._pair_rows("op", "y", torch.zeros((6, 1, 32), dtype=BF)[:, :, :16], 6, 1) == (16, 32)
    assert ops._pair_rows("op", "y", torch.zeros((1, 4, 16), dtype=BF)[:, 1:2], 1, 1) == (16, 16)
    assert ops._pair_rows("op", "y", torch.zeros((0, 2, 16), dtype=BF), 0, 2) == (16, 16)
    for bad in (y[:5], y.reshape(12, 16)[:11], torch.zeros((6, 4, 16), dtype=BF)[:, :2], torch.zeros((2, 6, 16), dtype=BF).transpose(0, 1),
                torch.zeros((6, 2, 12), dtype=BF), torch.zeros((6, 2, 0), dtype=BF), torch.zeros((6, 16, 2), dtype=BF).transpose(1, 2),
                torch.zeros((6, 2, 20), dtype=BF)[:, :, :16], torch.zeros((1, 1, 16), dtype=BF).expand(6, 2, 16), torch.zeros(192, dtype=BF)):
        with pytest.raises(ValueError):
            pairs(bad)
    for bad in (torch.zeros((16, 12), dtype=BF), torch.zeros((12, 16), dtype=BF), torch.zeros((8, 32), dtype=BF)[:, :16], torch.zeros((0, 16), dtype=BF),
                torch.zeros((16, 8), dtype=BF).T):
        with pytest.raises(ValueError):
            ops._shared_weight("op", bad, BF, 16)
    ops._shared_weight("op", torch.zeros((8, 16), dtype=BF), BF, 16)
    for good in (torch.zeros((3, 4)), torch.zeros((3, 4)).T, torch.zeros(0), torch.zeros((2, 3, 4)).permute(2, 0, 1), torch.zeros(())):
        assert ops._dense_layout(good)
    for bad in (torch.zeros(8)[::2], torch.zeros(1).expand(4), torch.zeros((4, 8))[:, :4]):
        assert not ops._dense_layout(bad)


def test_layer_shapes_and_constants_are_checked():
    x, wr = torch.zeros((4, 16), dtype=BF), torch.zeros((8, 16), dtype=BF)
    with pytest.raises(ValueError, match="do not fit"):
        dense.moe_layer(x, wr, torch.zeros((9, 16, 16), dtype=BF), torch.zeros((9, 16, 8), dtype=BF), 2)
    with pytest.raises(ValueError, match="bias has no gradient"):
        dense.route(torch.zeros((4, 8)), 2, bias=torch.zeros(8, requires_grad=True))


def test_parameters_without_gradients_have_the_norm_0():
    for parameters in ([], torch.zeros(4, requires_grad=True), iter([torch.zeros(4, requires_grad=True)])):
        norm = dense.clip_grad_norm(parameters, 1.0)
        assert norm.shape == () and norm.dtype == torch.float32 and float(norm) == 0.0


# ---- the reference that the GPU tests compare with, against loops over its definition ---------------------

def looped_route(row, k, score, bias, n_group, topk_group, group_best):
    """[(id, score)] of one token, by sorting tuples."""
    import math
    live = [not math.isnan(v) and v > -math.inf for v in row]
    top = max([v for v, ok in zip(row, live) if ok], default=0.0)
    e = [(1.0 if v == top else math.exp(v - top)) if ok else 0.0 for v, ok in zip(row, live)]
    s = [1 / (1 + math.exp(-v)) if ok else 0.0 for v, ok in zip(row, live)] if score == "sigmoid" else [v / (sum(e) or 1.0) for v in e]
    c = [v + b for v, b in zip(s, bias)] if bias is not None else list(row)
    live = [ok and not math.isnan(v) and v > -math.inf for ok, v in zip(live, c)]
    per, stay = len(row) // n_group, set(range(n_group))
    if n_group > 1:
        of = c if bias is not None or group_best == 1 else s
        value = []
        for g in range(n_group):
            best = sorted((of[i] for i in range(g * per, (g + 1) * per) if live[i]), reverse=True)[:group_best]
            value.append(sum(best) if best else -math.inf)
        stay = set(sorted(range(n_group), key=lambda g: (-value[g], g))[:topk_group])
    order = sorted((i for i in range(len(row)) if live[i] and i // per in stay), key=lambda i: (-c[i], i))
    return [(i, s[i]) for i in order[:k]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_reference_against_loops(score):
    import math

    import layer_ref as ref
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((30, 24), generator=g, dtype=torch.float64)
    logits[3] = logits[3].round()
    logits[4, ::2] = -math.inf
    logits[5] = -math.inf
    logits[6, 3:] = -math.inf
    bias = torch.randn(24, generator=g) * 0.2
    bias[7] = -math.inf
    for b in (None, bias):
        for n_group, topk_group, best in ((1, 1, 1), (4, 2, 1), (4, 2, 2), (24, 5, 2), (3, 3, 2)):
            for renorm in (True, False):
                ids, w = ref.route(logits, 5, score, b, n_group, topk_group, best, renorm, 1.5)
                for t, row in enumerate(logits.tolist()):
                    want = looped_route(row, 5, score, None if b is None else b.tolist(), n_group, topk_group, best)
                    total = sum(v for _, v in want) if renorm else 1.0
                    assert ids[t].tolist() == [i for i, _ in want] + [-1] * (5 - len(want))
                    assert w[t].tolist() == pytest.approx([1.5 * v / total for _, v in want] + [0.0] * (5 - len(want)), rel=1e-12)
    # a mistake in the rule shows: equals by the highest index, groups by one score where two are asked for
    flipped = 23 - ref.route(logits.flip(1), 5, score)[0]
    assert not torch.equal(flipped.clamp(max=23)[3], ref.route(logits, 5, score)[0][3])
    assert not torch.equal(ref.route(logits, 5, score, bias, 4, 2, 1)[0], ref.route(logits, 5, score, bias, 4, 2, 2)[0])


def test_the_reference_gradients_against_differences():
    import layer_ref as ref
    g = torch.Generator().manual_seed(2)
    logits, dw, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((8, 12), (8, 3), (8, 12)))
    ids = ref.route(logits, 3)[0]
    h = 1e-5
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            d, _ = ref.route_grad(dw, logits, ids, score, renorm, 2.0)
            f = [(ref.chosen_weights(logits + s * h * v, ids, ids >= 0, score, renorm, 2.0) * dw).sum() for s in (1, -1)]
            assert float((d * v).sum()) == pytest.approx(float(f[0] - f[1]) / (2 * h), rel=1e-7, abs=1e-9)
    x, w, z, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 8), (16, 8), (5, 16), (5, 16)))
    for act in (None, "silu", "gelu", "relu2"):
        diff = (ref.activation(z + h, act) - ref.activation(z - h, act)) / (2 * h)
        assert torch.allclose(ref.slope(z, act), diff, rtol=1e-6, atol=1e-6)


def test_route_arguments():
    good = (P, 512, 4, 512, 10, 0, 1, None, 8, 4, 2, 1.0, 2, P, P, None)
    for i, bad in ((0, None), (1, 511), (2, -1), (3, 0), (3, 1025), (4, 0), (4, 33), (5, 2), (5, -1), (6, 2), (8, 0), (8, 65), (8, 3), (9, 0),
                   (9, 9), (10, 0), (10, 3), (12, 3), (12, -1), (13, None), (14, None)):
        refused("moe_route", *swapped(good, i, bad))
    refused("moe_route", P, 4, 4, 4, 5, 0, 1, None, 1, 1, 1, 1.0, 2, P, P, None)          # more places than experts
    taken("moe_route", None, 512, 0, 512, 10, 0, 1, None, 8, 4, 2, 1.0, 2, None, None, None)
    good = (P, P, 512, P, 4, 512, 10, 0, 1, 1.0, 2, P, 512, None)
    for i, bad in ((0, None), (1, None), (2, 511), (3, None), (4, -1), (5, 0), (6, 0), (7, 2), (8, 2), (10, 3), (11, None), (12, 511)):
        refused("moe_route_grad", *swapped(good, i, bad))
    taken("moe_route_grad", *swapped(good, 4, 0))


def test_combine_arguments():
    good = (P, 64, P, P, 64, 4, 2, 64, 1, 0, P, 64, None)
    for i, bad in ((0, None), (0, P + 8), (1, 60), (1, 56), (2, None), (3, P + 8), (4, 8), (5, -1), (6, 0), (7, 0), (7, 12), (8, 2), (10, None),
                   (10, P + 2), (11, 12)):
        refused("moe_combine", *swapped(good, i, bad))
    refused("moe_combine", P, 64, P, None, 0, 1 << 20, 1 << 11, 64, 1, 0, P, 64, None)
    taken("moe_combine", *swapped(good, 5, 0))
    good = (P, 64, P, 64, P, 4, 2, 64, 1, P, 64, P, None)
    for i, bad in ((0, None), (1, 12), (2, P + 8), (3, 8), (4, None), (5, -1), (6, 0), (7, 12), (8, -1), (9, None), (10, 60), (11, None)):
        refused("moe_combine_grad", *swapped(good, i, bad))
    taken("moe_combine_grad", *swapped(good, 5, 0))


def test_linear_arguments():
    good = (P, 64, P, P, P, 128, 4, 64, 128, 1, 1, 0, None, P, 128, P, 128, None)
    for i, bad in ((0, None), (0, P + 8), (1, 56), (1, 68), (2, None), (2, P + 2), (3, P + 8), (4, P + 8), (5, 64), (6, -1), (7, 0), (7, 12), (8, 0),
                   (8, 12), (9, 4), (9, -1), (10, 2), (13, P + 8), (14, 64), (15, None), (15, P + 8), (16, 64)):
        refused("moe_linear", *swapped(good, i, bad))
    refused("moe_linear", P, 64, P, None, None, 0, (1 << 30) + 8, 64, 128, 0, 1, 0, None, None, 0, P, 128, None)
    assert "more than one launch" in refused("moe_linear", P, 8, P, None, None, 0, 1 << 30, 8, 1 << 30, 0, 1, 0, None, None, 0, P, 1 << 30, None)
    # few tiles of a long contraction take a workspace
    ws = _lib.lib().moe_linear_workspace_bytes
    assert ws(64, 4096, 4096) >= 2 * 4 * 64 * 4096 and ws(1, 4096, 4096) == 0 and ws(4096, 4096, 4096) == 0 and ws(0, 64, 64) == 0
    for bad in (None, P + 8):
        refused("moe_linear", P, 4096, P, None, None, 0, 64, 4096, 4096, 0, 1, 0, bad, None, 0, P, 4096, None)
    taken("moe_linear", *swapped(good, 6, 0))
    good = (P, 128, 0, P, 64, P, P, 128, 4, 64, 128, 1, 1, P, P, P, 0, P, None)
    for i, bad in ((0, None), (1, 64), (3, None), (4, 60), (5, None), (6, None), (7, 64), (8, -1), (8, (1 << 30) + 8), (9, 12), (10, 12), (11, 4), (12, 2),
                   (13, None), (13, P + 8), (14, P + 8), (15, P + 8)):
        refused("moe_linear_grad", *swapped(good, i, bad))
    ws = _lib.lib().moe_linear_grad_workspace_bytes
    assert ws(0, 64, 128, 0, 0, 0, 0) == 0 and ws(100, 64, 128, 0, 0, 0, 0) == 0 and ws(100, 64, 128, 1, 0, 0, 0) >= 2 * 100 * 128
    assert ws(100, 64, 128, 0, 1, 0, 0) >= 2 * 100 * 128 and ws(100, 64, 128, 0, 0, 0, 1) >= 4 * 128 and ws(1 << 20, 64, 4096, 1, 0, 0, 0) >= 1 << 33
    # few tiles of a long contraction: parts of their own
    assert ws(100, 64, 128, 0, 0, 1, 0) == 0 and ws(8192, 512, 64, 0, 0, 1, 0) >= 2 * 4 * 512 * 64


def clip(grads, outs, sizes, types, limit=1.0, ws=P, norm=P):
    n = len(sizes)
    u64, i64, i32 = ctypes.c_uint64 * max(n, 1), ctypes.c_int64 * max(n, 1), ctypes.c_int32 * max(n, 1)
    return n, u64(*grads), None if outs is None else u64(*outs), i64(*sizes), i32(*types), limit, ws, norm, None


def test_clip_arguments():
    a = 1 << 20
    for bad in (clip([a], [a], [4], [3]), clip([a], [a], [-1], [0]), clip([a], [a], [(1 << 40) + 1], [0]), clip([0], [a], [4], [0]), clip([a], [0], [4], [0]),
                clip([a + 1], [a + 1], [4], [0]), clip([a + 2], [a], [4], [2]), clip([a], [a + 2], [4], [2]), clip([a], [a], [4], [0], -1.0),
                clip([a], [a], [4], [0], float("nan")), clip([a], [a], [4], [0], ws=None), clip([a], [a], [4], [0], ws=P + 8),
                clip([a], [a], [4], [0], norm=None)):
        refused("moe_clip_grads", *bad)
    refused("moe_clip_grads", -1, None, None, None, None, 1.0, P, P, None)
    refused("moe_clip_grads", 1, None, None, None, None, 1.0, P, P, None)
    for bad in (clip([a, a], [a, a], [4, 4], [0, 0]), clip([a, a + 6], [a, a + 6], [4, 4], [0, 0]), clip([a], [a + 2], [4], [0]),
                clip([a, a + 8], [a + 8, a], [4, 4], [0, 0]), clip([a, a + 100], [a + 200, a + 206], [4, 4], [0, 0]),
                clip([a, a + 64, a + 2], [a, a + 64, a + 256], [32, 4, 4], [0, 0, 0])):
        assert "overlaps" in refused("moe_clip_grads", *bad)
    ws = _lib.lib().moe_clip_workspace_bytes
    assert ws(0, 0) >= 16 and ws(3, 1 << 20) >= 16 + 8 * 66
