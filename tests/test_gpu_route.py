"""Routing of a batch and its gradient against the definition in 64 bits: ids exactly, weights and gradients within the
bounds of layer_ref."""
import math

import pytest

import layer_ref as ref
from grouped_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"
INF = math.inf


def make(n_tok, n_exp, dtype, seed=0, spread=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((n_tok, n_exp), device=DEV, generator=g) * spread + torch.randn(n_exp, device=DEV, generator=g) * 0.5).to(dtype)


def compare(logits, k, **rule):
    from moe_offload import ops
    ids, w = ops.route(logits, k, **rule)
    want_ids, want_w = ref.route(logits, k, **rule)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.long(), want_ids), f"{int((ids.long() != want_ids).any(1).sum())} tokens' ids differ"
    nan = want_w.isnan()
    assert torch.equal(w.isnan(), nan)
    slack = ref.weight_slack(logits, k, want_w.nan_to_num(0.0))
    check(w.nan_to_num(0.0), want_w.nan_to_num(0.0), slack, "weights")
    return ids, w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n_tok,n_exp,k", [(1, 1, 1), (3, 2, 2), (7, 63, 8), (64, 64, 6), (65, 100, 32), (130, 512, 10), (33, 1024, 16), (5, 1000, 1)])
def test_plain(dtype, score, renorm, n_tok, n_exp, k):
    compare(make(n_tok, n_exp, dtype, n_tok + n_exp), k, score=score, renorm=renorm, scale=1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_exp,k,n_group,topk_group,group_best,bias", [
    (512, 10, 1, 1, 1, True), (240, 9, 8, 4, 2, True), (240, 9, 8, 4, 2, False), (256, 8, 8, 3, 1, True), (96, 6, 4, 2, 1, False),
    (64, 8, 64, 8, 2, True), (64, 4, 64, 4, 1, False), (1024, 32, 32, 5, 2, True), (36, 2, 12, 1, 2, True), (65, 5, 13, 13, 2, True),
    (1024, 16, 2, 1, 2, True), (1000, 16, 8, 4, 2, True)])
def test_bias_and_groups(dtype, score, n_exp, k, n_group, topk_group, group_best, bias):
    logits = make(131, n_exp, dtype, n_exp + k)
    b = torch.randn(n_exp, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) * 0.1 if bias else None
    for renorm in (True, False):
        compare(logits, k, score=score, bias=b, n_group=n_group, topk_group=topk_group, group_best=group_best, renorm=renorm, scale=2.5)


def test_many_tokens_differing_by_little():
    """Scores next to each other at the border: 64 bits decide."""
    logits = make(4096, 512, torch.float32, 5, spread=0.01)
    b = torch.randn(512, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) * 1e-4
    for score in ("softmax", "sigmoid"):
        compare(logits, 10, score=score, bias=b)
        compare(logits, 10, score=score, bias=b, n_group=16, topk_group=3, group_best=2)
        compare(logits, 10, score=score, n_group=16, topk_group=3, group_best=2)
    # a bias that puts the sums far from their scores: half of fp32's bits are the bias's
    for score in ("softmax", "sigmoid"):
        compare(logits, 10, score=score, bias=b + 1000.0)
        compare(logits, 10, score=score, bias=b * 1e7)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_to_the_lowest_index(dtype):
    logits = torch.zeros((9, 200), device=DEV, dtype=dtype)
    logits[1, 50:] = 1
    logits[2, ::7] = 2
    logits[3] = -0.0
    logits[3, ::2] = 0.0
    logits[4, 199] = 1
    g = torch.Generator(device=DEV).manual_seed(1)
    logits[5:] = torch.randint(-2, 3, (4, 200), device=DEV, generator=g).to(dtype)
    equal = torch.full((200,), 0.25, device=DEV)
    for score in ("softmax", "sigmoid"):
        compare(logits, 12, score=score)
        compare(logits, 12, score=score, bias=equal)
        compare(logits, 12, score=score, bias=equal, n_group=20, topk_group=5, group_best=2)
        compare(logits, 12, score=score, n_group=20, topk_group=5, group_best=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_masks_infinities_and_nan(dtype, score, renorm):
    lowest = torch.finfo(dtype).min
    logits = make(16, 96, dtype, 8)
    logits[0] = -INF                               # nobody
    logits[1, 5:] = -INF                           # fewer than k
    logits[2, ::2] = -INF
    logits[3] = lowest                             # everybody, evenly
    logits[4, 3:] = lowest
    logits[5, 7] = INF
    logits[6, 7], logits[6, 90] = INF, INF
    logits[7, 11] = math.nan
    logits[8] = math.nan
    logits[9] = INF
    logits[10] = -INF
    logits[10, 95] = 2
    logits[11] = torch.finfo(dtype).max
    logits[12, 1], logits[12, 2] = math.nan, INF
    bias = torch.randn(96, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) * 0.1
    masked = bias.clone()
    masked[20:40] = -INF
    masked[50] = math.nan
    masked[60] = INF
    for b in (None, bias, masked):
        compare(logits, 8, score=score, renorm=renorm, bias=b)
        for best in (1, 2):
            compare(logits, 8, score=score, renorm=renorm, bias=b, n_group=8, topk_group=3, group_best=best)


@pytest.mark.parametrize("shift", [-3000.0, -100.0, 0.0, 60.0, 3000.0])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_renormalised_weights_of_any_magnitude(score, shift):
    logits = make(40, 128, torch.float32, 9) + shift
    _, w = compare(logits, 8, score=score)
    assert float((w.double().sum(1) - 1).abs().max()) < 1e-6


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_and_given_outputs(dtype):
    from moe_offload import ops
    wide = make(50, 301, dtype, 10)
    for logits in (wide[:, :300], wide[:, 1:], wide[::3, 5:205], wide[4:5]):
        compare(logits, 7)
    ids, w = torch.full((50, 4), -7, dtype=torch.int32, device=DEV), torch.full((50, 4), -7.0, device=DEV)
    got = ops.route(wide, 4, ids=ids, weights=w)
    assert got[0] is ids and got[1] is w
    want = ref.route(wide, 4)
    assert torch.equal(ids.long(), want[0])
    assert ops.route(wide[:0], 4)[0].shape == (0, 4)


def test_more_tokens_than_blocks_hold():
    compare(make(70001, 16, torch.bfloat16, 11), 2, score="sigmoid")


# ---- the gradient ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n_tok,n_exp,k", [(1, 1, 1), (3, 2, 2), (70, 63, 8), (65, 100, 32), (130, 512, 10), (33, 1024, 16), (5, 1000, 1)])
def test_gradient(dtype, score, renorm, n_tok, n_exp, k):
    from moe_offload import ops
    logits = make(n_tok, n_exp, dtype, n_tok + n_exp + 1)
    ids, _ = ops.route(logits, k, score=score, renorm=renorm)
    dw = torch.randn((n_tok, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    got = ops.route_grad(dw, logits, ids, score=score, renorm=renorm, scale=2.5)
    want, slack = ref.route_grad(dw, logits, ids, score, renorm, 2.5)
    assert got.dtype == dtype
    check(got, want, slack, "dlogits")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(score, renorm):
    """(f(l + h v) - f(l - h v)) / 2h in 64 bits with h = 2^-12, the choice held: off by h^2 / 6 times a third derivative, which
    for sums of |dw| <= 4 and directions of |v| <= 4 stays below 4^4 x 20 per place: 2^-26 x 850 x k."""
    from moe_offload import ops
    logits, k = make(20, 48, torch.float32, 12), 6
    ids, _ = ops.route(logits, k, score=score, renorm=renorm)
    g = torch.Generator(device=DEV).manual_seed(13)
    dw = torch.randn((20, k), device=DEV, generator=g).clamp(-4, 4)
    got = ops.route_grad(dw, logits, ids, score=score, renorm=renorm, scale=1.0).double()
    has, h = ids >= 0, 2.0 ** -12
    for _ in range(5):
        v = torch.randn((20, 48), device=DEV, generator=g).clamp(-4, 4).double()
        f = [(ref.chosen_weights(logits.double() + s * h * v, ids.long(), has, score, renorm, 1.0) * dw.double()).sum(1) for s in (1, -1)]
        diff = (f[0] - f[1]) / (2 * h)
        along = (got * v).sum(1)
        assert float((diff - along).abs().max()) <= 2.0 ** -26 * 850 * k + 48 * 4 * 4e-5


def test_gradient_of_places_without_an_expert_and_of_one_twice():
    from moe_offload import ops
    logits = make(6, 40, torch.float32, 14)
    logits[1, 5:] = -INF
    ids = torch.tensor([[0, 1, 2, 3], [0, 1, -1, -1], [-1, -1, -1, -1], [4, 4, 5, 40], [7, 7, 7, 7], [2 ** 31 - 1, 3, -2 ** 31, 9]],
                       dtype=torch.int32, device=DEV)
    dw = torch.randn((6, 4), device=DEV, generator=torch.Generator(device=DEV).manual_seed(15))
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            out = torch.full((6, 40), math.nan, device=DEV)
            # what stands behind a place without an expert is not looked at
            poisoned = torch.where((ids >= 0) & (ids < 40), dw, math.nan)
            got = ops.route_grad(poisoned, logits, ids, score=score, renorm=renorm, out=out)
            assert got is out
            want, slack = ref.route_grad(dw, logits, ids, score, renorm, 1.0)
            check(got, want, slack, f"{score} {renorm}")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_at_extremes_is_finite(score, renorm):
    from moe_offload import ops
    logits = make(8, 64, torch.float32, 16)
    logits[0] = -INF
    logits[1, 3:] = -INF
    logits[2] = torch.finfo(torch.float32).min
    logits[3, 4] = INF
    logits[4] += 3000
    logits[5] -= 3000
    logits[6, 0], logits[6, 63] = INF, INF
    ids, _ = ops.route(logits, 5, score=score, renorm=renorm)
    got = ops.route_grad(torch.ones((8, 5), device=DEV), logits, ids, score=score, renorm=renorm)
    assert bool(got.isfinite().all())
    assert not bool(got[0].any())


def test_gradient_steps():
    from moe_offload import ops
    wide, out = make(30, 201, torch.bfloat16, 17), torch.full((30, 205), 7.0, dtype=torch.bfloat16, device=DEV)
    for renorm in (True, False):
        logits, o = wide[:, 1:], out[:, 3:203]
        ids, _ = ops.route(logits, 5, renorm=renorm)
        dw = torch.randn((30, 5), device=DEV, generator=torch.Generator(device=DEV).manual_seed(18))
        got = ops.route_grad(dw, logits, ids, renorm=renorm, out=o)
        want, slack = ref.route_grad(dw, logits, ids, "softmax", renorm, 1.0)
        check(got, want, slack)
        assert bool((out[:, :3] == 7).all()) and bool((out[:, 203:] == 7).all())


def test_captured_and_replayed():
    from moe_offload import ops
    logits = make(200, 512, torch.float32, 19)
    bias = torch.zeros(512, device=DEV)
    dw = torch.ones((200, 10), device=DEV)

    def both():
        ids, w = ops.route(logits, 10, score="sigmoid", bias=bias, n_group=8, topk_group=4, group_best=2)
        return ids, w, ops.route_grad(dw, logits, ids, score="sigmoid", renorm=False)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (1, 2, 3):
        logits.copy_(make(200, 512, torch.float32, seed))
        bias.normal_(0, 0.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, both()):
            assert torch.equal(a, b)


def test_on_another_stream():
    from moe_offload import ops
    logits = make(300, 512, torch.float32, 20)
    want = ops.route(logits, 10)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.route(logits, 10)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
