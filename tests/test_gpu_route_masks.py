"""Routing with finite biases of any size next to ordinary ones: the choice is that of the 64-bit sums."""
import math

import pytest

import layer_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"
LOWEST = torch.finfo(torch.float32).min


def compare(logits, k, **rule):
    from moe_offload import ops
    ids, w = ops.route(logits, k, **rule)
    want_ids, want_w = ref.route(logits, k, **rule)
    assert torch.equal(ids.long(), want_ids)
    slack = ref.weight_slack(logits, k, want_w)
    assert bool(((w.double() - want_w).abs() <= slack + want_w.abs() * ref.F32).all())


RULES = [(512, 10, 1, 1, 1), (512, 10, 8, 4, 2), (512, 10, 8, 4, 1), (240, 9, 8, 4, 2), (64, 6, 8, 2, 2), (1024, 32, 64, 5, 2), (100, 32, 1, 1, 1),
         (96, 8, 48, 20, 2)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_exp,k,n_group,topk_group,group_best", RULES)
@pytest.mark.parametrize("mask", [-1e4, -1e9, -3e38, LOWEST, 1e4, 1e9, 3e38, math.inf])
def test_a_few_experts_far_away(score, n_exp, k, n_group, topk_group, group_best, mask):
    g = torch.Generator(device=DEV).manual_seed(n_exp + k)
    logits = torch.randn((200, n_exp), device=DEV, generator=g) * 1.3
    for few in (1, 5, n_exp // 3):
        bias = torch.randn(n_exp, device=DEV, generator=g) * 0.05
        bias[torch.randperm(n_exp, device=DEV, generator=g)[:few]] = mask
        compare(logits, k, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_best=group_best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_exp,k,n_group,topk_group,group_best", RULES)
def test_values_a_step_apart_beside_far_ones(score, n_exp, k, n_group, topk_group, group_best):
    """Scores that fp32 sums do not tell apart, in every group, with masks of both kinds among them; biases of several magnitudes, whose
    sums round by different steps."""
    g = torch.Generator(device=DEV).manual_seed(n_exp)
    close = 0.25 + torch.randint(-3, 4, (300, n_exp), device=DEV, generator=g) * 2.0 ** -24
    mixed = torch.randn((300, n_exp), device=DEV, generator=g) * 0.01
    for logits in (close.float(), mixed):
        for scale in (1.0, 100.0, 1e5):
            bias = torch.randint(0, 2, (n_exp,), device=DEV, generator=g).float() * scale
            bias[::7] = -1e9
            bias[3::11] = LOWEST
            compare(logits, k, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_best=group_best)
        bias = torch.where(torch.rand(n_exp, device=DEV, generator=g) < 0.5, -1e9, -1e9 - 64)
        compare(logits, k, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_best=group_best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("large", [LOWEST, 3e38])
def test_group_sums_past_fp32(score, large):
    """Two values of a group whose sum fp32 does not hold: still more than a group that has none, and in the order of the 64-bit sums."""
    g = torch.Generator(device=DEV).manual_seed(4)
    logits = torch.randn((50, 32), device=DEV, generator=g)
    bias = torch.zeros(32, device=DEV)
    bias[:12] = -math.inf                              # groups 0 to 2 have nobody
    bias[20:24], bias[24:28] = large, large * 0.9
    for topk_group in (1, 2, 3, 4, 5, 6, 8):
        for k in (4, 20):
            compare(logits, k, score=score, bias=bias, n_group=8, topk_group=topk_group, group_best=2)
            compare(logits, k, score=score, bias=-bias.clamp(min=-3e38), n_group=8, topk_group=topk_group, group_best=2)
