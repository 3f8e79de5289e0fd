"""expert_plan (the row plan made on the GPU) against a stable sort: every entry equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _want(ids, k, n_exp):
    flat = ids.reshape(-1).astype(np.int64)
    cls = np.where((flat >= 0) & (flat < n_exp), flat, n_exp)
    order = np.argsort(cls, kind="stable")
    seg = np.searchsorted(cls[order], np.arange(n_exp + 1))
    return order // k, order, seg


def _check(ids, n_exp, **kw):
    from moe_offload import ops
    k = ids.shape[1] if ids.ndim == 2 else 1
    got = ops.expert_plan(torch.from_numpy(ids).cuda(), n_exp, **kw)
    for g, w, name in zip(got, _want(ids, k, n_exp), ("row_token", "row_out", "seg_start")):
        assert g.dtype == torch.int32
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)


@pytest.mark.parametrize("tokens,k,n_exp", [(1, 10, 512), (64, 10, 512), (1, 1, 1), (777, 6, 100), (63, 1, 2), (65, 3, 1024),
                                            (1000, 2, 1023), (4097, 10, 512), (16384, 10, 512), (40000, 7, 33),
                                            (6553, 10, 1024), (3277, 5, 7), (100000, 1, 5)])
def test_plan_matches_stable_sort(tokens, k, n_exp):
    rng = np.random.default_rng(tokens + k + n_exp)
    _check(rng.integers(0, n_exp, (tokens, k)).astype(np.int32), n_exp)


@pytest.mark.parametrize("tokens", [3, 1000, 30000])
def test_ids_outside_come_last_in_order(tokens):
    rng = np.random.default_rng(tokens)
    ids = rng.integers(-3, 70, (tokens, 4)).astype(np.int32)
    ids[0, 0], ids[0, 1] = -2 ** 31, 2 ** 31 - 1
    _check(ids, 64)
    _check(np.full((tokens, 2), -1, np.int32), 64)
    _check(np.full((tokens, 2), 1024, np.int32), 1024)


@pytest.mark.parametrize("tokens", [5, 20000])
def test_one_expert_takes_all(tokens):
    _check(np.full((tokens, 3), 511, np.int32), 512)
    _check(np.zeros((tokens, 3), np.int32), 512)


def test_no_tokens():
    _check(np.zeros((0, 10), np.int32), 512)


def test_one_dimension_and_given_outputs():
    ids = np.random.default_rng(0).integers(0, 9, 300).astype(np.int32)
    out = {n: torch.full((s,), -7, dtype=torch.int32, device="cuda")
           for n, s in (("row_token", 300), ("row_out", 300), ("seg_start", 10))}
    _check(ids, 9, **out)


def test_matches_resident_plan_and_feeds_the_2bit_products():
    """The same rows as prefill.resident_plan's, with one segment per expert; the 2-bit grouped products take it."""
    from moe_offload import ops, prefill, q2format, synth
    E, H, I, k = 24, 256, 128, 4
    ids, _ = synth.prefill_routing(50, k, E, seed=4)
    row_token, row_out, seg_start, seg_slot = (torch.from_numpy(a).cuda() for a in prefill.resident_plan(ids, k))
    mine = ops.expert_plan(torch.from_numpy(ids.astype(np.int32)).cuda(), E)
    assert torch.equal(mine[0], row_token) and torch.equal(mine[1], row_out)
    pool = torch.from_numpy(q2format.to_blobs(*synth.q2_experts(E, H, I, seed=2), H, I)).cuda()
    x = torch.from_numpy(synth.hidden_states(50, H, seed=5)).cuda()
    want = ops.q2_grouped_switch_glu(x, row_token, seg_start, pool, H, I, row_out=row_out, n_out_rows=200, seg_slot=seg_slot)
    got = ops.q2_grouped_switch_glu(x, mine[0], mine[2], pool, H, I, row_out=mine[1], n_out_rows=200)
    assert torch.equal(want, got)


@pytest.mark.parametrize("tokens", [64, 16384])
def test_replayed_graphs_and_two_streams(tokens):
    from moe_offload import ops
    ids = torch.randint(0, 512, (tokens, 10), dtype=torch.int32, device="cuda")
    ops.expert_plan(ids, 512)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.expert_plan(ids, 512)
        graphs.append((g, out))
    for n in range(3):
        ids.copy_(torch.randint(0, 512, (tokens, 10), dtype=torch.int32, device="cuda"))
        want = [t.clone() for t in ops.expert_plan(ids, 512)]
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), n
    side = torch.cuda.Stream()
    other = torch.randint(0, 512, (tokens, 10), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b = [ops.expert_plan(other, 512) for _ in range(5)]
    a = [ops.expert_plan(ids, 512) for _ in range(5)]
    torch.cuda.synchronize()
    for got, src in ((a, ids), (b, other)):
        want = _want(src.cpu().numpy(), 10, 512)
        for plan in got:
            for t, w in zip(plan, want):
                np.testing.assert_array_equal(t.cpu().numpy(), w)
