"""Low-rank adapters beside a shared projection against 64-bit forms (grouped_ref.py): one token to many, runs of a
request and tokens in any order, ranks and widths that end inside tiles, tokens without an adapter, strides, in
place, streams, replayed graphs, gradients."""
import pytest

import grouped_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def make(dtype, tokens, n_ad, rank, n_in, n_out, seed=0, runs=True):
    g = torch.Generator().manual_seed(seed)
    if runs:
        ids = torch.randint(-1, n_ad, (max(1, tokens // 37 + 1),), generator=g).repeat_interleave(37)[:tokens]
    else:
        ids = torch.randint(-1, n_ad + 1, (tokens,), generator=g)
    return (rnd((tokens, n_out), dtype, seed + 1), rnd((tokens, n_in), dtype, seed + 2), rnd((n_ad, rank, n_in), dtype, seed + 3, n_in ** -0.5),
            rnd((n_ad, n_out, rank), dtype, seed + 4, rank ** -0.5), ids.to(torch.int32).to(DEV),
            (torch.rand(n_ad, generator=g) + 0.5).to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("runs", [True, False])
@pytest.mark.parametrize("tokens,n_ad,rank,n_in,n_out", [
    (1, 1, 8, 8, 8), (1, 5, 16, 2048, 2048), (7, 3, 24, 264, 136), (16, 16, 64, 512, 520), (17, 40, 8, 1000, 72),
    (64, 4, 128, 128, 256), (65, 2, 40, 72, 1032), (333, 5, 8, 640, 2560), (500, 9, 256, 72, 264), (1500, 3, 48, 320, 200),
    (1100, 5, 16, 136, 264), (300, 1024, 8, 72, 40)])
def test_add(dtype, runs, tokens, n_ad, rank, n_in, n_out):
    from moe_offload import ops
    base, x, a, b, ids, scale = make(dtype, tokens, n_ad, rank, n_in, n_out, runs=runs)
    keep = base.clone()
    out = ops.lora_add(base, x, a, b, ids, scale=scale)
    assert torch.equal(base, keep)
    ref.check(out, *ref.lora(base, x, a, b, ids, scale), "add")
    none = (ids < 0) | (ids >= n_ad)
    assert torch.equal(out[none], base[none])
    ref.check(ops.lora_add(base, x, a, b, ids), *ref.lora(base, x, a, b, ids), "no scale")
    same = ops.lora_add(base, x, a, b, ids, scale=scale, out=base)
    assert same is base and torch.equal(base, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_no_adapters(dtype):
    from moe_offload import ops
    base, x, a, b, ids, scale = make(dtype, 50, 4, 16, 136, 72, runs=False)
    xs, bs = rnd((50, 200), dtype, 20)[:, 16:152], rnd((50, 88), dtype, 21)[:, 8:80]
    full = torch.full((50, 88), 7.0, dtype=dtype, device=DEV)
    a2 = rnd((4 * (16 * 136 + 8),), dtype, 22, 0.1).as_strided((4, 16, 136), (16 * 136 + 8, 136, 1))
    b2 = rnd((4 * (16 * 72 + 24),), dtype, 23, 0.2).as_strided((4, 72, 16), (16 * 72 + 24, 16, 1))
    ops.lora_add(bs, xs, a2, b2, ids, scale=scale, out=full[:, :72])
    ref.check(full[:, :72], *ref.lora(bs, xs, a2, b2, ids, scale))
    assert bool((full[:, 72:] == 7).all())
    assert torch.equal(ops.lora_add(base, x, a[:0], b[:0], ids), base)
    assert torch.equal(ops.lora_add(base, x, a, b, torch.full_like(ids, -1)), base)
    assert ops.lora_add(base[:0], x[:0], a, b, ids[:0]).shape == (0, 72)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_stays_in_its_token_and_adapter(dtype):
    from moe_offload import ops
    for tokens in (20, 300):
        base, x, a, b, ids, scale = make(dtype, tokens, 4, 16, 136, 72, runs=False)
        clean = ops.lora_add(base, x, a, b, ids, scale=scale)
        x2, a2 = x.clone(), a.clone()
        t = int((ids == 1).nonzero()[0])
        x2[t, 5] = float("nan")
        x2[ids < 0] = float("inf")                      # not read: these tokens have no adapter
        got = ops.lora_add(base, x2, a, b, ids, scale=scale)
        keep = torch.ones(tokens, dtype=torch.bool, device=DEV)
        keep[t] = False
        assert torch.equal(got[keep], clean[keep]) and bool(got[t].isnan().all())
        a2[2, 3, 4] = float("inf")
        got = ops.lora_add(base, x, a2, b, ids, scale=scale)
        assert torch.equal(got[ids != 2], clean[ids != 2]) and not bool(got[ids == 2].isfinite().any())


def test_v_is_not_rounded_to_16_bits():
    """A x beyond fp16's range, scaled back by B and the scale: finite, as the 32-bit intermediate is."""
    from moe_offload import ops
    for tokens in (1, 100):
        base = torch.zeros((tokens, 8), dtype=torch.float16, device=DEV)
        x = torch.full((tokens, 512), 64.0, dtype=torch.float16, device=DEV)
        a = torch.full((1, 8, 512), 64.0, dtype=torch.float16, device=DEV)
        b = torch.full((1, 8, 8), 2.0 ** -12, dtype=torch.float16, device=DEV)
        out = ops.lora_add(base, x, a, b, torch.zeros(tokens, dtype=torch.int32, device=DEV))
        assert bool((out == 8 * 2.0 ** 21 * 2.0 ** -12).all())          # 512 * 64 * 64 = 2^21, eight times 2^-12 of it


def test_offsets_past_32_bits():
    from moe_offload import ops
    dt, step = torch.bfloat16, 2 ** 31 + 64
    base, x, a, b, ids, scale = make(dt, 40, 3, 8, 72, 40, runs=False)
    buf = torch.empty(2 * step + 2 ** 16, dtype=dt, device=DEV)
    a2, b2 = buf.as_strided(a.shape, (step, 72, 1)), buf.as_strided(b.shape, (step, 8, 1), 2 ** 14)
    a2.copy_(a)
    b2.copy_(b)
    ref.check(ops.lora_add(base, x, a2, b2, ids, scale=scale), *ref.lora(base, x, a, b, ids, scale))


@pytest.mark.parametrize("tokens", [8, 700])
def test_replayed_graphs_and_streams(tokens):
    from moe_offload import ops
    dt = torch.bfloat16
    base, x, a, b, ids, scale = make(dt, tokens, 6, 16, 264, 136, runs=False)
    dy = rnd((tokens, 136), dt, 9)

    def step():
        return (ops.lora_add(base, x, a, b, ids, scale=scale), *ops.lora_grad(dy, x, a, b, ids, scale=scale))
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for n in range(3):
        x.copy_(rnd(x.shape, dt, 30 + n))
        ids.copy_(make(dt, tokens, 6, 8, 8, 8, seed=40 + n, runs=False)[4])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), n
    side = torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(side):
            got.append(step())
        got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g in got for p, q in zip(g, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,n_ad,rank,n_in,n_out", [(1, 3, 8, 64, 72), (50, 4, 24, 136, 264), (333, 5, 8, 640, 256), (100, 2, 96, 136, 72),
                                                         (1100, 3, 16, 136, 264), (1500, 2, 40, 264, 136), (40, 1024, 8, 24, 16),
                                                         (5000, 1, 8, 64, 72), (4500, 1, 136, 264, 136)])
def test_gradients(dtype, tokens, n_ad, rank, n_in, n_out):
    """(dx, da, db) against the formula in 64 bits.  v and dv are sums of two values of the type before the second product:
    the first is off by at most half a step, eps / 2 of the value, and the second by as much of that."""
    from moe_offload import dense, ops
    base, x, a, b, ids, scale = make(dtype, tokens, n_ad, rank, n_in, n_out, runs=False)
    dy = rnd((tokens, n_out), dtype, 40)
    half, tiny = (torch.finfo(dtype).eps / 2) ** 2, {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    dx, da, db = ops.lora_grad(dy, x, a, b, ids, scale=scale)
    wx, sx = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for j in range(n_ad):
        rows = (ids.cpu() == j).nonzero()[:, 0]
        xd, dyd, aj, bj, s = x.double().cpu()[rows], dy.double().cpu()[rows], a[j].double().cpu(), b[j].double().cpu(), float(scale[j])
        v, dv = xd @ aj.T, s * dyd @ bj
        ev = (n_in + 2) * ref.F32 * (xd.abs() @ aj.abs().T)
        ev = ev + half * (v.abs() + ev) + tiny
        edv = (n_out + 2) * ref.F32 * abs(s) * (dyd.abs() @ bj.abs())
        edv = edv + half * (dv.abs() + edv) + tiny
        m = rows.numel()
        wx[rows] = dv @ aj
        sx[rows] = edv @ aj.abs() + (rank + 2) * ref.F32 * ((dv.abs() + edv) @ aj.abs())
        ref.check(da[j], dv.T @ xd, edv.T @ xd.abs() + (m + 2) * ref.F32 * ((dv.abs() + edv).T @ xd.abs()), f"da {j}")
        ref.check(db[j], s * dyd.T @ v, abs(s) * (dyd.abs().T @ ev + (m + 2) * ref.F32 * (dyd.abs().T @ (v.abs() + ev))), f"db {j}")
    ref.check(dx, wx, sx, "dx")

    leaves = [t.clone().requires_grad_() for t in (base, x, a, b)]
    out = dense.lora_add(*leaves, ids, scale)
    out.backward(dy)
    for got, want in zip(leaves, (dy, dx, da, db)):
        assert torch.equal(got.grad, want)


def test_gradients_without_tokens():
    from moe_offload import ops
    base, x, a, b, ids, scale = make(torch.bfloat16, 3, 4, 16, 64, 72)
    dx, da, db = ops.lora_grad(base[:0], x[:0], a, b, ids[:0], scale=scale)
    assert dx.shape == (0, 64) and not bool(da.any()) and not bool(db.any())
    dx, da, db = ops.lora_grad(base, x, a, b, torch.full_like(ids, 4), scale=scale)
    assert not bool(dx.any()) and not bool(da.any()) and not bool(db.any())


def test_gradient_against_differences():
    from moe_offload import ops
    dtype = torch.float16
    base, x, a, b, ids, scale = make(dtype, 20, 3, 8, 40, 24, runs=False)
    dy = rnd((20, 24), dtype, 9)
    grads = ops.lora_grad(dy, x, a, b, ids, scale=scale)
    point = [t.double().cpu() for t in (x, a, b)]

    def f(v):
        total = 0.0
        for t, i in enumerate(ids.tolist()):
            if 0 <= i < 3:
                total += float(scale[i]) * float((dy[t].double().cpu() * (v[2][i] @ (v[1][i] @ v[0][t]))).sum())
        return total
    for i, g in enumerate(grads):
        d = torch.randn(point[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        up, dn = [p.clone() for p in point], [p.clone() for p in point]
        up[i] += 1e-3 * d
        dn[i] -= 1e-3 * d
        want = (f(up) - f(dn)) / 2e-3                       # f is linear in each argument: exact but for rounding
        room = 2 * torch.finfo(dtype).eps / 2 * float(g.double().cpu().norm() * d.norm()) + 1e-9
        assert abs(float((g.double().cpu() * d).sum()) - want) <= room, i


def test_beside_the_2bit_experts():
    """As served: the 2-bit grouped SwitchGLU, its rows combined, each request's adapter on top, and the gradient
    that trains the adapters over the frozen experts."""
    from moe_offload import ops, q2format, synth
    E, H, I, k, T = 16, 256, 128, 4, 40
    ids, scores = synth.prefill_routing(T, k, E, seed=6)
    pool = torch.from_numpy(q2format.to_blobs(*synth.q2_experts(E, H, I, seed=3), H, I)).cuda()
    x = torch.from_numpy(synth.hidden_states(T, H, seed=7)).cuda()
    tok, order, seg = ops.expert_plan(torch.from_numpy(ids.astype("int32")).cuda(), E)
    y = ops.q2_grouped_switch_glu(x, tok, seg, pool, H, I, row_out=order, n_out_rows=T * k)
    base = ops.pair_combine(y, torch.from_numpy(scores).cuda()).half()
    _, _, a, b, ad, scale = make(torch.float16, T, 3, 16, H, H, runs=True)
    out = ops.lora_add(base, x, a, b, ad, scale=scale)
    ref.check(out, *ref.lora(base, x, a, b, ad, scale))
    dx, da, db = ops.lora_grad(out, x, a, b, ad, scale=scale)
    assert da.shape == a.shape and db.shape == b.shape and bool(dx.isfinite().all())


def test_v_past_the_largest_rounded_value():
    # v = 2^127 (1 + 255/256) is finite in fp32 and rounds to infinity in bf16; times 2^-120 it is 255.5
    from moe_offload import ops
    x = torch.zeros((3, 8), dtype=torch.bfloat16, device=DEV)
    x[:, 0], x[:, 1] = 2.0 ** 63, 2.0 ** 62
    x[1] = -x[1]
    a = torch.zeros((1, 8, 8), dtype=torch.bfloat16, device=DEV)
    a[0, 0, 0], a[0, 0, 1] = 2.0 ** 64, 2.0 ** 65 * (255 / 256)
    b = torch.zeros((1, 16, 8), dtype=torch.bfloat16, device=DEV)
    b[0, :, 0] = 2.0 ** -120
    base = torch.full((3, 16), -128.0, dtype=torch.bfloat16, device=DEV)
    out = ops.lora_add(base, x, a, b, torch.zeros(3, dtype=torch.int32, device=DEV))
    # 127.5 and -383.5, exact in the sum, rounded once (127.5 is a value of the type; -383.5 lies between -382 and -384)
    assert out[0].tolist() == [127.5] * 16 and out[2].tolist() == [127.5] * 16 and out[1].tolist() == [-384.0] * 16
