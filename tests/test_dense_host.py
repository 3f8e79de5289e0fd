"""Refusals of the unquantised experts' operators and of the adapters, without a GPU: the tensor checks of
moe_offload.ops and the argument checks of the C entry points, none of which launches anything."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from moe_offload import _lib, dense, ops  # noqa: E402


def test_tensors_off_the_gpu_are_refused():
    x, w, seg = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros((2, 8, 16), dtype=torch.bfloat16), torch.tensor([0, 2, 4], dtype=torch.int32)
    ids = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.expert_plan(ids, 2), lambda: ops.grouped_mm(x, seg, w), lambda: ops.grouped_gate_up(x, None, seg, w),
                 lambda: ops.grouped_mm_dx(x[:, :8], seg, w), lambda: ops.grouped_mm_dw(x, x, seg),
                 lambda: ops.lora_add(x, x, w, w.transpose(1, 2).contiguous(), ids),
                 lambda: ops.lora_grad(x, x, w, w.transpose(1, 2).contiguous(), ids)):
        with pytest.raises(ValueError, match="not on a GPU"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        ops.grouped_mm([1.0], seg, w)


def test_matrix_checks():
    bf = torch.bfloat16
    rows = lambda t, **kw: ops._rows("op", "x", t, bf, kw.get("rows"), kw.get("width"))  # noqa: E731
    assert rows(torch.zeros((4, 16), dtype=bf)) == 16
    assert rows(torch.zeros((4, 24), dtype=bf)[:, :16]) == 24
    assert rows(torch.zeros((1, 24), dtype=bf)[:, 8:]) == 16
    with pytest.raises(TypeError):
        rows(torch.zeros((4, 16)))
    for bad in (torch.zeros((4, 12), dtype=bf), torch.zeros((4, 0), dtype=bf), torch.zeros(16, dtype=bf),
                torch.zeros((16, 8), dtype=bf).T, torch.zeros((1, 16), dtype=bf).expand(4, 16),
                torch.zeros((4, 20), dtype=bf)[:, :16], torch.zeros((64,), dtype=bf).as_strided((4, 16), (8, 1))):
        with pytest.raises(ValueError):
            rows(bad)
    with pytest.raises(ValueError):
        rows(torch.zeros((4, 16), dtype=bf), rows=5)
    mats = lambda t: ops._mats("op", "w", t, bf, (None, None, None))  # noqa: E731
    assert mats(torch.zeros((3, 8, 16), dtype=bf)) == 128
    assert mats(torch.zeros((3, 16, 16), dtype=bf)[:, :8]) == 256
    for bad in (torch.zeros((3, 8, 12), dtype=bf), torch.zeros((3, 4, 16), dtype=bf), torch.zeros((8, 16), dtype=bf),
                torch.zeros((3, 16, 8), dtype=bf).transpose(1, 2), torch.zeros((3, 8, 32), dtype=bf)[..., :16],
                torch.zeros((1, 8, 16), dtype=bf).expand(3, 8, 16)):
        with pytest.raises(ValueError):
            mats(bad)
    with pytest.raises(TypeError):
        ops._index("op", "ids", torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops._index("op", "ids", torch.zeros(8, dtype=torch.int32)[::2])
    with pytest.raises(TypeError):
        ops._half("op", torch.zeros(4))


def test_layer_shapes_are_checked():
    x, ids = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros((4, 2), dtype=torch.int32)
    up, down = torch.zeros((3, 16, 16), dtype=torch.bfloat16), torch.zeros((3, 16, 8), dtype=torch.bfloat16)
    for args in ((x, ids[:3], up, down), (x, ids[:, 0], up, down), (x, ids, up, down[:2]), (x, ids, up[:, :8], down), (x[:, :8], ids, up, down)):
        with pytest.raises(ValueError):
            dense.switch_glu(*args)
    with pytest.raises(ValueError, match="scale"):
        dense.lora_add(x, x, up, up, ids[:, 0], torch.ones(3, requires_grad=True))


# ---- C entry points: 64 stands for some aligned device address, which is never read here ----------

P = 64


def refused(name, *args):
    lib = _lib.lib()
    lib.c_clear_error()
    rc = getattr(lib, name)(*args)
    msg = _lib.last_error()
    lib.c_clear_error()
    assert rc == -1 and msg, (name, args)
    return msg


PLAN = dict(ids=P, n_ids=20, k=4, n_exp=8, workspace=None, row_token=P, row_out=P, seg_start=P, stream=None)
MM = dict(x=P, ldx=64, n_x=10, row_in=None, seg_start=P, seg_slot=None, n_seg=2, n_rows=10, w=P, w_stride=4096, n_slots=2, n=64, k=64,
          scale=None, y=P, ldy=64, n_y=10, row_out=None, dtype=1, fill=0, stream=None)
UP = dict(x=P, ldx=64, n_x=10, row_in=None, seg_start=P, seg_slot=None, n_seg=2, n_rows=10, w=P, w_stride=4096, n_slots=2, inter=32,
          hidden=64, h=P, ldh=32, gu=None, ldgu=0, dtype=1, fill=0, stream=None)
DX = dict(dy=P, lddy=64, n_dy=10, row_in=None, seg_start=P, seg_slot=None, n_seg=2, n_rows=10, w=P, w_stride=4096, n_slots=2, n=64, k=64,
          scale=None, gu=None, ldgu=0, dx=P, lddx=64, n_dx=10, row_out=None, dtype=1, fill=0, stream=None)
DW = dict(dy=P, lddy=64, n_dy=10, row_dy=None, x=P, ldx=64, n_x=10, row_x=None, seg_start=P, n_seg=2, n_rows=10, n=64, k=64, scale=None,
          dw=P, dw_stride=4096, out_f32=0, dtype=1, stream=None)
LORA = dict(base=P, ld_base=64, x=P, ldx=64, a=P, a_stride=512, b=P, b_stride=512, ids=P, scale=None, n_tok=4, n_ad=2, n_in=64, n_out=64,
            rank=8, dtype=1, workspace=P, out=P + 4096, ld_out=64, stream=None)
GRAD = dict(dy=P, lddy=64, x=P, ldx=64, a=P, a_stride=512, b=P, b_stride=512, ids=P, scale=None, n_tok=4, n_ad=2, n_in=64, n_out=64,
            rank=8, dtype=1, workspace=P, dx=P, lddx=64, da=P, db=P, stream=None)


@pytest.mark.parametrize("name,good,bad", [
    ("moe_expert_plan", PLAN, [dict(n_ids=-4), dict(k=0), dict(k=3), dict(n_exp=0), dict(n_exp=1025), dict(ids=None), dict(row_token=None),
                               dict(row_out=None), dict(seg_start=None), dict(n_ids=4100)]),
    ("moe_grouped_mm", MM, [dict(n_seg=-1), dict(n_seg=1025), dict(n_rows=-1), dict(n_rows=11), dict(n_x=9), dict(n_y=9), dict(dtype=2),
                            dict(k=60), dict(n=0), dict(n=-8), dict(n=12), dict(ldx=60), dict(ldx=56), dict(ldx=-64), dict(ldy=56), dict(w_stride=4088),
                            dict(w_stride=4100), dict(x=None), dict(x=P + 2), dict(w=None), dict(w=P + 8), dict(y=None), dict(y=P + 4),
                            dict(seg_start=None), dict(n_slots=-1)]),
    ("moe_grouped_gate_up", UP, [dict(inter=12), dict(inter=0), dict(hidden=36), dict(ldh=24), dict(h=None), dict(gu=P, ldgu=56), dict(gu=P + 2, ldgu=64),
                                 dict(w_stride=4088), dict(n_x=9), dict(dtype=-1), dict(inter=0x40000000)]),
    ("moe_grouped_mm_dx", DX, [dict(k=60), dict(n=60), dict(lddx=56), dict(lddy=56), dict(gu=P, ldgu=128), dict(gu=P, ldgu=120, lddx=128),
                               dict(dx=None), dict(dy=None), dict(n_dy=9), dict(n_dx=9), dict(w_stride=8)]),
    ("moe_grouped_mm_dw", DW, [dict(n=60), dict(k=60), dict(dw=None), dict(dw=P + 8), dict(dw_stride=4088), dict(n_dy=9), dict(n_x=9), dict(dtype=7),
                               dict(seg_start=None), dict(n_seg=1025)]),
    ("moe_lora_add", LORA, [dict(rank=12), dict(rank=0), dict(rank=264), dict(n_in=60), dict(n_out=60), dict(n_tok=-1), dict(n_ad=-1), dict(dtype=2),
                            dict(ldx=56), dict(ldx=60), dict(ld_base=56), dict(ld_out=56), dict(a_stride=504), dict(b_stride=504), dict(a=None),
                            dict(b=None), dict(ids=None), dict(out=None), dict(base=None), dict(workspace=None), dict(x=P + 2), dict(out=P + 8),
                             dict(out=P, ld_out=72), dict(n_out=1 << 23, ld_base=1 << 23, ld_out=1 << 23, b_stride=1 << 26)]),
    ("moe_lora_grad", GRAD, [dict(rank=12), dict(rank=264), dict(n_in=60), dict(n_out=60), dict(n_tok=-1), dict(n_ad=0), dict(n_ad=1025),
                             dict(dtype=2), dict(ldx=56), dict(lddy=56), dict(lddx=56), dict(a_stride=504), dict(b_stride=504), dict(a=None),
                             dict(b=None), dict(ids=None), dict(dx=None), dict(da=None), dict(db=P + 8), dict(workspace=None), dict(workspace=P + 4),
                             dict(dy=None), dict(x=P + 2)]),
])
def test_entry_points_refuse(name, good, bad):
    for change in bad:
        assert set(change) <= set(good)
        refused(name, *{**good, **change}.values())


def test_nothing_to_do_launches_nothing():
    lib = _lib.lib()
    lib.c_clear_error()
    for name, args in (("moe_grouped_mm", {**MM, "n_rows": 0}), ("moe_grouped_gate_up", {**UP, "n_rows": 0}),
                       ("moe_grouped_mm_dx", {**DX, "n_rows": 0}), ("moe_grouped_mm_dw", {**DW, "n_seg": 0}), ("moe_lora_add", {**LORA, "n_tok": 0})):
        assert getattr(lib, name)(*args.values()) == 0 and not _lib.last_error(), name
    assert lib.moe_expert_plan_workspace_bytes(4096, 512) == 0 and lib.moe_expert_plan_workspace_bytes(4097, 512) == 3 * 513 * 4
    assert lib.moe_expert_plan_workspace_bytes(2 ** 31 - 1, 1024) == 256 * 1025 * 4
    assert lib.moe_lora_grad_workspace_bytes(0, 3, 8) == 16
    assert lib.moe_lora_workspace_bytes(5, 16) == 320 and lib.moe_lora_workspace_bytes(0, 16) == 0
    assert ctypes.sizeof(ctypes.c_int64) == 8


BIG = 2 ** 30 + 8


@pytest.mark.parametrize("name,good,bad", [
    ("moe_grouped_mm", MM, [dict(n=BIG, ldy=BIG, w_stride=64 * BIG), dict(k=BIG, ldx=BIG, w_stride=64 * BIG), dict(n_rows=BIG, n_x=BIG, n_y=BIG)]),
    ("moe_grouped_gate_up", UP, [dict(hidden=BIG, ldx=BIG, w_stride=64 * BIG), dict(n_rows=BIG, n_x=BIG)]),
    ("moe_grouped_mm_dx", DX, [dict(n=BIG, lddy=BIG, w_stride=64 * BIG), dict(k=BIG, lddx=BIG, w_stride=64 * BIG), dict(n_rows=BIG, n_dy=BIG, n_dx=BIG)]),
    ("moe_grouped_mm_dw", DW, [dict(n=BIG, lddy=BIG, dw_stride=64 * BIG), dict(k=BIG, ldx=BIG, dw_stride=64 * BIG), dict(n_rows=BIG, n_dy=BIG, n_x=BIG)]),
    ("moe_lora_add", LORA, [dict(n_in=BIG, ldx=BIG, a_stride=8 * BIG), dict(n_tok=BIG)]),
    ("moe_lora_grad", GRAD, [dict(n_in=BIG, ldx=BIG, lddx=BIG, a_stride=8 * BIG), dict(n_tok=BIG)]),
])
def test_sizes_whose_sums_would_pass_31_bits_are_refused(name, good, bad):
    for change in bad:
        assert set(change) <= set(good)
        refused(name, *{**good, **change}.values())


def test_sizes_past_the_library_s_integers_are_refused():
    big, bf = 2 ** 31 + 8, torch.bfloat16
    for check, t in ((lambda t: ops._rows("op", "x", t, bf, None, None), torch.empty((big, 8), dtype=bf, device="meta")),
                     (lambda t: ops._rows("op", "x", t, bf, None, None), torch.empty((1, big), dtype=bf, device="meta")),
                     (lambda t: ops._mats("op", "w", t, bf, (None, None, None)), torch.empty((big, 8, 8), dtype=bf, device="meta")),
                     (lambda t: ops._mats("op", "w", t, bf, (None, None, None)), torch.empty((1, 8, big), dtype=bf, device="meta")),
                     (lambda t: ops._index("op", "ids", t), torch.empty(big, dtype=torch.int32, device="meta"))):
        with pytest.raises(ValueError, match="2\\^30"):
            check(t)


def test_adapters_past_the_gradients_limit_are_refused_where_the_call_is_made():
    base, x, ids = torch.zeros((2, 8)), torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int32)
    a, b = torch.zeros((1025, 8, 8)), torch.zeros((1025, 8, 8))
    for i in range(3):
        args = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, a, b))]
        with pytest.raises(ValueError, match="1024"):
            dense.lora_add(base, *args, ids)
        with torch.no_grad(), pytest.raises(ValueError, match="not on a GPU"):       # forward alone has no such limit
            dense.lora_add(base, *args, ids)
    with pytest.raises(ValueError, match="not on a GPU"):
        dense.lora_add(base.requires_grad_(), x, a, b, ids)


def test_pair_combine_takes_contiguous_fp16():
    """Other types, and rows that do not follow each other, would be read as if they were."""
    y, scores, res, out = (torch.zeros((6, 16), dtype=torch.float16), torch.zeros((3, 2), dtype=torch.float16),
                           torch.zeros((3, 16), dtype=torch.float16), torch.zeros((3, 16)))
    for args in ((y.bfloat16(), scores), (y, scores.float()), (y, scores.bfloat16(), res), (y, scores, res.float()),
                 (y, scores, res, out.half())):
        with pytest.raises(TypeError, match="pair_combine"):
            ops.pair_combine(*args)
    for args in ((torch.zeros((6, 32), dtype=torch.float16)[:, :16], scores), (y[:5], scores), (y, torch.zeros((2, 3), dtype=torch.float16).T),
                 (y, scores, res[:2]), (y, scores, res, out[:2])):
        with pytest.raises(ValueError, match="pair_combine"):
            ops.pair_combine(*args)


TOKENS = 32 * (2 ** 24 - 1)                                    # 2^24 - 1 blocks of 256 threads


@pytest.mark.parametrize("name,good,change", [
    ("moe_grouped_mm", MM, dict(n_rows=2 ** 30, n_x=2 ** 30, n_y=2 ** 30, n=8192, ldy=8192, k=4096, ldx=4096, w_stride=8192 * 4096)),
    ("moe_grouped_gate_up", UP, dict(n_rows=2 ** 30, n_x=2 ** 30, inter=4096, ldh=4096, hidden=4096, ldx=4096, w_stride=8192 * 4096)),
    ("moe_grouped_mm_dx", DX, dict(n_rows=2 ** 30, n_dy=2 ** 30, n_dx=2 ** 30, n=4096, lddy=4096, k=8192, lddx=8192, w_stride=8192 * 4096)),
    ("moe_grouped_mm_dw", DW, dict(n_seg=1024, n=2 ** 16, lddy=2 ** 16, k=2 ** 16, ldx=2 ** 16, dw_stride=2 ** 32)),
    ("moe_lora_add", LORA, dict(n_tok=TOKENS + 1)),
    ("moe_lora_grad", GRAD, dict(n_tok=TOKENS + 1)),
    ("moe_lora_grad", GRAD, dict(n_tok=2 ** 28, n_in=8192, ldx=8192, lddx=8192, rank=256, a_stride=2 ** 21, b_stride=2 ** 14)),
    ("moe_lora_grad", GRAD, dict(n_ad=1024, n_in=2 ** 30, ldx=2 ** 30, lddx=2 ** 30, a_stride=2 ** 33)),
])
def test_calls_that_one_launch_does_not_take_are_refused_before_any(name, good, change):
    """gridDim.x * blockDim.x stays below 2^32; without a GPU, a call that gets as far as a launch says something else."""
    assert set(change) <= set(good)
    msg = refused(name, *{**good, **change}.values())
    assert "more than one launch takes" in msg or "n_tok" in msg and str(TOKENS) in msg, msg
