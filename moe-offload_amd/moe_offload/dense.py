"""Unquantised experts and adapters in training: the operators of `ops` with their gradients under autograd.

    plan rows by expert -> gate and up projections, silu(g) * u -> down projections, one row per (token, k)

and back, each product and each gradient one launch of libmoe_offload.so.  What the forward pass keeps is the
row plan, (g, u) and h.  The score-weighted sum over a token's experts is the caller's, in torch operations, and
so is the scores' gradient (ops.pair_combine has none, and takes fp16 rows only).

A graph capture of a forward or backward pass through autograd is refused: an eager graph of the same leaves
that is still alive would end the process.  Programs that capture call ops.grouped_* and ops.lora_* themselves.
"""
from __future__ import annotations

import torch

from . import ops


def _refuse_capture(who: str) -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{who}: autograd is not captured into a graph; call the operators in moe_offload.ops")


def _operand(t: torch.Tensor) -> torch.Tensor:
    """A gradient as the operators take it: autograd may hand down a view that starts anywhere."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _SwitchGlu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, w_gate_up, w_down):
        n_tok, k = ids.shape
        row_token, row_out, seg_start = ops.expert_plan(ids, w_gate_up.shape[0])
        gu = torch.empty((n_tok * k, w_gate_up.shape[1]), dtype=x.dtype, device=x.device)
        h = ops.grouped_gate_up(x, row_token, seg_start, w_gate_up, gu_out=gu)
        y = ops.grouped_mm(h, seg_start, w_down, row_out=row_out)
        ctx.save_for_backward(x, w_gate_up, w_down, row_token, row_out, seg_start, gu, h)
        return y.view(n_tok, k, w_down.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("switch_glu")
        x, w_gate_up, w_down, row_token, row_out, seg_start, gu, h = ctx.saved_tensors
        n_tok, k, hidden = dy.shape
        dy = _operand(dy.reshape(n_tok * k, hidden))
        dx = dw_gate_up = dw_down = None
        if ctx.needs_input_grad[3]:
            dw_down = ops.grouped_mm_dw(dy, h, seg_start, row_dy=row_out)
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[2]:
            dgu = ops.grouped_mm_dx(dy, seg_start, w_down, row_in=row_out, gu=gu)
            if ctx.needs_input_grad[2]:
                dw_gate_up = ops.grouped_mm_dw(dgu, x, seg_start, row_x=row_token)
            if ctx.needs_input_grad[0]:
                # a row per (token, k), rounded to the inputs' type as every operator's result is; their sum is fp32
                rows = ops.grouped_mm_dx(dgu, seg_start, w_gate_up, row_out=row_out)
                dx = rows.view(n_tok, k, x.shape[1]).sum(1, dtype=torch.float32).to(x.dtype)
        return dx, None, dw_gate_up, dw_down


def switch_glu(x: torch.Tensor, ids: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """Per-(token, k) SwitchGLU outputs [n_tok, k, hidden] of unquantised experts, differentiable in x and the weights.

    x: fp16 or bf16 [n_tok, hidden]; ids: int32 [n_tok, k] (an id outside the experts gives a row of zeros and
    no gradient); w_gate_up: [n_exp, 2 * inter, hidden], gate rows before up rows; w_down: [n_exp, hidden, inter].
    """
    if ids.dim() != 2 or x.dim() != 2 or ids.shape[0] != x.shape[0]:
        raise ValueError(f"switch_glu: ids {tuple(ids.shape)} and x {tuple(x.shape)} must be [n_tok, k] and [n_tok, hidden]")
    if (w_gate_up.dim() != 3 or w_down.dim() != 3 or w_gate_up.shape[0] != w_down.shape[0]
            or w_gate_up.shape[1] != 2 * w_down.shape[2] or w_gate_up.shape[2] != x.shape[1]):
        raise ValueError(f"switch_glu: w_gate_up {tuple(w_gate_up.shape)} and w_down {tuple(w_down.shape)} do not fit")
    _refuse_capture("switch_glu")
    return _SwitchGlu.apply(x, ids, w_gate_up, w_down)


class _LoraAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, a, b, ids, scale):
        ctx.save_for_backward(x, a, b, ids, scale)
        return ops.lora_add(base, x, a, b, ids, scale=scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("lora_add")
        x, a, b, ids, scale = ctx.saved_tensors
        dx = da = db = None
        if a.shape[0] == 0:
            dx, da, db = torch.zeros_like(x), torch.empty_like(a), torch.empty_like(b)
        elif any(ctx.needs_input_grad[1:4]):
            dx, da, db = ops.lora_grad(_operand(dy), x, a, b, ids, scale=scale)
        return dy, dx, da, db, None, None


def lora_add(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
             scale: torch.Tensor | None = None) -> torch.Tensor:
    """ops.lora_add, differentiable in base, x, a and b (the scale is a constant); at most 1024 adapters where a gradient
    in x, a or b is wanted."""
    if scale is not None and scale.requires_grad:
        raise ValueError("lora_add: scale has no gradient here")
    if a.dim() == 3 and a.shape[0] > 1024 and torch.is_grad_enabled() and any(t.requires_grad for t in (x, a, b)):
        raise ValueError(f"lora_add: {a.shape[0]} adapters (gradients for up to 1024)")
    _refuse_capture("lora_add")
    return _LoraAdd.apply(base, x, a, b, ids, scale)
