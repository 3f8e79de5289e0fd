"""Layers of unquantised experts and adapters in training: the operators of `ops` with their gradients under autograd.

    logits (linear) -> ids and weights (route) -> rows by expert, gate and up, silu(g) * u, down (switch_glu)
    -> weighted sum onto the residual (combine);   moe_layer is all of them

and back, each product and each gradient one launch of libmoe_offload.so, or a few.  What switch_glu's forward pass keeps
is the row plan, (g, u) and h.  clip_grad_norm limits the gradients' norm before the optimizer's step.

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


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, bias, n_group, topk_group, group_best, renorm, scale):
        ids, weights = ops.route(logits, k, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_best=group_best,
                                 renorm=renorm, scale=scale)
        ctx.save_for_backward(logits, ids)
        ctx.rule = {"score": score, "renorm": renorm, "scale": scale}
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dweights):
        _refuse_capture("route")
        logits, ids = ctx.saved_tensors
        return (ops.route_grad(dweights.contiguous(), logits, ids, **ctx.rule),) + (None,) * 8


def route(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0):
    """ops.route, its weights differentiable in the logits.  The bias, which only the choice sees, has no gradient."""
    if bias is not None and bias.requires_grad:
        raise ValueError("route: the bias has no gradient here")
    _refuse_capture("route")
    return _Route.apply(logits, k, score, bias, n_group, topk_group, group_best, renorm, scale)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual):
        ctx.save_for_backward(y, weights)
        return ops.combine(y, weights, residual=residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _refuse_capture("combine")
        y, weights = ctx.saved_tensors
        dy = dweights = None
        if any(ctx.needs_input_grad[:2]):
            dy, dweights = ops.combine_grad(_operand(dout), y, weights)
        return dy, dweights, dout if ctx.needs_input_grad[2] else None


def combine(y, weights, residual=None):
    """ops.combine, differentiable in y, weights and residual."""
    _refuse_capture("combine")
    return _Combine.apply(y, weights, residual)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, act, residual, dtype, training):
        z = None
        if training and act is not None and any(ctx.needs_input_grad[:3]):
            z = torch.empty((x.shape[0], w.shape[0]), dtype=x.dtype, device=x.device)
        ctx.save_for_backward(x, w, z)
        ctx.act = act
        return ops.linear(x, w, bias=bias, act=act, residual=residual, z_out=z, dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("linear")
        x, w, z = ctx.saved_tensors
        want_dx, want_dw, want_db, _, want_dr, _, _ = ctx.needs_input_grad
        dx = dw = db = None
        if want_dx or want_dw or want_db:
            dx, dw, db = ops.linear_grad(_operand(dy), x, w, z=z, act=ctx.act, bias=want_db, want_dx=want_dx, want_dw=want_dw)
        return dx, dw, db, None, dy.to(x.dtype) if want_dr else None, None, None


def linear(x, w, bias=None, act=None, residual=None, dtype=None):
    """ops.linear, differentiable in x, w, bias and residual; with an activation the pre-activations are kept in the
    inputs' type for the backward pass."""
    _refuse_capture("linear")
    return _Linear.apply(x, w, bias, act, residual, dtype, torch.is_grad_enabled())


def moe_layer(x, w_router, w_gate_up, w_down, k, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True,
              scale=1.0, residual=None):
    """A layer of unquantised experts from its tokens to its output, [n_tok, hidden], differentiable in x, the three weights
    and the residual: the router's logits in fp32, each token's k experts (the arguments of ops.route), their SwitchGLU, the
    weighted sum plus the residual.

    x: fp16 or bf16 [n_tok, hidden]; w_router: same type [n_exp, hidden], n_exp a multiple of 8; w_gate_up, w_down as
    switch_glu.
    """
    if w_router.dim() != 2 or w_gate_up.dim() != 3 or w_router.shape[0] != w_gate_up.shape[0]:
        raise ValueError(f"moe_layer: w_router {tuple(w_router.shape)} and w_gate_up {tuple(w_gate_up.shape)} do not fit")
    logits = linear(x, w_router, dtype=torch.float32)
    ids, weights = route(logits, k, score, bias, n_group, topk_group, group_best, renorm, scale)
    return combine(switch_glu(x, ids, w_gate_up, w_down), weights, residual)


def clip_grad_norm(parameters, max_norm):
    """ops.clip_grad_norm of the parameters' gradients, in place (those without one are left out; 0 if all are); returns the norm
    before."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=parameters[0].device if parameters else None)
    return ops.clip_grad_norm(grads, max_norm)
