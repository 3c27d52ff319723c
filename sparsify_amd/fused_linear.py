"""A dense layer in one pass, ``act(x W^T + b) + residual``, with a backward that can run from 8-bit checkpoints.

The dense counterpart of ``fused_encoder``: the skip connection of a transcoder (sparse_coder.py:219-222,
``sae_out += x @ W_skip.mT``) is ``fused_linear(x, W_skip, residual=sae_out)``, which a SparseCoder with ``checkpoint``
calls (without it, its SkipProduct)."""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops, parallel
from .checkpoint8 import Checkpoint8, as_rows
from .fused_encoder import _autocast_bf16


def _operands(input: Tensor, weight: Tensor):
    """(x rows, weight) in the dtype the product runs in: bf16 under bf16 autocast or when both are bf16, else fp32."""
    parallel.wait_for(weight)                      # an overlapped optimizer update (sign_sgd.py)
    x = as_rows(input)
    if x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16:
        return x, as_rows(weight)
    for t, name in ((input, "input"), (weight, "weight")):
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}: sparsify_amd runs on the MI355X HIP path only (no CPU fallback)")
        ops._dt(t)
    if _autocast_bf16():
        if x.dtype != torch.bfloat16:
            x = ops.center_cast(x.contiguous(), None, False, True)[1] if x.numel() else x.bfloat16()
        # cast by every call, on its stream and inside its graph (4096 x 4096: 64 MiB read): a copy kept between calls would
        # be the old weight in the replays of a graph
        return x, as_rows(weight) if weight.dtype == torch.bfloat16 else ops.cast_bf16(weight.detach().contiguous())
    if weight.dtype != torch.float32:
        raise TypeError(f"fused_linear: weight is {weight.dtype} and input {input.dtype}; bf16 products need both in bf16 "
                        "or bf16 autocast")
    if x.dtype != torch.float32:
        x = ops.center_cast(x.contiguous(), None, True, False)[0] if x.numel() else x.float()
    return x, as_rows(weight)


class FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation: str, checkpoint):
        x, w = _operands(input, weight)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        made = checkpoint if isinstance(checkpoint, Checkpoint8) else None
        fmt = made.fmt if made is not None else checkpoint
        keep_z = None
        if activation != "none" and (need_x or need_w or need_b):
            keep_z = x.dtype if fmt is None else fmt
        y, z, codes = ops.linear(x, w, None if bias is None else bias.contiguous(),
                                 None if residual is None else as_rows(residual), activation, keep_z=keep_z,
                                 keep_x=fmt if need_w and made is None else None)
        kept_x = None
        if need_w:
            kept_x = x if fmt is None else codes if made is None else made.data
        # dx reads the weight the product ran with; dW and db only its shape
        ctx.save_for_backward(w if need_x and w.dtype != weight.dtype else weight, kept_x, z)
        ctx.fmt, ctx.activation, ctx.compute, ctx.w_dtype = fmt, activation, x.dtype, weight.dtype
        ctx.like = (input.shape, input.dtype, None if bias is None else bias.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return y if input.ndim == 2 else y.reshape(*input.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if g is None:
            return None, None, None, None, None, None
        weight, x, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        in_shape, in_dtype, b_dtype, r_dtype = ctx.like
        dx = dW = db = None
        if need_x or need_w or need_b:
            dx, dW, db = ops.linear_backward(as_rows(g), as_rows(weight), z, x, ctx.activation, z_fmt=ctx.fmt, x_fmt=ctx.fmt,
                                             dx_dtype=in_dtype if need_x else None, dw_dtype=ctx.w_dtype if need_w else None,
                                             db_dtype=b_dtype if need_b else None, dtype=ctx.compute)
            if need_x and len(in_shape) != 2:
                dx = dx.reshape(in_shape)
        dr = None
        if need_r:
            dr = g if g.dtype == r_dtype else g.to(r_dtype)
        return dx, dW, db, dr, None, None


def fused_linear(input: Tensor, weight: Tensor, bias: Tensor | None = None, *, residual: Tensor | None = None,
                 activation: str = "none", checkpoint: str | Checkpoint8 | None = None) -> Tensor:
    """act(input @ weight.T + bias) + residual, with one rounding at the end.

    input (..., D), weight (M, D), bias (M), residual (..., M); fp32 or bf16. The product runs in bf16 (fp32 sums) under
    bf16 autocast or when input and weight are bf16, else in exact fp32; the result has the wider dtype of the product
    and the residual. activation: "none", "relu", "gelu" (exact) or "silu". Under autocast an fp32 weight is cast in every
    call (4096 x 4096: 13 us); hold it in bf16 where it does not change.

    Gradients: dz = grad act'(z) in fp32, rounded once to the product's dtype (a bf16 product: to bf16, also where the
    result and its gradient are fp32); from it the input's and the weight's with fp32 sums, while the bias's sums dz
    unrounded. The residual's is grad itself.

    checkpoint: what the backward keeps of the input and of the activation's argument. None: as they are in the
    product's dtype. "int8" / "e4m3": 8-bit checkpoints (checkpoint8.py); gradients are those at the restored values. The
    backward reads z's codes as they are and, for the weight's gradient, restores the input's into scratch of the input's
    size in the product's dtype. A Checkpoint8 of this very input (already made for another layer that reads it) is kept
    instead of a second one."""
    ops._act(activation)
    in_shape, w_shape = input.shape, weight.shape
    if len(w_shape) != 2 or not in_shape or in_shape[-1] != w_shape[1] or 0 in w_shape:
        raise ValueError(f"fused_linear: input {tuple(in_shape)} does not go with weight {tuple(w_shape)}")
    M = w_shape[0]
    out_shape = (*in_shape[:-1], M)
    if bias is not None and bias.shape != (M,):
        raise ValueError(f"fused_linear: bias must be ({M},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != out_shape:
        raise ValueError(f"fused_linear: residual must be {out_shape}, got {tuple(residual.shape)}")
    if isinstance(checkpoint, Checkpoint8):
        if checkpoint.shape != input.shape or checkpoint.device != input.device:
            raise ValueError(f"fused_linear: the checkpoint holds {tuple(checkpoint.shape)} on {checkpoint.device}, "
                             f"input is {tuple(input.shape)} on {input.device}")
    elif checkpoint is not None:
        ops._code(checkpoint)
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return FusedLinear.apply(input, weight, bias, residual, activation, checkpoint)
    if forward_ad._current_level >= 0 or torch.jit.is_tracing():
        # the Function refuses an input with a tangent (there is no forward-mode derivative) and is what a trace records: the
        # kernels' launches are in neither's sight
        return FusedLinear.apply(input, weight, bias, residual, activation, checkpoint)
    x, w = _operands(input, weight)
    y = ops.linear(x, w, None if bias is None else bias.contiguous(), None if residual is None else as_rows(residual),
                   activation)[0]
    return y if len(out_shape) == 2 else y.reshape(out_shape)
