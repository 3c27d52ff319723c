"""A dense layer in one pass, ``act(x W^T + b) + residual``, with a backward that can run from 8-bit checkpoints.

The dense counterpart of ``fused_encoder``: the skip connection of a transcoder (sparse_coder.py:219-222,
``sae_out += x @ W_skip.mT``) is ``fused_linear(x, W_skip, residual=sae_out)``."""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import ops, parallel
from .checkpoint8 import Checkpoint8, as_rows, checkpoint8
from .fused_encoder import _autocast_bf16, bf16_shadow


def _prepare(input: Tensor, weight: Tensor):
    """(x rows, weight) in the dtype the product runs in: bf16 under bf16 autocast or when both are bf16, else fp32."""
    for t, name in ((input, "input"), (weight, "weight")):
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}: sparsify_amd runs on the MI355X HIP path only (no CPU fallback)")
        ops._dt(t)
    x2 = as_rows(input)
    if _autocast_bf16() or (input.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16):
        if x2.dtype != torch.bfloat16:
            x2 = ops.center_cast(x2.contiguous(), None, False, True)[1] if x2.numel() else x2.bfloat16()
        return x2, as_rows(bf16_shadow(weight))
    if weight.dtype != torch.float32:
        raise TypeError(f"fused_linear: weight is {weight.dtype} and input {input.dtype}; bf16 products need both in bf16 "
                        "or bf16 autocast")
    if x2.dtype != torch.float32:
        x2 = ops.center_cast(x2.contiguous(), None, True, False)[0] if x2.numel() else x2.float()
    return x2, as_rows(weight)


def _check(input: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str) -> None:
    ops._act(activation)
    if weight.ndim != 2 or input.ndim < 1 or input.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"fused_linear: input {tuple(input.shape)} does not go with weight {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"fused_linear: bias must be ({weight.shape[0]},), got {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != (*input.shape[:-1], weight.shape[0]):
        raise ValueError(f"fused_linear: residual must be {(*input.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")


class FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation: str, checkpoint):
        parallel.wait_for(weight)                  # an overlapped optimizer update (sign_sgd.py)
        x, w = _prepare(input.detach(), weight)
        lead, M = input.shape[:-1], weight.shape[0]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        fmt = checkpoint.fmt if isinstance(checkpoint, Checkpoint8) else checkpoint
        keep_z = activation != "none" and (need_x or need_w or need_b)
        # z on its way into 8 bits is kept in fp32: one rounding
        z_dtype = None if not keep_z else torch.float32 if fmt is not None else x.dtype
        b = None if bias is None else bias.detach().contiguous()
        r = None if residual is None else as_rows(residual.detach())
        y, z = ops.linear(x, w.detach(), b, r, activation, z_dtype=z_dtype)
        kept_x, kept_z = (), ()
        ctx.x_codes = ctx.z_codes = None
        if need_w:
            if fmt is None:
                kept_x = (x,)
            else:
                c = checkpoint if isinstance(checkpoint, Checkpoint8) else checkpoint8(x, fmt)
                kept_x, ctx.x_codes = (c.codes, c.scales), (fmt, c.shape, c.dtype)
        if keep_z:
            if fmt is None:
                kept_z = (z,)
            else:
                c = checkpoint8(z, fmt, keep_sign=activation == "relu")
                kept_z, ctx.z_codes = (c.codes, c.scales), (fmt, c.shape, c.dtype)
        ctx.save_for_backward(weight, *kept_x, *kept_z)
        ctx.kept = (len(kept_x), len(kept_z))
        ctx.activation, ctx.compute, ctx.in_shape, ctx.in_dtype = activation, x.dtype, input.shape, input.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.res_dtype = None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return y.reshape(*lead, M)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if g is None:
            return None, None, None, None, None, None
        weight, *kept = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        nx, nz = ctx.kept

        def unpack(tensors, codes):
            if not tensors:
                return None
            return tensors[0] if codes is None else Checkpoint8(*tensors, *codes)

        x, z = unpack(kept[:nx], ctx.x_codes), unpack(kept[nx:], ctx.z_codes)
        g2 = as_rows(g)
        dx = dW = dz = db = None
        products = need_x or need_w
        if products and ctx.activation == "none" and g2.dtype == ctx.compute:
            dz = g2                                # the gradient is dz already: only its sums are left to take
            db = ops.linear_grad_preact(g2, None, "none", None, ctx.bias_dtype)[1] if need_b else None
        elif products or need_b:
            dz, db = ops.linear_grad_preact(g2, z, ctx.activation, ctx.compute if products else None,
                                            ctx.bias_dtype if need_b else None)
        if need_x:
            w = as_rows(bf16_shadow(weight).detach() if ctx.compute == torch.bfloat16 else weight.detach())
            dx = ops.linear_grad_input(dz, w, ctx.in_dtype).reshape(ctx.in_shape)
        if need_w:
            dW = ops.linear_grad_weight(dz, x, weight.dtype)
        dr = None
        if need_r:
            dr = g if g.dtype == ctx.res_dtype else g.to(ctx.res_dtype)
        return dx, dW, db, dr, None, None


def fused_linear(input: Tensor, weight: Tensor, bias: Tensor | None = None, *, residual: Tensor | None = None,
                 activation: str = "none", checkpoint: str | Checkpoint8 | None = None) -> Tensor:
    """act(input @ weight.T + bias) + residual, with one rounding at the end.

    input (..., D), weight (M, D), bias (M), residual (..., M); fp32 or bf16. The product runs in bf16 (fp32 sums) under
    bf16 autocast or when input and weight are bf16, else in exact fp32; the result has the wider dtype of the product
    and the residual. activation: "none", "relu", "gelu" (exact) or "silu".

    checkpoint: what the backward keeps of the input and of the activation's argument. None: as they are in the
    product's dtype. "int8" / "e4m3": 8-bit checkpoints (checkpoint8.py); the weight's gradient then reads the codes, and
    gradients are those at the restored values. A Checkpoint8 of this very input (already made for another layer that
    reads it) is kept instead of a second one."""
    _check(input, weight, bias, residual, activation)
    if isinstance(checkpoint, Checkpoint8):
        if checkpoint.shape != input.shape or checkpoint.device != input.device:
            raise ValueError(f"fused_linear: the checkpoint holds {tuple(checkpoint.shape)} on {checkpoint.device}, "
                             f"input is {tuple(input.shape)} on {input.device}")
    elif checkpoint is not None:
        ops._code(checkpoint)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in (input, weight, bias, residual)):
        parallel.wait_for(weight)
        x, w = _prepare(input.detach(), weight)
        b = None if bias is None else bias.detach().contiguous()
        r = None if residual is None else as_rows(residual.detach())
        return ops.linear(x, w.detach(), b, r, activation)[0].reshape(*input.shape[:-1], weight.shape[0])
    return FusedLinear.apply(input, weight, bias, residual, activation, checkpoint)
