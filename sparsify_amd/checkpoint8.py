"""8-bit checkpoints: what a backward pass keeps of an activation, in half (bf16) or a quarter (fp32) of its bytes.

32 consecutive tokens of one feature share a power-of-two scale: the large values of a residual stream sit in a few
features at nearly all tokens, so a group holds values of one size. ``"int8"`` rounds to 255 even steps (at most 1/127 of
the group's largest value off), ``"e4m3"`` to 8-bit floats with 4 exponent bits (at most 2^-4 of each value off, or half the
smallest code's step). Both hold above the smallest scale, 2^-126 or 2^-117; the last step below 2^128 rounds down (1/64 off in
int8). Values times scales are exact in bf16 and fp32. A group that holds an infinity or a NaN restores as NaN."""
from __future__ import annotations

import torch
from torch import Tensor

from . import ops


class Checkpoint8:
    """An activation held in 8 bits: ``checkpoint8(x, fmt)``, read back by ``restore()`` or by the gradients of
    ``fused_linear(..., checkpoint=...)`` and ``fused_encoder(..., kept=...)``, which restore it for as long as they run.

    data: the buffer ops.checkpoint8_save writes; fmt: "int8" / "e4m3"; shape, dtype: of what was saved."""

    __slots__ = ("data", "fmt", "shape", "dtype")

    def __init__(self, data: Tensor, fmt: str, shape: torch.Size, dtype: torch.dtype):
        self.data, self.fmt, self.shape, self.dtype = data, fmt, torch.Size(shape), dtype

    @property
    def columns(self) -> int:
        return self.shape[-1]

    @property
    def rows(self) -> int:
        return self.shape[:-1].numel()

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def restore(self, dtype: torch.dtype | None = None) -> Tensor:
        """The values the codes stand for, in the dtype of what was saved or another one (exact in fp32 and bf16). New
        values: no gradient leads from them to what was saved."""
        _not_in_a_trace()
        out = ops.checkpoint8_restore(self.data, self.fmt, self.rows, self.columns, self.dtype if dtype is None else dtype)
        return out if len(self.shape) == 2 else out.reshape(self.shape)


def checkpoint8(x: Tensor, fmt: str = "int8", *, keep_sign: bool = False) -> Checkpoint8:
    """x (..., D), fp32 or bf16, in 8 bits; the leading dims are the tokens, groups of 32 in their order.
    fmt: "int8" or "e4m3". keep_sign: a value other than zero never becomes zero (a ReLU's mask survives)."""
    _not_in_a_trace()
    if x.ndim < 1:
        raise ValueError("checkpoint8: expected (..., D), got a scalar")
    return Checkpoint8(ops.checkpoint8_save(as_rows(x), fmt, keep_sign), fmt, x.shape, x.dtype)


def _not_in_a_trace() -> None:
    if torch.jit.is_tracing():
        raise RuntimeError("8-bit checkpoints cannot be traced: the trace would hold the codes of this input, or memory that "
                           "nothing fills")


def as_rows(t: Tensor) -> Tensor:
    """(..., D) as (tokens, D) with columns next to each other: t itself or a view where the strides allow one. For kernels,
    which read addresses: no autograd history is wanted of it."""
    if t.ndim != 2:
        t = t.detach().reshape(t.shape[:-1].numel(), t.shape[-1])
    return t if ops.is_rows(t) else t.detach().contiguous()
