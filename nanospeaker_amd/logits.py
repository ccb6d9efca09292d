"""
Between the head's logits and the choice of a token: penalties for repeated tokens, a bias and
a grammar mask, in one pass of the library's kernel (nsmoe_penalize_logits).  Forward only.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _native as nat
from .moe_kernel import _DT, call_on


def _vector(name: str, t: Optional[Tensor], n: int, dtype, device) -> int:
    """The address of a [n] operand, 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"penalize_logits: {name} must be a contiguous {dtype} [{n}] on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(name: str, t: Tensor, b: int, n: int, dtype, device) -> "tuple[int, int]":
    """(address, row stride) of a [b, n] operand, or of one row [n] or [1, n] for all."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if (t.dtype is not dtype or t.dim() != 2 or t.shape[0] not in (1, b) or t.shape[1] != n
            or t.device != device or (t.stride(1) != 1 and n > 1)):
        raise ValueError(f"penalize_logits: {name} must be {dtype} [{b}, {n}] or [{n}] on {device} "
                         f"with contiguous rows, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr(), t.stride(0) if t.shape[0] == b and b > 1 else 0


def penalize_logits(logits: Tensor, history: Optional[Tensor] = None,
                    lens: Optional[Tensor] = None, *, prompt_lens: Optional[Tensor] = None,
                    repetition: Optional[Tensor] = None, frequency: Optional[Tensor] = None,
                    presence: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                    mask: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """
    The logits [batch, vocab] (bf16, fp16 or fp32) with, in this order,

      * `repetition` [batch] fp32: tokens of the row's history divided by it where positive and
        multiplied by it where negative (1: no change; it must be positive);
      * `frequency` and `presence` [batch] fp32: frequency times the token's count and, where
        the count is not 0, presence subtracted; counted over the history after its first
        `prompt_lens` [batch] int32 tokens (all of it without);
      * `bias` fp32 [batch, vocab] or [vocab] added;
      * `mask` int32 [batch, ceil(vocab / 32)] or [ceil(vocab / 32)]: -inf where bit v % 32 of
        word v / 32 is 0, whatever the logit was.  A row that allows nothing is all -inf.

    history: int64 [batch, n], of which row b holds lens[b] (int32; n without) tokens; ids
    outside the vocabulary count nothing, so -1 may pad.  Computed in fp32 and rounded once, to
    the logits' type or to that of `out` (that type or fp32; logits itself writes in place).
    """
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DT:
        raise ValueError("penalize_logits: logits must be a bf16, fp16 or fp32 [batch, vocab] GPU "
                         f"tensor, got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    if torch.is_grad_enabled() and (logits.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise ValueError("penalize_logits: forward only, and logits or out requires a gradient "
                         "(call it under torch.no_grad, or detach)")
    b, v = logits.shape
    dev = logits.device
    given = out
    if v > 1 and logits.stride(1) != 1:
        raise ValueError("penalize_logits: the rows of logits must be contiguous")
    if out is None:
        out = logits.new_empty((b, v))
    elif (out.shape != (b, v) or out.device != dev or out.dtype not in (logits.dtype, torch.float32)
          or (v > 1 and out.stride(1) != 1) or (b > 1 and out.stride(0) < v)):
        raise ValueError(f"penalize_logits: out must be [{b}, {v}] with contiguous rows of the "
                         f"logits' type or fp32 on {dev}, got {out.dtype} {tuple(out.shape)}")
    elif out is not logits and out.numel() and _overlap(out, logits) and not (
            out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype
            and (b == 1 or out.stride(0) == logits.stride(0))):
        raise ValueError("penalize_logits: out overlaps logits without being them")
    n = hist = hist_s = 0
    if history is None:
        if any(t is not None for t in (repetition, frequency, presence, lens, prompt_lens)):
            raise ValueError("penalize_logits: penalties and lengths need a history")
    else:
        if history.dim() != 2:
            raise ValueError(f"penalize_logits: history {tuple(history.shape)}, expected [{b}, n]")
        n = history.shape[1]
        if history.shape[0] != b:
            raise ValueError(f"penalize_logits: history of {history.shape[0]} rows for {b}")
        hist, hist_s = _rows("history", history, b, n, torch.int64, dev)
    i32, f32 = torch.int32, torch.float32
    a = nat.logits_args(
        _DT[logits.dtype], _DT[out.dtype], b, v, 0, logits.data_ptr(), out.data_ptr(),
        logits.stride(0), out.stride(0), hist, hist_s, n, _vector("lens", lens, b, i32, dev),
        _vector("prompt_lens", prompt_lens, b, i32, dev),
        _vector("repetition", repetition, b, f32, dev),
        _vector("frequency", frequency, b, f32, dev), _vector("presence", presence, b, f32, dev),
        *((0, 0) if bias is None else _rows("bias", bias, b, v, f32, dev)),
        *((0, 0) if mask is None else _rows("mask", mask, b, (v + 31) // 32, i32, dev)))
    nat.check(call_on(dev, nat.lib().nsmoe_penalize_logits, a), "nsmoe_penalize_logits")
    if given is not None:
        increment_version(given)
    return out


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether the address ranges of two 2-d tensors with contiguous rows meet."""
    def span(t):
        last = (t.shape[0] - 1) * t.stride(0) + t.shape[1]
        return t.data_ptr(), t.data_ptr() + last * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
