"""
Rotary positions as an operator (reference: src/model/rope.py), for heads that do not go
through the prefill's attention kernel: a decode step's, a training step's, another model's.

`rotary_embed` turns query and key heads in one launch of the library's kernel (nsmoe_rope):
planes of half the head apart ("rotate half", as `decoder.Rotary` pairs them) or of
neighbouring dims (`interleaved`), over the whole head or its first dims, at any positions,
with autograd.  `rotary_frequencies` gives the planes' frequencies, stretched for contexts
longer than a model was trained on when asked.

`decoder.Rotary` rounds each product of the rotation to the tensor's dtype, as the reference's
tensor ops do; `rotary_embed` computes in fp32 from fp64 angles and rounds once.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _native as nat
from .moe_kernel import _DT, call_on

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rot_dim: int, base: float = 10_000.0, scaling: "str | None" = None,
                       factor: float = 1.0, original_length: int = 4096,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> "tuple[Tensor, float]":
    """
    (freqs [rot_dim / 2] fp64 in radians per position, amplitude) for rotary_embed:
    base^(-2 j / rot_dim), stretched by `factor` as `scaling` says:

      * None: unchanged.
      * "linear": every frequency divided by the factor (position interpolation).
      * "ntk": the base raised to base * factor^(rot_dim / (rot_dim - 2)), which divides the
        slowest plane's frequency by the factor and leaves the fastest as it is.
      * "yarn" (Peng et al., 2023): a plane that makes fewer than `beta_slow` turns over
        `original_length` positions is divided by the factor, one that makes more than
        `beta_fast` is left, those between are blended linearly in their turns; the amplitude
        is 0.1 ln(factor) + 1 (1 otherwise).
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary_frequencies: rot_dim {rot_dim} must be even and at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling {scaling!r}, expected one of {SCALINGS}")
    if not (base > 0 and factor >= 1.0):
        raise ValueError(f"rotary_frequencies: base {base} must be positive, factor {factor} at "
                         "least 1")
    if scaling == "ntk":
        if rot_dim == 2:
            raise ValueError("rotary_frequencies: ntk needs rot_dim > 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    j = torch.arange(rot_dim // 2, dtype=torch.float64)
    freqs = base ** (-2.0 * j / rot_dim)
    amplitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if not (original_length > 0 and beta_fast > beta_slow):
            raise ValueError("rotary_frequencies: yarn needs original_length > 0 and beta_fast > "
                             "beta_slow")
        turns = original_length * freqs / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        freqs = keep * freqs + (1.0 - keep) * freqs / factor
        amplitude = 0.1 * math.log(factor) + 1.0
    return freqs.to(device), amplitude


def _writable(t: Tensor) -> bool:
    """Whether no two elements of t share memory (an in-place kernel's operand)."""
    dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
    reach = 1
    for s, n in dims:
        if s < reach:
            return False
        reach = s * n if s * n > reach else reach
    return True


def _meet(a: Tensor, b: Tensor) -> bool:
    """Whether the heads of two [batch, tokens, heads, dim] tensors share elements: column blocks
    of one row are told apart, other views of common memory count as sharing."""
    def span(t, dims):
        return sum((t.shape[i] - 1) * t.stride(i) for i in dims) * t.element_size()
    size = a.element_size()
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + span(a, range(4)) + size <= pb or pb + span(b, range(4)) + size <= pa:
        return False
    row_a, row_b = span(a, (2, 3)) + size, span(b, (2, 3)) + size
    far = min((t.stride(i) * size for t in (a, b) for i in (0, 1) if t.shape[i] > 1),
              default=None)
    apart = pb - pa if pb >= pa else pa - pb
    first = row_a if pb >= pa else row_b
    rest = row_b if pb >= pa else row_a
    same = all(a.stride(i) == b.stride(i) or a.shape[i] == 1 for i in (0, 1))
    return not (same and apart >= first and (far is None or apart + rest <= far))


_NO_STRIDES = (0, 0, 0)


def _launch(q: Optional[Tensor], k: Optional[Tensor], positions: Tensor, freqs: Tensor,
            interleaved: bool, amplitude: float, inverse: bool, inplace: bool):
    """The kernel over 4-d q and k (either may be None): their rotations."""
    some = k if q is None else q
    dev = some.device
    b, n, _, d = some.shape
    hq = hk = qp = kp = op = okp = 0
    sq = sk = soq = sok = _NO_STRIDES
    oq = ok = None
    if q is not None:
        if q.stride(3) != 1 and d > 1:
            q = q.contiguous()
        oq = q if inplace else q.new_empty(q.shape)
        hq, qp, op = q.shape[2], q.data_ptr(), oq.data_ptr()
        sq, soq = q.stride()[:3], oq.stride()[:3]
    if k is not None:
        if k.stride(3) != 1 and d > 1:
            k = k.contiguous()
        ok = k if inplace else k.new_empty(k.shape)
        hk, kp, okp = k.shape[2], k.data_ptr(), ok.data_ptr()
        sk, sok = k.stride()[:3], ok.stride()[:3]
    a = nat.rope_args(_DT[some.dtype], interleaved, inverse, amplitude, b, n, hq, hk, d,
                      2 * freqs.shape[0], qp, kp, op, okp, *sq, *sk, *soq, *sok,
                      positions.data_ptr(), *positions.stride(), freqs.data_ptr())
    nat.check(call_on(dev, nat.lib().nsmoe_rope, a), "nsmoe_rope")
    return oq, ok


class _Rotate(torch.autograd.Function):
    """The rotation; its gradient is the rotation the other way."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, interleaved, amplitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        ctx.how = (interleaved, amplitude, inverse)
        return _launch(q, k, positions, freqs, interleaved, amplitude, inverse, False)

    @staticmethod
    def backward(ctx, gq, gk):
        dq = dk = None
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is not None or gk is not None:
            interleaved, amplitude, inverse = ctx.how
            dq, dk = _Rotate.apply(gq, gk, *ctx.saved_tensors, interleaved, amplitude,
                                   not inverse)
        return dq, dk, None, None, None, None, None


def rotary_embed(q: Tensor, k: Optional[Tensor], positions: Tensor, freqs: Tensor, *,
                 interleaved: bool = False, amplitude: float = 1.0,
                 inplace: bool = False) -> "tuple[Tensor, Optional[Tensor]]":
    """
    q [batch, tokens, query heads, dim] and k [batch, tokens, key heads, dim] (or both without
    the batch; k may be None) with plane j of every head turned by positions * freqs[j].

    positions: int64, broadcastable to [batch, tokens]; freqs: fp64 [rot_dim / 2], rot_dim at
    most dim (rotary_frequencies); the dims from rot_dim on are left as they are.  Any strides
    with a contiguous last dim (column blocks of a fused projection are taken as they are);
    bf16, fp16 or fp32 GPU tensors; computed in fp32 and rounded once.  Differentiable in q and
    k.  `inplace` writes into q and k themselves (which must not share elements) and returns
    them; it is for calls that nothing differentiates.
    """
    if q.dim() not in (3, 4) or not q.is_cuda or q.dtype not in _DT:
        raise ValueError("rotary_embed: q must be a bf16, fp16 or fp32 [batch, tokens, heads, dim] "
                         "or [tokens, heads, dim] GPU tensor, got "
                         f"{q.dtype} {tuple(q.shape)} on {q.device}")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2]
                          or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype
                          or k.device != q.device):
        raise ValueError(f"rotary_embed: k {tuple(k.shape)} {k.dtype} does not go with q "
                         f"{tuple(q.shape)} {q.dtype}")
    flat = q.dim() == 3
    q4, k4 = q, k
    if flat:
        q4, k4 = q.unsqueeze(0), None if k is None else k.unsqueeze(0)
    b, n, _, d = q4.shape
    if positions.dtype is not torch.int64 or positions.device != q.device:
        raise ValueError(f"rotary_embed: positions must be int64 on {q.device}, got "
                         f"{positions.dtype} on {positions.device}")
    if positions.shape != (b, n):
        positions = positions.expand(b, n)
    if freqs.dtype is not torch.float64 or freqs.device != q.device or freqs.dim() != 1 or not (
            2 <= 2 * freqs.shape[0] <= d):
        raise ValueError(f"rotary_embed: freqs must be fp64 [rot_dim / 2] on {q.device}, rot_dim "
                         f"2 .. {d}; got {freqs.dtype} {tuple(freqs.shape)} on {freqs.device}")
    if freqs.stride(0) != 1:
        freqs = freqs.contiguous()
    amplitude = float(amplitude)
    grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    if inplace:
        if grad:
            raise ValueError("rotary_embed: inplace is for calls that nothing differentiates")
        for t in (q4, k4):
            if t is not None and t.numel() and (t.stride(3) != 1 or not _writable(t)):
                raise ValueError("rotary_embed: inplace needs a contiguous last dim and elements "
                                 "that share no memory")
        if k4 is not None and k4.numel() and q4.numel() and _meet(q4, k4):
            raise ValueError("rotary_embed: inplace with q and k that share elements")
        _launch(q4, k4, positions, freqs, interleaved, amplitude, False, True)
        increment_version(q if k is None else (q, k))
        return q, k
    if grad:
        yq, yk = _Rotate.apply(q4, k4, positions, freqs, interleaved, amplitude, False)
    else:
        yq, yk = _launch(q4, k4, positions, freqs, interleaved, amplitude, False, False)
    if flat:
        yq, yk = yq.squeeze(0), None if yk is None else yk.squeeze(0)
    return yq, yk
