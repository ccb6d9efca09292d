"""
Decoding against key/value caches: attention of a batch's new tokens over a prefix that all
its sequences share and over each sequence's own cache, and eviction from those caches by
accumulated attention weight (reference: the grouped-query attention of src/model/mha.py:245-287
with a cache; the reference decodes with one cache per sequence and evicts nothing).

Keys lie in the caches as attention multiplies them: normalised and rotated (`rotary_embed`,
or the prefill, whose key heads `decoder.attn_prefill` leaves that way in its projection).
Forward only.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import _native as nat
from .moe_kernel import _stream, _ws, on_device

_DT16 = {torch.bfloat16: nat.BF16, torch.float16: nat.F16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _lens(op: str, lens: Tensor, b: int, device) -> None:
    _need(lens.dtype == torch.int32 and lens.shape == (b,) and lens.device == device
          and lens.is_contiguous(),
          f"{op}: lens must be a contiguous int32 [{b}] on {device}, got {lens.dtype} "
          f"{tuple(lens.shape)} on {lens.device}")


def _wide(t: Tensor) -> bool:
    """Whether a 16-bit tensor's rows can be read 16 bytes at a time: a contiguous last dim,
    every other stride and the address a multiple of 16 bytes."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1))


def _strides(t: Tensor) -> "tuple[int, ...]":
    """The strides before the last dim, 0 where a dim has one element (any stride fits it)."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape))


def shared_prefix_attention(q: Tensor, k_prefix: Optional[Tensor], v_prefix: Optional[Tensor],
                            k: Tensor, v: Tensor, lens: Tensor, *, window: "int | None" = None,
                            scale: "float | None" = None, weights: Optional[Tensor] = None,
                            weights_out: Optional[Tensor] = None, return_lse: bool = False):
    """
    Attention of the last n tokens of each sequence, q [batch, n, query heads, dim], over the
    prefix k_prefix, v_prefix [prefix rows, key heads, dim] shared by the batch (None: no
    prefix) and the sequence's own cache k, v [batch, rows, key heads, dim], of which it has
    lens[b] (int32) rows, the n new ones last.  The prefix is read once for the whole batch.

    Query i stands at its own row lens[b] - n + i, behind the prefix, and sees every row before
    it and itself, or the last `window` of them.  A query without a row (lens[b] < n: a padded
    batch, an idle slot) gets zeros, and -inf as lse.  Rows from lens[b] on are never read.
    bf16 or fp16, dim 64 or 128, query heads a multiple of key heads; any strides of 16 bytes
    with a contiguous last dim.  scale: 1 / sqrt(dim) by default, positive.

    Returns out [batch, n, query heads, dim]; with `return_lse` or `weights` / `weights_out` a
    tuple of it, the log-sum-exp of each query's scores [batch, n, query heads] fp32 (if asked
    for), and the accumulated weights [batch, key heads, rows] fp32 (if given): `weights` plus
    the softmax weight that each cached row got from the new queries, summed over them and over
    the query heads of its key head -- what cache_evict evicts by.  They are written to
    `weights_out` if given (weights itself accumulates in place; alone, it starts from zero),
    and rows from lens[b] on keep theirs.  At most 64 queries (n times query heads per key
    head) with weights.
    """
    op = "shared_prefix_attention"
    _need(q.dim() == 4 and q.is_cuda and q.dtype in _DT16,
          f"{op}: q must be a bf16 or fp16 [batch, n, heads, dim] GPU tensor, got {q.dtype} "
          f"{tuple(q.shape)} on {q.device}")
    b, n, hq, d = q.shape
    dev = q.device
    _need(k.dim() == 4 and k.shape == v.shape and k.shape[0] == b and k.shape[3] == d
          and k.shape[2] >= 1 and hq % k.shape[2] == 0,
          f"{op}: k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
    s, hk = k.shape[1], k.shape[2]
    _need((k_prefix is None) == (v_prefix is None), f"{op}: k_prefix without v_prefix")
    caches = [k, v]
    p = 0
    if k_prefix is not None:
        _need(k_prefix.dim() == 3 and k_prefix.shape == v_prefix.shape
              and k_prefix.shape[1:] == (hk, d),
              f"{op}: prefix {tuple(k_prefix.shape)}, {tuple(v_prefix.shape)}, expected "
              f"[rows, {hk}, {d}]")
        p = k_prefix.shape[0]
        caches += [k_prefix, v_prefix]
    for t in caches:
        _need(t.dtype == q.dtype and t.device == dev, f"{op}: caches and q differ in type or "
              "device")
        _need(t.numel() == 0 or _wide(t), f"{op}: caches need a contiguous last dim, and strides "
              "and addresses that are multiples of 16 bytes")
    _lens(op, lens, b, dev)
    _need(window is None or window >= 1, f"{op}: window {window}")
    if not _wide(q):
        q = q.contiguous() if q.data_ptr() % 16 == 0 else q.clone(
            memory_format=torch.contiguous_format)
    out = torch.empty((b, n, hq, d), dtype=q.dtype, device=dev)
    lse = torch.empty((b, n, hq), dtype=torch.float32, device=dev) if return_lse else None
    if weights is not None or weights_out is not None:
        for name, t in (("weights", weights), ("weights_out", weights_out)):
            _need(t is None or (t.dtype == torch.float32 and t.shape == (b, hk, s)
                                and t.device == dev and t.is_contiguous()),
                  f"{op}: {name} must be a contiguous fp32 {(b, hk, s)} on {dev}")
        _need(n * (hq // hk) <= 64, f"{op}: weights for at most 64 queries per key head, got "
              f"{n * (hq // hk)}")
        if weights_out is None:
            weights_out = torch.empty_like(weights)
    a = nat.PrefixAttnArgs(
        dtype=_DT16[q.dtype], head_dim=d, n_heads=hq, n_kv_heads=hk, batch=b, n_new=n,
        prefix_len=p, cap=s, window=0 if window is None else min(int(window), (1 << 30) - 1),
        scale=1.0 / math.sqrt(d) if scale is None else float(scale),
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=_strides(q),
        k_stride=_strides(k), v_stride=_strides(v), lens=lens.data_ptr(), out=out.data_ptr(),
        lse=None if lse is None else lse.data_ptr(),
        weights=None if weights is None else weights.data_ptr(),
        weights_out=None if weights_out is None else weights_out.data_ptr())
    if p:
        a.k_prefix, a.v_prefix = k_prefix.data_ptr(), v_prefix.data_ptr()
        a.kp_stride, a.vp_stride = _strides(k_prefix), _strides(v_prefix)
    if b and n:
        lib = nat.lib()
        with on_device(dev):
            ws = _ws(lib.nsmoe_prefix_attention_workspace_size(a), dev)
            nat.check(lib.nsmoe_prefix_attention(a, ws.data_ptr(), ws.numel(),
                                                 _stream(dev.index)), "nsmoe_prefix_attention")
    elif weights_out is not None and weights_out is not weights:
        weights_out.zero_() if weights is None else weights_out.copy_(weights)
    if lse is None and weights_out is None:
        return out
    return tuple(t for t in (out, lse, weights_out) if t is not None)


def cache_evict(k: Tensor, v: Tensor, weights: Tensor, lens: Tensor, budget: int, *,
                recent: int = 0, sinks: int = 0, out: "tuple[Tensor, Tensor, Tensor] | None" = None):
    """
    The caches k, v [batch, rows, key heads, dim] cut down to `budget` rows a sequence.  Of a
    sequence with more (lens[b], int32), each key head keeps its first `sinks` rows, its last
    `recent` ones and the heaviest others by weights [batch, key heads, rows] fp32 (what
    shared_prefix_attention accumulated; ties keep the earlier row, a NaN counts as the
    heaviest); shorter sequences keep all.  Kept rows move to the front in their order.

    Returns (k, v, weights, index, lens): caches and weights of `budget` rows, zero behind the
    kept ones; index [batch, key heads, budget] int32, the row that each came from (-1 behind
    them); lens [batch] int32.  With `out` = (k, v, weights) of at least `budget` rows, apart
    from the inputs, those are written instead, and their rows behind the kept ones left alone.
    Any 2- or 4-byte type and strides with a contiguous last dim.
    """
    op = "cache_evict"
    _need(k.dim() == 4 and k.is_cuda and k.element_size() in (2, 4) and k.shape == v.shape
          and v.dtype == k.dtype and v.device == k.device,
          f"{op}: k and v must be [batch, rows, heads, dim] GPU tensors of one 2- or 4-byte type, "
          f"got {k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)} on {k.device}")
    b, s, hk, d = k.shape
    dev = k.device
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    _need(budget >= 1 and recent >= 0 and sinks >= 0 and recent + sinks <= budget,
          f"{op}: budget {budget} with {sinks} sinks and {recent} recent rows")
    _need(weights.shape == (b, hk, s) and weights.dtype == torch.float32 and weights.device == dev,
          f"{op}: weights must be fp32 {(b, hk, s)} on {dev}, got {weights.dtype} "
          f"{tuple(weights.shape)} on {weights.device}")
    _lens(op, lens, b, dev)
    if out is None:
        k_out = torch.empty((b, budget, hk, d), dtype=k.dtype, device=dev)
        v_out = torch.empty_like(k_out)
        w_out = torch.empty((b, hk, budget), dtype=torch.float32, device=dev)
    else:
        k_out, v_out, w_out = out
        rows = k_out.shape[1] if k_out.dim() == 4 else -1
        _need(rows >= budget and k_out.shape == v_out.shape == (b, rows, hk, d)
              and w_out.shape == (b, hk, rows) and k_out.dtype == v_out.dtype == k.dtype
              and w_out.dtype == torch.float32
              and k_out.device == v_out.device == w_out.device == dev,
              f"{op}: out must be k, v {(b, f'>= {budget}', hk, d)} and weights "
              f"{(b, hk, f'>= {budget}')} of the inputs' types")
        for t in out:
            for i in (k, v, weights):
                _need(not _share(t, i), f"{op}: out shares memory with the inputs")
    for t in (k, v, k_out, v_out, weights, w_out):
        _need(t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1,
              f"{op}: the last dim must be contiguous")
    index = torch.empty((b, hk, budget), dtype=torch.int32, device=dev)
    lens_out = torch.empty_like(lens)
    if b and hk and d:
        a = nat.EvictArgs(
            elem_bytes=k.element_size(), n_kv_heads=hk, head_dim=d, zero_tail=int(out is None),
            batch=b, cap=s, out_cap=k_out.shape[1], budget=budget, recent=recent, sinks=sinks,
            k=k.data_ptr(), v=v.data_ptr(), k_out=k_out.data_ptr(), v_out=v_out.data_ptr(),
            k_stride=_strides(k), v_stride=_strides(v), k_out_stride=_strides(k_out),
            v_out_stride=_strides(v_out), weights=weights.data_ptr(),
            weights_out=w_out.data_ptr(), weights_stride=_strides(weights),
            weights_out_stride=_strides(w_out), lens=lens.data_ptr(),
            lens_out=lens_out.data_ptr(), index=index.data_ptr())
        with on_device(dev):
            nat.check(nat.lib().nsmoe_cache_evict(a, _stream(dev.index)), "nsmoe_cache_evict")
    return k_out, v_out, w_out, index, lens_out


def _share(a: Tensor, b: Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if not (a.numel() and b.numel()):
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
