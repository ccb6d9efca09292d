"""
Decoding against key/value caches: attention of a batch's new tokens over a prefix that all
its sequences share and over each sequence's own cache, and eviction from those caches by
accumulated attention weight (reference: the grouped-query attention of src/model/mha.py:245-287
with a cache; the reference decodes with one cache per sequence and evicts nothing).

Keys lie in the caches as attention multiplies them: normalised and rotated (`rotary_embed`,
or the prefill, whose key heads `decoder.attn_prefill` leaves that way in its projection).
`DecodeCache` holds them for a decoder (`Decoder.prefix`, `Decoder.step`).  Forward only.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _native as nat
from .moe_kernel import call_on
from .rope import _writable

_DT16 = {torch.bfloat16: nat.BF16, torch.float16: nat.F16}


def _fail(op: str, what: str):
    raise ValueError(f"{op}: {what}")


def _forward_only(op: str, *tensors) -> None:
    if torch.is_grad_enabled() and True in [t is not None and t.requires_grad for t in tensors]:
        _fail(op, "forward only: an operand requires a gradient (call it under torch.no_grad, or "
                  "detach)")


def _lens(op: str, lens: Tensor, b: int, device) -> None:
    if (lens.dtype is not torch.int32 or lens.shape != (b,) or lens.device != device
            or not lens.is_contiguous()):
        _fail(op, f"lens must be a contiguous int32 [{b}] on {device}, got {lens.dtype} "
                  f"{tuple(lens.shape)} on {lens.device}")


def _strides(t: Tensor) -> "tuple[int, ...]":
    """The strides before the last dim, 0 where a dim has one element (any stride fits it)."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape))


def _rows16(t: Tensor) -> "Optional[tuple[int, ...]]":
    """The strides before the last dim of a 16-bit tensor whose rows can be read 16 bytes at a
    time (a contiguous last dim, every other stride and the address a multiple of 16 bytes);
    None of one whose rows cannot."""
    s = t.stride()[:-1]
    bits = 0
    for x in s:
        bits |= x
    if bits & 7:  # a stride of a dim of one element may be anything
        s = _strides(t)
        bits = 0
        for x in s:
            bits |= x
    if t.numel() == 0:
        return s
    return None if bits & 7 or t.stride(-1) != 1 or t.data_ptr() & 15 else s


def _attend(a, dev, stream: int) -> None:
    lib = nat.lib()
    size = lib.nsmoe_prefix_attention_workspace_size(a)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    nat.check(lib.nsmoe_prefix_attention(a, None if ws is None else ws.data_ptr(), size, stream),
              "nsmoe_prefix_attention")


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
    if q.dim() != 4 or not q.is_cuda or q.dtype not in _DT16:
        _fail(op, "q must be a bf16 or fp16 [batch, n, heads, dim] GPU tensor, got "
                  f"{q.dtype} {tuple(q.shape)} on {q.device}")
    b, n, hq, d = q.shape
    dev, dt = q.device, q.dtype
    if (k.dim() != 4 or k.shape != v.shape or k.shape[0] != b or k.shape[3] != d
            or k.shape[2] < 1 or hq % k.shape[2]):
        _fail(op, f"k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
    s, hk = k.shape[1], k.shape[2]
    if (k_prefix is None) != (v_prefix is None):
        _fail(op, "k_prefix without v_prefix, or v_prefix without k_prefix")
    p = kp = vp = bits = 0
    skp = svp = (0, 0, 1)
    if k_prefix is not None:
        if (k_prefix.dim() != 3 or k_prefix.shape != v_prefix.shape or k_prefix.shape[1] != hk
                or k_prefix.shape[2] != d):
            _fail(op, f"prefix {tuple(k_prefix.shape)}, {tuple(v_prefix.shape)}, expected [rows, "
                      f"{hk}, {d}]")
        if (k_prefix.dtype is not dt or v_prefix.dtype is not dt or k_prefix.device != dev
                or v_prefix.device != dev):
            _fail(op, f"the prefix has another type or device than q's {dt} on {dev}")
        p = k_prefix.shape[0]
        kp, vp = k_prefix.data_ptr(), v_prefix.data_ptr()
        skp, svp = k_prefix.stride(), v_prefix.stride()
        bits = (kp | vp) >> 1 | skp[0] | skp[1] | svp[0] | svp[1]
    if k.dtype is not dt or v.dtype is not dt or k.device != dev or v.device != dev:
        _fail(op, f"a cache has another type or device than q's {dt} on {dev}")
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    ka, va = k.data_ptr(), v.data_ptr()
    bits |= ((ka | va | q.data_ptr()) >> 1 | sk[0] | sk[1] | sk[2] | sv[0] | sv[1] | sv[2] | sq[0]
             | sq[1] | sq[2])
    if bits & 7 or not sq[3] == sk[3] == sv[3] == skp[2] == svp[2] == 1:
        # something is off 16 bytes, or only a stride that does not matter
        sk, sv = _rows16(k), _rows16(v)
        if p:
            skp, svp = _rows16(k_prefix), _rows16(v_prefix)
        if sk is None or sv is None or skp is None or svp is None:
            _fail(op, "caches need a contiguous last dim, and strides and addresses that are "
                      "multiples of 16 bytes")
        sq = _rows16(q)
        if sq is None:
            q = q.clone(memory_format=torch.contiguous_format)
            sq = q.stride()
    _lens(op, lens, b, dev)
    if torch.is_grad_enabled():
        _forward_only(op, q, k, v, k_prefix, v_prefix, weights, weights_out)
    if window is None:
        window = 0
    elif window < 1:
        _fail(op, f"window {window}")
    out = q.new_empty((b, n, hq, d))
    lse = q.new_empty((b, n, hq), dtype=torch.float32) if return_lse else None
    if weights is not None or weights_out is not None:
        for name, t in (("weights", weights), ("weights_out", weights_out)):
            if t is not None and (t.dtype is not torch.float32 or t.shape != (b, hk, s)
                                  or t.device != dev or not t.is_contiguous()):
                _fail(op, f"{name} must be a contiguous fp32 {(b, hk, s)} on {dev}")
        if n * (hq // hk) > 64:
            _fail(op, f"weights for at most 64 queries per key head, got {n * (hq // hk)}")
        if weights_out is None:
            weights_out = torch.empty_like(weights)
        elif weights is not None and weights_out.data_ptr() != weights.data_ptr() and _share(
                weights, weights_out):
            _fail(op, "weights_out overlaps weights without being them")
    if b and n:
        a = nat.prefix_attn_args(
            _DT16[dt], d, hq, hk, b, n, p, s, min(int(window), (1 << 30) - 1),
            1.0 / math.sqrt(d) if scale is None else float(scale), q.data_ptr(), kp, vp,
            ka, va, *sq[:3], *skp[:2], *svp[:2], *sk[:3], *sv[:3], lens.data_ptr(),
            out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            0 if weights is None else weights.data_ptr(),
            0 if weights_out is None else weights_out.data_ptr())
        call_on(dev, _attend, a, dev)
        if weights_out is not None:
            increment_version(weights_out)
    elif weights_out is not None and weights_out is not weights:
        weights_out.zero_() if weights is None else weights_out.copy_(weights)
    if lse is None and weights_out is None:
        return out
    return tuple(t for t in (out, lse, weights_out) if t is not None)


def cache_evict(k: Tensor, v: Tensor, weights: Tensor, lens: Tensor, budget: int, *,
                recent: int = 0, sinks: int = 0,
                out: "tuple[Tensor, Tensor, Tensor] | None" = None):
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
    if (k.dim() != 4 or not k.is_cuda or k.element_size() not in (2, 4) or k.shape != v.shape
            or v.dtype is not k.dtype or v.device != k.device):
        _fail(op, "k and v must be [batch, rows, heads, dim] GPU tensors of one 2- or 4-byte type, "
                  f"got {k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)} on {k.device}")
    b, s, hk, d = k.shape
    dev = k.device
    if hk < 1 or d < 1:
        _fail(op, f"caches {tuple(k.shape)} without heads or dims")
    _forward_only(op, k, v, weights, *(out or ()))
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        _fail(op, f"budget {budget} with {sinks} sinks and {recent} recent rows")
    if weights.shape != (b, hk, s) or weights.dtype is not torch.float32 or weights.device != dev:
        _fail(op, f"weights must be fp32 {(b, hk, s)} on {dev}, got {weights.dtype} "
                  f"{tuple(weights.shape)} on {weights.device}")
    _lens(op, lens, b, dev)
    rows = budget
    if out is None:
        k_out = k.new_empty((b, budget, hk, d))
        v_out = torch.empty_like(k_out)
        w_out = weights.new_empty((b, hk, budget))
    else:
        k_out, v_out, w_out = out
        rows = k_out.shape[1] if k_out.dim() == 4 else -1
        if (rows < budget or not k_out.shape == v_out.shape == (b, rows, hk, d)
                or w_out.shape != (b, hk, rows) or not k_out.dtype == v_out.dtype == k.dtype
                or w_out.dtype is not torch.float32
                or not k_out.device == v_out.device == w_out.device == dev):
            _fail(op, f"out must be k, v {(b, f'>= {budget}', hk, d)} and weights "
                      f"{(b, hk, f'>= {budget}')} of the inputs' types")
        for i, t in enumerate(out):
            if any(_share(t, o) for o in (k, v, weights, *out[:i])):
                _fail(op, "out shares memory with the inputs or with itself")
            if not _writable(t):
                _fail(op, "out has elements that share memory")
    for t in (k, v, weights) if out is None else (k, v, weights, *out):
        if t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel():
            _fail(op, "the last dim must be contiguous")
    index = torch.empty((b, hk, budget), dtype=torch.int32, device=dev)
    lens_out = torch.empty_like(lens)
    if b:
        a = nat.evict_args(
            k.element_size(), hk, d, out is None, b, s, rows, budget, recent, sinks,
            k.data_ptr(), v.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), *k.stride()[:3],
            *v.stride()[:3], *k_out.stride()[:3], *v_out.stride()[:3], weights.data_ptr(),
            w_out.data_ptr(), *weights.stride()[:2], *w_out.stride()[:2], lens.data_ptr(),
            lens_out.data_ptr(), index.data_ptr())
        nat.check(call_on(dev, nat.lib().nsmoe_cache_evict, a), "nsmoe_cache_evict")
        if out is not None:
            increment_version(out)
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


class DecodeCache:
    """
    What a decoder keeps of a batch of sequences behind one prefix: the prefix's keys and values
    of each layer once (prefix_kv, [P, key heads, dim]), each sequence's own (k, v [batch, rows,
    key heads, dim]) with each layer's lengths (lens int32 [batch]), the accumulated weights of
    the layers without a window (weights, or None), and the position of the next token
    (positions int64 [batch]).  Made by Decoder.prefix, filled by Decoder.step.

    `filled` bounds every length from above without asking the device; a step that would pass
    the cache's rows is refused.  So are steps under graph capture, whose replays this count
    would miss, and steps after one that raised part way, which left its rows in some layers.
    """

    def __init__(self, windows, prefix_kv, prefix_len: int, batch: int, rows: int, n_kv_heads: int,
                 dim: int, dtype, device, weights: bool = False):
        n = len(windows)
        if rows < 1 or batch < 1:
            raise ValueError(f"DecodeCache: {batch} sequences of {rows} rows")
        if prefix_len and len(prefix_kv) != n:
            raise ValueError(f"DecodeCache: prefix of {len(prefix_kv)} layers for {n}")
        self.windows, self.rows, self.batch, self.filled = list(windows), rows, batch, 0
        self._open = False  # a step has written rows and not come to its end
        self.prefix_kv = list(prefix_kv) if prefix_len else [(None, None)] * n
        shape = (batch, rows, n_kv_heads, dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n)]
        self.lens = [torch.zeros(batch, dtype=torch.int32, device=device) for _ in range(n)]
        self.weights = [torch.zeros((batch, n_kv_heads, rows), dtype=torch.float32, device=device)
                        if weights and w is None else None for w in windows]
        self.positions = torch.full((batch,), prefix_len, dtype=torch.int64, device=device)
        self._seq = torch.arange(batch, device=device)[:, None]

    def reserve(self, idx: Tensor) -> None:
        """Refuses a step of tokens idx [batch, n] that the cache cannot hold or count."""
        if idx.dim() != 2 or idx.shape[0] != self.batch or idx.shape[1] < 1:
            raise ValueError(f"DecodeCache: tokens {tuple(idx.shape)}, expected [{self.batch}, n]")
        if self.filled + idx.shape[1] > self.rows:
            raise ValueError(f"DecodeCache: {idx.shape[1]} tokens more than the {self.rows} rows "
                             f"hold ({self.filled} used)")
        if self._open:
            raise RuntimeError("DecodeCache: a step raised before its end and left its rows in "
                               "some layers; make the cache anew")
        if self.positions.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("DecodeCache: a step under graph capture (its replays would not "
                               "count the rows they fill)")

    def next_positions(self, n: int) -> Tensor:
        """The positions [batch, n] of the next n tokens."""
        return self.positions[:, None] + torch.arange(n, device=self.positions.device)

    def append(self, layer: int, k: Tensor, v: Tensor) -> None:
        """Keys and values [batch, n, key heads, dim] behind a layer's rows."""
        n = k.shape[1]
        self._open = True
        at = self.lens[layer][:, None] + torch.arange(n, device=k.device)
        self.k[layer].index_put_((self._seq, at), k)
        self.v[layer].index_put_((self._seq, at), v)
        self.lens[layer] += n

    def attend(self, layer: int, q: Tensor, window: "int | None") -> Tensor:
        """Attention of the last tokens' q [batch, n, heads, dim] in a layer."""
        w, lens, n = self.weights[layer], self.lens[layer], q.shape[1]
        args = (*self.prefix_kv[layer], self.k[layer], self.v[layer])
        if w is None:
            return shared_prefix_attention(q, *args, lens, window=window)
        # weights are accumulated over at most 64 queries a call: a prompt goes in pieces, each
        # with the rows up to its own last token
        m = max(1, 64 * w.shape[1] // q.shape[2])
        o = [shared_prefix_attention(q[:, i:i + m], *args,
                                     lens - (n - i - m) if i + m < n else lens, window=window,
                                     weights=w, weights_out=w)[0] for i in range(0, n, m)]
        return o[0] if len(o) == 1 else torch.cat(o, dim=1)

    def advance(self, n: int) -> None:
        """Ends the step of n tokens."""
        self.positions += n
        self.filled += n
        self._open = False

    def evict(self, budget: int, recent: int = 0, sinks: int = 0) -> None:
        """Cuts the layers that accumulate weights down to `budget` rows a sequence (cache_evict).
        Layers with a window keep all of theirs: a window counts rows."""
        if all(w is None for w in self.weights):
            raise ValueError("DecodeCache: nothing to evict by, made without weights")
        for i, w in enumerate(self.weights):
            if w is None:
                continue
            k, v = torch.empty_like(self.k[i]), torch.empty_like(self.v[i])
            new = torch.zeros_like(w)
            r = cache_evict(self.k[i], self.v[i], w, self.lens[i], budget, recent=recent,
                            sinks=sinks, out=(k, v, new))
            for t in (self.k[i], self.v[i], w, self.lens[i]):
                t.record_stream(torch.cuda.current_stream(t.device))  # it may be of another
            self.k[i], self.v[i], self.weights[i], self.lens[i] = k, v, new, r[4]
        if all(w is not None for w in self.weights):
            self.filled = min(self.filled, budget)
