"""
The operators a program needs to generate from the decoder, as measurable cases: rotary
positions, attention over a shared prefix and each sequence's own cache, eviction from that
cache by accumulated attention weight, and the penalties, bias and grammar mask between the
logits and the choice of a token.

    listed()            the cases, plain dicts
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form in torch, or with `own` the package's operators
    exact(case, seed)   the same outputs from the definition, in 64 bits
    work(case)          the bytes and operations a pass cannot do without

Head layouts are this package's decoder (9 query and 3 key/value heads of 64) and a generic
wide one (32 and 8 heads of 128).
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
HEADS = {"narrow": (9, 3, 64), "wide": (32, 8, 128)}
NEG = float("-inf")


def listed():
    return [
        # One decode step of 64 sequences, far into a long context.
        _rope("rope_decode_64", 64, 1, "narrow", "bf16", far=500_000, base=500_000.0),
        # One layer of the prefill: q and k are column blocks of the fused projection.
        _rope("rope_prefill_4x8192", 4, 8192, "narrow", "bf16", base=500_000.0),
        # A training step of a model with interleaved planes over half of each head and a
        # context stretched by four, in fp32; one token short of a whole tile.
        _rope("rope_train_4x2047", 4, 2047, "wide", "fp32", part=64, interleaved=True,
              scaling="yarn", factor=4.0, train=True),
        # The smallest attention call: four answers just begun after a short prompt.
        _attn("attn_4x512", 4, 1, 512, 64, "narrow", "bf16"),
        # A serving step: 64 ragged sequences (one slot idle) behind a long system prompt.
        _attn("attn_64x8192", 64, 1, 8192, 1024, "wide", "bf16"),
        # A windowed layer verifying four draft tokens of 32 sequences; odd lengths.
        _attn("attn_window_32x2047", 32, 4, 2047, 777, "narrow", "fp16", window=512),
        # A long decode that also accumulates each cached key's weight for the eviction.
        _attn("attn_weights_48x1000", 48, 1, 1000, 8191, "narrow", "bf16", weights=True),
        # The questions of eight users, prefilled behind the prompt they share.
        _attn("attn_questions_8x8192", 8, 256, 8192, 300, "narrow", "bf16"),
        # Eviction as it comes up in a decode loop: a few rows over the budget.
        _evict("evict_8x1100", 8, 1100, 1024, 64, 4, "narrow", "bf16"),
        # Eviction of long ragged prompts down to a quarter.
        _evict("evict_32x8192", 32, 8192, 2048, 256, 4, "wide", "fp16"),
        # One sequence's next token.
        _logits("logits_1", 1, 32768, 512, "bf16", bias=False, mask=True),
        # A full batch with long histories, a bias and a grammar mask per row.
        _logits("logits_256", 256, 131072, 4096, "fp32", bias=True, mask=True),
    ]


def _rope(name, batch, tokens, heads, dtype, far=0, base=10_000.0, part=0, interleaved=False,
          scaling="none", factor=1.0, train=False):
    """far: positions start anywhere below it; part: width of the rotated part (0: all)."""
    return _named(name, what="rope", batch=batch, tokens=tokens, heads=heads, dtype=dtype,
                  far=far, base=base, part=part, interleaved=interleaved, scaling=scaling,
                  factor=factor, train=train)


def _attn(name, batch, new, prefix, cap, heads, dtype, window=0, weights=False):
    """new: query tokens per sequence; cap: rows of the cache, ragged lengths up to it."""
    return _named(name, what="attn", batch=batch, new=new, prefix=prefix, cap=cap, heads=heads,
                  dtype=dtype, window=window, weights=weights)


def _evict(name, batch, cap, budget, recent, sinks, heads, dtype):
    return _named(name, what="evict", batch=batch, cap=cap, budget=budget, recent=recent,
                  sinks=sinks, heads=heads, dtype=dtype)


def _logits(name, batch, vocab, history, dtype, bias, mask):
    return _named(name, what="logits", batch=batch, vocab=vocab, history=history, dtype=dtype,
                  bias=bias, mask=mask)


def _named(name, **case):
    return {"name": name, **case} if name else case


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    what = rng.choice(["rope", "attn", "attn", "evict", "logits"])
    heads = rng.choice(["narrow", "wide"])
    hq, hk, d = HEADS[heads]
    if what == "rope":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        batch = _log_int(rng, 1, 64)
        # no more than the prefill's elements
        tokens = _log_int(rng, 1, max(1, 25_000_000 // (batch * (hq + hk) * d)))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return _rope(None, batch, tokens, heads, dtype, far=rng.choice([0, 100_000, 1_000_000]),
                     base=rng.choice([10_000.0, 500_000.0]), part=rng.choice([0, d // 2, 24]),
                     interleaved=rng.random() < 0.5, scaling=scaling,
                     factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                     train=rng.random() < 0.4)
    if what == "attn":
        batch = _log_int(rng, 1, 64)
        prefix = _log_int(rng, 1, 8192) if rng.random() < 0.9 else 0
        # no more cached elements than 64 sequences of 1024 rows in the wide layout
        cap = _log_int(rng, 1, min(8192, 67_000_000 // (batch * hk * d)))
        new = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 256)])
        # no more products than the questions' prefill
        new = max(1, min(new, 39_000_000_000 // (4 * batch * hq * d * (prefix + cap))))
        weights = new * (hq // hk) <= 64 and rng.random() < 0.3
        return _attn(None, batch, min(new, cap), prefix, cap, heads, rng.choice(["bf16", "fp16"]),
                     window=rng.choice([0, 0, 512]), weights=weights)
    if what == "evict":
        batch = _log_int(rng, 1, 32)
        cap = _log_int(rng, 8, min(32768, 67_000_000 // (batch * hk * d)))
        budget = rng.randint(max(1, cap // 8), cap)
        sinks = min(rng.choice([0, 1, 4]), budget)
        return _evict(None, batch, cap, budget, rng.randint(0, (budget - sinks) // 2), sinks,
                      heads, rng.choice(["bf16", "fp16"]))
    batch = _log_int(rng, 1, 256)
    return _logits(None, batch, _log_int(rng, 1000, 131072), _log_int(rng, 1, 4096),
                   rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * int(seed) + 29)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _randint(gen, lo, hi, *shape, dtype=torch.int64):
    return torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=dtype)


def _lengths(gen, batch, least, cap):
    """Ragged lengths from a quarter of the cache up to all of it."""
    low = max(least, cap // 4)
    return _randint(gen, low, cap + 1, batch, dtype=torch.int32)


def prepare(case, seed):
    gen, dt = _gen(seed), DTYPES.get(case["dtype"])
    return {"case": case, **_PREPARE[case["what"]](case, gen, dt)}


def _prepare_rope(c, gen, dt):
    hq, hk, d = HEADS[c["heads"]]
    b, t = c["batch"], c["tokens"]
    # the fused projection's rows: q heads, k heads, v heads
    qkv = _randn(gen, b, t, hq + 2 * hk, d, dtype=dt)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    start = _randint(gen, 0, max(1, c["far"]), b, 1)
    s = {"q": q, "k": k, "positions": start + torch.arange(t, device=DEV),
         "freqs": _frequencies(c).to(DEV), "amplitude": _amplitude(c)}
    if c["train"]:
        s["q"], s["k"] = q.detach().requires_grad_(), k.detach().requires_grad_()
        s["gq"], s["gk"] = _randn(gen, b, t, hq, d, dtype=dt), _randn(gen, b, t, hk, d, dtype=dt)
    return s


def _prepare_attn(c, gen, dt):
    hq, hk, d = HEADS[c["heads"]]
    b, n, p, s = c["batch"], c["new"], c["prefix"], c["cap"]
    lens = _lengths(gen, b, n, s)
    if b >= 8:
        lens[b // 2] = 0  # an idle slot of the batch
    st = {"q": _randn(gen, b, n, hq, d, dtype=dt, scale=1.5),
          "kp": _randn(gen, p, hk, d, dtype=dt), "vp": _randn(gen, p, hk, d, dtype=dt),
          "k": _randn(gen, b, s, hk, d, dtype=dt), "v": _randn(gen, b, s, hk, d, dtype=dt),
          "lens": lens}
    if c["weights"]:
        st["weights"] = torch.rand(b, hk, s, generator=gen, device=DEV)
    return st


def _prepare_evict(c, gen, dt):
    _, hk, d = HEADS[c["heads"]]
    b, s = c["batch"], c["cap"]
    # accumulated weights: heavy-tailed, with keys that never got any (exact ties)
    w = torch.exp(_randn(gen, b, hk, s, scale=2.0)) * 1e-3
    w = torch.where(torch.rand(b, hk, s, generator=gen, device=DEV) < 0.2, 0.0, w)
    return {"k": _randn(gen, b, s, hk, d, dtype=dt), "v": _randn(gen, b, s, hk, d, dtype=dt),
            "weights": w, "lens": _lengths(gen, b, 1, s)}


def _prepare_logits(c, gen, dt):
    b, v, n = c["batch"], c["vocab"], c["history"]
    lens = _lengths(gen, b, 0, n)
    # token ids fall off like a language's: many repeats of few tokens
    ids = (v ** torch.rand(b, n, generator=gen, device=DEV, dtype=torch.float64)).long() - 1
    ids = ids.clamp(0, v - 1)
    pad = torch.arange(n, device=DEV)[None] >= lens[:, None]
    st = {"logits": _randn(gen, b, v, dtype=dt, scale=3.0), "history": ids.masked_fill(pad, -1),
          "lens": lens, "prompt_lens": (lens // 2).to(torch.int32),
          "repetition": 1.0 + torch.rand(b, generator=gen, device=DEV),
          "frequency": torch.rand(b, generator=gen, device=DEV),
          "presence": torch.rand(b, generator=gen, device=DEV), "bias": None, "mask": None}
    if c["bias"]:
        st["bias"] = _randn(gen, b, v, scale=0.5)
    if c["mask"]:
        # a grammar allows about one token in eight (three random bits agree)
        bits = _randint(gen, -2 ** 31, 2 ** 31, 3, b, (v + 31) // 32, dtype=torch.int64)
        st["mask"] = (bits[0] & bits[1] & bits[2]).to(torch.int32)
    return st


_PREPARE = {"rope": _prepare_rope, "attn": _prepare_attn, "evict": _prepare_evict,
            "logits": _prepare_logits}


def _amplitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "yarn" else 1.0


def _frequencies(c):
    """Radians per position of each plane, fp64: base^(-2j / part), stretched by `factor`."""
    part, f = c["part"] or HEADS[c["heads"]][2], c["factor"]
    j = torch.arange(part // 2, dtype=torch.float64)
    base = c["base"] * (f ** (part / (part - 2)) if c["scaling"] == "ntk" else 1.0)
    freq = base ** (-2.0 * j / part)
    if c["scaling"] == "linear":
        freq = freq / f
    if c["scaling"] == "yarn":
        # planes of fewer than 1 turn in the original 4096 positions are interpolated, of
        # more than 32 turns kept, the others in between
        turns = 4096 * freq / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * freq / f
    return freq


# ---- one pass -------------------------------------------------------------------------------

def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["what"]](s)


def _own_rope(s):
    from nanospeaker_amd import rotary_embed

    c = s["case"]
    q, k = rotary_embed(s["q"], s["k"], s["positions"], s["freqs"],
                        interleaved=c["interleaved"], amplitude=s["amplitude"])
    if not c["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _own_attn(s):
    from nanospeaker_amd import shared_prefix_attention

    c = s["case"]
    r = shared_prefix_attention(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["lens"],
                                window=c["window"] or None, weights=s.get("weights"),
                                return_lse=True)
    return dict(zip(("out", "lse", "weights"), r))


def _own_evict(s):
    from nanospeaker_amd import cache_evict

    c = s["case"]
    r = cache_evict(s["k"], s["v"], s["weights"], s["lens"], c["budget"], recent=c["recent"],
                    sinks=c["sinks"])
    return dict(zip(("k", "v", "weights", "index", "lens"), r))


def _own_logits(s):
    from nanospeaker_amd import penalize_logits

    return penalize_logits(s["logits"], s["history"], s["lens"], prompt_lens=s["prompt_lens"],
                           repetition=s["repetition"], frequency=s["frequency"],
                           presence=s["presence"], bias=s["bias"], mask=s["mask"])


_OWN = {"rope": _own_rope, "attn": _own_attn, "evict": _own_evict, "logits": _own_logits}


def _rotate(x, cos, sin, part, interleaved):
    """One tensor [B, T, H, D] turned by the tables [B, T, 1, part / 2], rounded once."""
    xf = x.float()
    rot = xf[..., :part]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = rot[..., :part // 2], rot[..., part // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((y, xf[..., part:]), dim=-1).to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[..., None, None] * s["freqs"]  # far positions: 64 bits
    cos = (angle.cos() * s["amplitude"]).float()
    sin = (angle.sin() * s["amplitude"]).float()
    part = 2 * s["freqs"].numel()
    q = _rotate(s["q"], cos, sin, part, c["interleaved"])
    k = _rotate(s["k"], cos, sin, part, c["interleaved"])
    if not c["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _plain_attn(s):
    c = s["case"]
    q, kp, vp, k, v = (s[n].float() for n in ("q", "kp", "vp", "k", "v"))
    b, n, hq, d = q.shape
    cap, hk = k.shape[1], k.shape[2]
    p, g = kp.shape[0], hq // hk
    qh = (q / math.sqrt(d)).view(b, n, hk, g, d).permute(0, 2, 1, 3, 4)  # [b, hk, n, g, d]
    # the prefix in one product for the whole batch, the caches in one per sequence
    sp = qh.permute(1, 0, 2, 3, 4).reshape(hk, b * n * g, d) @ kp.permute(1, 2, 0)
    sp = sp.view(hk, b, n, g, p).transpose(0, 1)
    ss = (qh.reshape(b, hk, n * g, d) @ k.permute(0, 2, 3, 1)).view(b, hk, n, g, cap)
    sc = torch.cat((sp, ss), dim=-1)
    row = s["lens"].long()[:, None] - n + torch.arange(n, device=q.device)  # [b, n]
    at = torch.arange(p + cap, device=q.device)
    far = (row + p)[..., None] - at                                         # [b, n, p + cap]
    seen = (far >= 0) & (row >= 0)[..., None]
    if c["window"]:
        seen = seen & (far < c["window"])
    sc = sc.masked_fill(~seen[:, None, :, None, :], NEG)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == NEG, 0.0, top)
    e = torch.exp(sc - top)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    o = (w[..., :p].transpose(0, 1).reshape(hk, b * n * g, p) @ vp.transpose(0, 1))
    o = o.view(hk, b, n, g, d).transpose(0, 1)
    o = o + (w[..., p:].reshape(b, hk, n * g, cap) @ v.transpose(1, 2)).view(b, hk, n, g, d)
    lse = (torch.log(total) + top).squeeze(-1)                              # [b, hk, n, g]
    r = {"out": o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, d).to(s["q"].dtype),
         "lse": lse.permute(0, 2, 1, 3).reshape(b, n, hq)}
    if c["weights"]:
        r["weights"] = s["weights"] + w[..., p:].sum((2, 3))
    return r


def _plain_evict(s):
    c = s["case"]
    k, w = s["k"], s["weights"]
    b, cap, hk, d = k.shape
    lens, budget = s["lens"].long(), c["budget"]
    j = torch.arange(cap, device=k.device)
    n = lens[:, None]
    held = (j < c["sinks"]) | (j >= n - c["recent"])
    rank = torch.where(held[:, None], float("inf"), w)
    rank = torch.where((j < n)[:, None], rank, NEG)
    idx = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    idx = torch.where(idx < n[..., None], idx, cap)  # fewer rows than the budget
    idx = torch.sort(idx, dim=-1).values
    live = idx < cap
    at = torch.where(live, idx, 0)
    rows = at.transpose(1, 2)[..., None].expand(b, budget, hk, d)
    keep = live.transpose(1, 2)[..., None]
    return {"k": torch.where(keep, torch.gather(k, 1, rows), 0),
            "v": torch.where(keep, torch.gather(s["v"], 1, rows), 0),
            "weights": torch.where(live, torch.gather(w, 2, at), 0.0),
            "index": torch.where(live, idx, -1).to(torch.int32),
            "lens": lens.clamp(max=budget).to(torch.int32)}


def _plain_logits(s):
    x = s["logits"].float()
    b, v = x.shape
    ids, n = s["history"], s["history"].shape[1]
    j = torch.arange(n, device=x.device)
    live = (j < s["lens"][:, None]) & (ids >= 0) & (ids < v)
    new = live & (j >= s["prompt_lens"][:, None])
    at = torch.where(live, ids, 0)
    zero = torch.zeros(b, v, device=x.device)
    seen = zero.scatter_add(1, at, live.float()) > 0
    count = zero.scatter_add(1, at, new.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        bit = torch.arange(32, device=x.device, dtype=torch.int32)
        on = ((s["mask"][..., None] >> bit) & 1).reshape(s["mask"].shape[0], -1)[:, :v]
        x = torch.where(on != 0, x, NEG)
    return x.to(s["logits"].dtype)


_PLAIN = {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict,
          "logits": _plain_logits}


# ---- 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["what"]](case, prepare(case, seed))


def _exact_rope(c, s):
    part = c["part"] or HEADS[c["heads"]][2]
    freq, amp = _frequencies(c).to(DEV), _amplitude(c)
    turn = torch.polar(torch.full((), amp, dtype=torch.float64, device=DEV),
                       s["positions"].double()[..., None] * freq)[:, :, None]  # [B, T, 1, part/2]

    def spin(x, t):
        x = x.double()
        r = x[..., :part]
        z = torch.complex(r[..., 0::2], r[..., 1::2]) if c["interleaved"] else \
            torch.complex(r[..., :part // 2], r[..., part // 2:])
        z = z * t
        y = torch.view_as_real(z).flatten(-2) if c["interleaved"] else \
            torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., part:]), -1)

    r = {"q": spin(s["q"], turn), "k": spin(s["k"], turn)}
    if c["train"]:
        r["dq"], r["dk"] = spin(s["gq"], turn.conj()), spin(s["gk"], turn.conj())
    return r


def _exact_attn(c, s):
    b, n, hq, d = s["q"].shape
    hk, p, cap = s["k"].shape[2], s["kp"].shape[0], s["k"].shape[1]
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=DEV)
    lse = torch.full((b, n, hq), NEG, dtype=torch.float64, device=DEV)
    w = s["weights"].double() if c["weights"] else None
    for i in range(b):
        ln = int(s["lens"][i])
        if ln == 0:
            continue
        k = torch.cat((s["kp"], s["k"][i, :ln])).double().transpose(0, 1)     # [hk, p + ln, d]
        v = torch.cat((s["vp"], s["v"][i, :ln])).double().transpose(0, 1)
        key = torch.arange(p + ln, device=DEV)
        me = p + ln - n + torch.arange(n, device=DEV)[:, None]
        ok = (key <= me) & (me >= p)
        if c["window"]:
            ok &= key > me - c["window"]
        for h in range(hq):
            kv = h * hk // hq
            sc = (s["q"][i, :, h].double() @ k[kv].t().contiguous()) / math.sqrt(d)
            sc = sc.masked_fill(~ok, NEG)
            lse[i, :, h] = torch.logsumexp(sc, -1)
            pr = torch.exp(sc - lse[i, :, h, None]).nan_to_num(0.0)
            out[i, :, h] = pr @ v[kv]
            if w is not None:
                w[i, kv, :ln] += pr[:, p:].sum(0)
    r = {"out": out, "lse": lse}
    if w is not None:
        r["weights"] = w
    return r


def _exact_evict(c, s):
    b, cap, hk, d = s["k"].shape
    m = c["budget"]
    k = torch.zeros(b, m, hk, d, dtype=torch.float64, device=DEV)
    v, w = torch.zeros_like(k), torch.zeros(b, hk, m, dtype=torch.float64, device=DEV)
    index = torch.full((b, hk, m), -1, dtype=torch.int32, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        for h in range(hk):
            if n <= m:
                keep = list(range(n))
            else:
                x = s["weights"][i, h, :n].tolist()
                mid = range(c["sinks"], n - c["recent"])
                best = sorted(mid, key=lambda j: (-x[j], j))[:m - c["sinks"] - c["recent"]]
                keep = [*range(c["sinks"]), *sorted(best), *range(n - c["recent"], n)]
            at = torch.tensor(keep, dtype=torch.int64, device=DEV)
            index[i, h, :len(keep)] = at
            k[i, :len(keep), h], v[i, :len(keep), h] = s["k"][i, at, h].double(), \
                s["v"][i, at, h].double()
            w[i, h, :len(keep)] = s["weights"][i, h, at].double()
    return {"k": k, "v": v, "weights": w, "index": index,
            "lens": torch.minimum(s["lens"], torch.full_like(s["lens"], m))}


def _exact_logits(c, s):
    x = s["logits"].double()
    b, v = x.shape
    for i in range(b):
        n, p = int(s["lens"][i]), int(s["prompt_lens"][i])
        ids = s["history"][i, :n]
        r = float(s["repetition"][i])
        some = torch.unique(ids)
        x[i, some] = torch.where(x[i, some] > 0, x[i, some] / r, x[i, some] * r)
        made, times = torch.unique(ids[p:], return_counts=True)
        x[i, made] -= float(s["frequency"][i]) * times + float(s["presence"][i])
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["mask"] is not None:
        col = torch.arange(v, device=DEV)
        x[(s["mask"][:, col // 32].long() >> (col % 32)) & 1 == 0] = NEG
    return x


_EXACT = {"rope": _exact_rope, "attn": _exact_attn, "evict": _exact_evict,
          "logits": _exact_logits}


# ---- the work a pass cannot do without --------------------------------------------------------

def work(c):
    """Ragged lengths count at their mean, five eighths of the cache."""
    size = SIZE[c["dtype"]]
    if c["what"] == "rope":
        hq, hk, d = HEADS[c["heads"]]
        rows = c["batch"] * c["tokens"] * (hq + hk)
        ways = 2 if c["train"] else 1
        part = c["part"] or d
        return {"bytes": ways * (2 * rows * d * size) + 8 * c["batch"] * c["tokens"],
                "flops": ways * rows * 3 * part}
    if c["what"] == "attn":
        hq, hk, d = HEADS[c["heads"]]
        b, n = c["batch"], c["new"]
        own_rows, pre = 0.625 * c["cap"], c["prefix"]
        if c["window"]:
            own_rows = min(own_rows, c["window"] + n)
            pre = min(pre, c["window"])
        io = 2 * b * n * hq * d * size + 4 * b * n * hq
        kv = 2 * hk * d * size * (pre + b * own_rows)
        w = 2 * 4 * b * hk * c["cap"] if c["weights"] else 0
        return {"bytes": io + kv + w, "flops": 4 * b * n * hq * d * (pre + own_rows)}
    if c["what"] == "evict":
        _, hk, d = HEADS[c["heads"]]
        kept = c["batch"] * hk * min(c["budget"], 0.625 * c["cap"])
        out = c["batch"] * hk * c["budget"]
        return {"bytes": 4 * c["batch"] * hk * 0.625 * c["cap"] + 2 * kept * d * size
                + 2 * out * d * size + 8 * out, "flops": 0}
    b, v = c["batch"], c["vocab"]
    return {"bytes": 2 * b * v * size + (4 * b * v if c["bias"] else 0)
            + (b * v / 8 if c["mask"] else 0) + 8 * b * 0.625 * c["history"], "flops": 4 * b * v}
