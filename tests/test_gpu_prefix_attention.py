"""
shared_prefix_attention (nsmoe_prefix_attention) against attention in 64 bits: every form a
part takes (few and many columns), both head dims and types, grouped heads, windows, ragged and
idle sequences, caches with NaN behind their rows, the accumulated weights and the lse.

Bounds, for an element o = sum p v of a query with scores s:
  * a score is an fp32 sum of D products: at most D 2^-24 of sum |q k|, times the scale; call
    the largest over the query's keys ds.  exp2 of the scaled difference rounds twice more at
    magnitude |s| and once itself: 2^-21 covers differences up to 2^2 and far keys weigh less.
    So a weight p, a sum and a quotient are off by at most dp = 2 ds + 2^-20, relatively.
  * p enters the product rounded to the type: half a step of it, relatively.
  * o is rounded once to the type.
  |error| <= step/2 |o| + (step/2 + dp) sum p |v|;  lse: ds + 2^-20 max(1, |lse|);
  weights: dp sum p + 2^-23 |w|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import shared_prefix_attention  # noqa: E402

DEV = "cuda"
NEG = float("-inf")
NAN = float("nan")


def ref(q, kp, vp, k, v, lens, window, scale, weights=None):
    """{out, lse, weights} in fp64 on the CPU and each one's bound (without the last rounding)."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    b, n, hq, d = q.shape
    s, hk = k.shape[1], k.shape[2]
    if kp is None:
        kp = vp = torch.zeros(0, hk, d)
    kp, vp, lens = kp.double().cpu(), vp.double().cpu(), lens.cpu()
    p, step = kp.shape[0], 0.0
    out = torch.zeros(b, n, hq, d, dtype=torch.float64)
    lse = torch.full((b, n, hq), NEG, dtype=torch.float64)
    rel, av = torch.zeros(b, n, hq, dtype=torch.float64), torch.zeros_like(out)
    w = torch.zeros(b, hk, s, dtype=torch.float64) if weights is None else weights.double().cpu()
    wsum = torch.zeros_like(w)
    wrel = torch.zeros_like(w)
    for i in range(b):
        ln = max(0, min(int(lens[i]), s))
        kk, vv = torch.cat((kp, k[i, :ln])), torch.cat((vp, v[i, :ln]))
        key = torch.arange(p + ln)
        for t in range(n):
            me = ln - n + t
            if me < 0:
                continue
            ok = key <= p + me
            if window is not None:
                ok &= p + me - key < window
            for h in range(hq):
                g = h // (hq // hk)
                sc = (kk[ok, g] @ q[i, t, h]) * scale
                size = (kk[ok, g].abs() @ q[i, t, h].abs()) * scale
                lse[i, t, h] = torch.logsumexp(sc, 0)
                pr = torch.softmax(sc, 0)
                out[i, t, h] = pr @ vv[ok, g]
                av[i, t, h] = pr @ vv[ok, g].abs()
                rel[i, t, h] = d * 2.0 ** -24 * float(size.max())
                full = torch.zeros(p + ln, dtype=torch.float64)
                full[ok] = pr
                wsum[i, g, :ln] += full[p:]
                wrel[i, g, :ln] += full[p:] * (2 * rel[i, t, h] + 2.0 ** -20)
    return dict(out=out, lse=lse, weights=w + wsum, av=av, rel=rel,
                wbound=wrel + 2.0 ** -23 * (w + wsum).abs() + 1e-38)


def check(got, want, dtype):
    step = torch.finfo(dtype).eps / 2
    out = got[0].double().cpu()
    assert not out.isnan().any()
    bound = step * want["out"].abs() + (step + 2 * want["rel"] + 2.0 ** -20)[..., None] * want["av"]
    bound = bound * (1 + 2 * step) + torch.finfo(dtype).smallest_normal
    err = (out - want["out"]).abs()
    print(f"  out: {float((err / bound).max()):.2f} of the bound", flush=True)
    assert (err <= bound).all(), float((err - bound).max())
    lse, ref_lse = got[1].double().cpu(), want["lse"]
    none = ref_lse == NEG
    assert torch.equal(lse == NEG, none) and not out[none].any()
    e = (lse - ref_lse).abs()[~none]
    lim = (want["rel"] + 2.0 ** -20 * ref_lse.abs().clamp(min=1.0))[~none]
    assert (e <= lim).all(), float((e - lim).max())
    if len(got) == 3:
        e = (got[2].double().cpu() - want["weights"]).abs()
        assert (e <= want["wbound"]).all(), float((e - want["wbound"]).max())


def make(b, n, p, s, hq, hk, d, dtype, lens=None, seed=0, junk=NAN):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g)
    if lens is None:
        lens = torch.randint(min(n, s), s + 1, (b,), generator=g)
        if b > 2:
            lens[b // 2] = 0
        lens[-1] = s
    lens = torch.as_tensor(lens, dtype=torch.int32)
    q = (1.5 * r(b, n, hq, d)).to(dtype)
    kp, vp = r(p, hk, d).to(dtype), r(p, hk, d).to(dtype)
    k, v = r(b, s, hk, d).to(dtype), r(b, s, hk, d).to(dtype)
    for i in range(b):  # rows behind a sequence were never written
        k[i, max(0, int(lens[i])):] = junk
        v[i, max(0, int(lens[i])):] = junk
    return tuple(t.to(DEV) for t in (q, kp, vp, k, v, lens))


def clean(t):
    return t.nan_to_num(nan=0.0)


def run(case, window=None, scale=None, weights=None, dtype=None):
    q, kp, vp, k, v, lens = case
    sc = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = ref(q, kp, vp, clean(k), clean(v), lens, window, sc, weights)
    got = shared_prefix_attention(q, kp, vp, k, v, lens, window=window, scale=scale,
                                  weights=weights, return_lse=True)
    check(got, want, q.dtype)
    return got


# batch, new, prefix, cap, heads, kv heads, dim, window: each form of both parts, edges of the
# tiles (32 and 64 keys) and of the splits
CASES = [
    (1, 1, 0, 1, 1, 1, 64, None), (1, 1, 1, 1, 9, 3, 64, None), (2, 1, 31, 33, 9, 3, 64, None),
    (4, 1, 512, 64, 9, 3, 64, None), (5, 1, 130, 700, 9, 3, 64, None),
    (3, 1, 1000, 300, 32, 8, 128, None), (16, 1, 700, 40, 9, 3, 64, None),
    (33, 1, 513, 65, 8, 2, 128, None), (40, 1, 257, 20, 12, 1, 64, None),
    (2, 4, 300, 100, 9, 3, 64, None), (3, 5, 64, 70, 8, 8, 128, None),
    (2, 13, 200, 50, 16, 2, 64, None), (2, 30, 100, 95, 9, 3, 128, None),
    (2, 100, 150, 130, 9, 3, 64, None), (1, 200, 65, 200, 8, 2, 128, None),
    (2, 3, 0, 2100, 6, 2, 64, None), (1, 1, 5000, 5, 4, 4, 128, None),
    (4, 1, 100, 700, 9, 3, 64, 512), (4, 3, 100, 200, 9, 3, 64, 64),
    (3, 2, 700, 37, 8, 2, 128, 50), (20, 2, 200, 37, 9, 3, 64, 33), (2, 70, 90, 80, 6, 2, 64, 17),
    (2, 5, 40, 60, 4, 2, 128, 1), (1, 1, 64, 64, 20, 1, 64, None), (1, 2, 10, 10, 40, 1, 128, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,n,p,s,hq,hk,d,window", CASES)
def test_against_64_bits(dtype, b, n, p, s, hq, hk, d, window):
    print(f"[prefix] {dtype} {(b, n, p, s, hq, hk, d, window)}", flush=True)
    case = make(b, n, p, s, hq, hk, d, dtype, seed=p + s)
    w = None
    if n * (hq // hk) <= 64:
        w = torch.rand(b, hk, s, generator=torch.Generator().manual_seed(1)).to(DEV)
    run(case, window, weights=w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,n,p,s,hq,hk,d,window", CASES)
def test_without_weights_against_64_bits(dtype, b, n, p, s, hq, hk, d, window):
    """Short contexts are not split where nobody asks for weights."""
    print(f"[prefix] {dtype} {(b, n, p, s, hq, hk, d, window)}", flush=True)
    run(make(b, n, p, s, hq, hk, d, dtype, seed=p + s + 1), window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,g", [(1, 1), (5, 3), (16, 2)])
@pytest.mark.parametrize("p,s", [(0, 40), (1, 33), (31, 64), (32, 31), (33, 1), (95, 97), (500, 520)])
def test_short_contexts(d, n, g, p, s):
    """Tiles that end with the prefix, with the window and with the sequence, in fewer tiles than
    waves and in more."""
    print(f"[prefix] short {(d, n, g, p, s)}", flush=True)
    case = make(3, n, p, s, 2 * g, 2, d, torch.bfloat16, lens=[s, max(1, s // 2), min(s, n // 2)])
    for window in (None, 1, 30, 70, p + 5):
        run(case, window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [1, 2, 4, 9])
@pytest.mark.parametrize("n,g", [(5, 2), (5, 4), (10, 5), (20, 5), (25, 9)])
def test_every_pair_of_forms(d, b, n, g):
    """Own parts of 10, 20, 50, 100 and 225 columns beside prefix parts of one to nine times as
    many, over lengths that end inside tiles, with a window that cuts both."""
    print(f"[prefix] forms {(d, b, n, g)}", flush=True)
    case = make(b, n, 150, 135, g, 1, d, torch.bfloat16, seed=b * n)
    run(case)
    run(case, window=140)


@pytest.mark.parametrize("n,g", [(1, 3), (4, 3), (12, 4), (40, 5)])
@pytest.mark.parametrize("weights", [False, True])  # which keep the call in parts
def test_rows_that_no_query_sees_may_hold_anything(n, g, weights):
    """NaN in every prefix and cache row before the oldest query's window."""
    q, kp, vp, k, v, lens = make(3, n, 100, 90, g, 1, 64, torch.bfloat16, lens=[90, 77, 50])
    k, v = clean(k), clean(v)
    kw = dict(window=8, return_lse=True)
    if weights and n * g <= 64:
        kw["weights_out"] = torch.empty(3, 1, 90, device=DEV)
    want = shared_prefix_attention(q, kp, vp, k, v, lens, **kw)
    for i, ln in enumerate((90, 77, 50)):
        oldest = max(0, ln - n - 7)
        k[i, :oldest], v[i, :oldest] = NAN, NAN
    kp[:], vp[:] = NAN, NAN
    got = shared_prefix_attention(q, kp, vp, k, v, lens, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("lens", [[0, 0, 0], [1, 2, 3], [4, 3, 40], [-7, 41, 2 ** 31 - 1]])
@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("window", [None, 3])
def test_queries_without_a_row_and_lengths_out_of_range(lens, n, window):
    case = make(3, n, 50, 40, 6, 2, 64, torch.bfloat16, lens=lens)
    w = torch.ones(3, 2, 40, device=DEV)
    got = run(case, window, weights=w)
    for i, ln in enumerate(lens):
        assert (got[2][i, :, max(0, min(ln, 40)):] == 1).all()  # rows behind keep theirs


@pytest.mark.parametrize("lens", [[0, 0, 0], [1, 2, 3], [-7, 41, 2 ** 31 - 1]])
@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("p", [50, 1700])  # in one launch, in parts
def test_lengths_out_of_range_without_weights(lens, n, p):
    case = make(3, n, p, 40, 6, 2, 64, torch.bfloat16, lens=lens)
    run(case)
    run(case, window=3)


def test_prefix_of_zero_rows_and_cache_of_zero_rows():
    q, kp, vp, k, v, lens = make(2, 1, 0, 9, 6, 2, 64, torch.bfloat16)
    a = run((q, kp, vp, k, v, lens))
    b = shared_prefix_attention(q, None, None, k, v, lens)
    assert torch.equal(a[0], b)
    none = shared_prefix_attention(q, None, None, k[:, :0], v[:, :0], lens * 0, return_lse=True)
    assert not none[0].any() and (none[1] == NEG).all()
    r = shared_prefix_attention(q[:0], None, None, k[:0], v[:0], lens[:0])
    assert r.shape == (0, 1, 6, 64)


def test_one_visible_key_returns_its_value():
    q, kp, vp, k, v, lens = make(2, 3, 20, 30, 6, 2, 128, torch.bfloat16)
    lens.fill_(30)
    k, v = clean(k), clean(v)
    o = shared_prefix_attention(q, kp, vp, k, v, lens, window=1)
    want = v[:, 27:30].repeat_interleave(3, dim=2)
    assert torch.equal(o, want)


def test_large_scores_and_a_given_scale():
    """Scores in the hundreds (one key takes all), and a scale of 1."""
    q, kp, vp, k, v, lens = make(2, 1, 300, 200, 6, 2, 64, torch.bfloat16)
    run((q * 20, kp, vp, k, v, lens))
    run((q, kp, vp, k, v, lens), scale=1.0)
    far = (q, kp * 8, vp, k, v, lens)  # the prefix towers over the cache
    run(far)


def test_scores_that_grow_along_the_keys():
    """A running maximum that moves in every tile."""
    q, kp, vp, k, v, lens = make(3, 1, 700, 500, 6, 2, 64, torch.float16)
    q = torch.ones_like(q)
    ramp = lambda t, dim: t * 0.1 + torch.linspace(0, 6, t.shape[dim], device=DEV).view(
        [-1 if i == dim else 1 for i in range(t.dim())])
    run((q, ramp(kp, 0).half(), vp, ramp(k, 1).half(), v, lens))


@pytest.mark.parametrize("p", [90, 1700])  # in one launch, in parts
def test_strided_operands(p):
    """Keys and values as column blocks of a fused projection, heads before rows, a strided q."""
    q, kp, vp, k, v, lens = make(3, 2, p, 70, 9, 3, 64, torch.bfloat16)
    want = shared_prefix_attention(q, kp, vp, k, v, lens, return_lse=True)
    fused = torch.full((p, 15, 64), NAN, dtype=q.dtype, device=DEV)
    fused[:, 9:12], fused[:, 12:] = kp, vp
    caches = torch.full((3, 70, 15, 64), NAN, dtype=q.dtype, device=DEV)
    caches[:, :, 9:12], caches[:, :, 12:] = k, v
    wide_q = torch.zeros(3, 2, 15, 64, dtype=q.dtype, device=DEV)
    wide_q[:, :, :9] = q
    got = shared_prefix_attention(wide_q[:, :, :9], fused[:, 9:12], fused[:, 12:],
                                  caches[:, :, 9:12], caches[:, :, 12:], lens, return_lse=True)
    t = lambda x, a, c: x.transpose(a, c).contiguous().transpose(a, c)
    other = shared_prefix_attention(t(q, 1, 2), t(kp, 0, 1), t(vp, 0, 1), t(k, 1, 2), t(v, 1, 2),
                                    lens, return_lse=True)
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)  # a query off the 16-byte alignment is copied
    third = shared_prefix_attention(odd, kp, vp, k, v, lens, return_lse=True)
    every = torch.zeros(3, 2, 9, 64 * 9, dtype=q.dtype, device=DEV)[..., ::9]
    every.copy_(q)  # and one whose last dim is strided
    fourth = shared_prefix_attention(every, kp, vp, k, v, lens, return_lse=True)
    for r in (got, other, third, fourth):
        assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])


def test_weights_accumulate_in_place_or_apart():
    case = make(3, 2, 90, 70, 9, 3, 64, torch.bfloat16)
    zero = shared_prefix_attention(*case, weights_out=torch.empty(3, 3, 70, device=DEV))
    start = torch.rand(3, 3, 70, device=DEV)
    apart = shared_prefix_attention(*case, weights=start)[1]
    kept = start.clone()
    same = shared_prefix_attention(*case, weights=kept, weights_out=kept)[1]
    assert same is kept and torch.equal(apart, kept)
    assert torch.equal(start + zero[1], apart)
    # each query gives each key head's group a weight of one in all, prefix included
    rows = (case[5] > 0).float() * 2 * 3
    assert (zero[1].sum(-1) <= rows[:, None] * (1 + 1e-5)).all()


def test_offsets_past_32_bits():
    """A cache whose last sequence lies more than 2^32 bytes behind the first one's."""
    b, s, hk, d = 3, 2_200_000, 8, 64
    cache = torch.empty(b, s, hk, d, dtype=torch.bfloat16, device=DEV)
    lens = torch.tensor([3, 0, s], dtype=torch.int32, device=DEV)
    cache[0, :3].normal_()
    cache[2].normal_()
    k = cache
    q = torch.randn(b, 1, hk, d, dtype=torch.bfloat16, device=DEV)
    got = shared_prefix_attention(q, None, None, k, k, lens, window=100, return_lse=True)
    small = shared_prefix_attention(q[2:], None, None, k[2:, s - 100:].contiguous(),
                                    k[2:, s - 100:].contiguous(),
                                    torch.tensor([100], dtype=torch.int32, device=DEV),
                                    return_lse=True)
    tail = ref(q[2:], None, None, k[2:, s - 100:], k[2:, s - 100:], torch.tensor([100]), None,
               1 / 8)
    check((got[0][2:], got[1][2:]), tail, q.dtype)
    check(small, tail, q.dtype)


@pytest.mark.parametrize("p", [300, 1700])  # in one launch, in parts
def test_another_stream_and_two_calls_at_once(p):
    a = make(4, 1, p, 200, 9, 3, 64, torch.bfloat16, seed=1)
    b = make(4, 1, p, 200, 9, 3, 64, torch.bfloat16, seed=2)
    want = [shared_prefix_attention(*c) for c in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = shared_prefix_attention(*a)
        with torch.cuda.stream(s2):
            y = shared_prefix_attention(*b)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_two_captured_graphs_replay_with_new_inputs():
    """Two graphs of one pool, replayed in turn with eager calls between."""
    kw = dict(window=None, return_lse=True)
    held = make(4, 1, 300, 200, 9, 3, 64, torch.bfloat16)
    w = torch.zeros(4, 3, 200, device=DEV)
    shared_prefix_attention(*held, weights=w, **kw)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(shared_prefix_attention(*held, weights=w, **kw))
        graphs.append(g)
    for seed in range(4):
        new = make(4, 1, 300, 200, 9, 3, 64, torch.bfloat16, seed=seed + 3)
        for x, y in zip(held, new):
            x.copy_(y)
        for g, o in zip(graphs, outs):
            g.replay()
            got = [t.clone() for t in o]
            want = shared_prefix_attention(*new, weights=w, **kw)
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y), seed


@pytest.mark.parametrize("p", [300, 1700])  # in one launch, in parts
def test_captured_without_weights(p):
    held = make(4, 1, p, 200, 9, 3, 64, torch.bfloat16)
    shared_prefix_attention(*held, return_lse=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = shared_prefix_attention(*held, return_lse=True)
    for seed in range(3):
        new = make(4, 1, p, 200, 9, 3, 64, torch.bfloat16, seed=seed + 3)
        for x, y in zip(held, new):
            x.copy_(y)
        g.replay()
        got = [t.clone() for t in outs]
        want = shared_prefix_attention(*new, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), seed


@pytest.mark.parametrize("p", [800, 1700])  # in one launch, in parts
def test_same_inputs_same_bits(p):
    case = make(9, 2, p, 300, 9, 3, 64, torch.bfloat16)
    first = shared_prefix_attention(*case, return_lse=True)
    for _ in range(4):
        again = shared_prefix_attention(*case, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_refusals():
    q, kp, vp, k, v, lens = make(2, 1, 20, 30, 6, 2, 64, torch.bfloat16)
    w = torch.zeros(2, 2, 30, device=DEV)
    q80 = torch.zeros(2, 1, 6, 80, dtype=q.dtype, device=DEV)
    k80 = torch.zeros(2, 30, 2, 80, dtype=q.dtype, device=DEV)
    bad = [
        (dict(q=q.cpu()), "GPU"), (dict(q=q.float()), "bf16"), (dict(q=q[0]), "q must"),
        (dict(q=q[:1]), "go with"), (dict(v=v[:, :20]), "go with"), (dict(q=q[:, :, :5]), "go with"),
        (dict(k=k.half()), "type"), (dict(k_prefix=kp.half()), "type"),
        (dict(k_prefix=None), "prefix"), (dict(v_prefix=vp[:10]), "prefix"),
        (dict(k_prefix=kp[:, :1], v_prefix=vp[:, :1]), "prefix"),
        (dict(lens=lens.long()), "lens"), (dict(lens=lens[:1]), "lens"), (dict(lens=lens.cpu()), "lens"),
        (dict(window=0), "window"), (dict(weights=w.half()), "weights"),
        (dict(weights=w[..., :20]), "weights"), (dict(weights_out=w.transpose(0, 1)), "weights"),
        (dict(k=torch.zeros(k.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(k.shape)), "16 bytes"),
        (dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)), "16 bytes"),
        (dict(v=torch.zeros(2, 30, 2, 64 * 9, dtype=q.dtype, device=DEV)[..., ::9]), "16 bytes"),
        (dict(k_prefix=torch.zeros(20, 2, 64 * 17, dtype=q.dtype, device=DEV)[..., ::17]), "16 bytes"),
    ]
    for change, needle in bad:
        args = dict(q=q, k_prefix=kp, v_prefix=vp, k=k, v=v, lens=lens) | change
        with pytest.raises(ValueError, match=needle):
            shared_prefix_attention(*[args.pop(n) for n in ("q", "k_prefix", "v_prefix", "k", "v",
                                                            "lens")], **args)
    both = torch.zeros(2 * 60 + 8, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        shared_prefix_attention(q, kp, vp, k, v, lens, weights=both[:120].view(2, 2, 30),
                                weights_out=both[8:].view(2, 2, 30))
    with pytest.raises(ValueError, match="forward only"):
        shared_prefix_attention(q.clone().requires_grad_(), kp, vp, k, v, lens)
    big = make(1, 33, 5, 40, 2, 1, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="at most 64"):
        shared_prefix_attention(*big, weights=torch.zeros(1, 1, 40, device=DEV))
    with pytest.raises(RuntimeError, match="head_dim"):
        shared_prefix_attention(q80, None, None, k80, k80, lens)
    with pytest.raises(RuntimeError, match="scale"):
        shared_prefix_attention(q, kp, vp, k, v, lens, scale=-1.0)
