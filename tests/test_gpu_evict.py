"""
cache_evict (nsmoe_cache_evict) against a plain sort: which rows stay (ties to the earlier row),
what moves with them, and what is left alone.  Every output is exact.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import cache_evict  # noqa: E402

DEV = "cuda"


def keep(w, n, budget, recent, sinks):
    """The rows that stay of one (sequence, head): w a list of floats."""
    if n <= budget:
        return list(range(n))
    big = lambda j: float("inf") if w[j] != w[j] else w[j]
    mid = sorted(range(sinks, n - recent), key=lambda j: (not w[j] != w[j], -big(j), j))
    return [*range(sinks), *sorted(mid[:budget - sinks - recent]), *range(n - recent, n)]


def make(b, s, h, d, dtype=torch.bfloat16, seed=0, ties=True):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, s, h, d, generator=g).to(dtype).to(DEV)
    v = torch.randn(b, s, h, d, generator=g).to(dtype).to(DEV)
    w = torch.exp(2 * torch.randn(b, h, s, generator=g)) * 1e-3
    if ties:
        w = torch.where(torch.rand(b, h, s, generator=g) < 0.4, w.mean(), w)
    lens = torch.randint(0, s + 1, (b,), generator=g, dtype=torch.int32)
    lens[0] = s
    return k, v, w.to(DEV), lens.to(DEV)


def check(k, v, w, lens, got, budget, recent, sinks):
    ko, vo, wo, idx, ln = (t.cpu() for t in got)
    k, v, w = k.cpu(), v.cpu(), w.cpu()
    for b, n in enumerate(lens.tolist()):
        n = max(0, min(n, k.shape[1]))
        m = min(n, budget)
        assert int(ln[b]) == m
        for h in range(k.shape[2]):
            at = torch.tensor(keep(w[b, h, :n].tolist(), n, budget, recent, sinks),
                              dtype=torch.int64)
            assert idx[b, h, :m].tolist() == at.tolist(), (b, h)
            assert (idx[b, h, m:] == -1).all()
            assert torch.equal(ko[b, :m, h], k[b, at, h]) and torch.equal(vo[b, :m, h], v[b, at, h])
            assert torch.equal(wo[b, h, :m].nan_to_num(nan=7.0), w[b, h, at].nan_to_num(nan=7.0))
        assert not ko[b, m:].any() and not vo[b, m:].any() and not wo[b, :, m:].any()


@pytest.mark.parametrize("b,s,h,d,budget,recent,sinks", [
    (1, 1, 1, 64, 1, 0, 0), (3, 50, 3, 64, 20, 5, 2), (2, 64, 2, 64, 64, 3, 1),
    (2, 63, 1, 64, 62, 62, 0), (2, 63, 1, 64, 62, 0, 62), (4, 1100, 3, 64, 1024, 64, 4),
    (2, 5000, 2, 128, 1, 0, 0), (2, 5000, 2, 128, 1, 1, 0), (1, 40_001, 2, 64, 3333, 77, 4),
    (2, 1000, 3, 63, 100, 7, 3), (2, 300, 2, 1, 17, 0, 1), (9, 129, 5, 80, 128, 10, 0)])
def test_rows_that_stay(b, s, h, d, budget, recent, sinks):
    print(f"[evict] {(b, s, h, d, budget, recent, sinks)}", flush=True)
    k, v, w, lens = make(b, s, h, d, seed=s)
    check(k, v, w, lens, cache_evict(k, v, w, lens, budget, recent=recent, sinks=sinks),
          budget, recent, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.int16])
def test_types(dtype):
    k, v, w, lens = make(2, 200, 2, 64)
    k, v = (k * 100).to(dtype), (v * 100).to(dtype)
    check(k, v, w, lens, cache_evict(k, v, w, lens, 90, recent=9), 90, 9, 0)


@pytest.mark.parametrize("value", [0.0, 1.5, -2.0])
def test_all_weights_equal_keeps_the_earliest(value):
    k, v, w, _ = make(2, 3000, 2, 64)
    w.fill_(value)
    lens = torch.full((2,), 3000, dtype=torch.int32, device=DEV)
    idx = cache_evict(k, v, w, lens, 700, recent=100, sinks=10)[3]
    want = [*range(600), *range(2900, 3000)]
    assert (idx.cpu() == torch.tensor(want, dtype=torch.int32)).all()


def test_weights_of_every_kind():
    """Negative, zero of both signs, denormal, infinite and NaN weights."""
    k, v, _, _ = make(1, 400, 1, 64)
    kinds = torch.tensor([float("nan"), float("inf"), float("-inf"), -1.0, -0.0, 0.0, 1e-42,
                          -1e-42, 3.0, 3.0000002])
    g = torch.Generator().manual_seed(3)
    w = kinds[torch.randint(0, 10, (1, 1, 400), generator=g)].to(DEV)
    lens = torch.tensor([400], dtype=torch.int32, device=DEV)
    for budget in (1, 39, 40, 41, 80, 150, 201, 240, 399):
        got = cache_evict(k, v, w, lens, budget)
        flat = [0.0 if x == 0 else x for x in w[0, 0].tolist()]  # -0 equals +0
        assert got[3][0, 0].tolist() == keep(flat, 400, budget, 0, 0), budget


def test_lengths_out_of_range_are_the_caches_ends():
    k, v, w, _ = make(3, 60, 2, 64)
    lens = torch.tensor([-5, 61, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    check(k, v, w, lens, cache_evict(k, v, w, lens, 30, recent=3), 30, 3, 0)


def test_given_buffers_keep_what_lies_behind():
    k, v, w, lens = make(3, 100, 2, 64)
    lens[1] = 7
    out = (torch.full((3, 55, 2, 64), 9.0, dtype=k.dtype, device=DEV),
           torch.full((3, 55, 2, 64), 9.0, dtype=k.dtype, device=DEV),
           torch.full((3, 2, 55), 9.0, device=DEV))
    r = cache_evict(k, v, w, lens, 40, recent=4, out=out)
    assert r[0] is out[0] and r[1] is out[1] and r[2] is out[2]
    fresh = cache_evict(k, v, w, lens, 40, recent=4)
    assert torch.equal(r[3], fresh[3]) and torch.equal(r[4], fresh[4])
    for b, m in enumerate(r[4].tolist()):
        for i in range(2):
            assert torch.equal(r[i][b, :m], fresh[i][b, :m]) and (r[i][b, m:] == 9).all()
        assert torch.equal(r[2][b, :, :m], fresh[2][b, :, :m]) and (r[2][b, :, m:] == 9).all()


def test_strides_and_alignment():
    """Heads before rows, column blocks of a wider row, and rows off the 16-byte alignment."""
    k, v, w, lens = make(2, 150, 3, 64)
    want = cache_evict(k, v, w, lens, 60, recent=6, sinks=1)
    wide = torch.zeros(2, 150, 3, 2, 65, dtype=k.dtype, device=DEV)
    wide[..., 0, 1:], wide[..., 1, 1:] = k, v
    for kk, vv in ((k.transpose(1, 2).contiguous().transpose(1, 2),
                    v.transpose(1, 2).contiguous().transpose(1, 2)),
                   (wide[..., 0, 1:], wide[..., 1, 1:])):
        ww = torch.zeros(2, 3, 2, 150, device=DEV)
        ww[:, :, 1] = w
        got = cache_evict(kk, vv, ww[:, :, 1], lens, 60, recent=6, sinks=1)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_empty_batch_and_empty_cache():
    k, v, w, lens = make(2, 10, 2, 64)
    r = cache_evict(k[:0], v[:0], w[:0], lens[:0], 5)
    assert r[0].shape == (0, 5, 2, 64) and r[4].shape == (0,)
    r = cache_evict(k[:, :0], v[:, :0], w[..., :0], lens, 5)
    assert not r[0].any() and (r[3] == -1).all() and not r[4].any()


def test_captured_call_replays_with_new_inputs():
    k, v, w, lens = make(3, 500, 2, 64)
    held = [t.clone() for t in (k, v, w, lens)]
    cache_evict(*held, 200, recent=20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache_evict(*held, 200, recent=20)
    for seed in (1, 2, 3):
        new = make(3, 500, 2, 64, seed=seed)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        want = cache_evict(*new, 200, recent=20)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), seed


def test_refusals():
    k, v, w, lens = make(2, 30, 2, 64)
    one, flat = k.clone(), k[:1].clone().expand(2, 30, 2, 64)
    bad = [
        (dict(k=k.cpu()), "GPU"), (dict(k=k.double(), v=v.double()), "byte"),
        (dict(v=v[:, :20]), "one 2- or 4-byte"), (dict(v=v.half()), "one 2- or 4-byte"),
        (dict(weights=w.double()), "weights"), (dict(weights=w[..., :20]), "weights"),
        (dict(lens=lens.long()), "lens"), (dict(lens=lens[:1]), "lens"),
        (dict(budget=0), "budget"), (dict(budget=3, recent=2, sinks=2), "budget"),
        (dict(recent=-1), "budget"), (dict(k=k.transpose(2, 3), v=v.transpose(2, 3)), "weights"),
        (dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
        (dict(out=(k, v, w)), "shares memory"), (dict(out=(one, one, w.clone())), "shares memory"),
        (dict(out=(flat, v.clone(), w.clone())), "share memory"),
        (dict(k=k[..., :0], v=v[..., :0]), "without"),
        (dict(weights=w.clone().requires_grad_()), "forward only"),
        (dict(out=(k[:, :5].clone(), v[:, :5].clone(), w[..., :5].clone())), "out must"),
    ]
    for change, needle in bad:
        args = dict(k=k, v=v, weights=w, lens=lens, budget=10) | change
        with pytest.raises(ValueError, match=needle):
            cache_evict(args.pop("k"), args.pop("v"), args.pop("weights"), args.pop("lens"),
                        args.pop("budget"), **args)
