"""
penalize_logits (nsmoe_penalize_logits) against the definition in 64 bits: every term alone and
all together, histories that are empty, full, one token long, all one token or out of the
vocabulary, rows that the mask empties, NaN and infinities in masked places, odd vocabularies.

Bound: the penalty's product or quotient, the frequency's product, two subtractions and the
bias's sum round once each, at most 2^-24 of the largest intermediate value; the result is
rounded to the output's type, half a step.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import penalize_logits  # noqa: E402

DEV = "cuda"
NEG = float("-inf")


def ref(x, history, lens, prompt, rep, freq, pres, bias, mask):
    """(values in fp64, the largest intermediate value of each) on the CPU."""
    x = x.double().cpu().clone()
    b, v = x.shape
    big = x.abs()
    for i in range(b):
        if history is not None:
            n = history.shape[1] if lens is None else int(lens[i])
            p = 0 if prompt is None else int(prompt[i])
            ids = history[i, :n].cpu()
            for at, part in ((0, ids), (1, ids[p:])):
                part = part[(part >= 0) & (part < v)]
                tok, num = torch.unique(part, return_counts=True)
                if at == 0 and rep is not None:
                    r = float(rep[i])
                    x[i, tok] = torch.where(x[i, tok] > 0, x[i, tok] / r, x[i, tok] * r)
                if at == 1:
                    f = 0.0 if freq is None else float(freq[i])
                    q = 0.0 if pres is None else float(pres[i])
                    big[i, tok] = big[i, tok] + x[i, tok].abs() + f * num + abs(q)
                    x[i, tok] -= f * num + q
        big[i] = torch.maximum(big[i], x[i].abs())
    if bias is not None:
        x = x + bias.double().cpu()
        big = big + bias.double().abs().cpu()
    if mask is not None:
        col = torch.arange(v)
        on = (mask.cpu().long()[..., col // 32] >> (col % 32)) & 1
        x = torch.where(on.expand(b, v) != 0, x, NEG)
    return x, big


def check(got, want, big):
    fi = torch.finfo(got.dtype)
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    bound = (5 * 2.0 ** -24 * big + fi.eps / 2 * want.abs()) * (1 + 2 * fi.eps) + fi.smallest_normal
    err = (got - want).abs()
    assert (err[fine] <= bound[fine]).all(), float((err - bound)[fine].max())


def make(b, v, n, dtype, seed=0, terms="rfpbm"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, v, generator=g) * 3).to(dtype).to(DEV)
    ids = (v ** torch.rand(b, n, generator=g, dtype=torch.float64)).long() - 1
    ids = torch.where(torch.rand(b, n, generator=g) < 0.05, torch.tensor(-1), ids)
    ids[:, n // 2:n // 2 + 1] = v  # one past the vocabulary
    lens = torch.randint(0, n + 1, (b,), generator=g, dtype=torch.int32)
    kw = dict(history=ids.to(DEV), lens=lens.to(DEV), prompt_lens=(lens // 2).int().to(DEV))
    if "r" in terms:
        kw["repetition"] = (0.5 + 2 * torch.rand(b, generator=g)).to(DEV)
    if "f" in terms:
        kw["frequency"] = torch.randn(b, generator=g).to(DEV)
    if "p" in terms:
        kw["presence"] = torch.randn(b, generator=g).to(DEV)
    if "b" in terms:
        kw["bias"] = torch.randn(b, v, generator=g).to(DEV)
    if "m" in terms:
        w = torch.randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), generator=g)
        w[b // 2] = 0  # a row that allows nothing
        kw["mask"] = w.to(torch.int32).to(DEV)
    return x, kw


def run(x, kw, **more):
    kw = dict(kw)
    h, l = kw.pop("history", None), kw.pop("lens", None)
    return penalize_logits(x, h, l, **kw, **more)


def want(x, kw):
    return ref(x, *(kw.get(n) for n in ("history", "lens", "prompt_lens", "repetition",
                                        "frequency", "presence", "bias", "mask")))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,v,n", [(1, 32768, 512), (3, 1001, 40), (2, 1, 3), (5, 8, 1),
                                   (2, 33, 300), (300, 1030, 17), (2, 131072, 5000),
                                   (4, 17000, 2)])
def test_all_terms(dtype, b, v, n):
    print(f"[logits] {dtype} {(b, v, n)}", flush=True)
    x, kw = make(b, v, n, dtype, seed=v)
    check(run(x, kw), *want(x, kw))


@pytest.mark.parametrize("terms", ["", "r", "f", "p", "b", "m", "rp", "bm"])
def test_each_term_alone(terms):
    x, kw = make(4, 5003, 64, torch.float32, seed=7, terms=terms)
    check(run(x, kw), *want(x, kw))


def test_without_history_lengths_or_prompt():
    x, kw = make(3, 2000, 50, torch.bfloat16, seed=3)
    for gone in (("lens",), ("prompt_lens",), ("lens", "prompt_lens")):
        some = {k: t for k, t in kw.items() if k not in gone}
        check(run(x, some), *want(x, some))
    only = {k: kw[k] for k in ("bias", "mask")}
    check(run(x, only), *want(x, only))
    none = dict(kw, history=kw["history"][:, :0], lens=torch.zeros_like(kw["lens"]))
    check(run(x, none), *want(x, none))


def test_lengths_past_the_history_stop_at_its_end():
    x, kw = make(3, 500, 20, torch.float32, seed=5, terms="rfp")
    over = dict(kw, lens=torch.tensor([21, 1 << 30, -4], dtype=torch.int32, device=DEV))
    fits = dict(kw, lens=torch.tensor([20, 20, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(run(x, over), run(x, fits))


def test_one_token_many_times_counts_exactly():
    x = torch.zeros(1, 64, device=DEV)
    h = torch.full((1, 70_000), 5, device=DEV)
    one = torch.ones(1, device=DEV)
    y = penalize_logits(x, h, frequency=one)
    assert float(y[0, 5]) == -70_000.0 and int((y != 0).sum()) == 1


def test_masked_places_may_hold_anything():
    x, kw = make(2, 777, 8, torch.float32, seed=9, terms="m")
    on = (kw["mask"].cpu().long()[:, torch.arange(777) // 32] >> (torch.arange(777) % 32)) & 1
    junk = torch.tensor([float("nan"), float("inf"), NEG])[torch.arange(777) % 3].to(DEV)
    x = torch.where(on.to(DEV) == 0, junk, x)
    y = run(x, kw)
    assert torch.equal(y == NEG, on.to(DEV) == 0) and not y.isnan().any()


def test_infinities_and_nan_that_are_allowed_stay():
    x = torch.tensor([[float("nan"), float("inf"), NEG, 1.0]], device=DEV)
    h = torch.tensor([[0, 1, 2, 3]], device=DEV)
    f = lambda v: torch.full((1,), v, device=DEV)
    y = penalize_logits(x, h, repetition=f(2.0), frequency=f(0.5), presence=f(0.25))
    assert y[0, 0].isnan() and y[0, 1] == float("inf") and y[0, 2] == NEG and y[0, 3] == -0.25


def test_strides_broadcast_rows_and_outputs():
    x, kw = make(4, 1000, 30, torch.bfloat16, seed=11)
    wide = torch.zeros(4, 1011, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:1003] = x
    view = wide[:, 3:1003]
    base = run(x, kw)
    assert torch.equal(run(view, kw), base)
    row = dict(kw, bias=kw["bias"][0], mask=kw["mask"][0])
    full = dict(kw, bias=kw["bias"][:1].expand(4, -1).contiguous(),
                mask=kw["mask"][:1].expand(4, -1).contiguous())
    assert torch.equal(run(x, row), run(x, full))
    f32 = torch.empty(4, 1000, device=DEV)
    assert run(x, kw, out=f32) is f32
    check(f32, *want(x, kw))
    assert torch.equal(f32.to(torch.bfloat16), base)
    # in place in a wider buffer: the columns beside it stay
    assert run(view, kw, out=view) is view
    assert torch.equal(view, base) and not wide[:, :3].any() and not wide[:, 1003:].any()


def test_captured_call_replays_with_new_inputs():
    x, kw = make(8, 4096, 100, torch.bfloat16, seed=13)
    held = {k: t.clone() for k, t in kw.items()}
    sx = x.clone()
    run(sx, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(sx, held)
    for seed in (14, 15, 16):
        x2, kw2 = make(8, 4096, 100, torch.bfloat16, seed=seed)
        sx.copy_(x2)
        for k, t in kw2.items():
            held[k].copy_(t)
        graph.replay()
        eager = run(x2, kw2)
        torch.cuda.synchronize()
        assert torch.equal(y, eager), seed


def test_refusals():
    x, kw = make(2, 100, 5, torch.float32, seed=1)
    bad = [
        (dict(x=x.cpu()), "GPU"), (dict(x=x[0]), "batch, vocab"), (dict(x=x.double()), "bf16"),
        (dict(x=x.t()), "contiguous"), (dict(history=kw["history"].int()), "history"),
        (dict(history=kw["history"][:1]), "rows"), (dict(history=kw["history"][0]), "history"),
        (dict(lens=kw["lens"].long()), "lens"), (dict(lens=kw["lens"][:1]), "lens"),
        (dict(prompt_lens=kw["lens"].cpu()), "prompt_lens"),
        (dict(repetition=kw["repetition"].double()), "repetition"),
        (dict(bias=kw["bias"].half()), "bias"), (dict(bias=kw["bias"][:, :99]), "bias"),
        (dict(mask=kw["mask"][:, :3]), "mask"), (dict(mask=kw["mask"].long()), "mask"),
        (dict(out=torch.empty(2, 100, device=DEV, dtype=torch.float16)), "out"),
        (dict(out=torch.empty(100, device=DEV).expand(2, 100)), "out"),
    ]
    for change, needle in bad:
        args = dict(kw, x=x) | change
        with pytest.raises(ValueError, match=needle):
            run(args.pop("x"), args)
    with pytest.raises(ValueError, match="forward only"):
        penalize_logits(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="need a history"):
        penalize_logits(x, frequency=kw["frequency"])
    big = torch.zeros(2 * 100 + 8, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        penalize_logits(big[:200].view(2, 100), bias=kw["bias"], out=big[8:].view(2, 100))
