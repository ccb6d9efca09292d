"""
The generation operators run together, as a decoder uses them: Decoder.prefix and Decoder.step
against the whole sequence run at once, eviction in mid-sequence, and penalties on the logits.

The yardstick for the decoder's logits: the prefill path (Decoder.forward on the kernels) and
the step path round at the same places (the projections, the norms, the probabilities, the
experts; the step's rotation rounds once where the prefill's rounds each product), so against
the same decoder in fp32 torch their errors are of one size; a factor of 2 covers the spread of
two such errors.  All experts are routed (top_k = n_experts), so no rounding can change an
expert's choice.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import (cache_evict, penalize_logits, rotary_embed,  # noqa: E402
                             rotary_frequencies, shared_prefix_attention)
from nanospeaker_amd.decoder import Decoder, DecoderConfig  # noqa: E402

DEV = "cuda"


def decoders(dtype, layers=3, window=24, seed=0):
    """(the decoder in `dtype` on the kernels, the same weights in fp32 torch)."""
    torch.manual_seed(seed)
    cfg = DecoderConfig(vocab_size=512, n_layers=layers, n_experts=6, top_k=6, window=window,
                        global_every=2)
    d = Decoder(cfg)
    with torch.no_grad():
        for name, p in d.named_parameters():
            if name.endswith("gamma"):
                p.copy_(1 + 0.2 * torch.randn_like(p))
            elif "embed" in name:
                p.mul_(20)
    d = d.to(dtype)
    plain = Decoder(cfg, kernel=False)
    plain.load_state_dict({k: v.float() for k, v in d.state_dict().items()})
    return d.to(DEV).eval(), plain.to(DEV).eval()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,steps", [(40, [1, 1, 3, 1, 7, 1]), (130, [5, 1, 30]), (0, [2, 1, 1]),
                                     (1, [1])])
def test_steps_match_the_whole_sequence(dtype, P, steps):
    print(f"[generation] {dtype} prefix {P} steps {steps}", flush=True)
    d, plain = decoders(dtype)
    B, n = 5, sum(steps)
    g = torch.Generator().manual_seed(1)
    pre = torch.randint(0, 512, (P,), generator=g).to(DEV)
    new = torch.randint(0, 512, (B, n), generator=g).to(DEV)
    whole = torch.cat((pre.expand(B, P), new), dim=1)
    with torch.no_grad():
        exact = plain(whole)[:, P:]
        prefill = d(whole)[:, P:]
    cache = d.prefix(pre, B, rows=n, weights=True)
    got, at = [], 0
    for s in steps:
        got.append(d.step(new[:, at:at + s], cache))
        at += s
    got = torch.cat(got, dim=1)
    assert got.shape == exact.shape and got.dtype == dtype
    a, b = rel(got, exact), rel(prefill, exact)
    print(f"  steps {a:.2e}, prefill {b:.2e} off the fp32 decoder", flush=True)
    assert a <= 2 * b
    assert (cache.positions == P + n).all() and cache.filled == n
    for lens in cache.lens:
        assert (lens == n).all()


def test_eviction_in_mid_sequence():
    """After the eviction a layer attends to exactly the kept rows, heavy ones among them, and
    the steps go on; the kept rows and weights are the old cache's."""
    d, _ = decoders(torch.bfloat16)
    B, P = 3, 20
    g = torch.Generator().manual_seed(2)
    tok = lambda n: torch.randint(0, 512, (B, n), generator=g).to(DEV)
    cache = d.prefix(tok(P)[0], B, rows=64, weights=True)
    d.step(tok(30), cache)  # 90 queries a key head: accumulated in pieces
    for _ in range(4):
        d.step(tok(1), cache)
    evicted = [i for i, w in enumerate(cache.weights) if w is not None]
    assert evicted == [0, 2]
    old = {i: (cache.k[i].clone(), cache.v[i].clone(), cache.weights[i].clone()) for i in evicted}
    # every query gives each key head's three heads a weight of 1 each, prefix included
    for i in evicted:
        total = old[i][2].sum(-1)
        assert (total > 0).all() and (total <= 34 * 3 * (1 + 1e-4)).all()
    cache.evict(12, recent=4, sinks=1)
    for i in evicted:
        k, v, w = old[i]
        assert (cache.lens[i] == 12).all()
        for b in range(B):
            for h in range(3):
                heavy = w[b, h, 1:30].topk(7).values.min()
                keep = [0] + [j for j in range(1, 30) if w[b, h, j] >= heavy] + [30, 31, 32, 33]
                assert torch.equal(cache.k[i][b, :12, h], k[b, keep, h])
                assert torch.equal(cache.v[i][b, :12, h], v[b, keep, h])
                assert torch.equal(cache.weights[i][b, h, :12], w[b, h, keep])
                assert not cache.weights[i][b, h, 12:].any()
    assert (cache.lens[1] == 34).all() and cache.filled == 34
    logits = d.step(tok(1), cache)
    assert logits.isfinite().all()
    assert (cache.lens[0] == 13).all() and (cache.lens[1] == 35).all()
    assert (cache.positions == P + 35).all()


def test_greedy_loop_with_penalties():
    """A loop as a program writes it: step, penalise what was said, mask, choose."""
    d, _ = decoders(torch.bfloat16)
    B, V = 4, 512
    pre = torch.arange(10, device=DEV)
    cache = d.prefix(pre, B, rows=20)
    history = torch.full((B, 30), -1, dtype=torch.int64, device=DEV)
    history[:, :10] = pre
    lens = torch.full((B,), 10, dtype=torch.int32, device=DEV)
    prompt = lens.clone()
    tok = torch.arange(B, device=DEV)[:, None]
    one = torch.ones(B, device=DEV)
    allowed = torch.full((16,), -1, dtype=torch.int32, device=DEV)
    allowed[0] = 0  # the grammar forbids tokens 0 .. 31
    for _ in range(20):
        logits = d.step(tok, cache)[:, -1]
        out = penalize_logits(logits, history, lens, prompt_lens=prompt, presence=1e4 * one,
                              mask=allowed)
        tok = out.argmax(-1, keepdim=True)
        history.scatter_(1, lens[:, None].long(), tok)
        lens += 1
    said = history[:, 10:]
    assert (said >= 32).all()
    for row in said.tolist():  # a penalty that large lets no token come twice
        assert len(set(row)) == 20


def test_refusals():
    d, plain = decoders(torch.bfloat16)
    tok = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    cache = d.prefix(torch.arange(5, device=DEV), 2, rows=2)
    with pytest.raises(ValueError, match="expected"):
        d.step(tok[:1], cache)
    d.step(tok, cache)
    with pytest.raises(ValueError, match="more than"):
        d.step(tok.expand(2, 2), cache)
    d.step(tok, cache)
    with pytest.raises(ValueError, match="more than"):
        d.step(tok, cache)
    with pytest.raises(ValueError, match="without weights"):
        cache.evict(1)
    with pytest.raises(RuntimeError, match="kernel path"):
        plain.prefix(torch.arange(5, device=DEV), 2, rows=2)
    with pytest.raises(RuntimeError, match="kernel path"):
        plain.step(tok, plain.prefix(torch.arange(0, device=DEV), 2, rows=2))
    with pytest.raises(ValueError, match="expected \\[P\\]"):
        d.prefix(torch.zeros(1, 5, dtype=torch.int64, device=DEV), 2, rows=2)
    with pytest.raises(ValueError, match="0 rows"):
        d.prefix(torch.arange(5, device=DEV), 2, rows=0)


def test_a_captured_step_is_refused():
    d, _ = decoders(torch.bfloat16, layers=1)
    cache = d.prefix(torch.arange(4, device=DEV), 2, 8)
    idx = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    d.step(idx, cache)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(g):
            cache.reserve(idx)
    d.step(idx, cache)
    assert cache.filled == 2


def test_written_operands_are_known_to_autograd():
    """What a call writes into its operands counts as an in-place change: a backward that saved
    the old values raises rather than use the new ones."""
    leaf = torch.randn(1, 3, 2, 64, device=DEV, requires_grad=True)
    lens = torch.full((1,), 3, dtype=torch.int32, device=DEV)
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(3, device=DEV)[None]

    def turn(t):
        rotary_embed(t, None, pos, freqs, inplace=True)

    def penalize(t):
        penalize_logits(t[0, 0], out=t[0, 0])

    def attend(t):
        kv = torch.randn(1, 64, 2, 64, device=DEV, dtype=torch.bfloat16)
        shared_prefix_attention(kv[:, :3], None, None, kv, kv, lens,
                                weights_out=t.view(-1)[:128].view(1, 2, 64))

    def evict(t):
        kv = torch.randn(1, 3, 2, 64, device=DEV)
        cache_evict(kv, kv, torch.zeros(1, 2, 3, device=DEV), lens, 2,
                    out=(t, torch.empty_like(kv), torch.empty(1, 2, 3, device=DEV)))

    for write in (turn, penalize, attend, evict):
        print(f"[generation] {write.__name__}", flush=True)
        saved = leaf * 1.0
        loss = (saved * saved).sum()
        write(saved.detach())
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()


def test_outputs_that_want_a_gradient_are_refused():
    x = torch.zeros(2, 8, device=DEV)
    with pytest.raises(ValueError, match="gradient"):
        penalize_logits(x, out=torch.zeros_like(x).requires_grad_())
    kv = torch.zeros(1, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
    lens = torch.full((1,), 4, dtype=torch.int32, device=DEV)
    w = torch.zeros(1, 1, 4, device=DEV)
    with pytest.raises(ValueError, match="gradient"):
        shared_prefix_attention(kv[:, :1], None, None, kv, kv, lens,
                                weights_out=torch.zeros_like(w).requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        cache_evict(kv, kv, w, lens, 2, out=(torch.zeros_like(kv).requires_grad_(),
                                             torch.zeros_like(kv), torch.zeros_like(w)))
