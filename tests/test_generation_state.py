"""
What the generation operators keep track of, on the CPU: a decode cache whose step raised part
way, its count of rows, which heads a rotation's backward turns, and which attentions are split
into parts.
"""

import pytest
import torch

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import _native as nat, rope  # noqa: E402
from nanospeaker_amd.cache import DecodeCache  # noqa: E402


def make(rows=4, layers=2):
    return DecodeCache([None] * layers, [], 0, 2, rows, 1, 8, torch.float32, "cpu")


def step(cache, n, fail_at=None):
    cache.reserve(torch.zeros(2, n, dtype=torch.int64))
    for layer in range(2):
        if layer == fail_at:
            raise MemoryError
        cache.append(layer, torch.ones(2, n, 1, 8), torch.ones(2, n, 1, 8))
    cache.advance(n)


def test_rows_are_counted_and_bounded():
    cache = make()
    step(cache, 3)
    assert cache.filled == 3 and [t.tolist() for t in cache.lens] == [[3, 3], [3, 3]]
    with pytest.raises(ValueError, match="rows"):
        step(cache, 2)
    step(cache, 1)
    assert cache.filled == 4 and cache.positions.tolist() == [4, 4]


def test_a_step_that_raised_part_way_ends_the_cache():
    """Layer 0 has its rows and layer 1 has not: another step would write behind them, past the
    cache's rows at last, and give the wrong attention before."""
    cache = make()
    with pytest.raises(MemoryError):
        step(cache, 2, fail_at=1)
    with pytest.raises(RuntimeError, match="anew"):
        step(cache, 2)


def test_a_step_that_wrote_nothing_can_be_made_again():
    cache = make()
    with pytest.raises(MemoryError):
        step(cache, 2, fail_at=0)
    step(cache, 2)
    assert cache.filled == 2


@pytest.mark.parametrize("need", [(True, False), (False, True), (True, True)])
def test_backward_turns_the_heads_that_want_it(monkeypatch, need):
    calls = []

    def launch(q, k, positions, freqs, interleaved, amplitude, inverse, inplace):
        calls.append((q is not None, k is not None, inverse))
        return tuple(None if t is None else t * 2 for t in (q, k))

    monkeypatch.setattr(rope, "_launch", launch)
    q = torch.ones(1, 2, 1, 4, requires_grad=need[0])
    k = torch.ones(1, 2, 1, 4, requires_grad=need[1])
    pos, freqs = torch.arange(2)[None], torch.ones(2, dtype=torch.float64)
    yq, yk = rope._Rotate.apply(q, k, pos, freqs, False, 1.0, False)
    (yq.sum() + yk.sum()).backward()
    assert calls == [(True, True, False), (*need, True)]
    for t, want in zip((q, k), need):
        assert (t.grad is not None) == want
        if want:
            assert torch.equal(t.grad, torch.full_like(t, 2))


@pytest.mark.parametrize("kw,split", [
    (dict(), False), (dict(prefix_len=0), False), (dict(prefix_len=1520), False),
    (dict(prefix_len=1521), True), (dict(head_dim=128, prefix_len=752), False),
    (dict(head_dim=128, prefix_len=753), True), (dict(prefix_len=4096, window=1024), False),
    (dict(prefix_len=4096, window=1536, n_new=2), True), (dict(weights_out=16), True),
    (dict(n_new=10), False), (dict(n_new=11), True), (dict(batch=400), True), (dict(cap=0), True)])
def test_short_contexts_need_no_workspace(kw, split):
    """One launch, without parts, for up to 32 columns a head over a short context."""
    base = dict(dtype=0, head_dim=64, n_heads=9, n_kv_heads=3, batch=2, n_new=1, prefix_len=8,
                cap=16, window=0, scale=0.125)
    lib = nat.lib()
    size = lib.nsmoe_prefix_attention_workspace_size(nat.PrefixAttnArgs(**(base | kw)))
    assert (size > 0) == split
