"""
The generation operators' C boundary without a GPU: struct layouts, refusals before anything is
launched, calls of nothing, the rotary frequencies, and the attention's tile copies restated
lane by lane (where each 16-byte chunk of a tile lands, and that the fragment reads find it).
"""

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from nanospeaker_amd import _native as nat
from nanospeaker_amd import cache_evict, penalize_logits, rotary_embed, rotary_frequencies
from nanospeaker_amd import shared_prefix_attention

HEADER = Path(__file__).resolve().parents[1] / "include" / "nsmoe.h"
STRUCTS = {"nsmoe_rope_args": nat.RopeArgs, "nsmoe_logits_args": nat.LogitsArgs,
           "nsmoe_evict_args": nat.EvictArgs, "nsmoe_prefix_attn_args": nat.PrefixAttnArgs}


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layouts_match_the_header(name):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    fields = re.findall(r"^\s*(.+?)\b(\w+)(?:\[(\d)\])?;", body, re.M)
    size = {"int32_t": 4, "float": 4, "int64_t": 8}
    mirror, at = STRUCTS[name], 0
    assert [f for _, f, _ in fields] == [f for f, _ in mirror._fields_]
    for ctype, field, count in fields:
        n = 8 if "*" in ctype else size[ctype.strip()]
        at = -(-at // n) * n
        assert getattr(mirror, field).offset == at, field
        at += n * int(count or 1)
        assert getattr(mirror, field).size == n * int(count or 1), field
    assert ctypes.sizeof(mirror) == -(-at // 8) * 8


def refused(fn, args, needle, *more):
    assert fn(args, *more, None) == 1
    assert needle in nat.lib().nsmoe_last_error().decode()


def rope(**kw):
    s = (1024, 512, 64)
    base = dict(dtype=0, amplitude=1.0, batch=1, n_tokens=4, n_q=2, n_k=1, head_dim=64, rot_dim=64,
                q=16, k=16, q_out=32, k_out=32, q_stride=s, k_stride=s, q_out_stride=s,
                k_out_stride=s, positions=16, pos_stride=(4, 1), freqs=16)
    return nat.RopeArgs(**(base | kw))


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=3), "dtype"), (dict(head_dim=0), "head_dim"), (dict(head_dim=1025), "head_dim"),
    (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"),
    (dict(n_q=0, n_k=0), "n_q"), (dict(n_k=-1), "n_k"), (dict(batch=-1), "batch"),
    (dict(q=None), "NULL"), (dict(k_out=None), "NULL"), (dict(freqs=None), "NULL"),
    (dict(positions=None), "NULL"), (dict(q=17), "misaligned"), (dict(dtype=2, k=18), "misaligned")])
def test_rope_refuses(kw, needle):
    refused(nat.lib().nsmoe_rope, rope(**kw), needle)


def logits(**kw):
    base = dict(dtype=0, out_dtype=0, batch=2, vocab=100, logits=16, out=32, logits_stride=100,
                out_stride=100, history=16, history_stride=8, history_cap=8)
    return nat.LogitsArgs(**(base | kw))


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=3), "dtype"), (dict(dtype=0, out_dtype=1), "dtype"), (dict(batch=65536), "batch"),
    (dict(vocab=-1), "vocab"), (dict(history_cap=-1), "history"), (dict(logits=None), "NULL"),
    (dict(out=None), "NULL"), (dict(history=None), "NULL"), (dict(logits=17), "misaligned"),
    (dict(bias=18), "misaligned"), (dict(dtype=0, out_dtype=2, out=18), "misaligned")])
def test_logits_refuse(kw, needle):
    refused(nat.lib().nsmoe_penalize_logits, logits(**kw), needle)


def evict(**kw):
    s = (2048, 64, 32)
    base = dict(elem_bytes=2, n_kv_heads=2, head_dim=32, batch=2, cap=32, out_cap=16, budget=16,
                recent=2, sinks=2, k=16, v=16, k_out=16, v_out=16, k_stride=s, v_stride=s,
                k_out_stride=s, v_out_stride=s, weights=16, weights_out=16,
                weights_stride=(64, 32), weights_out_stride=(32, 16), lens=16, lens_out=16,
                index=16)
    return nat.EvictArgs(**(base | kw))


@pytest.mark.parametrize("kw,needle", [
    (dict(elem_bytes=1), "elements"), (dict(head_dim=0), "head_dim"), (dict(n_kv_heads=0), "heads"),
    (dict(cap=-1), "capacity"), (dict(budget=0), "budget"), (dict(budget=17), "budget"),
    (dict(recent=15), "exceed"), (dict(sinks=-1), "exceed"), (dict(k=None), "NULL"),
    (dict(index=None), "NULL"), (dict(lens=None), "NULL"), (dict(k=17), "misaligned"),
    (dict(weights=18), "misaligned")])
def test_evict_refuses(kw, needle):
    refused(nat.lib().nsmoe_cache_evict, evict(**kw), needle)


def attn(**kw):
    base = dict(dtype=0, head_dim=64, n_heads=9, n_kv_heads=3, batch=2, n_new=1, prefix_len=8,
                cap=16, window=0, scale=0.125, q=16, k_prefix=16, v_prefix=16, k=16, v=16,
                q_stride=(576, 576, 64), kp_stride=(192, 64), vp_stride=(192, 64),
                k_stride=(3200, 192, 64), v_stride=(3200, 192, 64), lens=16, out=16)
    return nat.PrefixAttnArgs(**(base | kw))


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=2), "16-bit"), (dict(head_dim=96), "head_dim"), (dict(n_kv_heads=2), "n_heads"),
    (dict(n_kv_heads=0), "n_heads"), (dict(batch=-1), "batch"), (dict(cap=1 << 29), "cache"),
    (dict(prefix_len=-1), "prefix"), (dict(window=-1), "window"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(n_new=22, weights_out=16), "at most 64"), (dict(n_new=0), "no new"),
    (dict(q=None), "NULL"), (dict(k_prefix=None), "NULL"), (dict(v=None), "NULL"),
    (dict(lens=None), "NULL"), (dict(k=24), "16 bytes"), (dict(kp_stride=(196, 64)), "16 bytes"),
    (dict(q_stride=(576, 576, 60)), "16 bytes")])
def test_prefix_attention_refuses(kw, needle):
    refused(nat.lib().nsmoe_prefix_attention, attn(**kw), needle, 16, 1 << 30)


def test_prefix_attention_wants_its_workspace():
    a = attn(prefix_len=4096)
    lib = nat.lib()
    need = lib.nsmoe_prefix_attention_workspace_size(a)
    assert need > 0
    assert lib.nsmoe_prefix_attention(a, 256, need - 1, None) == 3
    assert lib.nsmoe_prefix_attention(a, None, need, None) == 3
    assert lib.nsmoe_prefix_attention(a, 264, need, None) == 1
    with_weights = attn(prefix_len=4096, weights_out=16)
    assert lib.nsmoe_prefix_attention_workspace_size(with_weights) > need


def test_calls_of_nothing():
    lib = nat.lib()
    assert lib.nsmoe_rope(rope(batch=0, q=None), None) == 0
    assert lib.nsmoe_rope(rope(n_tokens=0, q=None), None) == 0
    assert lib.nsmoe_penalize_logits(logits(batch=0, logits=None), None) == 0
    assert lib.nsmoe_penalize_logits(logits(vocab=0, logits=None), None) == 0
    assert lib.nsmoe_cache_evict(evict(batch=0, k=None), None) == 0
    assert lib.nsmoe_prefix_attention(attn(batch=0, q=None), None, 0, None) == 0
    for fn, more in ((lib.nsmoe_rope, ()), (lib.nsmoe_penalize_logits, ()),
                     (lib.nsmoe_cache_evict, ()), (lib.nsmoe_prefix_attention, (None, 0))):
        assert fn(None, *more, None) == 1


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        rotary_embed(x, None, torch.zeros(1, 2, dtype=torch.int64), rotary_frequencies(64)[0])
    with pytest.raises(ValueError, match="GPU"):
        shared_prefix_attention(x[:, :1], None, None, x, x, one)
    with pytest.raises(ValueError, match="GPU"):
        cache_evict(x, x, torch.zeros(1, 2, 2), one, 1)
    with pytest.raises(ValueError, match="GPU"):
        penalize_logits(torch.zeros(1, 8))


# ---- the rotary frequencies -----------------------------------------------------------------

def test_plain_linear_and_ntk_frequencies():
    f, a = rotary_frequencies(64, 500_000.0)
    assert f.dtype == torch.float64 and a == 1.0
    for j in (0, 1, 17, 31):
        assert math.isclose(float(f[j]), 500_000.0 ** (-2 * j / 64), rel_tol=1e-14)
    assert torch.equal(rotary_frequencies(64, 500_000.0, "linear", 4.0)[0], f / 4)
    n, a = rotary_frequencies(64, 500_000.0, "ntk", 4.0)
    assert a == 1.0 and float(n[0]) == 1.0
    assert math.isclose(float(n[31]), float(f[31]) / 4, rel_tol=1e-12)


def test_yarn_frequencies():
    f, _ = rotary_frequencies(128, 10_000.0)
    y, a = rotary_frequencies(128, 10_000.0, "yarn", 8.0, original_length=2048)
    assert math.isclose(a, 0.1 * math.log(8.0) + 1.0)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32])
    assert torch.allclose(y[turns <= 1], f[turns <= 1] / 8, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any()
    g = (turns[mid] - 1) / 31
    assert torch.allclose(y[mid], f[mid] * (g + (1 - g) / 8), rtol=1e-13, atol=0)


@pytest.mark.parametrize("args", [(63,), (0,), (64, 0.0), (64, 1e4, "other"), (64, 1e4, "ntk", 0.5),
                                  (2, 1e4, "ntk", 2.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        rotary_frequencies(*args)


# ---- the attention's tile copies ------------------------------------------------------------

def swz(d, r):
    return ((((r >> 1) & 3) << 1) | ((r >> 3) & 1)) if d == 64 else ((r & 7) << 1) | ((r >> 3) & 1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keys", [32, 64])
def test_tile_copies_fill_the_tile_once_and_reads_find_their_chunks(d, keys):
    """Copy u of a tile: lane l fetches chunk (l % CPR) ^ swz(r) of row r = u RPC + l / CPR into
    bytes 1024 u + 16 l.  A read of chunk c of row r goes to r 2 d + 16 (c ^ swz(r))."""
    cpr, rpc = d // 8, 1024 // (2 * d)
    place = {}
    for u in range(keys // rpc):
        for lane in range(64):
            r = u * rpc + lane // cpr
            at = 1024 * u + 16 * lane
            assert at not in place and at + 16 <= keys * 2 * d
            place[at] = (r, (lane % cpr) ^ swz(d, r))
    assert len(place) == keys * cpr
    for r in range(keys):
        for c in range(cpr):
            assert place[r * 2 * d + 16 * (c ^ swz(d, r))] == (r, c)


@pytest.mark.parametrize("d", [64, 128])
def test_fragment_reads_spread_over_the_banks(d):
    """A K fragment read (16 rows, one chunk) touches each 16-byte slot of a 256-byte line as
    evenly as rows allow; a transposed V read (8 rows, two chunks) no slot twice."""
    for c in range(d // 8):
        slots = [(r * 2 * d + 16 * (c ^ swz(d, r))) % 256 // 16 for r in range(16)]
        assert max(slots.count(s) for s in slots) == 1
    for db in range(d // 16):
        slots = [(r * 2 * d + 16 * ((2 * db + e) ^ swz(d, r))) % 256 // 16
                 for r in range(8) for e in (0, 1)]
        assert len(set(slots)) == 16
