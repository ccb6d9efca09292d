"""
rotary_embed (nsmoe_rope) against the rotation in 64 bits: both plane layouts, part of the
head, far and negative positions, ragged and strided operands, in place, and the gradient
against the formula's and against differences.

Bound on an element y1 = a (x1 c - x2 s): the angle is reduced in fp64 and rounded to fp32 at
most 2^-26 of a turn (2 pi 2^-26 < 1.6 * 2^-24) off, sin and cos are good to 2 ulp (2^-23 at
most below 1), the amplitude's product, the two products and the sum each round once: less
than 8 * 2^-24 of amplitude (|x1| + |x2|), and the result is rounded to the type, half a step.
The angle t itself is an fp64 product on both sides: the kernel rounds freq / (2 pi) twice (the
constant and the product) and its product with the position once, the reference its one product,
each by at most 2^-53 |t|; together 4 * 2^-53 |t| of an angle, which turns a plane by as much.
That is 5e-10 at position 10^6, and only tells at 10^10 and beyond.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("nanospeaker_amd.moe_kernel")
from nanospeaker_amd import rotary_embed, rotary_frequencies  # noqa: E402

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ref(x, positions, freqs, interleaved, amplitude, inverse=False):
    """([B, T, H, D] in fp64 on the CPU, the bound on another's error but its last rounding)."""
    x = x.detach().double().cpu()
    b, t, _, d = x.shape
    half = freqs.numel()
    ang = positions.expand(b, t).double().cpu()[..., None, None] * freqs.double().cpu()
    c, s = ang.cos() * amplitude, ang.sin() * amplitude * (-1.0 if inverse else 1.0)
    y, size = x.clone(), torch.zeros_like(x)
    i1 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i2 = i1 + (1 if interleaved else half)
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    rel = 8 * 2.0 ** -24 + 4 * 2.0 ** -53 * ang.abs()
    size[..., i1] = size[..., i2] = rel * (x[..., i1].abs() + x[..., i2].abs()) * amplitude
    return y, size


def check(name, got, want, slack):
    """Half a step of the type on top of the slack (and the type's smallest step)."""
    fi = torch.finfo(got.dtype)
    step = fi.eps / 2 * want.abs() * (1 + 1e-6) + fi.smallest_normal * fi.eps
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= slack * (1 + fi.eps) + step).all(), (name, float((err - slack - step).max()))


def make(b, t, hq, hk, d, dtype, seed=0, far=1000):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, t, hq + 2 * hk, d, generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, far, (b, 1), generator=g) + torch.arange(t)
    return qkv[:, :, :hq], qkv[:, :, hq:hq + hk], pos.to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,hq,hk,d,rot", [
    (1, 1, 9, 3, 64, 64), (3, 5, 9, 3, 64, 64), (2, 33, 4, 4, 128, 64), (1, 1200, 3, 1, 64, 24),
    (2, 7, 5, 1, 80, 80), (2, 9, 2, 1, 50, 10), (1, 3, 1, 1, 2, 2), (1, 4, 2, 2, 7, 6),
    (1, 2, 2, 1, 1024, 1024), (5, 700, 32, 8, 128, 128)])
def test_rotation(dtype, interleaved, b, t, hq, hk, d, rot):
    print(f"[rope] {dtype} interleaved={interleaved} {(b, t, hq, hk, d, rot)}", flush=True)
    q, k, pos = make(b, t, hq, hk, d, dtype)
    freqs, _ = rotary_frequencies(rot, device=DEV)
    yq, yk = rotary_embed(q, k, pos, freqs, interleaved=interleaved)
    for name, x, y in (("q", q, yq), ("k", k, yk)):
        want, slack = ref(x, pos, freqs, interleaved, 1.0)
        assert y.shape == x.shape and y.dtype == x.dtype
        check(name, y, want, slack)
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [1_000_000, 40_000_000_000, -5_000_000])
def test_far_positions_keep_their_angle(dtype, first):
    q, k, _ = make(2, 19, 3, 1, 64, dtype)
    pos = torch.arange(19, device=DEV) + first
    freqs, amp = rotary_frequencies(64, 500_000.0, "yarn", 8.0, device=DEV)
    yq, yk = rotary_embed(q, k, pos, freqs, amplitude=amp)
    for x, y in ((q, yq), (k, yk)):
        want, slack = ref(x, pos[None], freqs, False, amp)
        check(first, y, want, slack)


def test_one_tensor_no_batch_and_broadcast_positions():
    q, k, _ = make(1, 6, 3, 2, 64, torch.bfloat16)
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.tensor([7], device=DEV)
    y, none = rotary_embed(q[0], None, pos, freqs)
    assert none is None and y.shape == q[0].shape
    want, slack = ref(q, pos[None], freqs, False, 1.0)
    check("q", y[None], want, slack)
    both = rotary_embed(q, k, torch.full((1, 6), 7, device=DEV), freqs)
    assert torch.equal(both[0][0], y)


def test_empty_calls():
    freqs, _ = rotary_frequencies(64, device=DEV)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        q = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        pos = torch.empty(shape[:2], dtype=torch.int64, device=DEV)
        y, _ = rotary_embed(q, None, pos, freqs)
        assert y.shape == q.shape


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 24), (20, 6)])
def test_in_place_leaves_the_rest_alone(interleaved, d, rot):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2, 37, 7, d, generator=g).to(torch.float16).to(DEV)
    before = qkv.clone()
    freqs, _ = rotary_frequencies(rot, device=DEV)
    pos = torch.arange(37, device=DEV)
    want = rotary_embed(before[:, :, :4], before[:, :, 4:6], pos, freqs, interleaved=interleaved)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    r = rotary_embed(q, k, pos, freqs, interleaved=interleaved, inplace=True)
    assert r[0] is q and r[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, :, 6:], before[:, :, 6:])


def test_operands_off_the_vector_alignment():
    """Storage offsets and strides that rule the wide vectors out, and a transposed layout."""
    g = torch.Generator().manual_seed(2)
    freqs, _ = rotary_frequencies(32, device=DEV)
    pos = torch.arange(11, device=DEV)
    flat = torch.randn(2 * 11 * 3 * 65 + 1, generator=g).to(torch.bfloat16).to(DEV)
    odd = flat[1:].view(2, 11, 3, 65)[..., :64]
    heads_first = odd.transpose(1, 2).contiguous().transpose(1, 2)
    last = odd.transpose(2, 3).contiguous().transpose(2, 3)  # last dim not contiguous
    for il in (False, True):
        want, slack = ref(odd, pos[None], freqs, il, 1.0)
        for x in (odd, heads_first, last):
            check("x", rotary_embed(x, None, pos, freqs, interleaved=il)[0], want, slack)
    shared = odd[:, :, :1].expand(2, 11, 3, 64)
    y, _ = rotary_embed(shared, None, pos, freqs)
    check("expanded", y, *ref(shared, pos[None], freqs, False, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 64), (False, 24), (True, 10)])
def test_gradients_are_the_rotation_back(dtype, interleaved, rot):
    q, k, pos = make(2, 13, 3, 2, 64, dtype)
    freqs, amp = rotary_frequencies(rot, 10_000.0, "yarn", 4.0, device=DEV)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = rotary_embed(q, k, pos, freqs, interleaved=interleaved, amplitude=amp)
    gen = torch.Generator().manual_seed(3)
    gq = torch.randn(yq.shape, generator=gen).to(dtype).to(DEV)
    gk = torch.randn(yk.shape, generator=gen).to(dtype).to(DEV)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)
    for name, g, got in (("dq", gq, dq), ("dk", gk, dk)):
        check(name, got, *ref(g, pos, freqs, interleaved, amp, inverse=True))
    # one output alone, and an upstream gradient that is one value for all
    (only,) = torch.autograd.grad(yk, k, gk, retain_graph=True)
    assert torch.equal(only, dk)
    (ones,) = torch.autograd.grad(yq.sum(), q)
    check("ones", ones, *ref(torch.ones_like(yq), pos, freqs, interleaved, amp, inverse=True))


def test_gradient_against_differences():
    """fp32, central differences with a step of 2^-3: the rotation is linear, so they are exact
    but for the two values' errors (8 * 2^-24 of a loss of magnitude sum |w| |y| each way)."""
    q, _, pos = make(1, 3, 2, 1, 16, torch.float32)
    freqs, _ = rotary_frequencies(8, device=DEV)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).double().to(DEV)
    x = q.detach().contiguous().requires_grad_()
    loss = lambda v: float((rotary_embed(v, None, pos, freqs)[0].double() * w).sum())
    (g,) = torch.autograd.grad((rotary_embed(x, None, pos, freqs)[0].double() * w).sum(), x)
    h = 2.0 ** -3
    size = float((w.abs() * (x.detach().abs() + h + 1)).sum())
    for at in [(0, 0, 0, 0), (0, 1, 1, 5), (0, 2, 0, 7), (0, 2, 1, 15)]:
        e = torch.zeros_like(x)
        e[at] = h
        with torch.no_grad():
            diff = (loss(x + e) - loss(x - e)) / (2 * h)
        assert abs(diff - float(g[at])) <= 2 * 16 * 2.0 ** -24 * size / (2 * h)


def test_second_derivative_is_the_rotation_again():
    q, _, pos = make(1, 5, 2, 1, 64, torch.float32)
    freqs, _ = rotary_frequencies(64, device=DEV)
    x = q.detach().requires_grad_()
    y, _ = rotary_embed(x, None, pos, freqs)
    up = torch.randn_like(y).requires_grad_()
    (g,) = torch.autograd.grad(y, x, up, create_graph=True)
    v = torch.randn_like(g)
    (back,) = torch.autograd.grad(g, up, v)
    check("double", back, *ref(v, pos, freqs, False, 1.0))


def test_heads_that_share_memory_in_place():
    """Column blocks of one row in either order, and blocks of separate tensors, are no overlap."""
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    base = torch.randn(2, 5, 7, 64, device=DEV)
    for q, k in ((slice(0, 4), slice(4, 7)), (slice(3, 7), slice(0, 3)), (slice(0, 2), slice(5, 7))):
        x = base.clone()
        want = rotary_embed(base[:, :, q], base[:, :, k], pos, freqs)
        rotary_embed(x[:, :, q], x[:, :, k], pos, freqs, inplace=True)
        assert torch.equal(x[:, :, q], want[0]) and torch.equal(x[:, :, k], want[1])


def test_gradient_of_a_broadcast_operand():
    """One key head expanded to four: its gradient is the sum over them (fp32; three additions
    of values of at most |sum| of their sizes on top of the rotation's bound)."""
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(6, device=DEV)
    leaf = torch.randn(2, 6, 1, 64, device=DEV, requires_grad=True)
    y, _ = rotary_embed(leaf.expand(2, 6, 4, 64), None, pos, freqs)
    g = torch.randn_like(y)
    (got,) = torch.autograd.grad(y, leaf, g)
    want, slack = ref(g, pos[None], freqs, False, 1.0, inverse=True)
    size = want.abs().sum(2, keepdim=True)
    check("leaf", got, want.sum(2, keepdim=True), slack.sum(2, keepdim=True) + 4 * 2.0 ** -24 * size)


def test_captured_training_step():
    """Forward and backward in one graph, replayed with new inputs between eager steps."""
    freqs, amp = rotary_frequencies(32, 10_000.0, "yarn", 2.0, device=DEV)
    pos = torch.arange(9, device=DEV)

    def step(q, k, gq, gk):
        yq, yk = rotary_embed(q, k, pos, freqs, amplitude=amp)
        return (yq, yk, *torch.autograd.grad((yq, yk), (q, k), (gq, gk)))

    def inputs(seed):
        q, k, _ = make(2, 9, 3, 1, 64, torch.float32, seed=seed)
        gq, gk, _ = make(2, 9, 3, 1, 64, torch.float32, seed=seed + 50)
        return [q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_(),
                gq.clone(), gk.clone()]

    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for seed in (1, 2, 3):
        new = inputs(seed)
        with torch.no_grad():
            for a, b in zip(held, new):
                a.copy_(b)
        graph.replay()
        want = step(*new)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), seed


def test_captured_call_replays_with_new_inputs():
    q, k, pos = make(3, 8, 9, 3, 64, torch.bfloat16)
    freqs, _ = rotary_frequencies(64, device=DEV)
    sq, sk, sp = q.clone(), k.clone(), pos.clone()
    rotary_embed(sq, sk, sp, freqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = rotary_embed(sq, sk, sp, freqs)
    for seed in range(3):
        a, b, p = make(3, 8, 9, 3, 64, torch.bfloat16, seed=seed + 5)
        sq.copy_(a), sk.copy_(b), sp.copy_(p)
        graph.replay()
        wq, wk = rotary_embed(a, b, p, freqs)
        torch.cuda.synchronize()
        assert torch.equal(yq, wq) and torch.equal(yk, wk), seed


def test_refusals():
    q, k, pos = make(1, 4, 3, 1, 64, torch.bfloat16)
    freqs, _ = rotary_frequencies(64, device=DEV)
    fused = torch.zeros(1, 4, 6, 64, dtype=torch.bfloat16, device=DEV)
    bad = [
        (dict(q=q.cpu()), "GPU"), (dict(q=q.double()), "bf16"), (dict(q=q[..., 0]), "does not go"),
        (dict(k=k.float()), "does not go"), (dict(k=k[:, :2]), "does not go"),
        (dict(positions=pos.int()), "int64"), (dict(positions=pos.cpu()), "positions"),
        (dict(freqs=freqs.float()), "fp64"), (dict(freqs=freqs[None]), "fp64"),
        (dict(freqs=torch.cat((freqs, freqs))), "rot_dim"), (dict(freqs=freqs[:0]), "rot_dim"),
        (dict(q=q.clone().requires_grad_(), inplace=True), "inplace"),
        (dict(q=q[:, :, :1].expand(1, 4, 3, 64), inplace=True), "inplace"),
        (dict(k=q, inplace=True), "share elements"),
        (dict(q=fused[:, :, :4], k=fused[:, :, 3:5], inplace=True), "share elements"),
        (dict(q=fused[:, :, 3:5], k=fused[:, :, :4], inplace=True), "share elements"),
    ]
    for change, needle in bad:
        args = dict(q=q, k=k, positions=pos, freqs=freqs) | change
        with pytest.raises(ValueError, match=needle):
            rotary_embed(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("freqs"),
                         **args)
    with pytest.raises(RuntimeError):
        rotary_embed(q, k, torch.zeros(3, dtype=torch.int64, device=DEV), freqs)
