"""Rotary positions against plain implementations in 64 bits.

Tolerances. The angle: position * f in fixed point, off by the position times f's own rounding (2^-52 |f| with the division by 2 pi) and 2^-34 turns, then
2^-24 of at most pi / 4 from fp32; sine and cosine 2 ulp (2^-22 of at most 1), times the amplitude 2^-24; the two products and their sum
2^-24 each. Together below 2^-21 + 2^-50 |position f| of a (|x1| + |x2|). Then one rounding to the type, u = eps / 2 relative (bf16 2^-8, fp16 2^-11, fp32
2^-24), in fp16 at least half of its smallest step, 2^-25. Columns that are not turned, values and everything that is left alone are exact."""

import math

import pytest
import torch

from kohakufa_b200 import KVCache, Rotary, _lib, apply_rotary, attention_cached, cache_append, cache_append_rotary, rotary_frequencies

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def exact_rotary(x, at, f, interleaved, amplitude=1.0, back=False):
    """x [..., S, D] and positions [..., S] (any that broadcast) in 64 bits on the CPU: the turned rows and what their error may be."""
    x, f = x.detach().double().cpu(), f.double().cpu()
    pairs = f.numel()
    at = torch.as_tensor(at).cpu()
    angle = at.double().unsqueeze(-1) * f
    cos, sin = angle.cos() * amplitude, angle.sin() * (-amplitude if back else amplitude)
    i = torch.arange(pairs)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    y, room = x.clone(), torch.zeros_like(x)
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    off = abs(amplitude) * (x[..., lo].abs() + x[..., hi].abs()) * (2.0**-21 + 2.0**-50 * angle.abs())
    room[..., lo] = room[..., hi] = off
    return y, room


def check_close(got, want, room, dtype):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    u = torch.finfo(dtype).eps / 2
    room = room + (u * (want.abs() + room) + (2.0**-25 if dtype == torch.float16 else 0.0)) * (room > 0)
    off = (got - want).abs()
    assert bool((off <= room).all()), float((off / room.clamp_min(1e-300)).max())


def rows(*shape, dtype=torch.bfloat16, seed=0):
    """[B, H, S, D] views of [B, S, H, D] storage."""
    gen = torch.Generator().manual_seed(seed)
    b, h, s, d = shape
    return torch.randn(b, s, h, d, generator=gen).to(dtype).cuda().transpose(1, 2)


# ---- without a GPU -------------------------------------------------------------------------------------------------


def test_frequencies():
    f, a = rotary_frequencies(8, 100.0)
    assert a == 1.0 and torch.allclose(f, torch.tensor([1.0, 100.0**-0.25, 0.1, 100.0**-0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary_frequencies(8, 100.0, method="linear", factor=4.0)[0], f / 4)
    g, _ = rotary_frequencies(8, 100.0, method="base", factor=4.0)
    assert g[0] == f[0] and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-14)
    # 500 positions: 500 f / (2 pi) = 79.6, 25.2, 8.0, 2.5 turns; between 1 and 32 of them the ramp
    f2, a2 = rotary_frequencies(8, 100.0, method="yarn", factor=4.0, length=500)
    assert math.isclose(a2, 0.1 * math.log(4.0) + 1)
    turns = 500 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    assert float(keep[0]) == 1.0 and f2[0] == f[0] and torch.allclose(f2, keep * f + (1 - keep) * f / 4, rtol=1e-15)
    f3, a3 = rotary_frequencies(8, 100.0, method="ramp", factor=4.0, length=500, low=3.0, high=10.0)
    assert a3 == 1.0 and f3[3] == f[3] / 4 and f3[1] == f[1] and f[2] / 4 < f3[2] < f[2]


@pytest.mark.parametrize(
    "args,more",
    [((7,), {}), ((0,), {}), ((8, -1.0), {}), ((8,), {"method": "other"}), ((8,), {"method": "yarn"}), ((2,), {"method": "base", "factor": 2.0}),
     ((8,), {"factor": 0.0}), ((8,), {"method": "ramp", "length": 10, "low": 4.0, "high": 4.0}), ((2.5,), {}), ((8, math.inf), {})],
)  # fmt: skip
def test_frequencies_refuses(args, more):
    with pytest.raises(ValueError):
        rotary_frequencies(*args, **more)


def test_turns_are_fractions_of_a_turn():
    r = Rotary([math.pi, -math.pi / 2, 5 * math.pi, 0.0, 1.0], device="cpu")
    assert r.dim == 10 and r.turns.dtype == torch.int64
    assert r.turns[:4].tolist() == [-(2**63), -(2**62), -(2**63), 0]
    assert abs(int(r.turns[4]) / 2**64 - 1 / (2 * math.pi)) < 2.0**-54
    for bad in ([], [[1.0]], [math.nan], [math.inf]):
        with pytest.raises(ValueError):
            Rotary(bad, device="cpu")
    for bad in (math.nan, 1e39):
        with pytest.raises(ValueError):
            Rotary([1.0], amplitude=bad, device="cpu")


def test_refusals_without_a_gpu():
    r = Rotary.of(16, device="cpu")
    q, k = torch.zeros(2, 4, 3, 16, dtype=torch.bfloat16), torch.zeros(2, 2, 3, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        apply_rotary(q, k, r)
    with pytest.raises(TypeError):
        apply_rotary(q, k.float(), r)
    with pytest.raises(TypeError):
        apply_rotary(q.double(), None, r)
    with pytest.raises(ValueError, match="positions"):
        apply_rotary(q[0].transpose(0, 1), None, r)
    with pytest.raises(ValueError, match="batch"):
        apply_rotary(q, k[:, :, :2], r)


# ---- the pass of its own -------------------------------------------------------------------------------------------

# (batch, heads, K / V heads, tokens, head dim, turned columns, interleaved)
SHAPES = [
    (1, 8, 8, 1, 64, 64, False),
    (2, 4, 1, 33, 128, 128, False),
    (2, 4, 1, 33, 128, 128, True),
    (3, 5, 5, 7, 80, 32, False),
    (1, 3, 1, 300, 80, 20, True),
    (2, 2, 2, 17, 72, 72, False),  # halves of 36 columns
    (2, 2, 1, 9, 40, 18, False),  # of 9
    (1, 6, 2, 65, 96, 14, True),
    (1, 1, 1, 1500, 16, 16, False),  # one head: many tokens a block
    (1, 2, 1, 5, 24, 2, True),
    (1, 3, 3, 4, 25, 12, False),  # rows that begin anywhere
    (1, 3, 3, 4, 27, 26, True),
    (1, 2, 1, 3, 2, 2, False),
    (1, 1, 1, 5, 1024, 1024, False),
    (1, 1, 1, 5, 1023, 1022, True),
    (1, 300, 4, 2, 64, 32, False),
    (40, 1, 1, 1, 8, 8, True),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary(shape, dtype):
    b, h, hkv, s, d, turned, interleaved = shape
    f, _ = rotary_frequencies(turned, 1000.0)
    r = Rotary(f, interleaved=interleaved, amplitude=1.25)
    q, k = rows(b, h, s, d, dtype=dtype, seed=1), rows(b, hkv, s, d, dtype=dtype, seed=2)
    at = torch.arange(s)
    got = apply_rotary(q, k, r)
    assert _lib.device_status() == 0
    for x, y in zip((q, k), got):
        assert y.dtype == dtype and y.transpose(1, 2).is_contiguous()
        check_close(y, *exact_rotary(x, at, f, interleaved, 1.25), dtype)
    assert torch.equal(apply_rotary(q, None, r), got[0])
    # each row by itself gives the same bits
    one = apply_rotary(q[:, :, -1:], None, r, positions=torch.tensor([s - 1], device="cuda"))
    assert torch.equal(one[:, :, 0], got[0][:, :, -1])


@gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions(kind, interleaved):
    b, h, s, d = 3, 4, 11, 64
    f, _ = rotary_frequencies(48)
    r, q = Rotary(f, interleaved=interleaved), rows(3, 4, 11, 64, dtype=torch.float32)
    gen = torch.Generator().manual_seed(3)
    per = torch.randint(-500, 100000, (b, s), generator=gen).to(kind)
    offset = torch.tensor([5, -70, 123456], dtype=torch.int32)
    for at in (per, per[:1], per[0], per[:1].expand(b, s), per.T.contiguous().T, torch.stack([per, per], 2)[:, :, 1]):
        full = at if at.dim() == 2 else at[None]
        got = apply_rotary(q, None, r, positions=at.cuda())
        check_close(got, *exact_rotary(q, full[:, None], f, interleaved), torch.float32)
        got = apply_rotary(q, None, r, positions=at.cuda(), offset=offset.cuda())
        check_close(got, *exact_rotary(q, full[:, None].long() + offset[:, None, None], f, interleaved), torch.float32)
    got = apply_rotary(q, None, r, offset=offset.cuda())
    check_close(got, *exact_rotary(q, torch.arange(s)[None, None] + offset[:, None, None], f, interleaved), torch.float32)


@gpu
def test_far_positions_keep_their_angle():
    """Positions behind 2^31, where fp32 angles would be off by whole turns: quarter turns and thirds come out as such."""
    r = Rotary([math.pi / 2, 2 * math.pi / 3, 1.0])
    x = torch.zeros(1, 1, 4, 6, device="cuda")
    x[..., :3] = 1.0
    at = torch.tensor([2**40 + 1, -(2**40) + 3, 2**31 - 1, 3 * 2**38 + 1])
    y = apply_rotary(x, None, r, positions=at.cuda()).cpu()[0, 0].double()
    # (a frequency in 64 bits is off by 2^-53 of itself, 2^40 of those by 2^-12)
    for i, p in enumerate(at.tolist()):
        for j, turn in enumerate([(p % 4) / 4, (p % 3) / 3]):
            assert abs(y[i, j] - math.cos(2 * math.pi * turn)) < 2.0**-11 and abs(y[i, j + 3] - math.sin(2 * math.pi * turn)) < 2.0**-11
    f, _ = rotary_frequencies(128, 1e6, method="yarn", factor=64.0, length=8192)
    q = rows(1, 2, 64, 128, dtype=torch.float32)
    at = torch.arange(64) + 2**24 - 20
    got = apply_rotary(q, None, Rotary(f), positions=at.int().cuda())
    check_close(got, *exact_rotary(q, at, f, False), torch.float32)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Heads before tokens, rows cut out of wider ones, rows that begin between 16-byte boundaries, broadcast heads and tokens, packed sequences."""
    f, _ = rotary_frequencies(32)
    r, at = Rotary(f), torch.arange(13)
    qkv = torch.randn(2, 13, 12, 48, device="cuda").to(dtype)
    heads_first = torch.randn(2, 6, 13, 48, device="cuda").to(dtype)
    odd = torch.randn(2, 13, 6, 51, device="cuda").to(dtype)
    for x in (
        qkv.transpose(1, 2)[:, :8], heads_first, odd[..., 1:49].transpose(1, 2), odd[..., 2:42].transpose(1, 2), odd[..., 1:50].transpose(1, 2),
        qkv[:, :, :1].transpose(1, 2).expand(2, 5, 13, 48), qkv[:, :1].transpose(1, 2).expand(2, 12, 13, 48), qkv[:1].transpose(1, 2).expand(3, 12, 13, 48),
    ):  # fmt: skip
        got, again = apply_rotary(x, x[:, :1], r)
        check_close(got, *exact_rotary(x, at, f, False), dtype)
        assert torch.equal(got[:, :1], again)
    packed, where = qkv.flatten(0, 1), torch.cat([torch.arange(20), torch.arange(6)])
    q, k = apply_rotary(packed[:, :8], packed[:, 8:10], r, positions=where.int().cuda())
    for x, y in ((packed[:, :8], q), (packed[:, 8:10], k)):
        assert y.shape == x.shape and y.is_contiguous()
        want, room = exact_rotary(x.transpose(0, 1), where, f, False)
        check_close(y.transpose(0, 1), want, room, dtype)


@gpu
def test_what_is_not_turned_is_untouched():
    """NaN and infinities behind the turned columns, bit for bit, and inside them only in their pair."""
    for interleaved in (False, True):
        r = Rotary.of(16, interleaved=interleaved)
        x = rows(1, 2, 5, 40, dtype=torch.float16)
        clean = apply_rotary(x, None, r)
        x[0, 1, 2, 16], x[0, 1, 3, 39], x[0, 0, 4, 2] = math.nan, -math.inf, math.nan
        y = apply_rotary(x, None, r)
        assert torch.equal(y[..., 16:].view(torch.int16), x[..., 16:].view(torch.int16))
        touched = torch.zeros_like(y, dtype=torch.bool)
        touched[0, 0, 4, [2, 3] if interleaved else [2, 10]] = True
        assert bool(torch.isnan(y[touched]).all()) and torch.equal(y[..., :16][~touched[..., :16]], clean[..., :16][~touched[..., :16]])


@gpu
def test_no_tokens():
    r = Rotary.of(64)
    for shape in ((0, 4, 3, 64), (2, 4, 0, 64)):
        q, k = apply_rotary(torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda"), r)
        assert q.shape == k.shape == shape
    assert apply_rotary(torch.empty(0, 4, 64, device="cuda"), None, r, positions=torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


@gpu
def test_rows_beyond_32_bits():
    """4.6 GB of rows: byte offsets and cells beyond 2^32 / 2^31."""
    r = Rotary.of(128)
    s, h = 140000, 128
    q = torch.zeros(1, s, h, 128, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    for t in (0, s // 2 + 1, s - 1):
        q[0, :, t] = torch.randn(h, 128, device="cuda").to(torch.bfloat16)
    y = apply_rotary(q, None, r)
    f, _ = rotary_frequencies(128)
    for t in (0, s // 2 + 1, s - 1):
        check_close(y[:, :, t : t + 1], *exact_rotary(q[:, :, t : t + 1], torch.tensor([t]), f, False), torch.bfloat16)
    assert bool((y[0, :, 1] == 0).all()) and bool((y[0, :, s - 2] == 0).all())


# ---- gradients -----------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,turned", [(64, 64), (80, 20), (72, 36)])
def test_gradient(dtype, interleaved, dim, turned):
    f, _ = rotary_frequencies(turned)
    r = Rotary(f, interleaved=interleaved, amplitude=0.75)
    q, k = rows(2, 6, 19, dim, dtype=dtype).requires_grad_(), rows(2, 2, 19, dim, dtype=dtype, seed=1).requires_grad_()
    g = [rows(2, n, 19, dim, dtype=dtype, seed=5 + n) for n in (6, 2)]
    out = apply_rotary(q, k, r)
    got = torch.autograd.grad(out, (q, k), g)
    for x, gx, dx in zip((q, k), g, got):
        check_close(dx, *exact_rotary(gx, torch.arange(19), f, interleaved, 0.75, back=True), dtype)
    # one of the two only, and a gradient that is one number everywhere
    out = apply_rotary(q, k, r)
    (dk,) = torch.autograd.grad(out[1], k, g[1])
    assert torch.equal(dk, got[1])
    out = apply_rotary(q, k, r)
    (dq,) = torch.autograd.grad(out[0].sum(), q)
    check_close(dq, *exact_rotary(torch.ones_like(q), torch.arange(19), f, interleaved, 0.75, back=True), dtype)
    out = apply_rotary(q, None, r)
    assert torch.equal(torch.autograd.grad(out, q, g[0])[0], got[0])
    out = apply_rotary(q.detach(), k, r)
    out[1].backward(g[1])
    assert q.grad is None and torch.equal(k.grad, got[1]) and not out[0].requires_grad
    out = apply_rotary(q, k.detach(), r)
    assert out[0].requires_grad and not out[1].requires_grad and torch.equal(out[1], apply_rotary(q, k, r)[1])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    """The pass is linear: (y(x + h e) - y(x - h e)) / 2 h along a direction is the gradient's product with it, up to the roundings of fp32 outputs."""
    r = Rotary.of(12, interleaved=interleaved)
    x, e, w = (rows(1, 3, 8, 20, dtype=torch.float32, seed=s) for s in (0, 1, 2))
    x.requires_grad_()
    (g,) = torch.autograd.grad((apply_rotary(x, None, r) * w).sum(), x)
    with torch.no_grad():
        up, down = apply_rotary(x + 0.5 * e, None, r).double(), apply_rotary(x - 0.5 * e, None, r).double()
    by_differences, by_gradient = ((up - down) * w.double()).sum(), (g.double() * e.double()).sum()
    # 480 terms, each off by about 2^-20 of (|x1| + |x2|) |w| (inputs, outputs, gradient)
    room = 2.0**-20 * 2 * float((x.detach().abs().amax() + e.abs().amax()) * w.abs().sum())
    assert abs(float(by_differences - by_gradient)) <= room


@gpu
def test_gradient_of_broadcast_and_shared_inputs():
    r = Rotary.of(64)
    k = rows(2, 1, 9, 64, dtype=torch.float32).requires_grad_()
    y = apply_rotary(k.expand(2, 4, 9, 64), k, r)
    g = rows(2, 4, 9, 64, dtype=torch.float32, seed=3), rows(2, 1, 9, 64, dtype=torch.float32, seed=4)
    (dk,) = torch.autograd.grad(y, k, g)
    f, _ = rotary_frequencies(64)
    one, room = exact_rotary(torch.cat(g, 1), torch.arange(9), f, False, back=True)
    off = (dk.double().cpu() - one.sum(1, keepdim=True)).abs()
    assert bool((off <= room.sum(1, keepdim=True) + 8 * 2.0**-24 * one.abs().sum(1, keepdim=True)).all())


@gpu
def test_gradient_of_the_gradient():
    r = Rotary.of(32, interleaved=True)
    x, g = rows(1, 2, 4, 32, dtype=torch.float32).requires_grad_(), rows(1, 2, 4, 32, dtype=torch.float32, seed=1).requires_grad_()
    (dx,) = torch.autograd.grad(apply_rotary(x, None, r), x, g, create_graph=True)
    w = rows(1, 2, 4, 32, dtype=torch.float32, seed=2)
    (dg,) = torch.autograd.grad(dx, g, w)
    assert torch.equal(dg, apply_rotary(w, None, r))


@gpu
def test_positions_that_change_before_the_backward_are_noticed():
    r, x = Rotary.of(16), rows(1, 1, 4, 16, dtype=torch.float32).requires_grad_()
    at = torch.arange(4, device="cuda")
    y = apply_rotary(x, None, r, positions=at)
    at += 1
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


@gpu
def test_compiled():
    r = Rotary.of(64)
    q, k = rows(2, 4, 8, 64).requires_grad_(), rows(2, 2, 8, 64, seed=1).requires_grad_()
    at = torch.arange(8, device="cuda")

    def step(q, k):
        a, b = apply_rotary(q * 1.0, k * 1.0, r, positions=at)
        return a.float().square().sum() + b.float().sum()

    want = torch.autograd.grad(step(q, k), (q, k))
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(q, k), (q, k))
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@gpu
def test_capture_and_streams():
    """Forward and backward in a graph while an eager one of the same leaves lives (of the capture's stream: torch's engine ties a leaf to the
    stream it was first recorded on, and does not capture across two); replays follow the inputs."""
    r = Rotary.of(128)
    q, k = rows(2, 4, 50, 128).requires_grad_(), rows(2, 2, 50, 128, seed=1).requires_grad_()
    g = rows(2, 4, 50, 128, seed=2), rows(2, 2, 50, 128, seed=3)
    at = torch.arange(50, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = apply_rotary(q, k, r, positions=at)
        for _ in range(2):
            torch.autograd.grad(apply_rotary(q, k, r, positions=at), (q, k), g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = apply_rotary(q, k, r, positions=at)
        grads = torch.autograd.grad(out, (q, k), g)
    for step in range(3):
        with torch.no_grad():
            q.add_(0.5)
        at += 7
        graph.replay()
        want = apply_rotary(q.detach(), k.detach(), r, positions=at)
        for x, y in zip(out, want):
            assert torch.equal(x, y)
        back = torch.autograd.grad(apply_rotary(q, k, r, positions=at), (q, k), g)
        for x, y in zip(grads, back):
            assert torch.equal(x, y)
    del alive


@gpu
def test_refusals():
    r = Rotary.of(64)
    q, k = rows(2, 4, 8, 64), rows(2, 2, 8, 64)
    at = torch.arange(8, device="cuda")
    bad = [
        (ValueError, (q[..., :32], None), {}),  # more turned columns than there are
        (ValueError, (q, k[..., :40]), {}),
        (TypeError, (q, k.half()), {}),
        (TypeError, (q, None), {"positions": at.float()}),
        (ValueError, (q, None), {"positions": at[:7]}),
        (ValueError, (q, None), {"positions": at.expand(3, 8)}),
        (ValueError, (q, None), {"positions": at.cpu()}),
        (TypeError, (q, None), {"offset": torch.zeros(2, dtype=torch.int64, device="cuda")}),
        (ValueError, (q, None), {"offset": torch.zeros(3, dtype=torch.int32, device="cuda")}),
        (ValueError, (q.transpose(2, 3), None), {}),
        (ValueError, (q[0, 0], None), {"positions": at}),
        (ValueError, (q[:, :0], None), {}),
        (ValueError, (q, k.cpu()), {}),
    ]
    for error, args, more in bad:
        with pytest.raises(error):
            apply_rotary(*args, r, **more)
    with pytest.raises(ValueError, match="devices"):
        apply_rotary(q, k, r.to("cpu"))


# ---- into a cache --------------------------------------------------------------------------------------------------


def make_cache(lengths, kv_heads, dim, dtype, page, extra, seed=0):
    gen = torch.Generator().manual_seed(seed)
    batch, most = len(lengths), max(lengths) + extra
    if page is None:
        count, size, table = batch, most, None
    else:
        cols = -(-most // page)
        count, size = batch * cols + 2, page
        table = torch.randperm(count, generator=gen)[: batch * cols].view(batch, cols).to(torch.int32).cuda()
    k, v = (torch.randn(count, size, kv_heads, dim, generator=gen).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    return KVCache(k, v, torch.tensor(lengths, dtype=torch.int32).cuda(), table)


def clone(cache):
    return KVCache(cache.k.clone(), cache.v.clone(), cache.lengths.clone(), cache.table)


APPEND = [
    # lengths, page, heads, K / V heads, tokens, head dim, turned, interleaved
    ([100], None, 8, 8, 1, 64, 64, False),
    ([5, 0, 33], 16, 8, 2, 6, 128, 128, False),
    ([31, 32, 33, 127], 32, 4, 4, 3, 80, 20, True),
    ([7, 64], 8, 6, 1, 19, 72, 36, False),
    ([0, 0], 16, 5, 5, 130, 40, 18, False),
    ([1000], None, 32, 8, 1, 128, 64, True),
    ([3] * 50, 8, 2, 1, 2, 8, 8, False),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", APPEND, ids=str)
@pytest.mark.parametrize("ragged", [False, True])
def test_append(shape, dtype, ragged):
    lengths, page, heads, kv_heads, tokens, dim, turned, interleaved = shape
    batch = len(lengths)
    f, _ = rotary_frequencies(turned, 500.0)
    r = Rotary(f, interleaved=interleaved, amplitude=1.5)
    cache = make_cache(lengths, kv_heads, dim, dtype, page, tokens)
    q, k, v = rows(batch, heads, tokens, dim, dtype=dtype, seed=1), rows(batch, kv_heads, tokens, dim, dtype=dtype, seed=2), rows(batch, kv_heads, tokens, dim, dtype=dtype, seed=3)
    gen = torch.Generator().manual_seed(9)
    counts = torch.randint(0, tokens + 1, (batch,), generator=gen).to(torch.int32).cuda() if ragged else None
    offset = torch.randint(0, 5000, (batch,), generator=gen).to(torch.int32).cuda() if ragged else None
    want = clone(cache)
    if ragged:  # what is left out may be anything
        for b in range(batch):
            for t in (q, k, v):
                t[b, :, int(counts[b]) :] = math.nan
    got_q, got_k = cache_append_rotary(cache, q, k, v, r, counts=counts, offset=offset, return_keys=True)
    assert _lib.device_status() == 0
    at = torch.tensor(lengths)[:, None] + torch.arange(tokens) + (0 if offset is None else offset.cpu()[:, None])
    there = (torch.arange(tokens) < (tokens if counts is None else counts.cpu()[:, None])).expand(batch, tokens)
    for x, y in ((q, got_q), (k, got_k)):
        assert y.transpose(1, 2).is_contiguous()
        rest = ~there[:, None, :, None].expand_as(x)
        assert bool((y.cpu()[rest] == 0).all())
        y, x = y.cpu().masked_fill(rest, 0), x.cpu().masked_fill(rest, 0)
        check_close(y, *exact_rotary(x, at[:, None], f, interleaved, 1.5), dtype)
    # the cache has these keys, and nothing else changed
    cache_append(want, got_k, v, counts=counts)
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
    # without queries, without keys
    again = clone(want)
    again.k.zero_()
    assert cache_append_rotary(again, None, k, v, r, counts=counts, offset=offset) is None
    assert torch.equal(again.v, want.v)
    only = cache_append_rotary(clone(want), q, k, v, r, counts=counts, offset=offset)
    assert torch.equal(only, got_q)


@gpu
def test_append_with_an_index_and_positions():
    dtype, f = torch.bfloat16, rotary_frequencies(64)[0]
    r, cache = Rotary(f), make_cache([10, 0, 50], 2, 64, torch.bfloat16, 16, 8)
    k, v = rows(3, 2, 8, 64, dtype=dtype), rows(3, 2, 8, 64, dtype=dtype, seed=1)
    index = torch.tensor([[7, 0, 0], [1, 2, 3], [4, 4, 6]], dtype=torch.int32).cuda()
    counts = torch.tensor([3, 2, 1], dtype=torch.int32).cuda()
    depth = torch.tensor([[0, 1, 1, 2, 2, 2, 3, 1]]).cuda()
    for positions in (None, depth, depth.int()[0]):
        got, want = clone(cache), clone(cache)
        assert cache_append_rotary(got, None, k, v, r, index=index, counts=counts, positions=positions, offset=cache.lengths) is None
        if positions is None:
            at = cache.lengths[:, None] * 2 + torch.arange(3, device="cuda")
        else:
            at = cache.lengths[:, None] + depth[0][index.long()]
        taken = torch.stack([k[b][:, index[b].long()] for b in range(3)])
        cache_append(want, apply_rotary(taken, None, r, positions=at.int()), torch.stack([v[b][:, index[b].long()] for b in range(3)]), counts=counts)
        assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v)
    assert _lib.device_status() == 0


@gpu
def test_append_reports_what_has_no_place():
    dtype, r = torch.float16, Rotary.of(64)
    k, v, q = rows(2, 2, 4, 64, dtype=dtype), rows(2, 2, 4, 64, dtype=dtype, seed=1), rows(2, 4, 4, 64, dtype=dtype, seed=2)
    for what in ("capacity", "table", "negative", "index"):
        cache = make_cache([14, 5], 2, 64, dtype, 16, 6)
        table, lengths, index = cache.table.clone(), cache.lengths.clone(), None
        if what == "capacity":
            lengths[0] = cache.capacity - 2
        elif what == "table":
            table[1, 0] = 99
        elif what == "negative":
            lengths[1] = -1
        else:
            index = torch.tensor([[0, 4], [1, -1]], dtype=torch.int32).cuda()
        bad = KVCache(cache.k.clone(), cache.v.clone(), lengths, table)
        try:
            out = cache_append_rotary(bad, None if what == "index" else q, k, v, r, index=index)
            assert _lib.device_status() == _lib.DEV_BAD_CACHE
        finally:
            _lib.reset_device_status()
        keys = cache_append_rotary(clone(cache), None, k, v, r, return_keys=True)[1]
        assert _lib.device_status() == 0
        if what in ("capacity", "index"):  # what has a place is there
            page, slot = (bad.table[0, (cache.capacity - 2) // 16], (cache.capacity - 2) % 16) if what == "capacity" else (bad.table[0, 14 // 16], 14)
            assert torch.equal(bad.v[int(page), :, slot], v[0, :, 0])
        else:  # the other sequence's is
            assert torch.equal(bad.k[int(table[0, 0]), :, 14], keys[0][:, 0]) and torch.equal(bad.v[int(table[0, 0]), :, 15], v[0, :, 1])
        assert out is None or bool(torch.isfinite(out).all())


@gpu
def test_append_compiled():
    """Through the registered op, which a compiler sees."""
    r, cache = Rotary.of(64), make_cache([3, 20], 2, 64, torch.bfloat16, 16, 4)
    q, k, v = rows(2, 4, 4, 64), rows(2, 2, 4, 64, seed=1), rows(2, 2, 4, 64, seed=2)
    want = clone(cache)
    a, b = cache_append_rotary(want, q, k, v, r, return_keys=True)

    def step(kp, vp, q, k, v):
        x, y = cache_append_rotary(KVCache(kp, vp, cache.lengths, cache.table), q * 1.0, k, v, r, return_keys=True)
        return x + 0.0, y + 0.0

    with torch.no_grad():
        x, y = torch.compile(step, backend="aot_eager")(cache.k, cache.v, q, k, v)
    assert torch.equal(x, a) and torch.equal(y, b) and torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)


@gpu
def test_append_many_heads_and_long_prompts():
    """More tokens than one head a thread takes, with heads that are no multiple of three, against the pass of its own."""
    dtype, r = torch.bfloat16, Rotary.of(64, interleaved=True)
    for heads, kv_heads, tokens in ((7, 1, 3000), (4, 4, 2000), (40, 8, 500)):
        cache = make_cache([5, 100], kv_heads, 96, dtype, 32, tokens)
        q, k, v = (rows(2, h, tokens, 96, dtype=dtype, seed=s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
        want = clone(cache)
        got_q, got_k = cache_append_rotary(cache, q, k, v, r, return_keys=True)
        q2, k2 = apply_rotary(q, k, r, offset=cache.lengths)
        cache_append(want, k2, v)
        assert torch.equal(got_q, q2) and torch.equal(got_k, k2) and torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
    assert _lib.device_status() == 0


@gpu
def test_append_refusals():
    r, cache = Rotary.of(64), make_cache([3, 4], 2, 64, torch.bfloat16, 16, 4)
    q, k, v = rows(2, 4, 4, 64), rows(2, 2, 4, 64, seed=1), rows(2, 2, 4, 64, seed=2)
    index, ok = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for error, args, more in [
        (ValueError, (q, k, v, Rotary.of(72)), {}),
        (ValueError, (q, k, v, r), {"index": index}),
        (ValueError, (None, k, v, r), {"index": index, "return_keys": True}),
        (TypeError, (q.half(), k, v, r), {}),
        (ValueError, (q[:, :, :3], k, v, r), {}),
        (ValueError, (q[:, :3], k, v, r), {}),
        (ValueError, (q, k, v[:, :, :3], r), {}),
        (TypeError, (q, k, v, r), {"counts": ok.long()}),
        (TypeError, (q, k, v, r), {"offset": ok.float()}),
        (ValueError, (q, k, v, r), {"offset": ok[:1]}),
        (ValueError, (q, k, v, r), {"positions": torch.arange(3, device="cuda")}),
        (ValueError, (q, k, v, r), {"positions": torch.arange(4)}),
        (ValueError, (q, k, v, r.to("cpu")), {}),
        (RuntimeError, (q.clone().requires_grad_(), k, v, r), {}),
    ]:
        with pytest.raises(error):
            cache_append_rotary(cache, *args, **more)
    shared = KVCache(cache.k, cache.k, cache.lengths, cache.table)
    with pytest.raises(ValueError, match="memory of their own"):
        cache_append_rotary(shared, q, k, v, r)


@gpu
def test_append_far_into_a_pool():
    """A page whose bytes lie beyond 2^32, a length in the millions."""
    page, dim, dtype = 64, 128, torch.bfloat16
    k = torch.zeros(40000, page, 8, dim, dtype=dtype, device="cuda").transpose(1, 2)
    v = torch.zeros_like(k)
    n = 2_000_003
    table = torch.zeros(1, n // page + 2, dtype=torch.int32, device="cuda")
    table[0, -2:] = torch.tensor([39999, 39998], dtype=torch.int32)
    cache = KVCache(k, v, torch.tensor([n], dtype=torch.int32).cuda(), table)
    r = Rotary.of(dim)
    q, kn, vn = rows(1, 32, 70, dim), rows(1, 8, 70, dim, seed=1), rows(1, 8, 70, dim, seed=2)
    got, keys = cache_append_rotary(cache, q, kn, vn, r, return_keys=True)
    assert _lib.device_status() == 0
    at = torch.arange(70) + n
    check_close(got, *exact_rotary(q, at, rotary_frequencies(dim)[0], False), dtype)
    for i in (0, 63, 69):
        p = int(table[0, (n + i) // page])
        assert torch.equal(k[p, :, (n + i) % page], keys[0, :, i]) and torch.equal(v[p, :, (n + i) % page], vn[0, :, i])


@gpu
def test_generation_step_by_step_and_captured():
    """Decoding through cache_append_rotary and attention_cached gives what rotating and attending over the whole sequence gives; a captured
    step follows the lengths."""
    dtype, heads, kv_heads, dim, batch, steps = torch.float16, 4, 2, 64, 3, 12
    r = Rotary.of(dim, interleaved=True)
    q, k, v = rows(batch, heads, steps, dim, dtype=dtype), rows(batch, kv_heads, steps, dim, dtype=dtype, seed=1), rows(batch, kv_heads, steps, dim, dtype=dtype, seed=2)
    eager, captured = (KVCache.empty(batch, kv_heads, 32, dim, page=8, dtype=dtype) for _ in range(2))
    qs, ks, vs = (torch.empty_like(t[:, :, :1]) for t in (q, k, v))

    def step(cache, q, k, v):
        q, k = cache_append_rotary(cache, q, k, v, r, return_keys=True)
        out = attention_cached(q, cache, k, v)
        cache.lengths += 1
        return out

    for t, x in ((qs, q), (ks, k), (vs, v)):
        t.copy_(x[:, :, :1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, qs, ks, vs)
    torch.cuda.current_stream().wait_stream(side)
    captured.lengths.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured, qs, ks, vs)
    captured.lengths.zero_()
    # the whole sequence at once: as a prompt into an empty cache
    whole_q, whole_k = apply_rotary(q, k, r)
    whole = attention_cached(whole_q, KVCache.empty(batch, kv_heads, 8, dim, dtype=dtype), whole_k, v)
    for i in range(steps):
        for t, x in ((qs, q), (ks, k), (vs, v)):
            t.copy_(x[:, :, i : i + 1])
        want = step(eager, qs, ks, vs)
        graph.replay()
        assert torch.equal(out, want)
        # (P in 16 bits and the output's rounding on both sides: 4 u of values of order 1, at most 4)
        assert float((want - whole[:, :, i : i + 1]).abs().max()) <= 4 * 2.0**-11 * 4
    assert torch.equal(eager.k, captured.k) and torch.equal(eager.lengths, captured.lengths) and int(eager.lengths[0]) == steps
