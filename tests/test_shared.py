"""Attention behind shared prefixes against a plain implementation in 64 bits.

Tolerances are those of attention over a cache (test_cache.py): each part's P are rounded to 16 bits, u = eps / 2 relative, and the output once more; the parts are
joined in fp32 (factors and sums a few 2^-23 relative, inside the 2^-12). So |out - exact| <= (u + 2^-12) sum p |v| + u |out| + 2^-24."""

import ctypes
import math

import pytest
import torch

from kohakufa_b200 import KVCache, Rotary, _lib, apply_rotary, attention_cached, attention_shared, build, cache_append, cache_append_rotary
from tests.test_cache import logical, make_cache, random_tree, rows

gpu = pytest.mark.gpu


def group_of(starts, b):
    """The prefix that sequence b goes on from, None: none."""
    for p in range(len(starts) - 1):
        if starts[p] <= b < starts[p + 1]:
            return p
    return None


def exact_shared(q, prefix, cache, starts, k, v, tree, counts, scale):
    """out, sum p |v|, m, log2 l in 64 bits; rows that see nothing: 0, 0, +inf, 0. (On the GPU where the rows are many: nothing of the library.)"""
    device = "cuda"
    q = q.double()
    batch, heads, tokens, dim = q.shape
    kp, vp, kc, vc = (logical(c, w).to(device) for c in (prefix, cache) for w in ("k", "v"))
    n_prefix, n_own = prefix.lengths.tolist(), cache.lengths.tolist()
    kv_heads = kc.shape[1]
    group = heads // kv_heads
    out, size = torch.zeros(2, batch, heads, tokens, dim, dtype=torch.float64, device=device)
    m = torch.full((batch, heads, tokens), math.inf, dtype=torch.float64, device=device)
    log2l = torch.zeros(batch, heads, tokens, dtype=torch.float64, device=device)
    for b in range(batch):
        count = tokens if counts is None else int(counts[b])
        p = group_of(starts, b)
        keys, values = kc[b, :, : n_own[b]], vc[b, :, : n_own[b]]
        if p is not None:
            keys, values = torch.cat([kp[p, :, : n_prefix[p]], keys], 1), torch.cat([vp[p, :, : n_prefix[p]], values], 1)
        sees = torch.ones(count, keys.shape[1], dtype=torch.bool, device=device)
        if k is not None:
            among = torch.ones(tokens, tokens).tril().bool() if tree is None else (tree if tree.dim() == 2 else tree[b]).cpu()
            keys, values = torch.cat([keys, k[b, :, :count].double()], 1), torch.cat([values, v[b, :, :count].double()], 1)
            sees = torch.cat([sees, among[:count, :count].to(device)], 1)
        if count == 0 or keys.shape[1] == 0:
            continue
        x = q[b, :, :count].reshape(kv_heads, group * count, dim)
        s = (x @ keys.transpose(1, 2)).view(heads, count, -1).masked_fill(~sees, -math.inf)
        top = s.amax(-1)
        some = top > -math.inf
        e = torch.exp((s - torch.where(some, top, 0.0)[..., None]) * scale)
        l = torch.where(some, e.sum(-1), 1.0)
        w = (e / l[..., None]).view(kv_heads, group * count, -1)
        out[b, :, :count], size[b, :, :count] = (w @ values).view(heads, count, dim), (w @ values.abs()).view(heads, count, dim)
        m[b, :, :count], log2l[b, :, :count] = torch.where(some, top, math.inf), l.log2()
    return out, size, m, log2l


def check_shared(prefix, cache, starts, heads, tokens, dtype, new="causal", counts=None, seed=0, scale=None, q=None, k=None, v=None):
    batch, kv_heads, dim = cache.lengths.numel(), cache.k.shape[1], cache.k.shape[3]
    q = rows(batch, heads, tokens, dim, dtype, seed) if q is None else q
    tree = None
    if new != "none" and k is None:
        k, v = rows(batch, kv_heads, tokens, dim, dtype, seed + 1), rows(batch, kv_heads, tokens, dim, dtype, seed + 2)
    if isinstance(new, torch.Tensor):
        tree = new
    elif new == "tree":
        tree = random_tree(batch, tokens, seed)
    count = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    where = None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda()
    call = lambda: attention_shared(  # noqa: E731
        q, prefix, cache, k, v, starts=where, tree=None if tree is None else tree.cuda(), counts=count, scale=scale, return_stats=True
    )
    got, stats = call()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    again, again_stats = call()
    assert torch.equal(got.nan_to_num(7.0), again.nan_to_num(7.0)) and torch.equal(stats, again_stats)
    scale = dim**-0.5 if scale is None else scale
    out, size, m, log2l = exact_shared(q, prefix, cache, [0, batch] if starts is None else starts, k, v, tree, counts, scale)
    u = torch.finfo(dtype).eps / 2
    assert got.shape == q.shape and got.dtype == dtype and got.transpose(1, 2).is_contiguous()
    off = (got.double() - out).abs()
    room = (u + 2.0**-12) * size + u * out.abs() + 2.0**-24
    assert bool((off <= room).all()), float((off / room).max())
    stats = stats.double()
    fine = torch.isfinite(m)
    assert torch.equal(torch.isinf(stats[:, :, 0]), ~fine) and bool((stats[:, :, 1][~fine] == 0).all())
    assert torch.allclose(stats[:, :, 0][fine], m[fine], rtol=2.0**-18, atol=2.0**-16)
    assert torch.allclose(stats[:, :, 1], log2l, rtol=2.0**-16, atol=2.0**-13)
    return got


# prefix lengths, starts, own lengths, page, heads, K / V heads, tokens, head dim
SHAPES = [
    ([100], None, [3, 40], None, 8, 8, 1, 64),
    ([1], None, [1, 0, 33], None, 4, 2, 1, 64),
    ([257], None, [0] * 5, 16, 4, 1, 1, 128),
    ([31, 0, 129], [0, 2, 3, 6], [31, 32, 33, 127, 128, 129], 16, 4, 1, 1, 128),
    ([300, 64, 500], [0, 1, 1, 4], [257, 5, 0, 640], 32, 8, 2, 5, 64),
    ([700, 20], [1, 4, 5], [3, 300, 77, 9, 50, 12, 700], 48, 6, 3, 7, 80),
    ([1000], None, [70, 500, 3], 128, 8, 4, 33, 128),
    ([400], None, [513, 2], 64, 8, 1, 40, 128),  # more than 256 rows of a sequence
    ([90, 10, 200], [0, 0, 0, 2], [90, 10], 16, 3, 3, 2, 40),
    ([65], None, [130, 6] * 9, 24, 2, 1, 1, 16),
    ([2000], None, [20] * 70, 16, 8, 2, 1, 128),  # two tiles of sequences
    ([3000], None, [8, 0, 20, 100] * 10, 8, 12, 4, 3, 72),
    ([33, 50], [0, 2, 3], [33, 4, 5], 8, 130, 1, 1, 64),
    ([60], None, [5, 9], 16, 300, 1, 2, 64),  # more than 256 heads a K / V head
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{len(s[2])}x{s[4]}-{s[5]}-{s[6]}-{s[7]}")
@pytest.mark.parametrize("new", ["causal", "tree", "none"])
def test_shared(shape, new, dtype):
    before, starts, lengths, page, heads, kv_heads, tokens, dim = shape
    prefix, cache = make_cache(before, kv_heads, dim, dtype, page, seed=5), make_cache(lengths, kv_heads, dim, dtype, page, seed=6)
    check_shared(prefix, cache, starts, heads, tokens, dtype, new, seed=len(lengths))


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,tokens", [(2, 1), (5, 1), (12, 1), (30, 1), (64, 1), (130, 1), (9, 6), (3, 60)])
def test_rows_of_every_kernel(batch, tokens, dim):
    """8, 20, 48, 120, 256, 520, 216 and 720 rows a K / V head over a long prefix, which is cut, and caches long and short."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 900, (batch,), generator=gen).tolist()
    prefix = make_cache([9001], 2, dim, dtype, 16, seed=1)
    check_shared(prefix, make_cache(lengths, 2, dim, dtype, 16), None, 8, tokens, dtype, "tree", seed=tokens)
    check_shared(prefix, make_cache([n // 10 for n in lengths], 2, dim, dtype), None, 8, tokens, dtype, "causal")


@gpu
@pytest.mark.parametrize("batch,tokens,heads", [(5, 16, 4), (40, 12, 4), (200, 1, 4), (33, 5, 8), (2, 300, 2)])
def test_several_prefixes_with_many_rows(batch, tokens, heads):
    """Row tiles that take both halves of a CTA, of groups that do not fill them, beside own rows of each kind; prompts behind a prefix."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 300, (batch,), generator=gen).tolist()
    starts = [0, batch // 3, batch // 3, batch - 1, batch]
    for before in ([700, 50, 2500, 33], [64, 9000, 1, 0]):
        prefix, cache = make_cache(before, 1, 64, torch.bfloat16, 16, seed=1), make_cache(lengths, 1, 64, torch.bfloat16, 16)
        check_shared(prefix, cache, starts, heads, tokens, torch.bfloat16, "tree" if tokens < 100 else "causal")


@gpu
@pytest.mark.parametrize("dim", range(8, 129, 24))
@pytest.mark.parametrize("batch,tokens", [(3, 1), (3, 7), (50, 4)])
def test_head_dims(dim, batch, tokens):
    lengths = [40 * i % 333 for i in range(batch)]
    check_shared(make_cache([777], 2, dim, torch.float16, 16, seed=1), make_cache(lengths, 2, dim, torch.float16, 16), None, 8, tokens, torch.float16, "tree", seed=dim)


@gpu
def test_pages_far_into_a_pool():
    """Pages whose bytes lie beyond 2^32, of the prefix and of the caches."""
    dtype, page = torch.bfloat16, 64
    k = torch.zeros(140000, page, 2, 128, dtype=dtype, device="cuda").transpose(1, 2)
    v = torch.zeros_like(k)
    at = torch.tensor([139999 - 7 * i for i in range(60)], dtype=torch.int32)
    gen = torch.Generator().manual_seed(0)
    for t in (k, v):
        t[at.long().cuda()] = torch.randn(60, page, 2, 128, generator=gen).to(dtype).cuda().transpose(1, 2)
    far = [KVCache(k, v, torch.tensor(n, dtype=torch.int32).cuda(), table.cuda()) for n, table in (([3000], at[:47].view(1, 47)), ([100, 200, 3], at[47:59].view(3, 4)))]
    near = [KVCache(c.k[c.table.flatten().long()], c.v[c.table.flatten().long()], c.lengths, torch.arange(c.table.numel(), dtype=torch.int32, device="cuda").view(c.table.shape)) for c in far]
    q, kn, vn = (rows(3, h, 2, 128, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    assert torch.equal(attention_shared(q, *far, kn, vn), check_shared(*near, None, 8, 2, dtype, "causal", q=q, k=kn, v=vn))
    assert _lib.device_status() == 0


@gpu
def test_nobody_has_tokens():
    dtype = torch.bfloat16
    prefix, cache = make_cache([300], 2, 64, dtype, 16, seed=1), make_cache([5, 0, 90], 2, 64, dtype, 16)
    got = check_shared(prefix, cache, None, 8, 3, dtype, "causal", counts=[0, 0, 0])
    assert bool((got == 0).all())


@gpu
def test_compiled():
    dtype = torch.bfloat16
    prefix, cache = make_cache([300], 2, 64, dtype, 16, seed=1), make_cache([5, 0, 90], 2, 64, dtype, 16)
    q, k, v = (rows(3, h, 2, 64, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))

    def step(q, k, v):
        out, stats = attention_shared(q * 1.0, prefix, cache, k, v, return_stats=True)
        return out + 0.0, stats + 0.0

    with torch.no_grad():
        a, b = torch.compile(step, backend="aot_eager")(q, k, v)
        x, y = step(q, k, v)
    assert torch.equal(a, x) and torch.equal(b, y)


@gpu
def test_many_prefixes():
    """More prefixes than the GPU has SMs and a CTA has threads, most with few sequences or none; whole items and cut ones in one call."""
    dtype = torch.float16
    gen = torch.Generator().manual_seed(0)
    batch, prefixes = 500, 420
    cuts = torch.randint(0, batch + 1, (prefixes - 1,), generator=gen).sort().values.tolist()
    before = torch.randint(0, 60, (prefixes,), generator=gen).tolist()
    before[7] = 5000
    lengths = torch.randint(0, 50, (batch,), generator=gen).tolist()
    for heads, tokens in ((2, 1), (32, 3)):
        check_shared(make_cache(before, 1, 64, dtype, 8, seed=1), make_cache(lengths, 1, 64, dtype, 8), [0, *cuts, batch], heads, tokens, dtype, "causal")


@gpu
@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens,heads", [(6, 8), (1, 4), (40, 8)])
def test_what_is_behind_an_end_does_not_matter(page, fill, tokens, heads):
    """Behind the prefixes, behind the caches, and the rows that counts leaves out."""
    dtype = torch.bfloat16
    lengths, starts = [100, 0, 31, 257, 64], [0, 2, 5]
    counts = [min(c, tokens) for c in (5, 3, 0, 1, 6)]
    cols = {} if page is None else {"columns": 40}
    prefix = make_cache([70, 333], 2, 64, dtype, page, fill=fill, **cols)
    cache = make_cache(lengths, 2, 64, dtype, page, fill=fill, seed=3, **cols)
    q, k, v = (rows(5, h, tokens, 64, dtype, s) for h, s in ((heads, 1), (2, 2), (2, 3)))
    for b, n in enumerate(counts):
        for t in (q, k, v):
            t[b, :, n:] = fill
    got = check_shared(prefix, cache, starts, heads, tokens, dtype, "tree", counts, q=q, k=k, v=v)
    assert bool(torch.isfinite(got).all())
    for b, n in enumerate(counts):
        assert bool((got[b, :, n:] == 0).all())
    check_shared(prefix, cache, starts, heads, tokens, dtype, "none", counts, q=q)


@gpu
@pytest.mark.parametrize("tokens", [1, 40])
def test_a_nan_reaches_who_sees_it(tokens):
    dtype = torch.bfloat16
    prefix, cache = make_cache([200, 600], 2, 64, dtype, 16, seed=1), make_cache([50, 40, 30, 20, 10], 2, 64, dtype, 16)
    starts = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    q, k, v = (rows(5, h, tokens, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    call = lambda: attention_shared(q, prefix, cache, k, v, starts=starts)  # noqa: E731
    clean = call()
    prefix.k[int(prefix.table[1, 7]), 1, 3, 9] = math.nan
    got = call()
    assert bool(torch.isnan(got[2:4, 2:]).all())
    assert torch.equal(got[:2], clean[:2]) and torch.equal(got[4], clean[4]) and torch.equal(got[2:4, :2], clean[2:4, :2])
    prefix.k[int(prefix.table[1, 7]), 1, 3, 9] = 0.0
    prefix.v[int(prefix.table[0, 2]), 0, 5, 11] = math.inf
    got = call()
    assert bool((got[:2, :2, :, 11] == math.inf).all()) and bool(torch.isfinite(got[2:]).all()) and bool(torch.isfinite(got[:2, 2:]).all())
    assert bool(torch.isfinite(got[:2, :2, :, :11]).all())


@gpu
def test_scores_far_apart():
    """A prefix whose scores are far above the cache's, or far below: one part weighs nothing, the statistics are the other's."""
    dtype, f = torch.float16, 30.0
    prefix, cache = make_cache([150], 2, 64, dtype, 16, seed=1), make_cache([60, 500, 0], 2, 64, dtype, 16)
    q = rows(3, 4, 1, 64, dtype, 1)
    for near in (prefix, cache):
        near.k.mul_(f)
        check_shared(prefix, cache, None, 4, 1, dtype, "causal", q=q, scale=0.125)
        near.k.div_(f)
    check_shared(prefix, cache, None, 4, 1, dtype, "causal", q=q, scale=0.0)


@gpu
def test_layouts():
    """Heads before positions, both caches in one pool, rows cut out of wider ones, a part of a wider table, a batch whose sequences lie apart."""
    dtype, dim = torch.bfloat16, 64
    pool = torch.randn(60, 2, 16, 2 * dim, device="cuda").to(dtype)
    pages = torch.randperm(60, device="cuda").to(torch.int32)
    prefix = KVCache(pool[..., :dim], pool[..., dim:], torch.tensor([300, 55], dtype=torch.int32).cuda(), pages[:44].view(2, 22)[:, 1:21])
    cache = KVCache(pool[..., :dim], pool[..., dim:], torch.tensor([31, 0, 47], dtype=torch.int32).cuda(), pages[44:53].view(3, 3))
    qkv = torch.randn(2 * 3, 5, 8 + 2 + 2, dim, device="cuda").to(dtype)[::2].transpose(1, 2)
    check_shared(prefix, cache, [0, 2, 3], 8, 5, dtype, "causal", q=qkv[:, :8], k=qkv[:, 8:10], v=qkv[:, 10:])
    one = qkv[:, :, 1:2]
    check_shared(prefix, cache, [0, 2, 3], 8, 1, dtype, "causal", q=one[:, :8], k=one[:, 8:10], v=one[:, 10:])


@gpu
def test_is_what_the_whole_sequence_gets():
    """The same through attention_cached with the prefix's pages in every sequence's table, up to the roundings of both."""
    dtype, batch = torch.float16, 6
    prefix, own = make_cache([16 * 20], 2, 64, dtype, 16, seed=1), make_cache([40, 3, 0, 100, 17, 64], 2, 64, dtype, 16, columns=8)
    count = prefix.k.shape[0]
    k, v = (torch.cat([getattr(prefix, n).transpose(1, 2), getattr(own, n).transpose(1, 2)]).transpose(1, 2) for n in ("k", "v"))
    whole = KVCache(k, v, own.lengths + 320, torch.cat([prefix.table[:, :20].expand(batch, 20), own.table + count], 1).contiguous())
    q, kn, vn = (rows(batch, h, 3, 64, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    a, sa = attention_shared(q, prefix, own, kn, vn, return_stats=True)
    b, sb = attention_cached(q, whole, kn, vn, return_stats=True)
    # (values of order 1, at most 5; P and output rounded on both sides)
    assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0**-11 * 5 and torch.allclose(sa, sb, rtol=1e-5, atol=1e-4)


@gpu
def test_what_the_device_says_wrongly_is_reported():
    dtype = torch.bfloat16
    prefix, cache = make_cache([100, 90], 2, 64, dtype, 16, seed=1), make_cache([30, 20, 400], 2, 64, dtype, 16)
    q, k, v = (rows(3, h, 1, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    good = torch.tensor([0, 1, 3], dtype=torch.int32).cuda()
    clean = attention_shared(q, prefix, cache, k, v, starts=good)
    bad_table, bad_length = prefix.table.clone(), prefix.lengths.clone()
    bad_table[1, 2] = 1000
    bad_length[0] = prefix.capacity + 1
    for starts, p, c in [
        (torch.tensor([0, 3, 1], dtype=torch.int32).cuda(), prefix, cache),
        (torch.tensor([0, 1, 4], dtype=torch.int32).cuda(), prefix, cache),
        (torch.tensor([-1, 1, 3], dtype=torch.int32).cuda(), prefix, cache),
        (good, KVCache(prefix.k, prefix.v, prefix.lengths, bad_table), cache),
        (good, KVCache(prefix.k, prefix.v, bad_length, prefix.table), cache),
        (good, prefix, KVCache(cache.k, cache.v, torch.tensor([30, -5, 400], dtype=torch.int32).cuda(), cache.table)),
    ]:
        try:
            out, stats = attention_shared(q, p, c, k, v, starts=starts, return_stats=True)
            assert _lib.device_status() == _lib.DEV_BAD_CACHE
            if c is cache:
                assert bool(torch.isnan(out).all()) and bool(torch.isnan(stats).all())
        finally:
            _lib.reset_device_status()
    assert torch.equal(attention_shared(q, prefix, cache, k, v, starts=good), clean)


@gpu
def test_two_streams_and_capture():
    """Calls that overlap on two streams, each with scratch of its own; a captured call follows starts, lengths and contents."""
    dtype = torch.bfloat16
    prefix, cache = make_cache([3000, 500], 2, 128, dtype, 16, seed=1), make_cache([700, 20, 400, 90, 5, 61], 2, 128, dtype, 16, extra=40)
    starts = torch.tensor([0, 4, 6], dtype=torch.int32).cuda()
    qkv = [[rows(6, h, 2, 128, dtype, 10 * i + s) for h, s in ((8, 1), (2, 2), (2, 3))] for i in range(2)]
    want = [attention_shared(q, prefix, cache, k, v, starts=starts) for q, k, v in qkv]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, (q, k, v) in zip(streams, qkv):
            with torch.cuda.stream(s):
                got.append(attention_shared(q, prefix, cache, k, v, starts=starts))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, k, v = qkv[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = attention_shared(q, prefix, cache, k, v, starts=starts)
        second = attention_shared(q, prefix, cache, k, v, starts=starts)
    for step in range(3):
        starts[1] = 4 - step
        cache.lengths.add_(3)
        prefix.lengths[1] -= 7
        q.mul_(0.9)
        graph.replay()
        want = attention_shared(q, prefix, cache, k, v, starts=starts)
        assert torch.equal(first, want) and torch.equal(second, want)
    assert _lib.device_status() == 0


@gpu
def test_right_behind_the_writes_that_it_reads():
    """Kernels overlap the ends of those before them: keys, values, queries, lengths and prefixes that were written by the kernel just before are seen."""
    dtype, batch = torch.bfloat16, 24
    r = Rotary.of(128)
    prefix, cache = make_cache([900], 2, 128, dtype, 16, seed=1), make_cache([30] * batch, 2, 128, dtype, 16, extra=60)
    plain = KVCache(cache.k.clone(), cache.v.clone(), cache.lengths.clone(), cache.table)
    offset = torch.full((batch,), 900, dtype=torch.int32, device="cuda")
    for step in range(20):
        q, k, v = (rows(batch, h, 1, 128, dtype, 3 * step + s) for h, s in ((8, 1), (2, 2), (2, 3)))
        torch.cuda.synchronize()
        tq = cache_append_rotary(cache, q, k, v, r, offset=offset)
        cache.lengths += 1
        got = attention_shared(tq, prefix, cache)
        torch.cuda.synchronize()
        wq, wk = apply_rotary(q, k, r, offset=offset + plain.lengths)
        torch.cuda.synchronize()
        cache_append(plain, wk, v)
        torch.cuda.synchronize()
        plain.lengths += 1
        torch.cuda.synchronize()
        want = attention_shared(wq, prefix, plain)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_generation_from_a_shared_prompt():
    """A prompt stored once, several sequences that go on from it: every step equals attention over the whole rotated sequence."""
    dtype, heads, kv_heads, dim, batch, prompt, steps = torch.float16, 6, 2, 80, 4, 133, 9
    r = Rotary.of(40, interleaved=True)
    pq, pk, pv = (rows(1, h, prompt, dim, dtype, s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
    prefix, cache = KVCache.empty(1, kv_heads, 160, dim, page=16, dtype=dtype), KVCache.empty(batch, kv_heads, 32, dim, page=8, dtype=dtype)
    cache_append_rotary(prefix, pq, pk, pv, r)
    prefix.lengths += prompt
    offset = prefix.lengths.expand(batch).contiguous()
    q, k, v = (rows(batch, h, steps, dim, dtype, s) for h, s in ((heads, 4), (kv_heads, 5), (kv_heads, 6)))
    both = lambda a, b: torch.cat([a.expand(batch, -1, -1, -1), b], 2)  # noqa: E731
    wq, wk = apply_rotary(both(pq, q), both(pk, k), r)
    wv = both(pv, v)
    at = 0
    for tokens in (1, 1, 4, 1, 2):
        part = slice(at, at + tokens)
        tq, tk = cache_append_rotary(cache, q[:, :, part], k[:, :, part], v[:, :, part], r, offset=offset, return_keys=True)
        assert torch.equal(tq, wq[:, :, prompt + at : prompt + at + tokens]) and torch.equal(tk, wk[:, :, prompt + at : prompt + at + tokens])
        got = attention_shared(tq, prefix, cache, tk, v[:, :, part])
        cache.lengths += tokens
        n = prompt + at + tokens
        s = wq[:, :, n - tokens : n].double() @ wk[:, :, :n].double().repeat_interleave(heads // kv_heads, 1).transpose(2, 3) * dim**-0.5
        s = s.masked_fill(torch.arange(n, device="cuda") > torch.arange(n - tokens, n, device="cuda")[:, None], -math.inf)
        p, values = s.softmax(-1), wv[:, :, :n].double().repeat_interleave(heads // kv_heads, 1)
        room = (2.0**-11 + 2.0**-12) * (p @ values.abs()) + 2.0**-11 * (p @ values).abs() + 2.0**-24
        assert bool(((got.double() - p @ values).abs() <= room).all())
        at += tokens
    assert _lib.device_status() == 0


@gpu
def test_refusals():
    dtype = torch.bfloat16
    prefix, cache = make_cache([100, 90], 2, 64, dtype, 16, seed=1), make_cache([30, 20, 40], 2, 64, dtype, 16)
    q, k, v = (rows(3, h, 2, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    starts = torch.tensor([0, 1, 3], dtype=torch.int32).cuda()
    tree = torch.ones(2, 2, dtype=torch.bool, device="cuda")
    half = KVCache(prefix.k.half(), prefix.v.half(), prefix.lengths, prefix.table)
    for error, args, more in [
        (ValueError, (q, prefix, cache, k, v), {}),  # two prefixes without starts
        (ValueError, (q, prefix, cache, k, v), {"starts": starts[:2]}),
        (TypeError, (q, prefix, cache, k, v), {"starts": starts.long()}),
        (ValueError, (q, prefix, cache, k, v), {"starts": starts.cpu()}),
        (ValueError, (q, prefix, cache, k, None), {"starts": starts}),
        (ValueError, (q, prefix, cache), {"starts": starts, "tree": tree}),
        (TypeError, (q, half, cache, k, v), {"starts": starts}),
        (ValueError, (q, make_cache([9, 9], 1, 64, dtype, 16), cache, k, v), {"starts": starts}),
        (ValueError, (q, make_cache([9, 9], 2, 72, dtype, 16), cache, k, v), {"starts": starts}),
        (ValueError, (q[:, :3], prefix, cache, k, v), {"starts": starts}),
        (ValueError, (q[:2], prefix, cache, k[:2], v[:2]), {"starts": starts}),
        (ValueError, (q, prefix, cache, k, v), {"starts": starts, "scale": -1.0}),
        (TypeError, (q, prefix, cache, k, v), {"starts": starts, "counts": starts.float()}),
        (RuntimeError, (q.clone().requires_grad_(), prefix, cache, k, v), {"starts": starts}),
    ]:
        with pytest.raises(error):
            attention_shared(*args, **more)
    with torch.no_grad():
        attention_shared(q.clone().requires_grad_(), prefix, cache, k, v, starts=starts)


def test_refuses_without_a_gpu():
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    cache = KVCache(k, k.clone(), torch.zeros(2, dtype=torch.int32))
    prefix = KVCache(k[:1], k[:1].clone(), torch.zeros(1, dtype=torch.int32))
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attention_shared(q, prefix, cache)
    with pytest.raises(ValueError, match="starts"):
        attention_shared(q, cache, cache)
    with pytest.raises(TypeError):
        attention_shared(q.half(), prefix, cache)


def describe(cache):
    c = _lib.KfaCache()
    c.k, c.v = _lib.tensor4(cache.k), _lib.tensor4(cache.v)
    if cache.table is not None:
        c.table, c.table_stride, c.table_cols = cache.table.data_ptr(), cache.table.stride(0), cache.table.shape[1]
    c.lengths, c.batch = cache.lengths.data_ptr(), cache.lengths.numel()
    return ctypes.byref(c)


def ref(t):
    return ctypes.byref(_lib.tensor4(t))


@gpu
def test_the_c_entry_refuses():
    dtype, lib = torch.bfloat16, _lib.load()
    prefix, cache = make_cache([100, 90], 2, 64, dtype, 16, seed=1), make_cache([30, 20, 40], 2, 64, dtype, 16)
    other = make_cache([100, 90], 4, 64, dtype, 16, seed=1)
    q, k, v = (rows(3, h, 2, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    starts = torch.tensor([0, 1, 3], dtype=torch.int32).cuda()
    room = lib.kfa_cache_attend_shared_bytes(ref(q), describe(prefix), describe(cache), ref(k))
    scratch, out = torch.zeros(room // 4 + 8, device="cuda"), torch.zeros_like(q)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(q=q, prefix=prefix, starts=starts.data_ptr(), cache=cache, k=k, v=v, out=out, scratch=scratch.data_ptr(), scale=0.1, dtype=1, status=word.data_ptr()):
        return lib.kfa_cache_attend_shared(
            ref(q), describe(prefix), starts, describe(cache), None if k is None else ref(k), None if v is None else ref(v), None, None, None, ref(out), None,
            scratch, scale, dtype, status, _lib.stream_ptr(torch.device("cuda", 0)),
        )  # fmt: skip

    for bad in ({"starts": None}, {"prefix": other}, {"cache": other}, {"k": None}, {"scratch": None}, {"scratch": scratch.data_ptr() + 4}, {"scale": math.nan},
                {"dtype": 2}, {"status": None}, {"q": q[:, :3]}, {"out": out[:, :, :1]}):  # fmt: skip
        assert call(**bad) == -1, bad
        assert lib.kfa_last_error()
    assert call() == 0
    torch.cuda.synchronize()
    assert torch.equal(out, attention_shared(q, prefix, cache, k, v, starts=starts, scale=0.1)) and int(word.item()) == 0


@gpu
@pytest.mark.parametrize("tokens,columns", [(1, 4), (1, 80), (20, 80), (40, 80)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_wait_that_runs_out_is_reported_and_the_context_survives(tokens, columns, dim):
    """The library whose waits are a few hundred cycles (see test_cache_abort.py): each call ends, reports, and leaves NaN."""
    assert build.LIB_SHORT_WAIT.exists()
    short, shipped = ctypes.CDLL(str(build.LIB_SHORT_WAIT)), _lib.load()
    for name in ("kfa_cache_attend_shared", "kfa_cache_attend_shared_bytes"):
        getattr(short, name).argtypes, getattr(short, name).restype = getattr(shipped, name).argtypes, getattr(shipped, name).restype
    dtype = torch.bfloat16
    prefix = make_cache([16 * columns - 3], 2, dim, dtype, 16, seed=1)
    cache = make_cache([16 * columns - 40, 20], 2, dim, dtype, 16, columns=columns)
    q, k, v = (rows(2, h, tokens, dim, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, stats = torch.zeros_like(q), torch.zeros(2, 8, 2, tokens, device="cuda")
    room = short.kfa_cache_attend_shared_bytes(ref(q), describe(prefix), describe(cache), ref(k))
    scratch = torch.zeros(room // 4 + 8, device="cuda")
    rc = short.kfa_cache_attend_shared(ref(q), describe(prefix), None, describe(cache), ref(k), ref(v), None, None, None, ref(out), stats.data_ptr(),
                                       scratch.data_ptr(), dim**-0.5, 1, word.data_ptr(), _lib.stream_ptr(torch.device("cuda", 0)))  # fmt: skip
    assert rc == 0
    torch.cuda.synchronize()  # returns: nothing hangs
    assert 170 <= int(word.item()) <= 190, int(word.item())
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(stats).all())
    assert bool(torch.isfinite(attention_shared(q, prefix, cache, k, v)).all()) and _lib.device_status() == 0
