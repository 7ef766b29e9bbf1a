"""The operators on a cache of keys and values against plain implementations in 64 bits.

Tolerances. ``attention_cached``: P is rounded to 16 bits before the second product and the output once more, each by at most
u = eps / 2 relative (bf16 2^-8, fp16 2^-11); a row's P have the common factor 1 / l, so its error is at most u * sum_j p_j |v_j| from P and u |o| from
the output. Scores carry a few 2^-24 of sum |q_d k_d| from the tensor core's adder (D terms, truncated), which moves P by that times the scale: below
2^-15 for the inputs here (|q|, |k| of order 1, D <= 128) and covered by an extra 2^-12. So |out - exact| <= (u + 2^-12) * sum p |v| + u |out| + 2^-24.
``cache_weights``: fp32 throughout: an exponent off by 2^-24 * (sum |q_d k_d| + |m|) * scale * log2 e and the function's own 2^-22: 2^-13 relative.
Copies and selections are exact."""

import math

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_cached, cache_append, cache_evict, cache_weights, tree_mask

LOG2E = 1.4426950408889634


def make_cache(lengths, kv_heads, dim, dtype, page=None, extra=0, seed=0, columns=None, fill=None, spare=2):
    """A cache whose pages lie in random order, filled with random values everywhere (also behind the lengths), and the
    logical keys and values [B, Hkv, capacity, D] as float64 on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    batch, most = len(lengths), max(lengths) + extra
    if page is None:
        count, size, table = batch, max(columns or most, 1), None
    else:
        cols = columns or max(1, -(-most // page))
        count, size = batch * cols + spare, page
        table = torch.randperm(count, generator=gen)[: batch * cols].view(batch, cols).to(torch.int32)
    k, v = (torch.randn(count, size, kv_heads, dim, generator=gen).to(dtype) for _ in range(2))
    if fill is not None:  # what lies behind the lengths
        logical = torch.zeros(count, size, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for p in range(n + extra):
                at = (b, p) if table is None else (int(table[b, p // page]), p % page)
                logical[at] = True
        k[~logical], v[~logical] = fill, fill
    cache = KVCache(*(t.cuda().transpose(1, 2) for t in (k, v)), torch.tensor(lengths, dtype=torch.int32).cuda(),
                    None if table is None else table.cuda())  # fmt: skip
    return cache


def logical(cache, which="k"):
    pages = getattr(cache, which).detach().double().cpu()
    if cache.table is None:
        return pages
    return pages[cache.table.cpu().long().clamp(0, pages.shape[0] - 1)].transpose(1, 2).flatten(2, 3)


def rows(batch, heads, tokens, dim, dtype, seed):
    gen = torch.Generator().manual_seed(1000 + seed)
    return torch.randn(batch, tokens, heads, dim, generator=gen).to(dtype).cuda().transpose(1, 2)


def random_tree(batch, tokens, seed):
    gen = torch.Generator().manual_seed(seed)
    parents = torch.stack([torch.tensor([int(torch.randint(-1, t, (1,), generator=gen)) if t else -1 for t in range(tokens)]) for _ in range(batch)])
    return tree_mask(parents)


def exact_attention(q, cache, k, v, tree, counts, scale):
    """out, sum p |v|, m, log2 l in 64 bits on the CPU; rows that see nothing: 0, 0, +inf, 0."""
    q = q.double().cpu()
    batch, heads, tokens, dim = q.shape
    kc, vc, lengths = logical(cache, "k"), logical(cache, "v"), cache.lengths.tolist()
    group = heads // kc.shape[1]
    out, size = torch.zeros(2, batch, heads, tokens, dim, dtype=torch.float64)
    m, log2l = torch.full((batch, heads, tokens), math.inf, dtype=torch.float64), torch.zeros(batch, heads, tokens, dtype=torch.float64)
    for b in range(batch):
        count = tokens if counts is None else int(counts[b])
        for h in range(heads):
            for t in range(count):
                keys, values = kc[b, h // group, : lengths[b]], vc[b, h // group, : lengths[b]]
                if k is not None:
                    sees = torch.arange(tokens) <= t if tree is None else (tree if tree.dim() == 2 else tree[b])[t].cpu()
                    sees = sees & (torch.arange(tokens) < count)
                    keys = torch.cat([keys, k[b, h // group].double().cpu()[sees]])
                    values = torch.cat([values, v[b, h // group].double().cpu()[sees]])
                if not len(keys):
                    continue
                s = keys @ q[b, h, t]
                m[b, h, t] = s.max()
                e = torch.exp((s - s.max()) * scale)
                log2l[b, h, t] = e.sum().log2()
                p = e / e.sum()
                out[b, h, t], size[b, h, t] = p @ values, p @ values.abs()
    return out, size, m, log2l


def check_attention(cache, heads, tokens, dtype, new="causal", counts=None, seed=0, scale=None, k=None, v=None, q=None):
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
    got, stats = attention_cached(q, cache, k, v, tree=None if tree is None else tree.cuda(), counts=count, scale=scale, return_stats=True)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    scale = dim**-0.5 if scale is None else scale
    out, size, m, log2l = exact_attention(q, cache, k, v, tree, counts, scale)
    u = torch.finfo(dtype).eps / 2
    assert got.shape == q.shape and got.dtype == dtype
    off = (got.double().cpu() - out).abs()
    room = (u + 2.0**-12) * size + u * out.abs() + 2.0**-24
    assert bool((off <= room).all()), float((off / room).max())
    stats = stats.double().cpu()
    fine = torch.isfinite(m)
    assert torch.equal(torch.isinf(stats[:, :, 0]), ~fine) and bool((stats[:, :, 1][~fine] == 0).all())
    assert torch.allclose(stats[:, :, 0][fine], m[fine], rtol=2.0**-18, atol=2.0**-16)
    assert torch.allclose(stats[:, :, 1], log2l, rtol=2.0**-16, atol=2.0**-13)
    return got


# (lengths, page, heads, K / V heads, tokens, head dim)
SHAPES = [
    ([100], None, 8, 8, 1, 64),
    ([1, 0, 33], None, 4, 2, 1, 64),
    ([31, 32, 33, 127, 128, 129], 16, 4, 1, 1, 128),
    ([257, 5, 0, 640], 32, 8, 2, 5, 64),
    ([300, 77], 48, 6, 3, 7, 80),
    ([200, 64], 8, 16, 1, 3, 128),
    ([70, 500], 128, 8, 4, 33, 128),
    ([513, 2], 64, 8, 1, 40, 128),
    ([90, 10], 16, 3, 3, 2, 40),
    ([65, 130], 24, 2, 1, 17, 16),
    ([20, 6], None, 5, 5, 130, 8),
    ([1500], 16, 40, 2, 9, 72),
    ([33], 8, 130, 1, 2, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("new", ["causal", "tree", "none"])
def test_attention(shape, new, dtype):
    lengths, page, heads, kv_heads, tokens, dim = shape
    check_attention(make_cache(lengths, kv_heads, dim, dtype, page), heads, tokens, dtype, new, seed=len(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,lengths", [(1, [40000]), (6, [9000, 1, 20011, 0, 3000]), (1, [2000] * 40), (20, [700, 4100])])
def test_attention_split_over_the_keys(tokens, lengths):
    check_attention(make_cache(lengths, 2, 128, torch.bfloat16, 16), 8, tokens, torch.bfloat16, "tree")
    check_attention(make_cache(lengths, 1, 64, torch.float16), 2, tokens, torch.float16, "none")


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_what_lies_behind_a_sequence_does_not_matter(page, fill):
    """Stale cache positions, and the rows of new tokens that counts leaves out, hold NaN or infinities."""
    lengths, counts, dtype = [100, 0, 31, 257, 64], [5, 3, 0, 1, 6], torch.bfloat16
    cache = make_cache(lengths, 2, 64, dtype, page, fill=fill, columns=None if page is None else 40)
    q, k, v = (rows(5, h, 6, 64, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    for b, n in enumerate(counts):
        for t in (q, k, v):
            t[b, :, n:] = fill
    got = check_attention(cache, 8, 6, dtype, "tree", counts, q=q, k=k, v=v)
    assert bool(torch.isfinite(got).all())
    for b, n in enumerate(counts):
        assert bool((got[b, :, n:] == 0).all())
    check_attention(cache, 8, 6, dtype, "none", counts, q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_new_tokens_do_not_matter(dim):
    """A new token whose key and value are NaN or infinite reaches exactly the rows that see it."""
    dtype, tokens = torch.float16, 12
    cache = make_cache([50, 0], 2, dim, dtype, 16)
    q, k, v = (rows(2, h, tokens, dim, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    tree = random_tree(2, tokens, 5)
    clean = attention_cached(q, cache, k, v, tree=tree.cuda())
    for what, place in ((float("nan"), "k"), (float("nan"), "v"), (float("inf"), "v"), (-float("inf"), "v")):
        k2, v2 = k.clone(), v.clone()
        (k2 if place == "k" else v2)[0, 1, 4, 3] = what
        got = attention_cached(q, cache, k2, v2, tree=tree.cuda())
        touched = torch.zeros_like(clean, dtype=torch.bool)
        seen = tree[0, :, 4]
        if place == "k":
            touched[0, 2:, seen] = True
        else:
            touched[0, 2:, seen, 3] = True
        assert torch.equal(got[~touched], clean[~touched])
        if place == "k" or what != what:
            assert bool(torch.isnan(got[touched]).all())
        else:
            assert bool((got[touched] == what).all())


@pytest.mark.gpu
def test_rows_that_see_nothing():
    dtype, tokens = torch.bfloat16, 4
    tree = torch.zeros(tokens, tokens, dtype=torch.bool)
    tree[2, 1] = True
    got = check_attention(make_cache([0, 0], 2, 64, dtype, 16), 4, tokens, dtype, tree)
    assert bool((got[:, :, [0, 1, 3]] == 0).all()) and bool((got[:, :, 2] != 0).any())
    got = check_attention(make_cache([0, 10], 1, 128, dtype), 2, tokens, dtype, "none")
    assert bool((got[0] == 0).all())


@pytest.mark.gpu
def test_attention_layouts():
    """Pages with heads before positions, rows cut out of wider tensors, a transposed and an expanded tree, a table that is part of a
    larger one."""
    dtype, dim = torch.bfloat16, 64
    pool = torch.randn(30, 2, 16, 2 * dim, device="cuda").to(dtype)
    wide = torch.randperm(30, device="cuda")[:28].view(2, 14).to(torch.int32)
    cache = KVCache(pool[..., :dim], pool[..., dim:], torch.tensor([100, 37], dtype=torch.int32).cuda(), wide[:, 3:10])
    qkv = torch.randn(2, 5, 8 + 2 + 2, dim, device="cuda").to(dtype).transpose(1, 2)
    tree = random_tree(1, 5, 3)[0].T.contiguous().cuda().T
    check_attention(cache, 8, 5, dtype, tree, q=qkv[:, :8], k=qkv[:, 8:10], v=qkv[:, 10:])
    check_attention(cache, 8, 5, dtype, tree[None].expand(2, 5, 5), q=qkv[:, :8], k=qkv[:, 8:10], v=qkv[:, 10:])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", range(8, 129, 24))
@pytest.mark.parametrize("tokens", [1, 30])
def test_attention_head_dims(dim, tokens):
    """Head dims that are multiples of 8, in both kernels (4 and 120 rows a K / V head)."""
    check_attention(make_cache([333, 40, 0], 2, dim, torch.bfloat16, 16), 8, tokens, torch.bfloat16, "tree", seed=dim)


@pytest.mark.gpu
def test_attention_many_sequences():
    """More sequences than the threads of a CTA, most of them short, some empty."""
    gen = torch.Generator().manual_seed(0)
    lengths = torch.randint(0, 40, (900,), generator=gen).tolist()
    lengths[5], lengths[850], lengths[-1] = 1500, 700, 0
    check_attention(make_cache(lengths, 1, 64, torch.float16, 8), 4, 1, torch.float16, "causal")


@pytest.mark.gpu
def test_attention_many_heads_and_tokens():
    check_attention(make_cache([70], 1, 64, torch.bfloat16, 16), 300, 1, torch.bfloat16, "causal")  # two tiles of heads
    check_attention(make_cache([100, 3], 1, 32, torch.bfloat16, 16), 4, 200, torch.bfloat16, "causal")  # four of tokens
    check_attention(make_cache([2600], 1, 64, torch.float16, 16), 4, 20, torch.float16, "tree")  # 80 rows, cut


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40])
def test_a_nan_that_is_seen_is_passed_on(tokens):
    dtype = torch.bfloat16
    cache = make_cache([200, 600], 2, 64, dtype, 16)
    q, k, v = (rows(2, h, tokens, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    clean, stats = attention_cached(q, cache, k, v, return_stats=True)
    cache.k[int(cache.table[1, 7]), 1, 3, 9] = float("nan")
    got, got_stats = attention_cached(q, cache, k, v, return_stats=True)
    assert bool(torch.isnan(got[1, 2:]).all()) and bool(torch.isnan(got_stats[1, 2:, 1]).all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :2], clean[1, :2]) and torch.equal(got_stats[0], stats[0])
    q[0, 1] = float("nan")
    got = attention_cached(q, cache, k, v)
    assert bool(torch.isnan(got[0, 1]).all()) and torch.equal(got[0, [0, 2, 3]], clean[0, [0, 2, 3]])
    cache = make_cache([0, 0], 2, 64, dtype, 16)  # nothing but NaN to see
    assert bool(torch.isnan(attention_cached(q, cache, k, v)[0, 1]).all())


@pytest.mark.gpu
def test_large_scores_and_scales():
    dtype = torch.float16
    cache = make_cache([300, 40], 2, 64, dtype, 16)
    q = rows(2, 4, 3, 64, dtype, 9) * 8
    check_attention(cache, 4, 3, dtype, "causal", q=q, scale=0.25)
    check_attention(cache, 4, 3, dtype, "causal", scale=0.0)
    check_attention(cache, 4, 50, dtype, "tree", q=rows(2, 4, 50, 64, dtype, 9) * 8, scale=0.25)
    check_attention(cache, 4, 50, dtype, "tree", scale=0.0)
    check_attention(cache, 4, 3, dtype, "none", q=-q.abs(), scale=1.0)


def exact_weights(cache, q, stats, index, counts, scale):
    q, stats, keys, lengths = q.double().cpu(), stats.double().cpu(), logical(cache, "k"), cache.lengths.tolist()
    batch, heads, tokens, _ = q.shape
    total = torch.zeros(batch, keys.shape[1], keys.shape[2], dtype=torch.float64)
    group = heads // keys.shape[1]
    steps = tokens if index is None else index.shape[1]
    for b in range(batch):
        for i in range(steps if counts is None else int(counts[b])):
            t = i if index is None else int(index[b, i])
            last = lengths[b] + i + 1
            for h in range(heads):
                if stats[b, h, 0, t] == math.inf:
                    continue
                s = keys[b, h // group, :last] @ q[b, h, t]
                total[b, h // group, :last] += torch.exp((s - stats[b, h, 0, t]) * scale - stats[b, h, 1, t] / LOG2E)
    return total


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("accepted", [False, True])
def test_weights(shape, accepted):
    lengths, page, heads, kv_heads, tokens, dim = shape
    batch, dtype = len(lengths), torch.bfloat16
    cache = make_cache(lengths, kv_heads, dim, dtype, page, extra=tokens)
    q, k, v = (rows(batch, h, tokens, dim, dtype, s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
    gen = torch.Generator().manual_seed(3)
    index = counts = None
    if accepted:
        steps = max(1, tokens // 2)
        index = torch.stack([torch.randperm(tokens, generator=gen)[:steps].sort().values for _ in lengths]).to(torch.int32).cuda()
        counts = torch.randint(0, steps + 1, (batch,), generator=gen).to(torch.int32).cuda()
    _, stats = attention_cached(q, cache, k, v, return_stats=True)
    cache_append(cache, k, v, index=index, counts=counts)
    got = cache_weights(cache, q, stats, index=index, counts=counts)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    want = exact_weights(cache, q, stats, index, counts, dim**-0.5)
    assert got.shape == (batch, kv_heads, cache.capacity)
    assert torch.allclose(got.double().cpu(), want, rtol=2.0**-13, atol=2.0**-24)
    before = torch.rand(batch, kv_heads, cache.capacity + 3, device="cuda")
    sums = before.clone()
    assert cache_weights(cache, q, stats, index=index, counts=counts, weights=sums) is sums
    assert torch.allclose(sums[..., : cache.capacity], before[..., : cache.capacity] + got, rtol=2.0**-22, atol=0)
    for b, n in enumerate(lengths):
        last = 0 if counts is not None and int(counts[b]) == 0 else n + (tokens if counts is None else int(counts[b]))
        assert torch.equal(sums[b, :, last:], before[b, :, last:])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 90])
def test_weights_of_large_scores(tokens):
    """Scores of some hundreds, where a row's maximum and log2 sum do not fit into one fp32 number: the exponent's error stays 2^-24 of the
    score's terms (64 products of up to 8 * 4, summed: 2^-24 * 64 * 32 * 8 * 0.25 * log2 e = 2^-10.5)."""
    dtype = torch.float16
    cache = make_cache([300, 40], 2, 64, dtype, 16, extra=tokens)
    q, k, v = rows(2, 4, tokens, 64, dtype, 1) * 8, rows(2, 2, tokens, 64, dtype, 2), rows(2, 2, tokens, 64, dtype, 3)
    _, stats = attention_cached(q, cache, k, v, scale=0.25, return_stats=True)
    cache_append(cache, k, v)
    got = cache_weights(cache, q, stats, scale=0.25)
    want = exact_weights(cache, q, stats, None, None, 0.25)
    assert torch.allclose(got.double().cpu(), want, rtol=2.0**-10, atol=2.0**-24)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,tokens", [(4, 6), (8, 40)])
def test_weights_skip_what_is_not_there(heads, tokens):
    """Rows that counts leaves out, and rows that saw nothing (m = +inf), hold NaN; weights of a tensor with wider rows; a sequence without
    tokens; more sequences than the threads of a CTA."""
    dtype, batch = torch.bfloat16, 500
    gen = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 30, (batch,), generator=gen).tolist()
    cache = make_cache(lengths, 2, 64, dtype, 16, extra=tokens, fill=float("nan"))
    q, k, v = (rows(batch, h, tokens, 64, dtype, s) for h, s in ((heads, 1), (2, 2), (2, 3)))
    counts = torch.randint(0, tokens + 1, (batch,), generator=gen).to(torch.int32).cuda()
    _, stats = attention_cached(q, cache, k, v, counts=counts, return_stats=True)
    cache_append(cache, k, v, counts=counts)
    behind = torch.arange(tokens, device="cuda") >= counts[:, None]
    q.masked_fill_(behind[:, None, :, None], float("nan"))
    stats[:, :, 0, 1] = math.inf  # the second token saw nothing
    q[:, :, 1] = float("nan")
    wide = torch.full((batch, 2, cache.capacity + 40), 7.0, device="cuda")
    got = cache_weights(cache, q, stats, counts=counts, weights=wide)
    want = exact_weights(cache, torch.nan_to_num(q), stats, None, counts, 64**-0.5)
    assert torch.allclose(got[..., : cache.capacity].double().cpu(), want + 7, rtol=2.0**-13, atol=2.0**-13)
    assert bool((got[..., cache.capacity :] == 7).all())
    fresh = cache_weights(cache, q, stats, counts=counts)
    assert torch.allclose(fresh.double().cpu(), want, rtol=2.0**-13, atol=2.0**-24)
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [80, 64])
def test_weights_of_many_short_pieces(dim):
    """Sequences without tokens next to others: a CTA's two streams take a piece each, and while one waits for its keys the other is done
    with pieces that have none. Long sequences between them keep the memory busy."""
    batch, kv_heads = 200, 8
    gen = torch.Generator().manual_seed(4)
    counts = torch.randint(0, 2, (batch,), generator=gen).to(torch.int32).cuda()
    lengths = [(900, 639, 100, 30, 1)[int(i)] for i in torch.randint(0, 5, (batch,), generator=gen)]
    cache = make_cache(lengths, kv_heads, dim, torch.float16, extra=4)
    q, k, v = (rows(batch, kv_heads, 4, dim, torch.float16, s) for s in (1, 2, 3))
    _, stats = attention_cached(q, cache, k, v, return_stats=True)
    cache_append(cache, k, v, counts=counts)
    want = exact_weights(cache, q, stats, None, counts, dim**-0.5)
    other = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for n in range(60):
        if n % 2 == 0:
            other.fill_(n)  # (the keys come from memory, not from the cache of the device)
        got = cache_weights(cache, q, stats, counts=counts)
        first = got if first is None else first
        assert torch.equal(got, first), n
    assert torch.allclose(first.double().cpu(), want, rtol=2.0**-13, atol=2.0**-24)
    out = attention_cached(q, cache, k, v, counts=counts)
    for n in range(60):
        if n % 2 == 0:
            other.fill_(n)
        assert torch.equal(attention_cached(q, cache, k, v, counts=counts), out), n
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_weights_of_a_prompt_sum_to_its_rows():
    """Every row's weights add up to 1: with an empty cache all positions together got one per row and head."""
    dtype, tokens = torch.bfloat16, 700
    cache = make_cache([0, 0], 2, 64, dtype, 16, extra=tokens)
    q, k, v = (rows(2, h, tokens, 64, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    _, stats = attention_cached(q, cache, k, v, return_stats=True)
    cache_append(cache, k, v)
    got = cache_weights(cache, q, stats)
    assert torch.allclose(got.sum(-1), torch.full((2, 2), 4.0 * tokens, device="cuda"), rtol=2.0**-12)
    want = exact_weights(cache, q, stats, None, None, 64**-0.5)
    assert torch.allclose(got.double().cpu(), want, rtol=2.0**-13, atol=2.0**-24)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 8, 24])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append(page, dtype):
    lengths, tokens, dim = [0, 17, 40, 7], 9, 40
    cache = make_cache(lengths, 3, dim, dtype, page, extra=tokens)
    k, v = rows(4, 3, tokens, dim, dtype, 1), rows(4, 3, tokens, dim, dtype, 2)
    index = torch.tensor([[8, 2, 2, 0]] * 4, dtype=torch.int32).cuda()  # (a token may be taken twice)
    for idx, counts in ((None, None), (index, None), (index, [3, 0, 4, 9]), (None, [9, 1, 0, -2])):
        before = cache.k.clone(), cache.v.clone()
        count = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
        want = [t.clone() for t in before]
        steps = tokens if idx is None else 4
        for b, n in enumerate(lengths):
            for i in range(steps if counts is None else max(0, min(counts[b], steps))):
                p = n + i
                at = (b, p) if page is None else (int(cache.table[b, p // page]), p % page)
                for w, new in zip(want, (k, v)):
                    w[at[0], :, at[1]] = new[b, :, i if idx is None else int(idx[b, i])]
        cache_append(cache, k, v, index=idx, counts=count)
        assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])
    assert _lib.device_status() == 0


def expect_evicted(weights, lengths, keep, recent):
    """kept [B, Hkv, keep], from a sort."""
    batch, heads, _ = weights.shape
    kept = torch.full((batch, heads, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for g in range(heads):
            w = weights[b, g, :n].cpu()
            if n <= keep:
                stay = torch.arange(n)
            else:
                old = torch.sort(w[: n - recent], descending=True, stable=True).indices[: keep - recent]
                stay = torch.cat([old.sort().values, torch.arange(n - recent, n)])
            kept[b, g, : len(stay)] = stay.to(torch.int32)
    return kept


WEIGHTS = {
    "spread": lambda w: w.mul(3).exp(),
    "few values": lambda w: (w * 2).round(),
    "all equal": torch.zeros_like,
    "signed zeros": lambda w: torch.where(w > 0, 0.0, -0.0),
    "infinities and NaN": lambda w: torch.where(w > 1.5, math.nan, torch.where(w < -1, -math.inf, torch.where(w > 1, math.inf, w))),
    "tiny": lambda w: w.abs() * 1e-42,
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", WEIGHTS)
@pytest.mark.parametrize("keep,recent", [(64, 16), (1, 0), (1, 1), (100, 100), (300, 0), (5000, 7)])
def test_evict(kind, keep, recent):
    lengths, dtype, dim = [300, 0, 64, 65, 3000, 1], torch.bfloat16, 40
    cache = make_cache(lengths, 2, dim, dtype, 16)
    gen = torch.Generator().manual_seed(keep)
    weights = WEIGHTS[kind](torch.randn(6, 2, cache.capacity + 1, generator=gen)).cuda()
    want = expect_evicted(weights, lengths, keep, recent)
    k, v = logical(cache, "k"), logical(cache, "v")
    fresh = cache_evict(cache, weights, keep, recent=recent)
    target = make_cache([keep] * 6, 2, dim, dtype, 32, seed=5)
    before = logical(target, "k"), logical(target, "v")
    given = cache_evict(cache, weights, keep, recent=recent, out=target)
    assert given[0].k is target.k and given[0].table is target.table
    for (got, w_out, kept), behind in ((fresh, (torch.zeros_like(before[0]),) * 2), (given, before)):
        assert torch.equal(kept.cpu(), want)
        assert got.lengths.tolist() == [min(n, keep) for n in lengths]
        picked = weights.cpu().gather(2, want.clamp(min=0).long())
        picked[want < 0] = 0
        assert torch.equal(torch.nan_to_num(w_out.cpu(), 7.0, 8.0, -8.0), torch.nan_to_num(picked, 7.0, 8.0, -8.0))
        for pages, source, rest in ((logical(got, "k"), k, behind[0]), (logical(got, "v"), v, behind[1])):
            rows_ = source.gather(2, want.clamp(min=0).long()[..., None].expand(-1, -1, -1, dim))
            rest = rest[:, :, :keep].clone()
            rest[want >= 0] = rows_[want >= 0]
            assert torch.equal(pages[:, :, :keep], rest)
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 16])
def test_a_run_of_them(page):
    """Decoding by drafts with a bounded cache: every step's attention against a plain cache in 64 bits that is kept beside it."""
    batch, heads, kv_heads, dim, dtype, budget = 3, 4, 2, 64, torch.bfloat16, 48
    cache = KVCache.empty(batch, kv_heads, 96, dim, dtype=dtype, page=page)
    assert cache.capacity == 96 and cache.lengths.tolist() == [0, 0, 0]
    total = torch.zeros(batch, kv_heads, 96, device="cuda")
    gen = torch.Generator().manual_seed(0)
    for step in range(14):
        tokens = 20 if step == 0 else 6
        q, k, v = (rows(batch, h, tokens, dim, dtype, 10 * step + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
        tree = None if step == 0 else random_tree(batch, tokens, step)
        check_attention(cache, heads, tokens, dtype, "causal" if tree is None else tree, q=q, k=k, v=v)
        out, stats = attention_cached(q, cache, k, v, tree=None if tree is None else tree.cuda(), return_stats=True)
        if step == 0:
            index, counts = None, torch.tensor([20, 7, 13], dtype=torch.int32).cuda()
        else:  # a path of the tree: the last token and those it follows
            index = torch.zeros(batch, tokens, dtype=torch.int32)
            counts = torch.zeros(batch, dtype=torch.int32)
            for b in range(batch):
                path = tree[b, int(torch.randint(0, tokens, (1,), generator=gen))].nonzero().flatten()
                index[b, : len(path)], counts[b] = path.to(torch.int32), len(path)
            index, counts = index.cuda(), counts.cuda()
        cache_append(cache, k, v, index=index, counts=counts)
        old = total.clone()
        cache_weights(cache, q, stats, index=index, counts=counts, weights=total)
        want = exact_weights(cache, q, stats, index, counts, dim**-0.5)
        assert torch.allclose((total - old).double().cpu(), want, rtol=1e-3, atol=2.0**-20)
        cache.lengths += counts
        if int(cache.lengths.max()) > 80:
            kept_before = cache.lengths.tolist()
            smaller, weights, kept = cache_evict(cache, total, budget, recent=8, out=KVCache.empty(batch, kv_heads, 96, dim, dtype=dtype, page=page))
            assert torch.equal(kept.cpu(), expect_evicted(total, kept_before, budget, 8))
            cache = smaller
            total = torch.zeros(batch, kv_heads, 96, device="cuda")
            total[..., :budget] = weights
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    cache = make_cache([5000, 33, 900], 2, 128, torch.bfloat16, 16, extra=4)
    q, k, v = (rows(3, h, 4, 128, torch.bfloat16, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    first = attention_cached(q, cache, k, v, return_stats=True)
    cache_append(cache, k, v)
    weights = cache_weights(cache, q, first[1])
    for _ in range(5):
        again = attention_cached(q, cache, k, v, return_stats=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
        assert torch.equal(cache_weights(cache, q, first[1]), weights)


@pytest.mark.gpu
def test_captured_step_follows_lengths_and_table():
    """One captured decoding step, replayed: lengths and table are read when it runs. Two graphs in flight on two streams."""
    dtype = torch.bfloat16
    caches = [make_cache([0, 0], 2, 64, dtype, 16, columns=8, seed=s) for s in (1, 2)]
    data = [[rows(2, h, 1, 64, dtype, 10 * s + i) for i, h in enumerate((8, 2, 2))] for s in (1, 2)]
    totals = [torch.zeros(2, 2, 128, device="cuda") for _ in caches]
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    outs, graphs, streams = [None, None], [], [torch.cuda.Stream(), torch.cuda.Stream()]

    def step(i):
        q, k, v = data[i]
        outs[i], stats = attention_cached(q, caches[i], k, v, return_stats=True)
        cache_append(caches[i], k, v)
        cache_weights(caches[i], q, stats, weights=totals[i])
        caches[i].lengths.add_(one)

    for i in range(2):
        step(i)  # eager once
        caches[i].lengths.zero_()
        totals[i].zero_()
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i)
        graphs.append(g)
    shadow = [([], []) for _ in caches]
    gen = torch.Generator().manual_seed(9)
    for n in range(40):
        for i in range(2):
            for t in data[i]:
                t.copy_(torch.randn(t.shape, generator=gen).to(dtype))
            shadow[i][0].append(data[i][1].double().cpu())
            shadow[i][1].append(data[i][2].double().cpu())
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            keys, values = (torch.cat(x, 2).repeat_interleave(4, 1) for x in shadow[i])
            p = torch.softmax(data[i][0].double().cpu() @ keys.transpose(2, 3) * 64**-0.5, -1)
            off = (outs[i].double().cpu() - p @ values).abs()
            assert bool((off <= 2.0**-6 * (p @ values.abs()) + 2.0**-24).all())
            assert caches[i].lengths.tolist() == [n + 1] * 2
            assert torch.allclose(totals[i].sum(-1), torch.full((2, 2), 4.0 * (n + 1), device="cuda"), rtol=1e-4)
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_other_stream():
    cache = make_cache([700, 12], 2, 64, torch.float16, 16)
    q, k, v = (rows(2, h, 3, 64, torch.float16, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    want = attention_cached(q, cache, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attention_cached(q, cache, k, v)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_pool_of_more_than_32_bits():
    """Pages whose offsets pass 2^32 bytes, read and written; the pool's other pages hold whatever was there."""
    page, dim, count = 16, 128, 1_100_000  # 4.5 GB each
    k, v = (torch.empty(count, page, 1, dim, dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in range(2))
    gen = torch.Generator().manual_seed(0)
    table = torch.randint(1_060_000, count, (2, 24), generator=gen).unique()[:40].flip(0).view(2, 20).to(torch.int32).cuda()
    cache = KVCache(k, v, torch.tensor([200, 37], dtype=torch.int32).cuda(), table)
    for pages in (k, v):
        pages[table.long()] = torch.randn(2, 20, 1, page, dim, generator=gen).to(torch.bfloat16).cuda()
    small = KVCache(k[table.flatten().long()], v[table.flatten().long()], cache.lengths, torch.arange(40, dtype=torch.int32).view(2, 20).cuda())
    q, kn, vn = (rows(2, h, 5, dim, torch.bfloat16, s) for h, s in ((4, 1), (1, 2), (1, 3)))
    results = []
    for c in (cache, small):
        out, stats = attention_cached(q, c, kn, vn, return_stats=True)
        cache_append(c, kn, vn)
        weights = cache_weights(c, q, stats)
        left, w_left, kept = cache_evict(c, weights, 40, recent=3)
        results.append((out, stats, weights, left.k, left.v, w_left, kept, c.k[c.table.long()], c.v[c.table.long()]))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_eviction_inside_one_pool_captured():
    """Out of some pages of a pool into others, in a graph: positions, lengths and weights are read when it runs."""
    pool = make_cache([128] * 8, 2, 64, torch.float16, 16)
    lengths, tables = torch.tensor([100, 9, 40], dtype=torch.int32).cuda(), [pool.table[i : i + 3].clone() for i in (0, 3)]
    source, target = (KVCache(pool.k, pool.v, lengths, t) for t in tables)
    weights = torch.rand(3, 2, 128, device="cuda")
    cache_evict(source, weights, 24, recent=4, out=target)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, w_out, kept = cache_evict(source, weights, 24, recent=4, out=target)
    for n in ([100, 9, 40], [128, 0, 24], [25, 128, 1]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        weights.copy_(torch.rand(3, 2, 128))
        k, rest = logical(source, "k"), logical(pool, "k")[6:]
        graph.replay()
        want = expect_evicted(weights, n, 24, 4)
        assert torch.equal(kept.cpu(), want) and got.lengths.tolist() == [min(x, 24) for x in n]
        moved = k.gather(2, want.clamp(min=0).long()[..., None].expand(-1, -1, -1, 64))
        assert torch.equal(logical(got, "k")[:, :, :24][want >= 0], moved[want >= 0])
        assert torch.equal(logical(source, "k"), k) and torch.equal(logical(pool, "k")[6:], rest)
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_inference_mode():
    with torch.inference_mode():
        cache = KVCache.empty(2, 2, 64, 64)
        q, k, v = (rows(2, h, 3, 64, torch.bfloat16, s) for h, s in ((8, 1), (2, 2), (2, 3)))
        out, stats = attention_cached(q, cache, k, v, return_stats=True)
        cache_append(cache, k, v)
        weights = cache_weights(cache, q, stats)
        cache.lengths += 3
        less, _, _ = cache_evict(cache, weights, 2, out=KVCache.empty(2, 2, 8, 64))
        assert torch.equal(cache.k[:, :, :3], k) and less.lengths.tolist() == [2, 2]
    before = cache.k.clone()
    with pytest.raises(RuntimeError, match="nference"):  # as torch has it for every write
        cache_append(cache, k, v)
    assert torch.equal(cache.k, before)


@pytest.mark.gpu
def test_calls_one_behind_the_other_among_others():
    """A long run of calls on two streams between kernels of every other kind, without a wait on the host: each result as if alone."""
    cache = make_cache([900, 30, 2000], 2, 128, torch.bfloat16, 16, extra=70)
    cases = [(t, [rows(3, h, t, 128, torch.bfloat16, 7 * t + i) for i, h in enumerate((8, 2, 2))]) for t in (1, 5, 16, 64)]
    want = []
    for _, (q, k, v) in cases:
        out, stats = attention_cached(q, cache, k, v, return_stats=True)
        cache_append(cache, k, v)
        want.append((out, cache_weights(cache, q, stats)))
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    caches = [KVCache(cache.k.clone(), cache.v.clone(), cache.lengths, cache.table) for _ in streams]
    torch.cuda.synchronize()
    for n in range(24):
        for stream, c in zip(streams, caches):
            with torch.cuda.stream(stream):
                i = n % len(cases)
                q, k, v = cases[i][1]
                q = q * 1.0  # (a kernel of another library right before and behind)
                out, stats = attention_cached(q, c, k, v, return_stats=True)
                cache_append(c, k, v)
                got.append((i, out * 1.0, cache_weights(c, q, stats)))
    torch.cuda.synchronize()
    for i, out, weights in got:
        assert torch.equal(out, want[i][0]) and torch.equal(weights, want[i][1])
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_compiled_calls_take_the_custom_ops():
    cache = make_cache([60, 12], 2, 64, torch.bfloat16, 16, extra=3)
    q, k, v = (rows(2, h, 3, 64, torch.bfloat16, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    kp, vp = cache.k.clone(), cache.v.clone()
    counts = torch.tensor([3, 1], dtype=torch.int32).cuda()

    def step(q, k, v, kp, vp, lengths, table):
        c = KVCache(kp, vp, lengths, table)
        out, stats = attention_cached(q, c, k, v, counts=counts, return_stats=True)
        cache_append(c, k, v, counts=counts)
        w = cache_weights(c, q, stats, counts=counts)
        small, w_small, kept = cache_evict(c, w, 16, recent=4)
        return out, stats, w, small.k, small.v, w_small, kept

    want = step(q, k, v, cache.k, cache.v, cache.lengths, cache.table)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, kp, vp, cache.lengths, cache.table)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(kp, cache.k) and torch.equal(vp, cache.v)


@pytest.mark.gpu
def test_what_a_cache_says_wrongly_is_reported():
    """Pages that are not there, lengths beyond the capacity, rows that do not exist: a status, NaN or nothing written, and no access
    outside the pages (the kernels check before they look)."""
    dtype = torch.bfloat16
    q, k, v = (rows(2, h, 3, 64, dtype, s) for h, s in ((4, 1), (2, 2), (2, 3)))
    index = torch.tensor([[0, 3], [0, 1]], dtype=torch.int32).cuda()

    def reported(call):
        torch.cuda.synchronize()
        assert _lib.device_status() == 0
        result = call()
        torch.cuda.synchronize()
        status = _lib.device_status()
        _lib.reset_device_status()
        assert status == 90
        return result

    def cache_with(lengths=(40, 20), table=None):
        c = make_cache([40, 20], 2, 64, dtype, 16, columns=4)
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        if table is not None:
            c.table[0, 1] = table
        return c

    stats = torch.zeros(2, 4, 2, 3, device="cuda")
    for c in (cache_with(table=-1), cache_with(table=10), cache_with(table=2**31 - 1), cache_with(lengths=(65, 20)), cache_with(lengths=(-1, 20))):
        out = reported(lambda: attention_cached(q, c, k, v))
        assert bool(torch.isnan(out[0]).all())
        fine = attention_cached(q, cache_with(), k, v)  # (the other sequence: as ever, or NaN where the report came first)
        assert torch.equal(out[1], fine[1]) or bool(torch.isnan(out[1]).any())
        reported(lambda: cache_evict(c, torch.rand(2, 2, 64, device="cuda"), 16))
    for c in (cache_with(lengths=(62, 20)), cache_with(lengths=(-1, 20)), cache_with(lengths=(16, 20), table=10), cache_with(lengths=(16, 20), table=-5)):
        reported(lambda: cache_append(c, k, v))
        reported(lambda: cache_weights(c, q, stats))
    reported(lambda: cache_append(cache_with(), k, v, index=index))
    reported(lambda: cache_weights(cache_with(), q, stats, index=index))
    with pytest.raises(_lib.KfaError, match="KVCache"):
        attention_cached(q, cache_with(table=10), k, v)
        try:
            _lib.check_status()
        finally:
            _lib.reset_status()
    # entries that no position needs may be anything
    c = cache_with()
    c.table[1, 2:] = -7
    assert torch.equal(attention_cached(q, c, k, v), attention_cached(q, cache_with(), k, v))
    assert _lib.device_status() == 0


def cpu_cache(**change):
    a = dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), v=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16),
             lengths=torch.zeros(2, dtype=torch.int32), table=torch.zeros(2, 2, dtype=torch.int32))  # fmt: skip
    a.update(change)
    return KVCache(**a)


def test_refused_caches():
    f32 = torch.zeros(4, 2, 16, 64)
    for error, change in (
        (TypeError, dict(k=f32, v=f32)),
        (TypeError, dict(v=f32.half())),
        (TypeError, dict(lengths=torch.zeros(2, dtype=torch.int64))),
        (TypeError, dict(table=torch.zeros(2, 2, dtype=torch.int64))),
        (ValueError, dict(v=torch.zeros(4, 2, 16, 32, dtype=torch.bfloat16))),
        (ValueError, dict(k=f32[..., :60].bfloat16(), v=f32[..., :60].bfloat16())),
        (ValueError, dict(k=torch.zeros(4, 2, 16, 136).bfloat16(), v=torch.zeros(4, 2, 16, 136).bfloat16())),
        (ValueError, dict(k=f32[:, :, :12].bfloat16(), v=f32[:, :, :12].bfloat16())),
        (ValueError, dict(lengths=torch.zeros(3, dtype=torch.int32))),
        (ValueError, dict(lengths=torch.zeros(4, dtype=torch.int32)[::2])),
        (ValueError, dict(table=None)),
        (ValueError, dict(table=torch.zeros(2, 0, dtype=torch.int32))),
        (ValueError, dict(table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2])),
        (ValueError, dict(k=f32[:0].bfloat16(), v=f32[:0].bfloat16())),
    ):
        with pytest.raises(error, match="KVCache"):
            cpu_cache(**change)
    assert cpu_cache().capacity == 32


def test_refused_calls():
    """Every refusal comes before anything is launched, and so on the CPU too; a call that is right is refused for its device."""
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    q, k = bf(2, 4, 3, 64), bf(2, 2, 3, 64)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    tree = torch.ones(3, 3, dtype=torch.bool)
    c = cpu_cache()
    for error, args, more in (
        (ValueError, (q, c, k, k), {}),  # the device
        (TypeError, (q.half(), c, k, k), {}),
        (TypeError, (q, c, k.float(), k), {}),
        (ValueError, (bf(2, 3, 3, 64), c, k, k), {}),
        (ValueError, (bf(1, 4, 3, 64), c, k, k), {}),
        (ValueError, (bf(2, 4, 3, 32), c, k, k), {}),
        (ValueError, (bf(2, 4, 0, 64), c, bf(2, 2, 0, 64), bf(2, 2, 0, 64)), {}),
        (ValueError, (q[0], c, k, k), {}),
        (ValueError, (q, c, k, None), {}),
        (ValueError, (q, c, bf(2, 2, 4, 64), bf(2, 2, 4, 64)), {}),
        (ValueError, (q, c, q, q), {}),
        (ValueError, (bf(2, 4, 64, 3).transpose(2, 3), c, k, k), {}),
        (ValueError, (bf(1, 4, 3, 64).expand(2, 4, 3, 64), c, k, k), {}),
        (ValueError, (q, c), dict(tree=tree)),
        (TypeError, (q, c, k, k), dict(tree=tree.int())),
        (ValueError, (q, c, k, k), dict(tree=tree[:2])),
        (ValueError, (q, c, k, k), dict(tree=tree.expand(3, 3, 3))),
        (TypeError, (q, c, k, k), dict(counts=torch.zeros(2, dtype=torch.int64))),
        (ValueError, (q, c, k, k), dict(counts=ints(3))),
        (ValueError, (q, c, k, k), dict(scale=float("nan"))),
        (ValueError, (q, c, k, k), dict(scale=-1.0)),
        (RuntimeError, (q.clone().requires_grad_(), c, k, k), {}),
    ):
        with pytest.raises(error, match="attention_cached"):
            attention_cached(*args, **more)
    for error, args, more in (
        (ValueError, (c, k, k), {}),
        (ValueError, (c, q, q), {}),
        (ValueError, (c, k, bf(2, 2, 4, 64)), {}),
        (TypeError, (c, k.half(), k), {}),
        (TypeError, (c, k, k), dict(index=torch.zeros(2, 2, dtype=torch.int64))),
        (ValueError, (c, k, k), dict(index=ints(3, 2))),
        (ValueError, (c, k, k), dict(index=ints(2, 0))),
        (ValueError, (c, k, k), dict(counts=ints(1))),
        (ValueError, (KVCache(c.k, c.k, c.lengths, c.table), k, k), {}),
        (RuntimeError, (c, k.clone().requires_grad_(), k), {}),
    ):
        with pytest.raises(error, match="cache_append"):
            cache_append(*args, **more)
    stats, w = torch.zeros(2, 4, 2, 3), torch.zeros(2, 2, 32)
    for error, args, more in (
        (ValueError, (c, q, stats), {}),
        (TypeError, (c, q, stats.double()), {}),
        (ValueError, (c, q, stats[..., :2]), {}),
        (ValueError, (c, q, stats), dict(weights=w[..., :31])),
        (ValueError, (c, q, stats), dict(weights=w[:1])),
        (ValueError, (c, q, stats), dict(weights=w[:1].expand(2, 2, 32))),
        (TypeError, (c, q, stats), dict(weights=w.double())),
        (ValueError, (c, q, stats), dict(index=ints(2))),
        (ValueError, (c, q, stats), dict(scale=float("inf"))),
    ):
        with pytest.raises(error, match="cache_weights"):
            cache_weights(*args, **more)
    other, other_pages = cpu_cache(k=bf(4, 1, 16, 64), v=bf(4, 1, 16, 64)), cpu_cache()
    for error, args, more in (
        (ValueError, (c, w, 16), {}),
        (ValueError, (c, w, 0), {}),
        (ValueError, (c, w, 4), dict(recent=5)),
        (ValueError, (c, w, 4), dict(recent=-1)),
        (ValueError, (c, w[..., :31], 4), {}),
        (TypeError, (c, w.bfloat16(), 4), {}),
        (ValueError, (c, w, 4), dict(out=c)),
        (ValueError, (c, w, 4), dict(out=other)),
        (ValueError, (c, w, 33), dict(out=cpu_cache())),
        (ValueError, (c, w, 4), dict(out=KVCache(c.k, c.v, ints(2), c.table))),
        (ValueError, (c, w, 4), dict(out=KVCache(c.k, bf(4, 2, 16, 64), ints(2), c.table))),
        (ValueError, (c, w, 4), dict(out=KVCache(c.k[:2], c.v[:2], ints(2)))),
        (ValueError, (c, w, 4), dict(out=KVCache(other_pages.k, other_pages.k, ints(2), c.table))),
    ):
        with pytest.raises(error, match="cache_evict"):
            cache_evict(*args, **more)


def test_tree_mask():
    parents = torch.tensor([-1, 0, 0, 1, -1, 4, 3])
    want = torch.tensor([[t == 0, t in (0, 1), t in (0, 2), t in (0, 1, 3), t == 4, t in (4, 5), t in (0, 1, 3, 6)] for t in range(7)]).T
    assert torch.equal(tree_mask(parents), want)
    assert torch.equal(tree_mask(parents.expand(2, 7)), want.expand(2, 7, 7))
    assert torch.equal(tree_mask(torch.arange(40) - 1), torch.ones(40, 40, dtype=torch.bool).tril())
    assert tree_mask(torch.tensor([-1])).tolist() == [[True]]
    with pytest.raises(TypeError):
        tree_mask(torch.zeros(3))
