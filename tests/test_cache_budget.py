"""Generation with a bounded cache as the module's documentation writes it: the loop runs on behind its evictions. Tolerances as in test_cache.py;
a position's accumulated weight has up to 60 additions of fp32 behind it, each half a step off: 2^-24 * 60 relative, below the 2^-13 of the weights."""

import ctypes

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_cached, cache_append, cache_evict, cache_weights
from tests.test_cache import check_attention, cpu_cache, exact_weights, expect_evicted, logical, make_cache, random_tree, rows


@pytest.mark.gpu
@pytest.mark.parametrize("into", ["new", "plain", "pages"])
def test_the_loop_goes_on_behind_its_evictions(into):
    batch, heads, kv_heads, dim, dtype, keep, room = 3, 4, 2, 64, torch.bfloat16, 40, 72
    cache = KVCache.empty(batch, kv_heads, room, dim, dtype=dtype, page=8 if into == "pages" else None)
    w = torch.zeros(batch, kv_heads, room, device="cuda")
    total, gen, evictions = w.double().cpu(), torch.Generator().manual_seed(0), 0
    for step in range(60):
        tokens = 6
        q, k, v = (rows(batch, h, tokens, dim, dtype, 10 * step + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
        tree = random_tree(batch, tokens, step)
        check_attention(cache, heads, tokens, dtype, tree, q=q, k=k, v=v)
        out, stats = attention_cached(q, cache, k, v, tree=tree.cuda(), return_stats=True)
        accepted, n = torch.zeros(batch, tokens, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
        for b in range(batch):  # a path of the tree: a token and those it follows
            path = tree[b, int(torch.randint(0, tokens, (1,), generator=gen))].nonzero().flatten()
            accepted[b, : len(path)], n[b] = path.to(torch.int32), len(path)
        accepted, n = accepted.cuda(), n.cuda()
        cache_append(cache, k, v, index=accepted, counts=n)
        cache_weights(cache, q, stats, index=accepted, counts=n, weights=w)
        total += exact_weights(cache, q, stats, accepted, n, dim**-0.5)
        assert torch.allclose(w.double().cpu(), total, rtol=2.0**-13, atol=2.0**-20)
        cache.lengths += n
        if int(cache.lengths.max()) + tokens > room:
            lengths, k_all, w_all = cache.lengths.tolist(), logical(cache, "k"), w.cpu()
            target = None if into == "new" else KVCache.empty(batch, kv_heads, room, dim, dtype=dtype, page=8 if into == "pages" else None)
            cache, w, kept = cache_evict(cache, w, keep=keep, recent=8, room=room, out=target)
            assert cache.capacity == room and w.shape == (batch, kv_heads, room) and kept.shape == (batch, kv_heads, keep)
            want = expect_evicted(w_all, lengths, keep, 8)
            assert torch.equal(kept.cpu(), want)
            at = want.clamp(min=0).long()
            assert torch.equal(w[..., :keep].cpu(), w_all.gather(2, at).masked_fill(want < 0, 0.0)) and bool((w[..., keep:] == 0).all())
            there = want >= 0
            assert torch.equal(logical(cache, "k")[:, :, :keep][there], k_all.gather(2, at[..., None].expand(-1, -1, -1, dim))[there])
            assert into != "new" or bool((logical(cache, "k")[:, :, keep:] == 0).all())
            total = torch.zeros_like(total)
            total[..., :keep] = w[..., :keep].double().cpu()
            evictions += 1
    assert evictions >= 3 and _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("keep,room", [(1, 1), (5, 37), (64, 64), (64, 1000), (700, 701)])
def test_room(keep, room):
    """What lies behind the kept positions is zeros up to the room; without an argument the room is what is kept. Compiled calls too."""
    lengths, dim = [300, 0, 64, 650, 1], 40
    cache = make_cache(lengths, 2, dim, torch.float16, 16)
    weights = torch.rand(5, 2, cache.capacity, device="cuda")
    small, w_small, kept = cache_evict(cache, weights, keep)
    assert small.capacity == keep and w_small.shape == (5, 2, keep)

    def step(k, v, lengths, table, w):
        c, w, kept = cache_evict(KVCache(k, v, lengths, table), w, keep, room=room)
        return c.k, c.v, c.lengths, w, kept

    junk = [torch.full((5, room, 2, dim), 7.0, dtype=torch.float16, device="cuda") for _ in range(4)]  # (what the allocator gives next)
    del junk
    for call in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        k, v, left, w, kept_too = call(*cache._tensors(), weights)
        assert k.shape == v.shape == (5, 2, room, dim) and w.shape == (5, 2, room)
        assert torch.equal(kept_too, kept) and torch.equal(left, small.lengths)
        for got, less in ((k, small.k), (v, small.v), (w, w_small)):
            assert torch.equal(got[:, :, :keep], less) and bool((got[:, :, keep:] == 0).all())
    target = make_cache([keep] * 5, 2, dim, torch.float16, 32, seed=5)
    before = logical(target, "k")
    got, w, kept_too = cache_evict(cache, weights, keep, room=room, out=target)
    assert torch.equal(kept_too, kept) and torch.equal(w[..., :keep], w_small) and bool((w[..., keep:] == 0).all())
    behind = torch.ones(before.shape[:3], dtype=torch.bool)
    behind[:, :, :keep] = kept.cpu() < 0
    assert torch.equal(logical(got, "k")[behind], before[behind]) and _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("clear", [0, 1])
def test_the_c_entries(clear):
    """kfa_cache_evict is kfa_cache_evict_room with room for what is kept; rooms that do not fit are refused before a launch."""
    lib, keep = _lib.load(), 24
    cache = make_cache([300, 5], 2, 64, torch.float16, 16)
    weights = torch.rand(2, 2, cache.capacity, device="cuda")
    want = cache_evict(cache, weights, keep, recent=4)
    word, stream = _lib.status_word(weights.device), _lib.stream_ptr(weights.device)
    stride = (ctypes.c_int64 * 2)(weights.stride(0), weights.stride(1))

    def describe(c):
        d = _lib.KfaCache(_lib.tensor4(c.k), _lib.tensor4(c.v), None, 0, 0, c.lengths.data_ptr(), c.lengths.numel())
        if c.table is not None:
            d.table, d.table_stride, d.table_cols = c.table.data_ptr(), c.table.stride(0), c.table.shape[1]
        return ctypes.byref(d)

    for room in (None, keep, 40):
        out = KVCache(*(torch.full((2, 32, 2, 64), 7.0, dtype=torch.float16, device="cuda").transpose(1, 2) for _ in range(2)), cache.lengths)
        w, kept = torch.full((2, 2, room or keep), 7.0, device="cuda"), torch.empty(2, 2, keep, dtype=torch.int32, device="cuda")
        lengths = torch.empty_like(cache.lengths)
        behind = (describe(out), w.data_ptr(), kept.data_ptr(), lengths.data_ptr(), clear, word.data_ptr(), stream)
        if room is None:
            rc = lib.kfa_cache_evict(describe(cache), weights.data_ptr(), stride, keep, 4, *behind)
        else:
            rc = lib.kfa_cache_evict_room(describe(cache), weights.data_ptr(), stride, keep, 4, room, *behind)
        if room == 40 and clear:  # out has room for 32
            assert rc != 0 and b"room" in lib.kfa_last_error()
            continue
        assert rc == 0 and torch.equal(kept, want[2]) and lengths.tolist() == [24, 5]
        assert torch.equal(w[..., :keep], want[1]) and bool((w[..., keep:] == 0).all())
        there = want[2] >= 0
        assert torch.equal(out.k[:, :, :keep][there], want[0].k[there]) and bool((out.v[:, :, :keep][~there] == (0 if clear else 7)).all())
        assert bool((out.k[:, :, keep:] == 7).all())
    assert lib.kfa_cache_evict_room(describe(cache), weights.data_ptr(), stride, keep, 4, keep - 1, *behind) != 0
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def test_refused_rooms():
    c, w = cpu_cache(), torch.zeros(2, 2, 32)
    for room in (3, 0, -1, 2**31):
        with pytest.raises(ValueError, match="cache_evict"):
            cache_evict(c, w, 4, room=room)
    with pytest.raises(ValueError, match="cache_evict"):  # the device
        cache_evict(c, w, 4, room=40)
