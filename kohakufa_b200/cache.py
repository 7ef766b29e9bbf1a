"""A cache of keys and values, and what a program that generates from a model does with it in every layer:

    cache = KVCache(k_pages, v_pages, lengths, table)          # or KVCache.empty(...)
    w = torch.zeros(batch, kv_heads, cache.capacity, device="cuda")
    while generating:
        out, stats = attention_cached(q, cache, k, v, tree=tree, return_stats=True)   # drafted tokens, or one (T = 1)
        cache_append(cache, k, v, index=accepted, counts=n)         # the accepted ones go into the cache
        cache_weights(cache, q, stats, index=accepted, counts=n, weights=w)   # who was looked at, accumulated
        cache.lengths += n                                          # once a step where layers share their lengths
        if full:                                                    # back to the budget, with room for what comes
            cache, w, kept = cache_evict(cache, w, keep=2048, recent=256, room=4096)

Keys that are turned by their positions (``kohakufa_b200.rotary``) go in through ``cache_append_rotary``; sequences that go on from prefixes which are stored
once attend through ``attention_shared``.

All of it is for inference: there are no gradients, and a call on tensors that autograd would record is refused. The calls go to
``libkfa.so`` through the C++ launch path like ``attention``: current stream, no host synchronisation, scratch from the
caching allocator, CUDA-graph capture after one eager call on the device. ``lengths`` and ``table`` are read on the device,
so a captured step follows them; what they say wrongly (a page that is not there, a length beyond the capacity) is reported by
``check_status`` and touches no memory outside the pages. The reference has no counterpart.
"""

import torch
from torch import Tensor

from kohakufa_b200 import _lib
from kohakufa_b200.rotary import Rotary

__all__ = ["KVCache", "attention_cached", "attention_shared", "cache_append", "cache_append_rotary", "cache_evict", "cache_weights", "tree_mask"]


class KVCache:
    """Keys and values of a batch of sequences, in pages.

    ``k`` and ``v``: ``[N, Hkv, page, D]`` (fp16 or bf16; views of ``[N, page, Hkv, D]`` storage are usual: the last dim
    contiguous, the other strides multiples of 16 bytes, D a multiple of 8 up to 128). ``table``: int32 ``[B, M]``; position ``p`` of
    sequence ``b`` lies in page ``table[b, p // page]``, slot ``p % page`` (``page`` a multiple of 8; entries behind a sequence's end
    may be anything). Without a table page ``b`` is sequence ``b``'s, of any size. ``lengths``: int32 ``[B]``, how many positions of each
    sequence hold something; the calls read it and never change it."""

    __slots__ = ("k", "lengths", "table", "v")

    def __init__(self, k: Tensor, v: Tensor, lengths: Tensor, table: Tensor | None = None) -> None:
        if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype != k.dtype:
            raise TypeError("KVCache: pages of k and v must be fp16 or bf16 (both the same)")
        if k.dim() != 4 or k.shape != v.shape or 0 in k.shape:
            raise ValueError(f"KVCache: pages [N, Hkv, page, D], got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.shape[3] % 8 or k.shape[3] > 128:
            raise ValueError(f"KVCache: head_dim {k.shape[3]}: a multiple of 8 up to 128")
        if lengths.dtype != torch.int32 or (table is not None and table.dtype != torch.int32):
            raise TypeError("KVCache: lengths and table are int32")
        if lengths.dim() != 1 or not lengths.is_contiguous() or not lengths.numel():
            raise ValueError("KVCache: lengths is a contiguous vector, one entry per sequence")
        if table is None:
            if k.shape[0] != lengths.numel():
                raise ValueError(f"KVCache: without a table one page per sequence: {k.shape[0]} pages, {lengths.numel()} lengths")
        else:
            if table.dim() != 2 or table.shape[0] != lengths.numel() or not table.shape[1] or table.stride(1) != 1:
                raise ValueError("KVCache: table [B, M] with contiguous rows, one per sequence")
            if k.shape[2] % 8:
                raise ValueError(f"KVCache: pages of {k.shape[2]} positions: a multiple of 8")
        if any(t.device != k.device for t in (v, lengths, table) if t is not None):
            raise ValueError("KVCache: tensors on different devices")
        self.k, self.v, self.lengths, self.table = k, v, lengths, table

    @classmethod
    def empty(
        cls, batch: int, kv_heads: int, capacity: int, head_dim: int, *, page: int | None = None,
        dtype: torch.dtype = torch.bfloat16, device="cuda",
    ) -> "KVCache":  # fmt: skip
        """A cache with nothing in it: one stretch of memory per sequence, or (``page``) pages with a table that gives every
        sequence as many as it needs."""
        columns = 1 if page is None else -(-capacity // page)
        shape = (batch * columns, capacity if page is None else page, kv_heads, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
        lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        table = None if page is None else torch.arange(batch * columns, dtype=torch.int32, device=device).view(batch, columns)
        return cls(k, v, lengths, table)

    @property
    def capacity(self) -> int:
        """Positions that a sequence's pages have room for."""
        return self.k.shape[2] if self.table is None else self.table.shape[1] * self.k.shape[2]

    def _tensors(self):
        return self.k, self.v, self.lengths, self.table


def _new_cache(k: Tensor, v: Tensor, lengths: Tensor, table: Tensor | None) -> KVCache:
    """A cache of tensors that are known to fit."""
    cache = KVCache.__new__(KVCache)
    cache.k, cache.v, cache.lengths, cache.table = k, v, lengths, table
    return cache


def _refuse_autograd(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name}: has no gradient; call it under torch.no_grad() or on detached tensors")


def tree_mask(parents: Tensor) -> Tensor:
    """bool ``[..., T, T]``, which drafted tokens a drafted token sees (itself and those it follows), from the ``[..., T]`` indices of
    the token that each one continues (-1: the end of the cache)."""
    if parents.is_floating_point() or parents.dtype == torch.bool or parents.dim() < 1:
        raise TypeError("tree_mask: integer indices [..., T]")
    tokens = parents.shape[-1]
    one = torch.arange(tokens, device=parents.device)
    sees = (parents.unsqueeze(-1) == one) | (one[:, None] == one)
    reach = 1
    while reach < tokens:  # who is seen by the seen
        sees = (sees.float() @ sees.float()) > 0
        reach *= 2
    return sees


@torch.library.custom_op("kohakufa_b200::cached_attention", mutates_args=(), device_types="cuda")
def cached_attention_op(
    q: Tensor, k_pages: Tensor, v_pages: Tensor, lengths: Tensor, table: Tensor | None, k: Tensor | None, v: Tensor | None,
    tree: Tensor | None, counts: Tensor | None, scale: float,
) -> tuple[Tensor, Tensor]:  # fmt: skip
    word = _lib.status_word(q.device)
    return _lib.host().cached_attention(q, k_pages, v_pages, lengths, table, k, v, tree, counts, scale, True, word)


@cached_attention_op.register_fake
def _(q, k_pages, v_pages, lengths, table, k, v, tree, counts, scale):
    batch, heads, tokens, dim = q.shape
    return q.new_empty(batch, tokens, heads, dim).transpose(1, 2), q.new_empty(batch, heads, 2, tokens, dtype=torch.float32)


def attention_cached(
    q: Tensor,
    cache: KVCache,
    k: Tensor | None = None,
    v: Tensor | None = None,
    *,
    tree: Tensor | None = None,
    counts: Tensor | None = None,
    scale: float | None = None,
    return_stats: bool = False,
):
    """Attention of the newest tokens of each sequence to its cached keys and to one another.

    ``q`` is ``[B, H, T, D]``, ``k`` and ``v`` ``[B, Hkv, T, D]`` are the new tokens' own keys and values, not yet in the cache (``Hkv``
    divides ``H``). New token ``t`` sees every cached position and, of the new tokens, those that ``tree`` shows it: bool ``[T, T]`` or
    ``[B, T, T]``, True where row ``t`` sees token ``j`` (see ``tree_mask``); without ``tree`` tokens ``0 .. t``. ``T`` is 1 for plain
    decoding, the number of drafted tokens in a verification step, or the length of a prompt's chunk. Without ``k`` and ``v`` the
    cache is all there is to see: cross attention to an encoder's states. ``counts``: int32 ``[B]``, how many of the ``T`` tokens
    sequence ``b`` has; the others neither see nor are seen, and what their rows of q, k and v hold does not matter.

    Returns ``[B, H, T, D]`` laid out as ``[B, T, H, D]``, and with ``return_stats`` also fp32 ``[B, H, 2, T]``: the raw score's row
    maximum and the log2 of the sum of exponentials (for ``cache_weights``). A row that sees nothing has output 0 and statistics
    (+inf, 0). Results repeat bit for bit."""
    pages = cache._tensors()
    softmax_scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if _lib.plain_eager(q, *pages, k, v, tree, counts):
        return _lib.host().cached_attention(
            q, *pages, k, v, tree, counts, softmax_scale, return_stats, _lib.status_word(q.device) if q.is_cuda else None
        )
    _refuse_autograd("attention_cached", q, cache.k, cache.v, k, v)
    out, stats = cached_attention_op(q, *pages, k, v, tree, counts, softmax_scale)
    return (out, stats) if return_stats else out


@torch.library.custom_op("kohakufa_b200::shared_attention", mutates_args=(), device_types="cuda")
def shared_attention_op(
    q: Tensor, k_prefix: Tensor, v_prefix: Tensor, prefix_lengths: Tensor, prefix_table: Tensor | None, k_pages: Tensor, v_pages: Tensor,
    lengths: Tensor, table: Tensor | None, starts: Tensor | None, k: Tensor | None, v: Tensor | None, tree: Tensor | None,
    counts: Tensor | None, scale: float,
) -> tuple[Tensor, Tensor]:  # fmt: skip
    return _lib.host().shared_attention(
        q, k_prefix, v_prefix, prefix_lengths, prefix_table, k_pages, v_pages, lengths, table, starts, k, v, tree, counts, scale, True,
        _lib.status_word(q.device),
    )  # fmt: skip


@shared_attention_op.register_fake
def _(q, k_prefix, v_prefix, prefix_lengths, prefix_table, k_pages, v_pages, lengths, table, starts, k, v, tree, counts, scale):
    batch, heads, tokens, dim = q.shape
    return q.new_empty(batch, tokens, heads, dim).transpose(1, 2), q.new_empty(batch, heads, 2, tokens, dtype=torch.float32)


def attention_shared(
    q: Tensor,
    prefix: KVCache,
    cache: KVCache,
    k: Tensor | None = None,
    v: Tensor | None = None,
    *,
    starts: Tensor | None = None,
    tree: Tensor | None = None,
    counts: Tensor | None = None,
    scale: float | None = None,
    return_stats: bool = False,
):
    """``attention_cached`` for sequences that go on from prefixes which are stored, and read, once: a system prompt, a document with many
    questions, many samples of one prompt.

    ``prefix`` holds the prefixes, one per entry of its batch (pages of their own or of the same pool), ``cache`` what each sequence has behind its prefix.
    ``starts``: int32 ``[P + 1]`` on the device, ascending: sequences ``starts[p] .. starts[p + 1] - 1`` go on from prefix ``p``, those before ``starts[0]`` and from ``starts[P]`` on
    have none; so the batch is in the order of its prefixes. Without it there is one prefix, of all sequences. New token ``t`` of a sequence sees its
    whole prefix, all of the sequence's cached positions, and of the new tokens what ``attention_cached`` says, whose other arguments and results are these. The
    statistics are those over all that a row sees, as ``cache_weights`` wants them, for the cache's own positions.

    The rows of a prefix's sequences are put together, up to 256 of a K / V head, and the prefix is read once for them; what they get from it and from their own
    cache is joined in fp32. Results repeat bit for bit, but a sequence's last bits depend on how many are in the batch. Keys turned by their positions
    stand behind the prefix: ``cache_append_rotary(..., offset=lengths of the sequences' prefixes)``."""
    pages, shared = cache._tensors(), prefix._tensors()
    softmax_scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if _lib.plain_eager(q, *shared, *pages, starts, k, v, tree, counts):
        return _lib.host().shared_attention(
            q, *shared, *pages, starts, k, v, tree, counts, softmax_scale, return_stats, _lib.status_word(q.device) if q.is_cuda else None
        )
    _refuse_autograd("attention_shared", q, prefix.k, prefix.v, cache.k, cache.v, k, v)
    out, stats = shared_attention_op(q, *shared, *pages, starts, k, v, tree, counts, softmax_scale)
    return (out, stats) if return_stats else out


@torch.library.custom_op("kohakufa_b200::cache_append", mutates_args=("k_pages", "v_pages"), device_types="cuda")
def cache_append_op(
    k_pages: Tensor, v_pages: Tensor, lengths: Tensor, table: Tensor | None, k: Tensor, v: Tensor, index: Tensor | None,
    counts: Tensor | None,
) -> None:  # fmt: skip
    _lib.host().cache_append(k_pages, v_pages, lengths, table, k, v, index, counts, _lib.status_word(k.device))


def cache_append(cache: KVCache, k: Tensor, v: Tensor, *, index: Tensor | None = None, counts: Tensor | None = None) -> None:
    """Writes keys and values of new tokens behind the cached ones: position ``lengths[b] + i`` gets token ``index[b, i]`` of ``k`` and
    ``v`` ``[B, Hkv, T, D]`` (``index``: int32 ``[B, A]``, e.g. the accepted path of a draft; without it token ``i``), for ``i <
    counts[b]`` (int32 ``[B]``; without it all). ``lengths`` is left as it is: add the counts to it once all layers have appended. The pages that
    are written must belong to one sequence each, and ``k`` and ``v`` must not lie in the positions that are written. Positions beyond the
    capacity are dropped and reported by ``check_status``."""
    pages = cache._tensors()
    if _lib.plain_eager(*pages, k, v, index, counts):
        _lib.host().cache_append(*pages, k, v, index, counts, _lib.status_word(k.device) if k.is_cuda else None)
        return
    _refuse_autograd("cache_append", cache.k, cache.v, k, v)
    cache_append_op(*pages, k, v, index, counts)


@torch.library.custom_op("kohakufa_b200::cache_append_rotary", mutates_args=("k_pages", "v_pages"), device_types="cuda")
def cache_append_rotary_op(
    k_pages: Tensor, v_pages: Tensor, lengths: Tensor, table: Tensor | None, q: Tensor | None, k: Tensor, v: Tensor, index: Tensor | None,
    counts: Tensor | None, turns: Tensor, positions: Tensor | None, offset: Tensor | None, amplitude: float, interleaved: bool, keys: bool,
) -> tuple[Tensor, Tensor]:  # fmt: skip
    q_out, k_out = _lib.host().cache_append_rotary(
        k_pages, v_pages, lengths, table, q, k, v, index, counts, turns, positions, offset, amplitude, interleaved, keys, _lib.status_word(k.device)
    )
    return k.new_empty(0) if q_out is None else q_out, k.new_empty(0) if k_out is None else k_out


@cache_append_rotary_op.register_fake
def _(k_pages, v_pages, lengths, table, q, k, v, index, counts, turns, positions, offset, amplitude, interleaved, keys):
    like = lambda t: t.new_empty(t.shape[0], t.shape[2], t.shape[1], t.shape[3]).transpose(1, 2)  # noqa: E731
    return k.new_empty(0) if q is None else like(q), like(k) if keys else k.new_empty(0)


def cache_append_rotary(
    cache: KVCache, q: Tensor | None, k: Tensor, v: Tensor, rotary: Rotary, *, index: Tensor | None = None, counts: Tensor | None = None,
    positions: Tensor | None = None, offset: Tensor | None = None, return_keys: bool = False,
):  # fmt: skip
    """``cache_append`` for keys that are not turned yet (``apply_rotary``), with the new tokens' queries in the same pass: position
    ``lengths[b] + i`` gets token ``i`` of ``k``, turned, and of ``v``.

    Token ``i`` stands at ``offset[b] + lengths[b] + i``: ``offset`` (int32 ``[B]``) is what a sequence has before its cache begins, a prefix that is stored
    elsewhere or positions that were evicted. Or at ``offset[b] + positions[b, t]`` (int32 or int64, ``[B, T]``, ``[1, T]`` or ``[T]``), whatever the cache holds.
    ``q`` ``[B, H, T, D]`` or None. Returns the turned queries (None without ``q``), and with ``return_keys`` also the turned keys, for
    ``attention_cached`` or ``attention_shared`` in the same step, before ``lengths`` grows:

        q, k = cache_append_rotary(cache, q, k, v, rotary, return_keys=True)
        out = attention_cached(q, cache, k, v)

    Rows that ``counts`` leaves out are zeros there. ``index`` and what else is said of ``cache_append`` holds here too; with an index only the pages are written: ``q`` is
    None and no keys are returned."""
    pages = cache._tensors()
    tensors = (q, k, v, index, counts, rotary.turns, positions, offset)
    more = (rotary.amplitude, rotary.interleaved, bool(return_keys))
    if _lib.plain_eager(*pages, *tensors):
        q_out, k_out = _lib.host().cache_append_rotary(*pages, *tensors, *more, _lib.status_word(k.device) if k.is_cuda else None)
        return (q_out, k_out) if return_keys else q_out
    _refuse_autograd("cache_append_rotary", cache.k, cache.v, q, k, v)
    q_out, k_out = cache_append_rotary_op(*pages, *tensors, *more)
    q_out = None if q is None else q_out
    return (q_out, k_out) if return_keys else q_out


@torch.library.custom_op("kohakufa_b200::cache_weights", mutates_args=("weights",), device_types="cuda")
def cache_weights_op(
    k_pages: Tensor, v_pages: Tensor, lengths: Tensor, table: Tensor | None, q: Tensor, stats: Tensor, index: Tensor | None,
    counts: Tensor | None, weights: Tensor, add: bool, scale: float,
) -> None:  # fmt: skip
    word = _lib.status_word(q.device)
    _lib.host().cache_weights(k_pages, v_pages, lengths, table, q, stats, index, counts, weights, add, scale, word)


def cache_weights(
    cache: KVCache,
    q: Tensor,
    stats: Tensor,
    *,
    index: Tensor | None = None,
    counts: Tensor | None = None,
    weights: Tensor | None = None,
    scale: float | None = None,
) -> Tensor:
    """How much attention the newest tokens gave to every cached position: fp32 ``[B, Hkv, capacity]``, the softmax weights summed
    over those tokens and over the query heads of a K / V head.

    Call it after ``cache_append`` with the same ``index`` and ``counts`` and before ``lengths`` grows: the ``i``-th counted token stands
    at position ``lengths[b] + i`` and saw the positions up to its own. ``q`` ``[B, H, T, D]`` and ``stats`` ``[B, H, 2, T]`` are those of the
    ``attention_cached`` call. With ``weights`` (fp32 ``[B, Hkv, W]``, ``W`` at least the capacity) the sums are added to it, in place, and
    positions that no token saw keep theirs; without, a new tensor is returned, 0 where no token looked."""
    pages = cache._tensors()
    softmax_scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    add = weights is not None
    if weights is None:
        weights = torch.empty(q.shape[0], cache.k.shape[1], cache.capacity, dtype=torch.float32, device=q.device)
    if _lib.plain_eager(*pages, q, stats, index, counts, weights):
        word = _lib.status_word(q.device) if q.is_cuda else None
        _lib.host().cache_weights(*pages, q, stats, index, counts, weights, add, softmax_scale, word)
        return weights
    _refuse_autograd("cache_weights", cache.k, q, stats, weights)
    cache_weights_op(*pages, q, stats, index, counts, weights, add, softmax_scale)
    return weights


@torch.library.custom_op(
    "kohakufa_b200::cache_evict", mutates_args=("k_out", "v_out", "lengths_out", "weights_out", "kept"), device_types="cuda"
)
def cache_evict_op(
    k_pages: Tensor, v_pages: Tensor, lengths: Tensor, table: Tensor | None, weights: Tensor, keep: int, recent: int, k_out: Tensor,
    v_out: Tensor, table_out: Tensor | None, lengths_out: Tensor, weights_out: Tensor, kept: Tensor, clear: bool,
) -> None:  # fmt: skip
    word = _lib.status_word(weights.device)
    _lib.host().cache_evict(k_pages, v_pages, lengths, table, weights, keep, recent, k_out, v_out, table_out, lengths_out, weights_out, kept, clear, word)  # fmt: skip


def cache_evict(
    cache: KVCache, weights: Tensor, keep: int, *, recent: int = 0, room: int | None = None, out: KVCache | None = None
) -> tuple[KVCache, Tensor, Tensor]:
    """Reduces every sequence to at most ``keep`` positions: the ``recent`` newest, and of the others those with the largest accumulated
    ``weights`` (fp32 ``[B, Hkv, W]``, ``W`` at least the capacity). Each K / V head keeps positions of its own; of equal weights the
    lower position stays, NaN counts as the largest. What stays moves to positions ``0, 1, ...`` in ascending order.

    ``out``: the cache that takes it (other pages than those that are read, e.g. of the same pool; a capacity of ``keep`` or more; what
    lies behind the kept positions is left as it was); without it a new one of one stretch per sequence and a capacity of ``room`` positions, zeros behind
    the kept. ``cache`` itself is not changed. ``room`` (at least ``keep``, which it is by default): how many positions the returned weights are wide. Where
    generation goes on, ask for the tokens that come before the next eviction as well: a cache without room for them drops what is appended, and
    ``cache_weights`` wants weights as wide as the cache's capacity (``room=out.capacity``).
    Returns the cache that holds the rest, with lengths of its own, their weights, fp32 ``[B, Hkv, room]`` (0 behind the last), and the positions they
    had, int32 ``[B, Hkv, keep]`` (-1 behind the last)."""
    pages = cache._tensors()
    keep, recent = int(keep), int(recent)
    if not 0 <= recent <= keep or keep < 1:
        raise ValueError(f"cache_evict: keep {keep}, recent {recent}: 0 <= recent <= keep, keep at least 1")
    room = keep if room is None else int(room)
    if room < keep:
        raise ValueError(f"cache_evict: room {room}: at least keep, {keep}")
    if out is cache:
        raise ValueError("cache_evict: out must have pages of its own")
    k, target = cache.k, (None, None, None, None) if out is None else out._tensors()
    if _lib.plain_eager(*pages, weights, *target):
        word = _lib.status_word(k.device) if k.is_cuda else None
        k_out, v_out, lengths_out, weights_out, kept = _lib.host().evict(*pages, weights, keep, recent, room, *target, word)
        return _new_cache(k_out, v_out, lengths_out, target[3]), weights_out, kept
    _refuse_autograd("cache_evict", cache.k, cache.v, weights, *target[:2])
    batch, heads, dim = cache.lengths.numel(), k.shape[1], k.shape[3]
    k_out, v_out, _, table_out = target
    if out is None:
        k_out, v_out = (k.new_empty(batch, room, heads, dim).transpose(1, 2) for _ in range(2))
    lengths_out = cache.lengths.new_empty(batch)
    weights_out = k.new_empty(batch, heads, room, dtype=torch.float32)
    kept = cache.lengths.new_empty(batch, heads, keep)
    cache_evict_op(*pages, weights, keep, recent, k_out, v_out, table_out, lengths_out, weights_out, kept, out is None)
    return _new_cache(k_out, v_out, lengths_out, table_out), weights_out, kept
