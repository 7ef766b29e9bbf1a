"""What the operators on a cache leave where its table, lengths or an index say something that is not so: the status, NaN for what the fault
took part in, every other result as ever or NaN, and nothing outside the positions that a call writes. (The kernels check before they look.)"""

import pytest
import torch

from kohakufa_b200 import _lib, attention_cached, cache_append, cache_evict, cache_weights
from kohakufa_b200.cache import cache_evict_op
from tests.test_cache import exact_attention, logical, make_cache, rows

pytestmark = pytest.mark.gpu
DTYPE, DIM, HEADS, COLUMNS = torch.bfloat16, 64, 4, 16  # 256 positions


def reported(call):
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    result = call()
    torch.cuda.synchronize()
    status = _lib.device_status()
    _lib.reset_device_status()
    assert status == 90
    return result


def cache_with(lengths=(140, 60), page=None, columns=COLUMNS):
    """Sequence 0 says something wrong: its length, or its fourth page (positions 48 .. 63)."""
    c = make_cache([140, 60], 2, DIM, DTYPE, 16, columns=columns)
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    if page is not None:
        c.table[0, 3] = page
    return c


FAULTS = [dict(page=-1), dict(page=10_000), dict(page=2**31 - 1), dict(lengths=(257, 60)), dict(lengths=(-1, 60)), dict(lengths=(2**31 - 1, 60))]


@pytest.mark.parametrize("fault", FAULTS, ids=str)
@pytest.mark.parametrize("tokens,columns", [(3, 16), (3, 100), (40, 16), (100, 100)])
def test_attention(fault, tokens, columns):
    if fault.get("lengths", (0,))[0] == 257:
        fault = dict(lengths=(16 * columns + 1, 60))
    q, k, v = (rows(2, h, tokens, DIM, DTYPE, s) for h, s in ((HEADS, 1), (2, 2), (2, 3)))
    want, size, m, log2l = (t[1] for t in exact_attention(q, cache_with(columns=columns), k, v, None, None, DIM**-0.5))
    out, stats = reported(lambda: attention_cached(q, cache_with(**fault, columns=columns), k, v, return_stats=True))
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(stats[0]).all())
    # (not bit for bit: where the work is cut, and so the order of the sums, goes by all sequences' lengths; tolerances of test_cache.py)
    u, got, got_stats = torch.finfo(DTYPE).eps / 2, out[1].double().cpu(), stats[1].double().cpu()
    as_ever = ((got - want).abs() <= (u + 2.0**-12) * size + u * want.abs() + 2.0**-24).all(-1)
    as_ever &= torch.isclose(got_stats[:, 0], m, rtol=2.0**-18, atol=2.0**-16) & torch.isclose(got_stats[:, 1], log2l, rtol=2.0**-16, atol=2.0**-13)
    lost = torch.isnan(got).all(-1) & torch.isnan(got_stats).all(1)
    assert bool((as_ever | lost).all())


@pytest.mark.parametrize("fault", FAULTS, ids=str)
@pytest.mark.parametrize("tokens", [3, 50])  # 6 and 100 rows
@pytest.mark.parametrize("accepted", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_weights(fault, tokens, accepted, add):
    if fault.get("lengths", (0,))[0] == 257:
        fault = dict(lengths=(256 - tokens + 1, 60))
    q = rows(2, HEADS, tokens, DIM, DTYPE, 1)
    stats = torch.zeros(2, HEADS, 2, tokens, device="cuda")
    index = torch.arange(tokens, dtype=torch.int32).expand(2, tokens).contiguous().cuda() if accepted else None
    before = torch.rand(2, 2, 256, device="cuda")
    call = lambda c: cache_weights(c, q, stats, index=index, weights=before.clone() if add else None)  # noqa: E731
    fine = call(cache_with())
    got = reported(lambda: call(cache_with(**fault)))
    if "page" in fault:
        assert bool(torch.isnan(got[0, :, 48:64]).all())
        assert bool((torch.isnan(got[0]) | (got[0] == fine[0])).all())
    else:
        assert bool(torch.isnan(got[0, :, : min(max(fault["lengths"][0], 0) + tokens, 256)]).all())
    # (behind the last position nothing is written, or zeros)
    assert bool((torch.isnan(got[1]) | (got[1] == fine[1])).all())


@pytest.mark.parametrize("tokens", [3, 50])
@pytest.mark.parametrize("entry", [-1, "T", 2**31 - 1])
def test_weights_of_rows_that_are_not_there(tokens, entry):
    q = rows(2, HEADS, tokens, DIM, DTYPE, 1)
    stats = torch.zeros(2, HEADS, 2, tokens, device="cuda")
    index = torch.arange(tokens, dtype=torch.int32).repeat(2, 1)
    fine = cache_weights(cache_with(), q, stats, index=index.cuda())
    index[0, 1] = tokens if entry == "T" else entry
    got = reported(lambda: cache_weights(cache_with(), q, stats, index=index.cuda()))
    assert bool(torch.isnan(got[0, :, : 140 + tokens]).all())
    assert bool((torch.isnan(got[1]) | (got[1] == fine[1])).all())


@pytest.mark.parametrize("tokens", [3, 50])
@pytest.mark.parametrize("fault", [dict(lengths=(255, 60)), dict(lengths=(300, 60)), dict(lengths=(-1, 60)), dict(lengths=(46, 60), page=-1),
                                   dict(lengths=(46, 60), page=10_000), dict(lengths=(2**31 - 1, 60)), "index"], ids=str)  # fmt: skip
def test_append_writes_nothing_else(fault, tokens):
    k, v = rows(2, 2, tokens, DIM, DTYPE, 2), rows(2, 2, tokens, DIM, DTYPE, 3)
    c = cache_with(**({} if fault == "index" else fault))
    index = torch.arange(tokens, dtype=torch.int32).repeat(2, 1)
    if fault == "index":
        index[0, 1] = tokens
    want = [t.clone() for t in (c.k, c.v)]
    for b, n in enumerate(c.lengths.tolist()):
        for i in range(tokens):
            p, t = n + i, int(index[b, i])
            page = int(c.table[b, p // 16]) if n >= 0 and p < 256 else -1
            if 0 <= page < c.k.shape[0] and t < tokens:
                for w, new in zip(want, (k, v)):
                    w[page, :, p % 16] = new[b, :, t]
    reported(lambda: cache_append(c, k, v, index=index.cuda() if fault == "index" else None))
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])


@pytest.mark.parametrize("page", [-1, 10_000, 2**31 - 1])
@pytest.mark.parametrize("clear", [False, True])
def test_eviction_leaves_nan_where_a_page_is_not_there(page, clear):
    """Rows of a page that is not there read as NaN, whatever the memory held before that takes them."""
    c, keep = cache_with(page=page), 80
    weights = torch.rand(2, 2, 256, device="cuda")
    weights[0, :, 50:60] = 2.0  # (these stay)
    want = reported(lambda: cache_evict(c, weights, keep, recent=8))
    kept = want[2]
    assert kept[0, 0, 0] >= 0 and bool((kept[1, :, 60:] == -1).all())
    lost = (kept >= 48) & (kept < 64)
    lost[1] = False
    assert bool(lost[0, 0].sum() >= 10)
    if clear:  # a new cache, in memory of which is known what it held
        k_out, v_out = (torch.full((2, keep, 2, DIM), 7.0, dtype=DTYPE, device="cuda").transpose(1, 2) for _ in range(2))
        lengths, w_out, again = torch.empty_like(c.lengths), torch.empty_like(want[1]), torch.empty_like(kept)
        reported(lambda: cache_evict_op(*c._tensors(), weights, keep, 8, k_out, v_out, None, lengths, w_out, again, True))
        behind = torch.zeros(2, 2, keep, DIM, dtype=torch.float64)
    else:
        target = make_cache([keep, keep], 2, DIM, DTYPE, 16, seed=3)
        behind = logical(target, "k")[:, :, :keep]
        got, w_out, again = reported(lambda: cache_evict(c, weights, keep, recent=8, out=target))
        k_out, lengths = logical(got, "k")[:, :, :keep].to(DTYPE).cuda(), got.lengths
    assert torch.equal(again, kept) and torch.equal(w_out, want[1]) and lengths.tolist() == [keep, 60]
    assert bool(torch.isnan(k_out[lost]).all())
    here = (kept >= 0) & ~lost
    source = logical(c, "k").gather(2, kept.cpu().clamp(min=0).long()[..., None].expand(-1, -1, -1, DIM))
    assert torch.equal(k_out.double().cpu()[here.cpu()], source[here.cpu()])
    assert torch.equal(k_out.double().cpu()[kept.cpu() < 0], behind[kept.cpu() < 0])
    assert bool(torch.isnan(want[0].k[lost]).all()) and bool(torch.isnan(want[0].v[lost]).all())
