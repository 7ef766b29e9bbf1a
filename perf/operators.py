"""Attention over a cache of keys and values: what a program that generates from a model calls in each layer.

Four operators, which share one cache of pages:

  attend   the new tokens of each sequence (one, or a tree of drafted ones) attend to the cached keys and to each other;
  append   the accepted tokens' keys and values go into the cache;
  weigh    how much attention the accepted tokens gave to every cached position, summed over rows and heads;
  evict    each K / V head keeps the positions that got most, and the newest, and drops the rest.

A cache is ``k_pages`` and ``v_pages`` [N, Hkv, page, D] (views of [N, page, Hkv, D] storage), ``table`` int32 [B, M] (position p of
sequence b lies in page ``table[b, p // page]``; None: page b is sequence b's) and ``lengths`` int32 [B].
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
LOG2E = 1.4426950408889634


def _case(name, op, batch, heads, kv_heads, dim, dtype, page, longest, shortest, tokens, length_seed=1, **more):
    case = dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, longest=longest,
                shortest=shortest, tokens=tokens, length_seed=length_seed, **more)  # fmt: skip
    return dict(name=name, **case) if name else case


def _attend(name, *args, new="causal", ragged=False, stats=False, **more):
    return _case(name, "attend", *args, new=new, ragged=ragged, stats=stats, **more)


def _evict(name, *args, keep=0, recent=0, into=0, **more):
    return _case(name, "evict", *args, 0, keep=keep, recent=recent, into=into, **more)


def listed():
    return [
        # one user, one new token, a short conversation: launches and host time count
        _attend("decode_tiny", 1, 8, 8, 64, "fp16", 0, 100, 100, 1),
        # a serving batch generating one token each, grouped queries, small pages, lengths of all kinds
        _attend("decode_batch", 64, 32, 8, 128, "bf16", 16, 4096, 1, 1),
        # one user with a whole book in the cache
        _attend("decode_long", 1, 32, 8, 128, "bf16", 0, 131072, 131072, 1),
        # a few drafted tokens per sequence, some sequences with fewer of them than others
        _attend("draft_small", 8, 16, 4, 64, "fp16", 64, 2048, 300, 7, new="tree", ragged=True, stats=True),
        # a wide tree of drafted tokens over long caches: 256 rows per K / V head
        _attend("draft_wide", 16, 32, 8, 128, "bf16", 32, 4096, 2048, 64, new="tree", stats=True),
        # a decoder that looks at an encoder's states: nothing new among the keys, a head dim between the common ones, an empty text
        _attend("cross_states", 32, 12, 12, 80, "fp16", 0, 1500, 0, 3, new="none"),
        # after a verification step: up to 5 of 8 drafted tokens accepted
        _case("weigh_step", "weigh", 16, 32, 8, 128, "bf16", 16, 4096, 300, 8, accepted=5),
        # the weights that a whole prompt gave to itself
        _case("weigh_prompt", "weigh", 1, 32, 8, 128, "bf16", 64, 0, 0, 4096, accepted=0),
        # the accepted tokens of a serving batch
        _case("append_step", "append", 64, 32, 8, 128, "bf16", 16, 4096, 1, 8, accepted=5),
        # prompts of 4096 tokens into fresh pages
        _case("append_prompt", "append", 4, 32, 8, 128, "bf16", 64, 0, 0, 4096, accepted=0),
        # a small cache a little over its budget
        _evict("evict_small", 2, 8, 4, 64, "fp16", 0, 320, 250, keep=256, recent=32),
        # long prompts reduced to a budget, into the pages of the serving cache
        _evict("evict_prompt", 16, 32, 8, 128, "bf16", 16, 8192, 1500, keep=2048, recent=256, into=16),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {c["op"]: work(c) for c in listed()}  # the last listed case of an operator is its largest (attend: see below)
    most["attend"] = work([c for c in listed() if c["name"] == "draft_wide"][0])
    while True:
        op = rng.choice(["attend"] * 6 + ["weigh"] * 2 + ["append", "evict", "evict"])
        dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([64] * 4 + [128] * 6 + [96, 80, 40, 72, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
        batch = _log_uniform(rng, 1, 96)
        page = rng.choice([0, 0, 16, 16, 32, 64, 128, 48])
        longest = _log_uniform(rng, 16, 65536)
        shortest = rng.choice([longest, rng.randint(0, longest), 0])
        args = (batch, heads, kv_heads, dim, dtype, page, longest, shortest)
        seed = rng.randrange(1000)
        if op == "attend":
            tokens = rng.choice([1, 1, 1, _log_uniform(rng, 1, 80)])
            new = rng.choice(["causal", "tree", "tree", "none"])
            case = _attend(None, *args, tokens, new=new, ragged=rng.random() < 0.3, stats=rng.random() < 0.5, length_seed=seed)
        elif op in ("weigh", "append"):
            if rng.random() < 0.3:
                case = _case(None, op, batch, heads, kv_heads, dim, dtype, page, 0, 0, _log_uniform(rng, 64, 4096), seed, accepted=0)
            else:
                tokens = _log_uniform(rng, 1, 64)
                case = _case(None, op, *args, tokens, seed, accepted=rng.randint(1, tokens))
        else:
            longest = max(longest, 32)
            keep = _log_uniform(rng, 16, longest)
            case = _evict(None, *args[:6], longest, min(shortest, longest), keep=keep, recent=rng.randint(0, keep),
                          into=rng.choice([0, 0, 16, 32]), length_seed=seed)  # fmt: skip
        w = work(case)
        if w["flops"] <= most[op]["flops"] and w["bytes"] <= most[op]["bytes"] and _values(case) <= 2**31:
            return case


def _values(case):
    """What the plain form holds at once, in numbers: scores, and the cache in 32 bits."""
    keys = case["longest"] + case["tokens"]
    rows = case["heads"] * max(1, case["tokens"]) if case["op"] in ("attend", "weigh") else 0
    return case["batch"] * keys * (rows + 2 * case["kv_heads"] * case["dim"])


# ---- sizes that the case fixes -----------------------------------------------------------------------------------------


def _lengths(case):
    rng = random.Random(case["length_seed"])
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lengths[0] = case["longest"]
    return lengths


def _counts(case):
    """New (attend) or accepted (weigh, append) tokens of each sequence."""
    rng = random.Random(case["length_seed"] + 1)
    tokens = case["tokens"]
    if case["op"] == "attend":
        return [rng.randint(0, tokens) for _ in range(case["batch"])] if case["ragged"] else [tokens] * case["batch"]
    if case["accepted"] == 0:
        return [tokens] * case["batch"]
    return [rng.randint(1, case["accepted"]) for _ in range(case["batch"])]


def work(case):
    """Every cached key and value that is looked at, the new tokens' rows and the weights read once, every result written once;
    two products of the visible pairs (weigh: one)."""
    lengths, d, hkv, h = _lengths(case), case["dim"], case["kv_heads"], case["heads"]
    row = 2 * d  # bytes
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": float(hkv * (4 * sum(lengths) + 4 * row * kept + 8 * kept)), "flops": 0.0}
    counts = _counts(case)
    if case["op"] == "append":
        return {"bytes": float(4 * row * hkv * sum(counts)), "flops": 0.0}
    pairs = sum(c * n + c * (c + 1) // 2 for c, n in zip(counts, lengths))
    if case["op"] == "weigh":
        seen = sum(c + n for c, n in zip(counts, lengths))
        return {"bytes": float(hkv * seen * (row + 4) + h * sum(counts) * (row + 8)), "flops": 2.0 * h * d * pairs}
    if case["new"] == "none":
        pairs, new = sum(c * n for c, n in zip(counts, lengths)), 0
    else:
        new = sum(counts)
    moved = 2 * row * hkv * (sum(n for c, n in zip(counts, lengths) if c) + new) + (2 * row + 8 * case["stats"]) * h * sum(counts)
    return {"bytes": float(moved), "flops": 4.0 * h * d * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _pages(case, positions, page, gen):
    """Pages for so many positions of each sequence, each filled with keys and values, and the table that finds them."""
    std = 0.5 if case["dim"] == 128 else 1.0
    dtype, b = DTYPES[case["dtype"]], case["batch"]
    if page == 0:
        count, page, table = b, max(max(positions), 1), None
    else:
        need = [-(-n // page) for n in positions]
        count = sum(need) + 3
        order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
        first = torch.tensor([0, *need], device="cuda").cumsum(0)[:-1]
        cols = torch.arange(max(max(need), 1), device="cuda")
        table = order[(first[:, None] + cols).clamp_(max=count - 1)]
        table = torch.where(cols < torch.tensor(need, device="cuda")[:, None], table, torch.zeros_like(table)).contiguous()
    shape = (count, page, case["kv_heads"], case["dim"])
    one = lambda: torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(std).transpose(1, 2)  # noqa: E731
    return one(), one(), table


def _rows(case, heads, tokens, gen):
    std = 0.5 if case["dim"] == 128 else 1.0
    x = torch.randn(case["batch"], tokens, heads, case["dim"], generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])
    return x.mul_(std).transpose(1, 2)


def _tree(case, gen):
    """bool [B, T, T]: which drafted tokens a drafted token sees, itself and those it follows."""
    b, t = case["batch"], case["tokens"]
    parent = (torch.rand(b, t, generator=gen, device="cuda") * (torch.arange(t, device="cuda") + 1)).long() - 1  # -1 .. t - 1
    sees = torch.zeros(b, t, t, dtype=torch.bool, device="cuda")
    one = torch.arange(b, device="cuda")
    for i in range(t):
        sees[:, i] = sees[one, parent[:, i].clamp(min=0)] & (parent[:, i] >= 0)[:, None]
        sees[:, i, i] = True
    return sees


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, t = case["batch"], case["tokens"]
    lengths = _lengths(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": case, "lengths": ints(lengths), "scale": case["dim"] ** -0.5}
    if case["op"] == "evict":
        s["k_pages"], s["v_pages"], s["table"] = _pages(case, lengths, case["page"], gen)
        room = _room(s)
        # what heads give to positions: a few large ones, many small ones, and some that nothing has looked at
        w = torch.randn(b, case["kv_heads"], room, generator=gen, device="cuda").mul_(2).exp_()
        s["weights"] = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.1)
        if case["into"]:
            k, v, table = _pages(case, [case["keep"]] * b, case["into"], gen)
            s["out"] = (k, v, table)
        return s
    counts = _counts(case)
    if case["op"] == "attend":
        s["k_pages"], s["v_pages"], s["table"] = _pages(case, lengths, case["page"], gen)
        s["q"] = _rows(case, case["heads"], t, gen)
        s["counts"] = ints(counts) if case["ragged"] else None
        if case["new"] != "none":
            s["k"], s["v"] = _rows(case, case["kv_heads"], t, gen), _rows(case, case["kv_heads"], t, gen)
        if case["new"] == "tree":
            s["tree"] = _tree(case, gen)
        return s
    steps = case["accepted"] or t
    s["k_pages"], s["v_pages"], s["table"] = _pages(case, [n + steps for n in lengths], case["page"], gen)
    if case["accepted"]:
        s["index"] = torch.rand(b, t, generator=gen, device="cuda").argsort(1)[:, :steps].sort(1).values.to(torch.int32)
        s["counts"] = ints(counts)
    else:
        s["index"] = s["counts"] = None
    if case["op"] == "append":
        s["k"], s["v"] = _rows(case, case["kv_heads"], t, gen), _rows(case, case["kv_heads"], t, gen)
        return s
    s["q"] = _rows(case, case["heads"], t, gen)
    s["stats"] = torch.zeros(b, case["heads"], 2, t, device="cuda")
    scores = _scores(s)  # what the attention call before this one returned for the accepted rows
    m = scores.amax(-1)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    log2l = (((scores - m[..., None]) * (s["scale"] * LOG2E)).exp2_().sum(-1)).clamp_(min=1e-30).log2()
    both = torch.stack([m.flatten(1, 2), log2l.flatten(1, 2)], 2)  # [B, H, 2, steps]
    if s["index"] is None:
        s["stats"].copy_(both)
    else:
        s["stats"].scatter_(3, s["index"].long()[:, None, None].expand_as(both), both)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _room(s):
    """Positions that a sequence's pages have room for."""
    page = s["k_pages"].shape[2]
    return page if s["table"] is None else s["table"].shape[1] * page


def _cached(pages, table):
    """[B, Hkv, room, D] in 32 bits."""
    if table is None:
        return pages.float()
    return pages[table.long()].transpose(1, 2).flatten(2, 3).float()


def _scores(s):
    """Raw scores [B, Hkv, group, steps, room] of the accepted rows, -inf where a row does not see a position."""
    case, q = s["case"], s["q"].float()
    if s["index"] is not None:
        steps = s["index"].shape[1]
        q = q.gather(2, s["index"].long()[:, None, :, None].expand(-1, q.shape[1], -1, q.shape[3]))
    else:
        steps = case["tokens"]
    k = _cached(s["k_pages"], s["table"])
    b, h, _, d = q.shape
    hkv = case["kv_heads"]
    scores = (q.reshape(b, hkv, -1, d) @ k.transpose(2, 3)).view(b, hkv, h // hkv, steps, -1)
    row = torch.arange(steps, device="cuda")
    last = s["lengths"][:, None] + row  # the last position that a row sees: its own
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    if s["counts"] is not None:
        seen &= (row < s["counts"][:, None])[..., None]
    return scores.masked_fill_(~seen[:, None, None], -math.inf)


def _plain_attend(s):
    case, dtype = s["case"], s["q"].dtype
    q, k, v = s["q"].float(), _cached(s["k_pages"], s["table"]), _cached(s["v_pages"], s["table"])
    b, h, t, d = q.shape
    hkv, room = case["kv_heads"], k.shape[2]
    seen = (torch.arange(room, device="cuda") < s["lengths"][:, None])[:, None].expand(b, t, room)
    if case["new"] != "none":
        k, v = torch.cat([k, s["k"].float()], 2), torch.cat([v, s["v"].float()], 2)
        if case["new"] == "tree":
            among = s["tree"]
        else:
            among = torch.ones(t, t, dtype=torch.bool, device="cuda").tril().expand(b, t, t)
        seen = torch.cat([seen, among], 2)
    if s["counts"] is not None:
        there = torch.arange(t, device="cuda") < s["counts"][:, None]
        seen = seen & there[:, :, None]
        if case["new"] != "none":
            seen = seen & torch.cat([there.new_ones(b, room), there], 1)[:, None]
    scores = (q.reshape(b, hkv, -1, d) @ k.transpose(2, 3)).view(b, hkv, h // hkv, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    some = m > -math.inf
    m = torch.where(some, m, torch.zeros_like(m))
    p = scores.sub_(m).mul_(s["scale"] * LOG2E).exp2_()
    l = p.sum(-1, keepdim=True)
    out = (p.view(b, hkv, -1, p.shape[-1]) @ v).view(b, hkv, h // hkv, t, d) / torch.where(some, l, torch.ones_like(l))
    out = out.reshape(b, h, t, d).to(dtype)
    if not case["stats"]:
        return out
    m = torch.where(some, m, torch.full_like(m, math.inf)).reshape(b, h, t)
    log2l = torch.where(some, l, torch.ones_like(l)).log2().reshape(b, h, t)
    return out, torch.stack([m, log2l], 2)


def _plain_weigh(s):
    steps = s["index"].shape[1] if s["index"] is not None else s["case"]["tokens"]
    scores, stats = _scores(s), s["stats"]
    if s["index"] is not None:
        stats = stats.gather(3, s["index"].long()[:, None, None].expand(-1, stats.shape[1], 2, -1))
    m, log2l = (stats[:, :, i].view(*scores.shape[:3], steps, 1) for i in (0, 1))
    return scores.sub_(m).mul_(s["scale"] * LOG2E).sub_(log2l).exp2_().sum((2, 3))


def _places(lengths, table, page, steps):
    """Page and slot of the positions lengths[b] .. lengths[b] + steps - 1."""
    at = lengths.long()[:, None] + torch.arange(steps, device="cuda")
    if table is None:
        return torch.arange(at.shape[0], device="cuda")[:, None].expand_as(at), at
    return table.long().gather(1, at // page), at % page


def _plain_append(s):
    page = s["k_pages"].shape[2]
    steps = s["index"].shape[1] if s["index"] is not None else s["case"]["tokens"]
    at = _places(s["lengths"], s["table"], page, steps)
    row = torch.arange(steps, device="cuda")
    one = torch.arange(s["case"]["batch"], device="cuda")[:, None]
    index = s["index"].long() if s["index"] is not None else row.expand(one.shape[0], -1)
    k, v = s["k"].transpose(1, 2)[one, index], s["v"].transpose(1, 2)[one, index]  # [B, steps, Hkv, D]
    kp, vp = s["k_pages"].transpose(1, 2), s["v_pages"].transpose(1, 2)  # [N, page, Hkv, D]
    if s["counts"] is not None:
        there = (row < s["counts"][:, None])[..., None, None]
        k, v = torch.where(there, k, kp[at]), torch.where(there, v, vp[at])
    kp[at], vp[at] = k, v
    return s["k_pages"], s["v_pages"]


def _plain_evict(s):
    case, w = s["case"], s["weights"]
    keep, recent = case["keep"], case["recent"]
    b, hkv, room = w.shape
    pos, length = torch.arange(room, device="cuda"), s["lengths"][:, None, None].long()
    rank = torch.where(pos < length, torch.where(pos >= length - recent, math.inf, w), -math.inf)
    best = rank.sort(dim=2, descending=True, stable=True).indices[..., :keep]
    if room < keep:
        best = torch.cat([best, best.new_full((b, hkv, keep - room), room)], 2)
    left = length.clamp(max=keep)
    slot = torch.arange(keep, device="cuda")
    kept = torch.where(slot < left, best, room).sort(dim=2).values  # ascending; behind the new length: none
    there = slot < left
    at = kept.clamp(max=room - 1)
    page = s["k_pages"].shape[2]
    one, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[:, None]
    src = (one.expand_as(at), at) if s["table"] is None else (s["table"].long()[one, at // page], at % page)
    k, v = s["k_pages"][src[0], head, src[1]], s["v_pages"][src[0], head, src[1]]  # [B, Hkv, keep, D]
    out_w = torch.where(there, w.gather(2, at), torch.zeros_like(w[..., :1]))
    kept = torch.where(there, kept, -1).to(torch.int32)
    if case["into"]:
        ko, vo, table = s["out"]
        to = (table.long()[one, slot // ko.shape[2]], head, slot % ko.shape[2])
        ko[to], vo[to] = torch.where(there[..., None], k, ko[to]), torch.where(there[..., None], v, vo[to])
    else:
        ko, vo = (torch.where(there[..., None], x, torch.zeros_like(x)) for x in (k, v))
    return ko, vo, left.flatten().to(torch.int32), out_w, kept


def _handle(s):
    """The cache as the framework's programs hold it, made once and kept beside the tensors."""
    from kohakufa_b200 import KVCache

    if "cache" not in s:
        s["cache"] = KVCache(s["k_pages"], s["v_pages"], s["lengths"], s["table"])
        if "out" in s:
            k, v, table = s["out"]
            s["into"] = KVCache(k, v, torch.zeros_like(s["lengths"]), table)
    return s["cache"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"attend": _plain_attend, "weigh": _plain_weigh, "append": _plain_append, "evict": _plain_evict}[op](state)
    import kohakufa_b200 as kfa

    cache = _handle(state)
    if op == "attend":
        return kfa.attention_cached(
            state["q"], cache, state.get("k"), state.get("v"), tree=state.get("tree"), counts=state["counts"],
            scale=state["scale"], return_stats=state["case"]["stats"],
        )  # fmt: skip
    if op == "weigh":
        return kfa.cache_weights(cache, state["q"], state["stats"], index=state["index"], counts=state["counts"], scale=state["scale"])
    if op == "append":
        kfa.cache_append(cache, state["k"], state["v"], index=state["index"], counts=state["counts"])
        return state["k_pages"], state["v_pages"]
    out, weights, kept = kfa.cache_evict(
        cache, state["weights"], state["case"]["keep"], recent=state["case"]["recent"], out=state.get("into")
    )
    return out.k, out.v, out.lengths, weights, kept


# ---- 64 bits, from the definitions -----------------------------------------------------------------------------------


def _sequence(pages, table, b, n):
    """[Hkv, n, D]: the first n positions of sequence b."""
    if table is None:
        return pages[b, :, :n]
    page = pages.shape[2]
    return torch.cat([pages[p] for p in table[b, : -(-n // page)].tolist()] or [pages[0, :, :0]], 1)[:, :n]


def _exact_rows(q, k, visible, scale):
    """Softmax weights in 64 bits of [R, D] rows over [n, D] keys, the raw row maxima and the log2 of the sums."""
    raw = (q.double() @ k.double().T).masked_fill(~visible, -math.inf)
    empty = ~visible.any(1) if visible.shape[1] else torch.ones(visible.shape[0], dtype=torch.bool, device=visible.device)
    m = raw.amax(1) if visible.shape[1] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    e = torch.exp((raw - torch.where(empty, 0.0, m)[:, None]) * scale)
    l = e.sum(1)
    m, l = torch.where(empty, math.inf, m), torch.where(empty, 1.0, l)
    return e / l[:, None], m, l.log2()


def _exact_attend(s):
    case = s["case"]
    b, h, t, d = s["q"].shape
    group, counts = h // case["kv_heads"], _counts(case)
    out = torch.zeros(b, h, t, d, dtype=torch.float64, device="cuda")
    stats = torch.zeros(b, h, 2, t, dtype=torch.float64, device="cuda")
    stats[:, :, 0] = math.inf
    for i, (n, c) in enumerate(zip(_lengths(case), counts)):
        kc, vc = _sequence(s["k_pages"], s["table"], i, n), _sequence(s["v_pages"], s["table"], i, n)
        visible = torch.ones(c, n, dtype=torch.bool, device="cuda")
        if case["new"] != "none":
            kc, vc = torch.cat([kc, s["k"][i, :, :c]], 1), torch.cat([vc, s["v"][i, :, :c]], 1)
            among = s["tree"][i, :c, :c] if case["new"] == "tree" else torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
            visible = torch.cat([visible, among], 1)
        for g in range(h if c else 0):
            p, m, log2l = _exact_rows(s["q"][i, g, :c], kc[g // group], visible, s["scale"])
            out[i, g, :c], stats[i, g, 0, :c], stats[i, g, 1, :c] = p @ vc[g // group].double(), m, log2l
    return (out, stats) if case["stats"] else out


def _exact_weigh(s):
    case = s["case"]
    total = torch.zeros(case["batch"], case["kv_heads"], _room(s), dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        rows = s["index"][i, :c].long() if s["index"] is not None else torch.arange(c, device="cuda")
        keys = _sequence(s["k_pages"], s["table"], i, n + c)
        visible = torch.ones(c, n + c, dtype=torch.bool, device="cuda").tril(n)
        for g in range(case["heads"]):
            raw = s["q"][i, g, rows].double() @ keys[g // group].double().T
            m, log2l = (s["stats"][i, g, j, rows].double()[:, None] for j in (0, 1))
            p = torch.exp((raw - m) * s["scale"]) / torch.exp2(log2l)
            total[i, g // group, : n + c] += torch.where(visible, p, 0.0).sum(0)
    return total


def _exact_append(s):
    case, steps = s["case"], s["case"]["accepted"] or s["case"]["tokens"]
    got = []
    for pages, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pages = pages.double()
        for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
            rows = s["index"][i].tolist() if s["index"] is not None else None
            at = torch.arange(n, n + min(c, steps), device="cuda")
            page = torch.full_like(at, i) if s["table"] is None else s["table"][i].long()[at // pages.shape[2]]
            slot = at if s["table"] is None else at % pages.shape[2]
            x = new[i, :, :c] if rows is None else new[i][:, rows[:c]]
            pages[page, :, slot] = x.transpose(0, 1).double()
        got.append(pages)
    return tuple(got)


def _exact_evict(s):
    case = s["case"]
    keep, recent, b, hkv = case["keep"], case["recent"], case["batch"], case["kv_heads"]
    if case["into"]:
        ks, vs, table = s["out"][0].double(), s["out"][1].double(), s["out"][2]
    else:
        ks = torch.zeros(b, hkv, keep, case["dim"], dtype=torch.float64, device="cuda")
        vs, table = torch.zeros_like(ks), None
    weights = torch.zeros(b, hkv, keep, dtype=torch.float64, device="cuda")
    kept = torch.full((b, hkv, keep), -1, dtype=torch.int32, device="cuda")
    lengths = _lengths(case)
    for i, n in enumerate(lengths):
        k, v = _sequence(s["k_pages"], s["table"], i, n), _sequence(s["v_pages"], s["table"], i, n)
        left = min(n, keep)
        for g in range(hkv):
            w = s["weights"][i, g, :n].double()
            if n <= keep:
                stay = torch.arange(n, device="cuda")
            else:
                old = w[: n - recent].argsort(descending=True, stable=True)[: keep - recent]
                stay = torch.cat([old.sort().values, torch.arange(n - recent, n, device="cuda")])
            weights[i, g, :left], kept[i, g, :left] = w[stay], stay.to(torch.int32)
            slot = torch.arange(left, device="cuda")
            page = torch.full_like(slot, i) if table is None else table[i].long()[slot // ks.shape[2]]
            slot = slot if table is None else slot % ks.shape[2]
            ks[page, g, slot], vs[page, g, slot] = k[g, stay].double(), v[g, stay].double()
    return ks, vs, torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device="cuda"), weights, kept


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "weigh": _exact_weigh, "append": _exact_append, "evict": _exact_evict}[case["op"]](s)
