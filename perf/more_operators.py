"""Positions and shared prompts: what a program that trains or serves a model calls beside attention.

Three operators:

  rotary   queries and keys are turned by their positions' angles (two layouts, part of the head, frequencies scaled for
           long contexts), forward, or forward and backward;
  append   the same on the way into a cache of pages: keys turned and written behind the cached ones, values written, queries turned;
  shared   attention of new tokens whose sequences go on from a few prefixes that are stored once: each row sees its prefix, its
           sequence's own cache and the new tokens before it.

A cache is ``k_pages`` and ``v_pages`` [N, Hkv, page, D] (views of [N, page, Hkv, D] storage), ``table`` int32 [B, M] (position p of
sequence b lies in page ``table[b, p // page]``; None: page b is sequence b's) and ``lengths`` int32 [B].
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LOG2E = 1.4426950408889634
BASE = 10000.0


def _angles(rotated, interleaved=False, method="none", factor=1.0, trained=0):
    return dict(rotated=rotated, interleaved=interleaved, method=method, factor=factor, trained=trained)


def _named(name, case):
    return dict(name=name, **case) if name else case


def _rotary(name, batch, heads, kv_heads, tokens, dim, dtype, angles, first=0, packed=False, step=False, seed=1):
    """first: the position of the first token; packed: sequences of different lengths back to back, [T, H, D]; step: with the gradients."""
    return _named(name, dict(op="rotary", batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim, dtype=dtype, first=first,
                             packed=packed, step=step, length_seed=seed, **angles))  # fmt: skip


def _append(name, batch, heads, kv_heads, dim, dtype, page, longest, shortest, tokens, angles, ragged=False, far=0, keys=False, seed=1):
    """ragged: some sequences have fewer new tokens; far: positions that each sequence has besides those in the cache; keys: turned keys are
    wanted beside the pages."""
    return _named(name, dict(op="append", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, longest=longest,
                             shortest=shortest, tokens=tokens, ragged=ragged, far=far, keys=keys, length_seed=seed, **angles))  # fmt: skip


def _shared(name, batch, heads, kv_heads, dim, dtype, page, prefixes, prefix_longest, prefix_shortest, longest, shortest, tokens, new="causal",
            ragged=False, stats=False, seed=1):  # fmt: skip
    return _named(name, dict(op="shared", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, prefixes=prefixes,
                             prefix_longest=prefix_longest, prefix_shortest=prefix_shortest, longest=longest, shortest=shortest, tokens=tokens,
                             new=new, ragged=ragged, stats=stats, length_seed=seed))  # fmt: skip


def listed():
    return [
        # one user's next token: launch and host time count
        _rotary("rotary_token", 1, 8, 8, 1, 64, "fp16", _angles(64), first=100),
        # a packed batch of long documents, frequencies stretched 16 times over the trained length
        _rotary("rotary_packed", 6, 16, 16, 20000, 64, "fp16", _angles(64, method="yarn", factor=16.0, trained=4096), packed=True),
        # a training step of a small model in 32 bits, a quarter of the head turned, pairs next to one another
        _rotary("rotary_part_step", 3, 12, 12, 1537, 80, "fp32", _angles(20, interleaved=True), step=True),
        # a training step of grouped queries over full sequences
        _rotary("rotary_step", 4, 32, 8, 8192, 128, "bf16", _angles(128), step=True),
        # a serving batch, one token each
        _append("append_token", 64, 32, 8, 128, "bf16", 16, 4096, 1, 1, _angles(128)),
        # some verified tokens each, sequences that go on from a prefix, half of the head turned
        _append("append_ragged", 24, 16, 4, 80, "fp16", 32, 3000, 0, 6, _angles(40, interleaved=True), ragged=True, far=8000, keys=True),
        # prompts of 4096 tokens into fresh pages, stretched frequencies
        _append("append_prompt", 4, 32, 8, 128, "bf16", 64, 0, 0, 4096, _angles(128, method="ramp", factor=8.0, trained=8192), keys=True),
        # two answers to one short question
        _shared("shared_pair", 2, 8, 8, 64, "fp16", 0, 1, 100, 100, 40, 3, 1),
        # several system prompts of different popularity, groups between the powers of two, a head dim between the common ones, an empty cache
        _shared("shared_groups", 96, 12, 4, 80, "fp16", 16, 7, 3500, 0, 900, 0, 1),
        # drafted trees of 8 tokens behind one document
        _shared("shared_draft", 32, 32, 8, 128, "bf16", 32, 1, 8192, 8192, 1500, 10, 8, new="tree", ragged=True, stats=True),
        # a serving batch with one long instruction
        _shared("shared_batch", 64, 32, 8, 128, "bf16", 16, 1, 8192, 8192, 1024, 1, 1),
        # many samples of a long document
        _shared("shared_samples", 256, 32, 8, 128, "bf16", 64, 1, 32768, 32768, 2048, 200, 1),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_angles(rng, dim):
    interleaved = rng.random() < 0.4
    rotated = rng.choice([dim, dim, dim, dim // 2 // 2 * 2, dim // 4 // 2 * 2])
    method = rng.choice(["none", "none", "linear", "base", "ramp", "yarn"]) if rotated > 2 else "none"
    return _angles(max(rotated, 2), interleaved, method, 1.0 if method == "none" else rng.choice([2.0, 8.0, 32.0]), 4096)


def draw(rng):
    most = {c["op"]: work(c) for c in listed()}  # the last listed case of an operator is its largest
    while True:
        op = rng.choice(["rotary"] * 3 + ["append"] * 3 + ["shared"] * 6)
        dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([64] * 4 + [128] * 6 + [96, 80, 40, 72, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
        batch = _log_uniform(rng, 1, 192)
        page = rng.choice([0, 0, 16, 16, 32, 64, 128, 48])
        seed = rng.randrange(1000)
        if op == "rotary":
            batch = _log_uniform(rng, 1, 16)
            case = _rotary(None, batch, heads, kv_heads, _log_uniform(rng, 1, 16384), dim, rng.choice([dtype, dtype, "fp32"]),
                           _draw_angles(rng, dim), rng.choice([0, 0, 1000, 100000]), rng.random() < 0.3, rng.random() < 0.5, seed)  # fmt: skip
        elif op == "append":
            longest = _log_uniform(rng, 1, 16384)
            shortest = rng.choice([longest, rng.randint(0, longest), 0])
            tokens = rng.choice([1, _log_uniform(rng, 1, 64), _log_uniform(rng, 64, 4096)])
            case = _append(None, batch, heads, kv_heads, dim, dtype, page, longest, shortest, tokens, _draw_angles(rng, dim),
                           rng.random() < 0.4, rng.choice([0, 0, 500, 60000]), rng.random() < 0.5, seed)  # fmt: skip
        else:
            prefixes = min(rng.choice([1, 1, 1, 2, 5, 16]), batch)
            prefix = _log_uniform(rng, 16, 32768)
            longest = _log_uniform(rng, 1, 4096)
            case = _shared(None, batch, heads, kv_heads, dim, dtype, page, prefixes, prefix, rng.choice([prefix, rng.randint(0, prefix)]), longest,
                           rng.choice([longest, rng.randint(0, longest), 0]), rng.choice([1, 1, 1, _log_uniform(rng, 1, 24)]),
                           rng.choice(["causal", "tree", "none"]), rng.random() < 0.3, rng.random() < 0.5, seed)  # fmt: skip
        w = work(case)
        if w["flops"] <= most[op]["flops"] and w["bytes"] <= most[op]["bytes"] and _values(case) <= 2**31:
            return case


def _values(case):
    """What the plain form holds at once, in numbers."""
    b, h, hkv, t, d = (case[n] for n in ("batch", "heads", "kv_heads", "tokens", "dim"))
    if case["op"] == "rotary":
        return 2 * b * t * (h + hkv) * d
    if case["op"] == "append":
        return b * ((case["longest"] + t) * 2 * hkv + t * (h + 2 * hkv)) * d
    return b * (case["longest"] + t) * (h * t + 2 * hkv * d) + b * h * t * case["prefix_longest"]


# ---- sizes that the case fixes -----------------------------------------------------------------------------------------


def _lengths(case):
    """Cached positions of each sequence of its own (a packed batch: the lengths of its sequences)."""
    rng = random.Random(case["length_seed"])
    if case["op"] == "rotary":
        if not case["packed"]:
            return [case["tokens"]] * case["batch"]
        return [case["tokens"]] + [rng.randint(1, case["tokens"]) for _ in range(case["batch"] - 1)]
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lengths[0] = case["longest"]
    return lengths


def _counts(case):
    """New tokens of each sequence."""
    rng = random.Random(case["length_seed"] + 1)
    return [rng.randint(0, case["tokens"]) for _ in range(case["batch"])] if case["ragged"] else [case["tokens"]] * case["batch"]


def _groups(case):
    """Lengths of the prefixes, and where the sequences that go on from each begin: starts[p] .. starts[p + 1] - 1."""
    rng = random.Random(case["length_seed"] + 2)
    count = case["prefixes"]
    lengths = [case["prefix_longest"]] + [rng.randint(case["prefix_shortest"], case["prefix_longest"]) for _ in range(count - 1)]
    cuts = sorted(rng.randint(0, case["batch"]) for _ in range(count - 1))  # (some prefixes may have nobody)
    return lengths, [0, *cuts, case["batch"]]


def work(case):
    """Every input row read once and every result written once; attention: each prefix's and each own key and value once, two products of the visible pairs."""
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    row = d * (4 if case["dtype"] == "fp32" else 2)  # bytes
    if case["op"] == "rotary":
        rows = sum(_lengths(case)) * (h + hkv) * (2 if case["step"] else 1)
        return {"bytes": float(2 * row * rows), "flops": float(3 * case["rotated"] * rows)}
    counts = _counts(case)
    new = sum(counts)
    if case["op"] == "append":
        moved = row * (2 * (h + 2 * hkv) + case["keys"] * hkv) * new
        return {"bytes": float(moved), "flops": float(3 * case["rotated"] * (h + hkv) * new)}
    lengths, (prefix, starts) = _lengths(case), _groups(case)
    keys = sum(n for c, n in zip(counts, lengths) if c)
    pairs = sum(c * n for c, n in zip(counts, lengths))
    for p, n in enumerate(prefix):
        mine = sum(counts[starts[p] : starts[p + 1]])
        keys += n if mine else 0
        pairs += mine * n
    if case["new"] != "none":
        keys += new
        pairs += sum(c * (c + 1) // 2 for c in counts)
    return {"bytes": float(2 * row * hkv * keys + (2 * row + 8 * case["stats"]) * h * new), "flops": 4.0 * h * d * pairs}


# ---- angles ----------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Angle per position of each pair in 64 bits, and the amplitude of cosine and sine."""
    dim, method, s = case["rotated"], case["method"], case["factor"]
    base = BASE * s ** (dim / (dim - 2)) if method == "base" else BASE
    f = torch.tensor([base ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device="cuda")
    if method == "linear":
        f = f / s
    if method in ("ramp", "yarn"):  # what turns often over the trained length stays, what turns less than once is stretched
        low, high = (1.0, 4.0) if method == "ramp" else (1.0, 32.0)
        keep = ((case["trained"] * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / s
    return f, (0.1 * math.log(s) + 1.0 if method == "yarn" else 1.0)


def _turn(x, at, case, sign=1.0, dtype=torch.float32):
    """x [..., S, D] in `dtype`, turned by positions at [..., S] (one dimension less than x, broadcast)."""
    x = x.to(dtype)
    f, amplitude = _frequencies(case)
    angle = at.double()[..., None] * f
    cos, sin = (angle.cos() * amplitude).to(dtype), (angle.sin() * (sign * amplitude)).to(dtype)
    turned, rest = x[..., : case["rotated"]], x[..., case["rotated"] :]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


# ---- inputs --------------------------------------------------------------------------------------------------------


def _pages(case, positions, page, gen):
    """Pages for so many positions of each sequence, each filled with keys and values, and the table that finds them."""
    std = 0.5 if case["dim"] == 128 else 1.0
    dtype = DTYPES[case["dtype"]]
    if page == 0:
        count, page, table = len(positions), max(max(positions), 1), None
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


def _rows(case, heads, gen):
    std = 0.5 if case["dim"] == 128 else 1.0
    shape = (case["batch"], case["tokens"], heads, case["dim"])
    return torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]]).mul_(std).transpose(1, 2)


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
    lengths, s = _lengths(case), {"case": case}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "rotary":
        dtype, d = DTYPES[case["dtype"]], case["dim"]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            shape = (sum(lengths), heads, d) if case["packed"] else (case["batch"], case["tokens"], heads, d)
            make = lambda: torch.randn(shape, generator=gen, device="cuda", dtype=dtype)  # noqa: B023, E731
            s[name] = make() if case["packed"] else make().transpose(1, 2)
            if case["step"]:
                s["d" + name] = make() if case["packed"] else make().transpose(1, 2)
        if case["packed"]:
            s["positions"] = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in lengths]) + case["first"]
        else:
            s["positions"] = torch.arange(case["tokens"], dtype=torch.int32, device="cuda") + case["first"]
        return s
    counts = _counts(case)
    s["lengths"], s["counts"] = ints(lengths), ints(counts) if case["ragged"] else None
    s["q"], s["k"], s["v"] = (_rows(case, n, gen) for n in (case["heads"], case["kv_heads"], case["kv_heads"]))
    if case["op"] == "append":
        s["k_pages"], s["v_pages"], s["table"] = _pages(case, [n + case["tokens"] for n in lengths], case["page"], gen)
        far = random.Random(case["length_seed"] + 3)
        s["offset"] = ints([far.randint(0, case["far"]) for _ in lengths]) if case["far"] else None
        return s
    prefix, starts = _groups(case)
    s["k_pages"], s["v_pages"], s["table"] = _pages(case, lengths, case["page"], gen)
    s["prefix"] = (*_pages(case, prefix, case["page"], gen), ints(prefix))
    s["starts"] = ints(starts) if case["prefixes"] > 1 else None
    s["scale"] = case["dim"] ** -0.5
    if case["new"] == "none":
        s["k"] = s["v"] = None
    s["tree"] = _tree(case, gen) if case["new"] == "tree" else None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _heads_first(x, case):
    return x.transpose(0, 1) if case["packed"] else x


def _plain_rotary(s):
    case = s["case"]
    turn = lambda x, sign: _heads_first(_turn(_heads_first(x, case), s["positions"], case, sign), case).to(x.dtype)  # noqa: E731
    out = [turn(s["q"], 1.0), turn(s["k"], 1.0)]
    return out + [turn(s["dq"], -1.0), turn(s["dk"], -1.0)] if case["step"] else out


def _plain_append(s):
    case, page = s["case"], s["k_pages"].shape[2]
    step = torch.arange(case["tokens"], device="cuda")
    place = s["lengths"].long()[:, None] + step  # [B, T]
    stands = place if s["offset"] is None else place + s["offset"][:, None]
    q, k = (_turn(s[n], stands[:, None], case).to(s[n].dtype) for n in ("q", "k"))
    there = None if s["counts"] is None else (step < s["counts"][:, None])[:, None, :, None]
    if there is not None:
        q, k = torch.where(there, q, torch.zeros_like(q)), torch.where(there, k, torch.zeros_like(k))
    if s["table"] is None:
        at = torch.arange(case["batch"], device="cuda")[:, None].expand_as(place), place
    else:
        at = s["table"].long().gather(1, place // page), place % page
    kp, vp = s["k_pages"].transpose(1, 2), s["v_pages"].transpose(1, 2)  # [N, page, Hkv, D]
    ks, vs = k.transpose(1, 2), s["v"].transpose(1, 2)
    if there is not None:
        ks, vs = torch.where(there.transpose(1, 2), ks, kp[at]), torch.where(there.transpose(1, 2), vs, vp[at])
    kp[at], vp[at] = ks, vs
    return (q, s["k_pages"], s["v_pages"], k) if case["keys"] else (q, s["k_pages"], s["v_pages"])


def _cached(pages, table):
    """[B, Hkv, room, D] in 32 bits."""
    if table is None:
        return pages.float()
    return pages[table.long()].transpose(1, 2).flatten(2, 3).float()


def _part(raw, v, c):
    """Of masked raw scores: the row's maximum, sum of exponentials and their product with the values."""
    m = raw.amax(-1, keepdim=True) if raw.shape[-1] else raw.new_full((*raw.shape[:-1], 1), -math.inf)
    p = raw.sub_(torch.where(m > -math.inf, m, 0.0)).mul_(c).exp2_()
    return m, p.sum(-1, keepdim=True), p @ v


def _plain_shared(s):
    case, q, c = s["case"], s["q"].float(), s["scale"] * LOG2E
    b, h, t, d = q.shape
    hkv, group = case["kv_heads"], h // case["kv_heads"]
    # a sequence's own keys: cached, then new
    k, v = _cached(s["k_pages"], s["table"]), _cached(s["v_pages"], s["table"])
    seen = (torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None])[:, None].expand(b, t, -1)
    if case["new"] != "none":
        among = s["tree"] if case["new"] == "tree" else torch.ones(t, t, dtype=torch.bool, device="cuda").tril().expand(b, t, t)
        if s["counts"] is not None:
            among = among & (torch.arange(t, device="cuda") < s["counts"][:, None])[:, None]
        k, v, seen = torch.cat([k, s["k"].float()], 2), torch.cat([v, s["v"].float()], 2), torch.cat([seen, among], 2)
    rows = q.reshape(b, hkv, group, t, d)
    raw = rows.flatten(2, 3) @ k.transpose(2, 3)
    raw.view(b, hkv, group, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    parts = [tuple(x.view(b, hkv, group, t, -1) for x in _part(raw, v, c))]
    # the prefixes' keys, all rows of a prefix at once
    kp, vp, table, _ = s["prefix"]
    kp, vp = _cached(kp, table), _cached(vp, table)
    lengths, starts = _groups(case)
    m, l, o = (x.new_full(x.shape, fill) for x, fill in zip(parts[0], (-math.inf, 0.0, 0.0)))
    for p, n in enumerate(lengths):
        mine, n_rows = slice(starts[p], starts[p + 1]), starts[p + 1] - starts[p]
        if n == 0 or n_rows == 0:
            continue
        together = rows[mine].transpose(0, 1).reshape(hkv, -1, d)
        for whole, x in zip((m, l, o), _part(together @ kp[p, :, :n].transpose(1, 2), vp[p, :, :n], c)):
            whole[mine] = x.view(hkv, n_rows, group, t, -1).transpose(0, 1)
    parts.append((m, l, o))
    top = torch.maximum(parts[0][0], parts[1][0])
    some = top > -math.inf
    if s["counts"] is not None:
        some = some & (torch.arange(t, device="cuda") < s["counts"][:, None])[:, None, None, :, None]
    top = torch.where(some, top, 0.0)
    weights = [torch.where(some, ((part[0] - top) * c).exp2(), 0.0) for part in parts]
    l = sum(w * part[1] for w, part in zip(weights, parts))
    l = torch.where(some, l, 1.0)
    out = (sum(w * part[2] for w, part in zip(weights, parts)) / l).reshape(b, h, t, d).to(s["q"].dtype)
    if not case["stats"]:
        return out
    return out, torch.stack([torch.where(some, top, math.inf).reshape(b, h, t), l.log2().reshape(b, h, t)], 2)


# ---- the framework's calls ---------------------------------------------------------------------------------------------


def _handles(s):
    """What a program makes once and keeps: the angles, and the caches as the framework has them."""
    import kohakufa_b200 as kfa

    case = s["case"]
    if case["op"] != "shared" and "rotary" not in s:
        ramp = {"ramp": dict(length=case["trained"], low=1.0, high=4.0), "yarn": dict(length=case["trained"])}.get(case["method"], {})
        s["rotary"] = kfa.Rotary.of(
            case["rotated"], base=BASE, method=case["method"], factor=case["factor"], interleaved=case["interleaved"], **ramp
        )
    if case["op"] != "rotary" and "cache" not in s:
        s["cache"] = kfa.KVCache(s["k_pages"], s["v_pages"], s["lengths"], s["table"])
    if case["op"] == "shared" and "shared" not in s:
        k, v, table, lengths = s["prefix"]
        s["shared"] = kfa.KVCache(k, v, lengths, table)


def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "shared": _plain_shared}[case["op"]](state)
    import kohakufa_b200 as kfa

    _handles(state)
    if case["op"] == "rotary":
        if not case["step"]:
            return kfa.apply_rotary(state["q"], state["k"], state["rotary"], positions=state["positions"])
        q, k = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
        out = kfa.apply_rotary(q, k, state["rotary"], positions=state["positions"])
        return [x.detach() for x in out] + list(torch.autograd.grad(out, (q, k), (state["dq"], state["dk"])))
    if case["op"] == "append":
        out = kfa.cache_append_rotary(
            state["cache"], state["q"], state["k"], state["v"], state["rotary"], counts=state["counts"], offset=state["offset"],
            return_keys=case["keys"],
        )  # fmt: skip
        q, k = out if case["keys"] else (out, None)
        return (q, state["k_pages"], state["v_pages"], k) if case["keys"] else (q, state["k_pages"], state["v_pages"])
    return kfa.attention_shared(
        state["q"], state["shared"], state["cache"], state["k"], state["v"], starts=state["starts"], tree=state["tree"],
        counts=state["counts"], scale=state["scale"], return_stats=case["stats"],
    )  # fmt: skip


# ---- 64 bits, from the definitions -----------------------------------------------------------------------------------


def _exact_turn(x, at, case, back=False):
    """x [..., S, D] as complex numbers times amplitude * exp(i angle) of positions at [S]."""
    f, amplitude = _frequencies(case)
    n = case["rotated"]
    z = x[..., :n].double()
    z = torch.complex(z[..., 0::2], z[..., 1::2]) if case["interleaved"] else torch.complex(z[..., : n // 2], z[..., n // 2 :])
    angle = at.double()[:, None] * f
    z = z * torch.polar(torch.full_like(angle, amplitude), -angle if back else angle)
    y = torch.stack([z.real, z.imag], -1).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., n:].double()], -1)


def _exact_rotary(s):
    case = s["case"]
    out = []
    for name, back in (("q", False), ("k", False), ("dq", True), ("dk", True)):
        if name in s:
            out.append(_heads_first(_exact_turn(_heads_first(s[name], case), s["positions"], case, back), case))
    return out


def _exact_append(s):
    case = s["case"]
    q, k = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k"))
    pages = [s["k_pages"].double(), s["v_pages"].double()]
    far = [0] * case["batch"] if s["offset"] is None else s["offset"].tolist()
    for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        at = torch.arange(n, n + c, device="cuda")
        q[i, :, :c], k[i, :, :c] = (_exact_turn(s[x][i, :, :c], at + far[i], case) for x in ("q", "k"))
        size = pages[0].shape[2]
        page = torch.full_like(at, i) if s["table"] is None else s["table"][i].long()[at // size]
        slot = at if s["table"] is None else at % size
        pages[0][page, :, slot] = k[i, :, :c].transpose(0, 1)
        pages[1][page, :, slot] = s["v"][i, :, :c].transpose(0, 1).double()
    return (q, *pages, k) if case["keys"] else (q, *pages)


def _sequence(pages, table, b, n):
    """[Hkv, n, D]: the first n positions of sequence b."""
    if table is None:
        return pages[b, :, :n]
    page = pages.shape[2]
    return torch.cat([pages[p] for p in table[b, : -(-n // page)].tolist()] or [pages[0, :, :0]], 1)[:, :n]


def _exact_shared(s):
    case = s["case"]
    b, h, t, d = s["q"].shape
    hkv, group = case["kv_heads"], h // case["kv_heads"]
    out = torch.zeros(b, h, t, d, dtype=torch.float64, device="cuda")
    stats = torch.zeros(b, h, 2, t, dtype=torch.float64, device="cuda")
    stats[:, :, 0] = math.inf
    prefix, starts = _groups(case)
    kp, vp, table, _ = s["prefix"]
    lengths, counts = _lengths(case), _counts(case)
    for p, n in enumerate(prefix):
        before = [_sequence(x, table, p, n).double() for x in (kp, vp)]
        for i in range(starts[p], starts[p + 1]):
            c = counts[i]
            if c == 0:
                continue
            own_keys = [_sequence(x, s["table"], i, lengths[i]).double() for x in (s["k_pages"], s["v_pages"])]
            visible = torch.ones(c, n + lengths[i], dtype=torch.bool, device="cuda")
            keys, values = (torch.cat([x, y], 1) for x, y in zip(before, own_keys))
            if case["new"] != "none":
                keys, values = (torch.cat([x, s[name][i, :, :c].double()], 1) for x, name in ((keys, "k"), (values, "v")))
                among = s["tree"][i, :c, :c] if case["new"] == "tree" else torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
                visible = torch.cat([visible, among], 1)
            if keys.shape[1] == 0:
                continue
            rows = s["q"][i, :, :c].double().reshape(hkv, group * c, d)
            raw = (rows @ keys.transpose(1, 2)).view(hkv, group, c, -1).masked_fill(~visible, -math.inf)
            m = raw.amax(-1, keepdim=True)
            some = m > -math.inf
            e = torch.exp((raw - torch.where(some, m, 0.0)) * s["scale"])
            l = torch.where(some, e.sum(-1, keepdim=True), 1.0)
            o = (e / l).flatten(1, 2) @ values
            out[i, :, :c] = o.view(h, c, d)
            stats[i, :, 0, :c] = torch.where(some, m, math.inf).view(h, c)
            stats[i, :, 1, :c] = l.log2().view(h, c)
    return (out, stats) if case["stats"] else out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "shared": _exact_shared}[case["op"]](s)
