"""Decode attention over the quantized paged cache, and the cache's pages, as the framework's operators
are measured on them.

Operators (public entry points in `mcoplib.custom_ops` and `torch.ops._C`):
  attention  kv_cache_attention: one new token of every sequence over the sequence's cached keys and values
  copy       kv_cache_copy_pages: pages copied in the codes and scales of every layer
  fork       a step of parallel sampling: kv_cache_fork of prompts into samples, kv_cache_copy_pages of
             the part-filled pages that a fork gives its child, kv_cache_extend of every sample by its
             new tokens, and kv_cache_free of the samples, which leaves the pool as it was
  compact    kv_cache_compact of a pool with holes, and kv_cache_copy_pages of the pages that it moves

Queries, keys and values are N(0, 1) with two key channels of a head 4 times as large; caches hold what
kv_cache_write_quant gives for them, in pages of random order.  The page operators move an fp8 cache.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32  # values that share a 4-bit scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one user's chat of a thousand tokens, an 8B-class model's heads (the smallest call)
        dict(name="attention_t1", op="attention", sequences=1, tokens=1000, ragged=False, heads=8,
             group=4, key=128, value=128, cache="fp8", page=16, dtype="bf16", window=0, lse=False),
        # a decode step of 64 sequences with contexts of all lengths, a 70B-class model's heads
        dict(name="attention_t64_int8", op="attention", sequences=64, tokens=131072, ragged=True,
             heads=8, group=8, key=128, value=128, cache="int8", page=16, dtype="bf16", window=0,
             lse=False),
        # two documents of 128k tokens: the length has to fill the card
        dict(name="attention_long_fp8", op="attention", sequences=2, tokens=262144, ragged=False,
             heads=8, group=8, key=128, value=128, cache="fp8", page=64, dtype="fp16", window=0,
             lse=False),
        # a 4-bit cache whose keys are wider than its values
        dict(name="attention_mxfp4", op="attention", sequences=16, tokens=131072, ragged=False,
             heads=8, group=4, key=192, value=128, cache="mxfp4", page=16, dtype="bf16", window=0,
             lse=False),
        # odd everything: heads, widths, pages; fp32, with the row's log-sum for a later join
        dict(name="attention_ragged_fp32", op="attention", sequences=37, tokens=60013, ragged=True,
             heads=5, group=3, key=80, value=96, cache="int8", page=7, dtype="fp32", window=0,
             lse=True),
        # layers with a sliding window, wide heads, sixteen query heads a key head
        dict(name="attention_window", op="attention", sequences=48, tokens=48 * 8192, ragged=False,
             heads=4, group=16, key=256, value=256, cache="fp8", page=16, dtype="bf16", window=1024,
             lse=False),
        # pages handed from one part of a pool to another: a few of a small model
        dict(name="copy_few", op="copy", pairs=16, pages=256, layers=4, heads=4, width=128, page=16),
        # the largest: a long prompt's pages in 32 layers
        dict(name="copy_layers", op="copy", pairs=400, pages=1000, layers=32, heads=8, width=128,
             page=16),
        # one prompt into four samples, a first token each
        dict(name="fork_one", op="fork", prompts=1, forks=4, tokens=700, grow=1, spare=100, layers=2,
             heads=4, width=128, page=16),
        # 32 prompts into 128 samples, a chunk of drafted tokens each
        dict(name="fork_batch", op="fork", prompts=32, forks=128, tokens=16000, grow=40, spare=200,
             layers=16, heads=8, width=128, page=16),
        # a small pool after a few sequences ended
        dict(name="compact_small", op="compact", pages=500, used=0.5, sequences=9, layers=2, heads=4,
             width=64, page=8),
        # a pool of 8192 pages, nine tenths in use, before its end is given to something else
        dict(name="compact_pool", op="compact", pages=8192, used=0.9, sequences=64, layers=2, heads=8,
             width=128, page=16),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    """Any operator: 1 to 256 sequences of together 1 to 262144 tokens, heads of 16 to 256 in groups of
    1 to 16, pages of 1 to 64 tokens, pools of up to 8192 pages, every type."""
    op = rng.choice(("attention", "attention", "attention", "copy", "fork", "compact"))
    if op == "attention":
        cache = rng.choice(tuple(CACHES))
        step = BLOCK if cache == "mxfp4" else rng.choice((1, 8, 16))
        width = lambda: step * max(1, _log(rng, 16, 256) // step)  # noqa: E731
        key = width()
        value = key if rng.random() < 0.6 else width()
        heads, sequences = rng.randint(1, 16), _log(rng, 1, 256)
        most = min(262144, (1 << 29) // (heads * (key + value)))
        tokens = max(sequences, _log(rng, 1, most))
        ragged = rng.random() < 0.6
        window = 0 if ragged or rng.random() < 0.6 else _log(rng, 1, 4096)
        return dict(op=op, sequences=sequences, tokens=tokens, ragged=ragged, heads=heads,
                    group=rng.randint(1, 16), key=key, value=value, cache=cache,
                    page=rng.choice((1, 16, 16, 64, 7)), dtype=rng.choice(tuple(DTYPES)),
                    window=window, lse=rng.random() < 0.3)
    shape = dict(layers=_log(rng, 1, 32), heads=rng.randint(1, 8),
                 width=rng.choice((1, 8, 16)) * rng.randint(4, 16), page=rng.choice((1, 7, 16, 16)))
    slab = shape["layers"] * shape["heads"] * shape["page"] * (2 * shape["width"] + 8)
    most = min(8192, (1 << 29) // slab)  # pages of a pool of half a gigabyte
    if op == "copy":
        pages = _log(rng, 2, most)
        return dict(op=op, pairs=_log(rng, 1, pages // 2), pages=pages, **shape)
    if op == "fork":
        prompts, forks = _log(rng, 1, 32), _log(rng, 1, 64)
        tokens = max(prompts, _log(rng, 1, max(1, most // 4 * shape["page"])))
        return dict(op=op, prompts=prompts, forks=forks, tokens=tokens, grow=_log(rng, 1, 60),
                    spare=_log(rng, 1, 200), **shape)
    return dict(op=op, pages=_log(rng, 2, most), used=rng.uniform(0.05, 1.0),
                sequences=_log(rng, 1, 64), **shape)


# ------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _randint(g, low, high, *shape):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)


def _lengths(g, count, total, ragged):
    """count lengths (on the host) that are total together: equal but for one, or random cuts."""
    if not ragged:
        return torch.tensor([total // count + (i < total % count) for i in range(count)],
                            dtype=torch.int32)
    cuts = (torch.rand(count - 1, generator=g, device="cuda") * (total + 1)).to(torch.int32).cpu()
    edges = torch.cat([torch.zeros(1, dtype=torch.int32), cuts.sort().values,
                       torch.tensor([total], dtype=torch.int32)])
    return edges[1:] - edges[:-1]


def _table(g, lengths, page, columns, pages):
    """A table of the pages that the lengths take, in random order; -1 past them."""
    held = (lengths + page - 1) // page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((lengths.numel(), columns), -1, dtype=torch.int32)
    table[torch.arange(columns).expand_as(table) < held[:, None]] = order[:int(held.sum())]
    return table


def _vectors(g, pages, page, heads, width, kind, loud=False):
    """(codes, scales) of random vectors, a page's slots all in use."""
    codes, scales = [], []
    for part in range(0, pages, 4096):
        x = _randn(g, min(4096, pages - part), page, heads, width)
        if loud:
            x[..., :2] *= 4
        if kind == "mxfp4":
            code, scale = _packed(*_blocks(x))
        else:
            most = x.abs().amax(-1)
            scale = (most / (127 if kind == "int8" else 448)).clamp_min(1e-30)
            q = x / scale[..., None]
            code = (q.round().clamp(-127, 127) if kind == "int8" else q.clamp(-448, 448)).to(
                CACHES[kind])
        codes.append(code)
        scales.append(scale)
    return torch.cat([c.view(torch.uint8) for c in codes]).view(CACHES[kind]), torch.cat(scales)


def _prepare_attention(case, g, state):
    lengths = _lengths(g, case["sequences"], case["tokens"], case["ragged"])
    page = case["page"]
    pages = int(((lengths + page - 1) // page).sum()) + 3
    state["longest"] = int(lengths.max())
    columns = max(1, -(-state["longest"] // page))
    state["table"] = _table(g, lengths, page, columns, pages).cuda()
    state["lengths"] = lengths.cuda()
    for name in ("key", "value"):
        state[name + "_cache"], state[name + "_scale"] = _vectors(
            g, pages, page, case["heads"], case[name], case["cache"], loud=name == "key")
    # the queries as they lie in a fused projection's output, beside the new keys and values
    queries = case["heads"] * case["group"]
    qkv = _randn(g, case["sequences"],
                 queries * case["key"] + case["heads"] * (case["key"] + case["value"]),
                 dtype=DTYPES[case["dtype"]])
    state["query"] = qkv[:, :queries * case["key"]].unflatten(1, (queries, case["key"]))


def _layers(g, case, pages):
    """The codes of every layer's keys and values, and their scales."""
    sides = [_vectors(g, pages, case["page"], case["heads"], case["width"], "fp8")
             for _ in range(2 * case["layers"])]
    shape = (case["layers"], 2, pages)
    return [torch.stack([part.view(torch.uint8) for part in parts]).view(parts[0].dtype).unflatten(
        0, shape[:2]) for parts in zip(*sides)]


def _counts(table, pages):
    held = table[table >= 0].long()
    return torch.bincount(held, minlength=pages).to(torch.int32)


def _prepare_pages(case, g, state):
    page, op = case["page"], case["op"]
    if op == "copy":
        pages = case["pages"]
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        state["src"] = order[:case["pairs"]].clone()
        state["dst"] = order[case["pairs"]:2 * case["pairs"]].clone()
    elif op == "fork":
        longest = 4 * case["tokens"] // case["prompts"]
        lengths = _lengths(g, case["prompts"], case["tokens"], True).clamp_max(longest)
        # 1 to grow new tokens, together the same for every seed
        half = (torch.rand(case["forks"] // 2, generator=g, device="cuda") * case["grow"] + 1).to(
            torch.int32).cpu()
        middle = torch.full((case["forks"] % 2,), (case["grow"] + 1) // 2, dtype=torch.int32)
        grow = torch.cat([half, middle, case["grow"] + 1 - half])
        pages = (case["tokens"] // page + case["prompts"]
                 + case["forks"] * (case["grow"] // page + 2) + case["spare"])
        columns = (longest + case["grow"]) // page + 2
        table = torch.full((case["prompts"] + case["forks"], columns), -1, dtype=torch.int32)
        table[:case["prompts"]] = _table(g, lengths, page, columns, pages)
        state["lengths"] = torch.cat([lengths, torch.zeros(case["forks"], dtype=torch.int32)]).cuda()
        state["children"] = (case["prompts"] + torch.randperm(
            case["forks"], generator=g, device="cuda")).to(torch.int32)
        state["parents"] = _randint(g, 0, case["prompts"], case["forks"])
        state["cu"] = torch.cat([torch.zeros(1, dtype=torch.int32),
                                 grow.cumsum(0).to(torch.int32)]).cuda()
        state["new"] = int(state["cu"][-1])
        state["table"], state["counts"] = table.cuda(), _counts(table, pages).cuda()
    else:
        pages = case["pages"]
        used = max(1, int(pages * case["used"]))
        lengths = _lengths(g, case["sequences"], used * page, True)
        columns = min(pages, 4 * used // case["sequences"] + 1)
        lengths = lengths.clamp_max(columns * page)
        while int(((lengths + page - 1) // page).sum()) > pages:  # part-filled pages
            lengths[lengths.argmax()] -= min(page, int(lengths.max()))
        table = _table(g, lengths, page, columns, pages)
        table = torch.cat([table, table[:1]])  # two sequences on the same pages
        state["table"], state["counts"] = table.cuda(), _counts(table, pages).cuda()
    state["held"] = _layers(g, case, pages)
    state["caches"] = [t for codes, scales in zip(*state["held"]) for t in (*codes, *scales)]


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["op"] == "attention":
        _prepare_attention(case, g, state)
    else:
        _prepare_pages(case, g, state)
    return state


# ---------------------------------------------------------------------------------- plain form


def _blocks(x):
    """(codes 0..15, scale bytes) of x in blocks of 32, as the 4-bit cache holds them."""
    v = x.unflatten(-1, (-1, BLOCK))
    most = v.abs().amax(-1)
    byte = torch.where(most == 0, 0, (torch.frexp(most).exponent + 124).clamp_min(0))
    q = torch.ldexp(v.abs(), (127 - byte)[..., None])
    code = ((q > 0.25).int() + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5)
            + (q > 5))
    return (code + 8 * torch.signbit(v)).flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def _packed(code, byte):
    pairs = code.unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4), byte


def _values(codes, scale, kind):
    if kind != "mxfp4":
        return codes.float() * scale[..., None]
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = table[code.int()].unflatten(-1, (-1, BLOCK))
    return torch.ldexp(v, (scale.int() - 127)[..., None]).flatten(-2)


def _attention(state):
    page, heads, group = state["page"], state["heads"], state["group"]
    at = torch.arange(state["longest"], device="cuda", dtype=torch.int32)
    length = state["lengths"][:, None]
    live = at < length
    if state["window"]:
        live = live & (at >= length - state["window"])
    row = state["table"][:, at // page].long() * page + at % page
    row = torch.where(live, row, 0)
    k, v = (torch.where(live[..., None, None],
                        _values(state[n + "_cache"].view(torch.uint8).flatten(0, 1)[row].view(
                            CACHES[state["cache"]]),
                            state[n + "_scale"].flatten(0, 1)[row], state["cache"]), 0.0)
            .permute(0, 2, 1, 3).contiguous() for n in ("key", "value"))
    q = state["query"].float().unflatten(1, (heads, group)) / math.sqrt(state["key"])
    s = torch.matmul(q, k.transpose(2, 3))
    s = torch.where(live[:, None, None], s, -math.inf)
    most = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(s - most)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.flatten(1, 2).to(DTYPES[state["dtype"]])
    return [out, (most + total.log()).flatten(1)] if state["lse"] else out


def _copy(caches, src, dst):
    move = (src >= 0) & (dst >= 0)
    src, dst = src[move].long(), dst[move].long()
    for t in caches:
        t = t.view(torch.uint8)
        t[dst] = t[src]


def _free_pages(counts):
    """The free pages, the lowest first, and how many there are."""
    busy = counts > 0
    return torch.sort(busy.int(), stable=True).indices.to(torch.int32), (~busy).sum()


def _fork(state):
    table, lengths, counts, page = (state[n] for n in ("table", "lengths", "counts", "page"))
    parents, children = state["parents"].long(), state["children"].long()
    length = lengths[parents]
    full, part = length // page, length % page > 0
    free, many = _free_pages(counts)
    rank = part.cumsum(0) - 1
    got = ~part | (rank < many)
    copied = part & got
    dst = torch.where(copied, free[rank.clamp_min(0)], -1).to(torch.int32)
    src = torch.where(copied, table[parents, full.clamp_max(table.shape[1] - 1).long()], -1).to(
        torch.int32)
    rows = table[parents]
    column = torch.arange(table.shape[1], device="cuda")
    shared = (column < full[:, None]) & got[:, None]
    counts.scatter_add_(0, rows.clamp_min(0).long().flatten(), shared.int().flatten())
    counts.scatter_add_(0, dst.clamp_min(0).long(), copied.int())
    last = (column == full[:, None]) & copied[:, None]
    table[children] = torch.where(shared, rows, torch.where(last, dst[:, None], -1))
    lengths[children] = torch.where(got, length, 0)
    return src, dst


def _extend(state):
    table, lengths, counts, page = (state[n] for n in ("table", "lengths", "counts", "page"))
    sequences, cu = state["children"].long(), state["cu"]
    old = lengths[sequences]
    new = old + cu[1:] - cu[:-1]
    have = (old + page - 1) // page
    fits = new <= table.shape[1] * page
    need = torch.where(fits, (new + page - 1) // page - have, 0)
    first = need.cumsum(0) - need
    free, many = _free_pages(counts)
    got = fits & ((need == 0) | (first + need <= many))
    column = torch.arange(table.shape[1], device="cuda")
    taken = (column >= have[:, None]) & (column < (have + need)[:, None]) & got[:, None]
    index = (first[:, None] + column - have[:, None]).clamp(0, counts.numel() - 1)
    page_of = free[index]
    rows = torch.where(taken, page_of, table[sequences])
    table[sequences] = rows
    counts.scatter_add_(0, page_of.long().flatten(), taken.int().flatten())
    lengths[sequences] = torch.where(got, new, old)
    token = torch.arange(state["new"], device="cuda", dtype=torch.int32)
    owner = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    at = old[owner] + token - cu[owner]
    slots = rows[owner, (at // page).long()].long() * page + at % page
    return torch.where(got[owner], slots, -1), torch.where(got, old, -1).to(torch.int32)


def _free(state):
    table, lengths, counts, page = (state[n] for n in ("table", "lengths", "counts", "page"))
    sequences = state["children"].long()
    held = (lengths[sequences] + page - 1) // page
    live = torch.arange(table.shape[1], device="cuda") < held[:, None]
    counts.scatter_add_(0, table[sequences].clamp_min(0).long().flatten(), -live.int().flatten())
    table[sequences] = -1
    lengths[sequences] = 0


def _compact(table, counts):
    pages = counts.numel()
    index = torch.arange(pages, device="cuda")
    busy = counts > 0
    used = busy.sum()
    before = busy.cumsum(0) - busy.long()
    none = pages // 2  # one more than the lists hold
    src, dst = (torch.full((none + 1,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    moves, hole = busy & (index >= used), ~busy & (index < used)
    src[torch.where(moves, used - 1 - before, none)] = index.to(torch.int32)
    dst[torch.where(hole, index - before, none)] = index.to(torch.int32)
    place = torch.where(moves, dst[torch.where(moves, used - 1 - before, none)], index).to(torch.int32)
    table.copy_(torch.where(table >= 0, place[table.clamp_min(0).long()], table))
    held = torch.zeros_like(counts).scatter_add_(0, place.long(), torch.where(busy, counts, 0))
    counts.copy_(held)
    return src[:none], dst[:none], used.to(torch.int32).reshape(1)


def _plain(state):
    op = state["op"]
    if op == "attention":
        return _attention(state)
    if op == "copy":
        _copy(state["caches"], state["src"], state["dst"])
        return state["held"]
    if op == "fork":
        src, dst = _fork(state)
        _copy(state["caches"], src, dst)
        slots, starts = _extend(state)
        _free(state)
        return [src, dst, slots, starts, state["table"], state["lengths"], state["counts"],
                *state["held"]]
    # of a copy of the bookkeeping, so that a pass leaves the next one its holes
    table, counts = state["table"].clone(), state["counts"].clone()
    src, dst, used = _compact(table, counts)
    _copy(state["caches"], src, dst)
    return [src, dst, used, table, counts, *state["held"]]


# ------------------------------------------------------------------------- the framework's calls


def _framework(state):
    from mcoplib import custom_ops

    op = state["op"]
    if op == "attention":
        return custom_ops.kv_cache_attention(
            state["query"], state["key_cache"], state["value_cache"], state["key_scale"],
            state["value_scale"], state["table"], state["lengths"], window=state["window"],
            return_lse=state["lse"])
    if op == "copy":
        custom_ops.kv_cache_copy_pages(state["caches"], state["src"], state["dst"])
        return state["held"]
    if op == "fork":
        pool = (state["table"], state["lengths"], state["counts"])
        src, dst = custom_ops.kv_cache_fork(*pool, state["parents"], state["children"], state["page"])
        custom_ops.kv_cache_copy_pages(state["caches"], src, dst)
        slots, starts = custom_ops.kv_cache_extend(*pool, state["children"], state["cu"], state["new"],
                                                   state["page"])
        custom_ops.kv_cache_free(*pool, state["children"], state["page"])
        return [src, dst, slots, starts, *pool, *state["held"]]
    table, counts = state["table"].clone(), state["counts"].clone()
    src, dst, used = custom_ops.kv_cache_compact(table, counts)
    custom_ops.kv_cache_copy_pages(state["caches"], src, dst)
    return [src, dst, used, table, counts, *state["held"]]


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# ------------------------------------------------------------------------------ work and exact


def work(case):
    if case["op"] == "attention":
        held = case["tokens"]
        if case["window"]:
            held = case["sequences"] * min(case["window"], max(1, held // case["sequences"]))
        heads, values = case["heads"], case["key"] + case["value"]
        vector = values // 2 + values // BLOCK if case["cache"] == "mxfp4" else values + 8
        queries = case["sequences"] * heads * case["group"]
        return {"bytes": held * heads * vector + queries * values * BYTES[case["dtype"]],
                "flops": 2 * held * heads * case["group"] * values}
    slab = case["layers"] * case["heads"] * case["page"] * (2 * case["width"] + 8)
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * slab, "flops": 0}
    if case["op"] == "fork":  # nearly every prompt ends inside a page
        shared = case["forks"] * case["tokens"] // case["prompts"] // case["page"]
        part = 0 if case["page"] == 1 else case["forks"]
        return {"bytes": 2 * part * slab + 4 * 6 * shared, "flops": 0}
    moved = int(case["pages"] * case["used"] * (1 - case["used"]))
    return {"bytes": 2 * moved * slab + 8 * case["pages"], "flops": 0}


def _exact_vectors(codes, scale, kind):
    """The values of one head's vectors in 64 bits; 4-bit ones from their sign, exponent and fraction."""
    if kind != "mxfp4":
        return codes.double() * scale.double().unsqueeze(-1)
    both = torch.empty(*codes.shape, 2, dtype=torch.int32, device=codes.device)
    both[..., 0], both[..., 1] = codes % 16, codes // 16
    code = both.reshape(*codes.shape[:-1], -1)
    power, fraction = (code // 2) % 4, (code % 2).double()
    size = torch.where(power > 0, (1 + fraction / 2) * torch.exp2(power.double() - 1), fraction / 2)
    return torch.where(code >= 8, -size, size) * torch.exp2(scale.double() - 127).repeat_interleave(
        BLOCK, -1)


def _exact_attention(state):
    """A sequence and a key head at a time, its positions in one softmax."""
    page, group = state["page"], state["group"]
    queries = state["heads"] * group
    out = torch.zeros(state["sequences"], queries, state["value"], dtype=torch.float64, device="cuda")
    lse = torch.full((state["sequences"], queries), -math.inf, dtype=torch.float64, device="cuda")
    for s, n in enumerate(state["lengths"].tolist()):
        first = max(0, n - state["window"]) if state["window"] else 0
        if n == first:
            continue
        position = torch.arange(first, n, device="cuda")
        pages = state["table"][s].index_select(0, position // page).long()
        for h in range(state["heads"]):
            k, v = (_exact_vectors(
                state[name + "_cache"].view(torch.uint8)[pages, position % page, h].view(
                    CACHES[state["cache"]]),
                state[name + "_scale"][pages, position % page, h], state["cache"])
                for name in ("key", "value"))
            mine = slice(h * group, (h + 1) * group)
            logits = state["query"][s, mine].double() @ k.t().contiguous() * state["key"] ** -0.5
            lse[s, mine] = torch.logsumexp(logits, -1)
            out[s, mine] = torch.softmax(logits, -1) @ v
    return [out, lse] if state["lse"] else out


def _exact_copies(held, src, dst):
    pairs = [(a, b) for a, b in zip(src, dst) if a >= 0 and b >= 0]
    read = torch.tensor([a for a, _ in pairs], dtype=torch.int64, device="cuda")
    write = torch.tensor([b for _, b in pairs], dtype=torch.int64, device="cuda")
    outs = []
    for t in held:
        raw = t.clone().view(torch.uint8)
        raw.index_copy_(2, write, raw.index_select(2, read))
        outs.append(raw.view(t.dtype))
    return outs


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _exact_fork(state):
    """The pool as lists, one fork and one sequence after the other."""
    page = state["page"]
    table, lengths, counts = (state[n].tolist() for n in ("table", "lengths", "counts"))
    src, dst, slots, starts = [], [], [], []

    def take():
        found = counts.index(0)
        counts[found] = 1
        return found

    for parent, child in zip(state["parents"].tolist(), state["children"].tolist()):
        full, part = divmod(lengths[parent], page)
        for column in range(full):
            table[child][column] = table[parent][column]
            counts[table[parent][column]] += 1
        src.append(table[parent][full] if part else -1)
        dst.append(take() if part else -1)
        if part:
            table[child][full] = dst[-1]
        lengths[child] = lengths[parent]
    cu = state["cu"].tolist()
    for i, sequence in enumerate(state["children"].tolist()):
        starts.append(lengths[sequence])
        for _ in range(cu[i + 1] - cu[i]):
            column, offset = divmod(lengths[sequence], page)
            if offset == 0:
                table[sequence][column] = take()
            slots.append(table[sequence][column] * page + offset)
            lengths[sequence] += 1
    return [_ints(src), _ints(dst), _ints(slots, torch.int64), _ints(starts), state["table"],
            state["lengths"], state["counts"], *_exact_copies(state["held"], src, dst)]


def _exact_compact(state):
    table, counts = state["table"].tolist(), state["counts"].tolist()
    src, dst = [], []
    low, high = 0, len(counts) - 1
    while True:  # the last page in use to the first that is free
        while low < len(counts) and counts[low] > 0:
            low += 1
        while high >= 0 and counts[high] <= 0:
            high -= 1
        if low >= high:
            break
        src.append(high)
        dst.append(low)
        counts[low], counts[high] = counts[high], 0
    place = dict(zip(src, dst))
    table = [[place.get(p, p) for p in row] for row in table]
    short = [-1] * (len(counts) // 2 - len(src))
    used = sum(1 for c in counts if c > 0)
    return [_ints(src + short), _ints(dst + short), _ints([used]), _ints(table), _ints(counts),
            *_exact_copies(state["held"], src, dst)]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state)
    if case["op"] == "copy":
        return _exact_copies(state["held"], state["src"].tolist(), state["dst"].tolist())
    if case["op"] == "fork":
        return _exact_fork(state)
    return _exact_compact(state)
