"""The paged cache's operators as cases that can be timed and compared.

A search that branches games keeps the keys and values of their histories in pages that rows
share, and evaluates the events that may follow as a tree of drafted tokens.  Four operators
(`cugo_amd.paged_cache`):

  attend  `tree_attention`: the queries of drafted tokens over a row's cached tokens and, of the
          drafts behind them, their own ancestors (or, without a tree, all earlier ones)
  append  `append`: new keys and values into their rows' pages
  branch  `branch`: rows become copies of others, with room for more tokens: whole pages are
          shared, the one that will be written is copied, the old ones are given back
  accept  `accept`: of the drafted tokens the accepted ones move together, the pages behind
          them are given back; before it, `branch` in place makes the round's room

The plain forms below are the definitions in elementary torch operations.
"""

import types

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
MOST_KEYS = 600_000_000  # values of keys, padded to the longest row
MOST_SCORES = 600_000_000
MOST_MOVED = 150_000_000  # values of keys that a pass copies


def listed():
    return [
        # One game's next event: the call's own latency.
        {"name": "attend_one", "kind": "attend", "seqs": 1, "queries": 1, "context": 40,
         "heads": 8, "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16", "tree": False},
        # A wave of games, each with a tree of up to 16 events behind a history of up to 320.
        {"name": "attend_games", "kind": "attend", "seqs": 4096, "queries": 16, "context": 320,
         "heads": 8, "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16", "tree": True},
        # A few long rows of very different lengths with odd trees, four heads a key head.
        {"name": "attend_ragged_long", "kind": "attend", "seqs": 24, "queries": 33,
         "context": 32768, "heads": 32, "kv_heads": 8, "dh": 128, "page": 64, "dtype": "f16",
         "tree": True},
        # A single very long row with a full tree.
        {"name": "attend_single_long", "kind": "attend", "seqs": 1, "queries": 64,
         "context": 131000, "heads": 16, "kv_heads": 4, "dh": 64, "page": 32, "dtype": "bf16",
         "tree": True},
        # Chunks of prompts: many queries, each over all earlier tokens.
        {"name": "attend_chunk", "kind": "attend", "seqs": 4, "queries": 512, "context": 14336,
         "heads": 16, "kv_heads": 4, "dh": 128, "page": 128, "dtype": "bf16", "tree": False},
        # One layer's new tokens of a few games.
        {"name": "append_65", "kind": "append", "seqs": 13, "queries": 5, "context": 48,
         "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16"},
        # The wave's drafts.
        {"name": "append_games", "kind": "append", "seqs": 4096, "queries": 16, "context": 320,
         "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16"},
        # One game's expansion.
        {"name": "branch_16", "kind": "branch", "parents": 1, "children": 16, "context": 40,
         "room": 4, "layers": 4, "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16"},
        # A wave's expansion: 16 children of each of 512 games.
        {"name": "branch_games", "kind": "branch", "parents": 512, "children": 8192,
         "context": 48, "room": 16, "layers": 4, "kv_heads": 8, "dh": 32, "page": 16,
         "dtype": "bf16"},
        # Children of long rows: what is shared outweighs what is copied.
        {"name": "branch_long", "kind": "branch", "parents": 32, "children": 257,
         "context": 8187, "room": 24, "layers": 2, "kv_heads": 8, "dh": 128, "page": 64,
         "dtype": "f16"},
        # A round of a few games.
        {"name": "accept_32", "kind": "accept", "seqs": 32, "queries": 7, "context": 48,
         "layers": 4, "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16"},
        # A round of the wave.
        {"name": "accept_games", "kind": "accept", "seqs": 4096, "queries": 16, "context": 320,
         "layers": 4, "kv_heads": 8, "dh": 32, "page": 16, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "branch", "accept"])
    case = {"kind": kind, "kv_heads": rng.choice([1, 2, 3, 4, 8, 8, 16]),
            "dh": rng.choice([32, 32, 64, 128, 128, 256]),
            "page": rng.choice([16, 16, 32, 64, 128, 256]),
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    token = case["kv_heads"] * case["dh"]
    if kind == "attend":
        case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 4, 5, 8])
        case["tree"] = rng.random() < 0.6
        case["queries"] = _log_int(rng, 1, 130 if case["tree"] else 512)
        case["context"] = _log_int(rng, 1, 131072)
        longest = case["context"] + case["queries"]
        most = min(MOST_KEYS // (longest * token),
                   MOST_SCORES // (longest * case["queries"] * case["heads"]))
        case["seqs"] = _log_int(rng, 1, max(1, min(4096, most)))
        return case
    if kind == "append":
        case["queries"] = _log_int(rng, 1, 512)
        case["context"] = _log_int(rng, 1, 2048)
        most = MOST_MOVED // ((case["context"] + case["queries"] + case["page"]) * token)
        case["seqs"] = _log_int(rng, 1, max(1, min(8192, most)))
        return case
    case["layers"] = rng.randint(1, 6)
    if kind == "branch":
        case["context"] = _log_int(rng, 1, 8192)
        case["room"] = _log_int(rng, 1, 64)
        each = case["page"] * 2 + case["room"]
        most = MOST_MOVED // (each * token * case["layers"])
        case["children"] = _log_int(rng, 1, max(1, min(8192, most)))
        least = MOST_MOVED // ((case["context"] + case["page"]) * token * case["layers"])
        case["parents"] = _log_int(rng, 1, max(1, min(case["children"], least)))
        return case
    case["queries"] = _log_int(rng, 1, 64)
    case["context"] = _log_int(rng, 1, 2048)
    most = MOST_MOVED // ((case["context"] + case["queries"] + case["page"]) * token * case["layers"])
    case["seqs"] = _log_int(rng, 1, max(1, min(8192, most)))
    return case


def _spread(n, low, high):
    """n whole numbers spread evenly over low ... high, the same for every seed."""
    return [low + ((high - low) * (2 * i + 1) + n) // (2 * n) for i in range(n)]


def _lengths(case):
    """Each row's cached tokens, and how many drafted ones are behind them."""
    n = case["seqs"]
    drafts = _spread(n, (case["queries"] + 1) // 2, case["queries"])
    drafts[-1] = case["queries"]
    return _spread(n, case["context"] // 8, case["context"]), drafts


# ------------------------------------------------------------------------------ inputs


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen)
    return torch.tensor(values, dtype=torch.int64)[order]


def _cache(case, gen, dev_gen, lengths, rows, width, spare):
    """A cache whose first rows hold `lengths` tokens in pages anywhere in the pool, which has
    `spare` pages more than those can need."""
    page, layers = case["page"], case.get("layers", 1)
    need = (lengths + page - 1) // page
    used = int(need.sum())
    pages = int(lengths.sum()) // page + len(lengths) + spare  # the same for every seed
    place = torch.randperm(pages, generator=gen)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    inside = torch.zeros(rows, width, dtype=torch.bool)
    inside[:len(lengths)] = torch.arange(width)[None] < need[:, None]
    table[inside] = place[:used].int()
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[place[:used]] = 1
    bits = torch.zeros(-(-pages // 64) * 64, dtype=torch.int64)
    bits[:pages] = refs == 0
    free = (bits.view(-1, 64) << torch.arange(64)).sum(1)
    length = torch.zeros(rows, dtype=torch.int64)
    length[:len(lengths)] = lengths
    shape = (layers, pages, case["kv_heads"], page, case["dh"])

    def values():
        x = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda")
        return x.normal_(generator=dev_gen)

    return types.SimpleNamespace(k=values(), v=values(), table=table.cuda(), length=length.cuda(),
                                 refs=refs.cuda(), free=free.cuda())


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev_gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    page = case["page"]
    if case["kind"] == "branch":
        parents, children = case["parents"], case["children"]
        lengths = _shuffled(_spread(parents, (case["context"] + 1) // 2, case["context"]), gen)
        rows = parents + children
        width = -(-(case["context"] + case["room"]) // page)
        # room for the children's own pages
        spare = children * (-(-case["room"] // page) + 2)
        state["cache"] = _cache(case, gen, dev_gen, lengths, rows, width, spare)
        src = _shuffled([i * parents // children for i in range(children)], gen)
        state["src"] = src.cuda()
        state["dst"] = (parents + torch.randperm(children, generator=gen)).cuda()
        state["want"] = (lengths[src] + case["room"]).cuda()
        return state
    cached, drafts = _lengths(case)
    prefix, drafts = _shuffled(cached, gen), _shuffled(drafts, gen)
    n = case["seqs"]
    rows = n + 3
    width = -(-(case["context"] + case["queries"]) // page)
    total = int(drafts.sum())
    offsets = torch.zeros(n + 1, dtype=torch.int64)
    offsets[1:] = drafts.cumsum(0)
    held = prefix if case["kind"] == "accept" else prefix + drafts
    spare = n * (-(-case["queries"] // page) + 1) if case["kind"] == "accept" else 5
    cache = _cache(case, gen, dev_gen, held, rows, width, spare)
    state["cache"] = cache
    # the sequences' rows, in another order than the cache's
    rows_of = torch.randperm(n, generator=gen)
    prefix, drafts = prefix[rows_of], drafts[rows_of]
    offsets[1:] = drafts.cumsum(0)
    state["rows"], state["prefix"] = rows_of.cuda(), prefix.cuda()
    if case["kind"] == "attend":
        state["offsets"] = offsets.cuda()
        state["most"] = case["queries"]
        state["q"] = torch.empty(total, case["heads"], case["dh"], dtype=DTYPES[case["dtype"]],
                                 device="cuda").normal_(generator=dev_gen)
        state["mask"] = _tree(case, gen, drafts).cuda() if case["tree"] else None
        return state
    which = torch.repeat_interleave(torch.arange(n), drafts)
    index = torch.arange(total) - offsets[which]
    if case["kind"] == "append":
        state["token_rows"] = rows_of[which].cuda()
        state["pos"] = (prefix[which] + index).cuda()
        for name in ("k_new", "v_new"):
            state[name] = torch.empty(total, case["kv_heads"], case["dh"],
                                      dtype=DTYPES[case["dtype"]], device="cuda")
            state[name].normal_(generator=dev_gen)
        return state
    # accept: a path through the tree, 1 to about 5 of the drafts; one row in 8 accepts none
    most = case["queries"]
    chance = torch.rand(n, most, generator=gen)
    chance[torch.arange(most)[None] >= drafts[:, None]] = 2.0
    picked = chance < 3.0 / most
    picked &= torch.rand(n, 1, generator=gen) > 0.125
    place = torch.where(picked, torch.arange(most)[None].expand(n, most), 1 << 40)
    keep = place.sort(1).values
    state["keep"] = torch.where(keep < 1 << 40, keep, -1).cuda()
    state["want"] = (prefix + drafts).cuda()
    return state


def _tree(case, gen, drafts):
    """Each drafted token's ancestors and itself as bits; its parent is an earlier token, one of
    the latest more often, or none."""
    n, most = case["seqs"], case["queries"]
    words = -(-most // 64)
    near = torch.rand(n, most, generator=gen).pow(3)
    parent = torch.arange(most)[None] - 1 - (near * (torch.arange(most)[None] + 1)).long()
    bits = torch.zeros(n, most + 1, words, dtype=torch.int64)  # the last: no ancestors
    one = torch.arange(n)
    for j in range(most):
        bits[:, j] = bits[one, torch.where(parent[:, j] < 0, most, parent[:, j])]
        bits[:, j, j // 64] |= torch.tensor(1, dtype=torch.int64) << (j % 64)
    return bits[:, :most][torch.arange(most)[None] < drafts[:, None]].contiguous()


# ------------------------------------------------------------------------------ one pass


def run(state):
    kind = state["case"]["kind"]
    if kind == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if kind == "append":
        return _own_append(state) if own else _plain_append(state)
    if kind == "branch":
        return _own_branch(state) if own else _plain_branch(state)
    return _own_accept(state) if own else _plain_accept(state)


def _ext():
    from cugo_amd import load_extension

    return load_extension()


def _whole(c, ok):
    return {"ok": ok, "k": c.k, "v": c.v, "table": c.table, "length": c.length, "refs": c.refs,
            "free": c.free}


def _own_attend(s):
    from cugo_amd import paged_cache

    return paged_cache.tree_attention(_ext(), s["cache"], 0, s["q"], s["prefix"], mask=s["mask"],
                                      rows=s["rows"], offsets=s["offsets"])


def _own_append(s):
    from cugo_amd import paged_cache

    paged_cache.append(_ext(), s["cache"], 0, s["k_new"], s["v_new"], s["pos"], s["token_rows"])
    return s["cache"].k, s["cache"].v


def _own_branch(s):
    from cugo_amd import paged_cache

    ok = paged_cache.branch(_ext(), s["cache"], s["dst"], s["src"], s["want"])
    return _whole(s["cache"], ok)


def _own_accept(s):
    from cugo_amd import paged_cache

    ext = _ext()
    room = paged_cache.branch(ext, s["cache"], s["rows"], s["rows"], s["want"])
    ok = paged_cache.accept(ext, s["cache"], s["rows"], s["prefix"], s["keep"])
    return {"room": room, **_whole(s["cache"], ok)}


def _plain_attend(s):
    """Every sequence padded to the longest, in 32 bits."""
    case, c = s["case"], s["cache"]
    page, dh, kv_heads = case["page"], case["dh"], case["kv_heads"]
    group = case["heads"] // kv_heads
    n, most = case["seqs"], s["most"]
    longest = c.table.shape[1] * page
    # the queries, [n, kv_heads, most * group, dh]
    count = s["offsets"][1:] - s["offsets"][:-1]
    index = torch.arange(most, device="cuda")
    real = index < count[:, None]
    token = torch.where(real, s["offsets"][:-1, None] + index, 0)
    q = s["q"][token].float().view(n, most, kv_heads, group, dh)
    q = q.transpose(1, 2).reshape(n, kv_heads, most * group, dh)
    # the keys and values, [n, kv_heads, longest, dh]
    position = torch.arange(longest, device="cuda")
    pages = c.table[s["rows"]].clamp_min(0).long()
    k = c.k[0][pages].transpose(1, 2).reshape(n, kv_heads, longest, dh).float()
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * dh**-0.5
    del k
    # what a query sees, [n, most, longest]
    draft = position - s["prefix"][:, None]
    if s["mask"] is None:
        seen = draft[:, None] <= index[:, None]
    else:
        words = s["mask"].shape[1]
        mask = s["mask"][token]
        at = draft.clamp(0, 64 * words - 1)
        word = mask.gather(2, (at >> 6)[:, None].expand(n, most, longest))
        seen = (word >> (at & 63)[:, None]) & 1 != 0
        seen = (draft < 0)[:, None] | (seen & (draft < 64 * words)[:, None])
    seen = seen & (position < c.length[s["rows"]][:, None])[:, None] & real[:, :, None]
    scores = scores.view(n, kv_heads, most, group, longest)
    scores.masked_fill_(~seen[:, None, :, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -torch.inf, top, 0.0))
    del scores
    total = e.sum(-1, keepdim=True)
    v = c.v[0][pages].transpose(1, 2).reshape(n, kv_heads, longest, dh).float()
    v = torch.where((position < c.length[s["rows"]][:, None])[:, None, :, None], v, 0.0)
    out = torch.matmul(e.view(n, kv_heads, most * group, longest), v)
    out = out.view(n, kv_heads, most, group, dh) / torch.where(total > 0, total, 1.0)
    out = out.transpose(1, 2).reshape(n, most, case["heads"], dh)
    return out[real].to(s["q"].dtype)


def _plain_append(s):
    c, page = s["cache"], s["case"]["page"]
    pos, rows = s["pos"], s["token_rows"]
    width = c.table.shape[1]
    where = c.table[rows, (pos // page).clamp(0, width - 1)].long()
    safe = where.clamp(0, c.refs.numel() - 1)
    fits = (pos >= 0) & (pos < c.length[rows]) & (where == safe) & (c.refs[safe] == 1)
    where, slot = where[fits], (pos % page)[fits]
    c.k[0][where, :, slot] = s["k_new"][fits]
    c.v[0][where, :, slot] = s["v_new"][fits]
    return c.k, c.v


def _release(c, pages, given):
    """One reference less of each page in `given`'s places."""
    c.refs.index_add_(0, torch.where(given, pages, 0).flatten().long(), -given.flatten().int())


def _set_free(c):
    pages = c.refs.numel()
    bits = torch.zeros(c.free.numel() * 64, dtype=torch.int64, device="cuda")
    bits[:pages] = c.refs == 0
    c.free.copy_((bits.view(-1, 64) << torch.arange(64, device="cuda")).sum(1))


def _branched(c, page, dst, src, want):
    """`branch`: entries whose row is out of range or used by another entry are refused, then the
    old pages are given back, then the lowest free pages handed out in the entries' order."""
    rows, width = c.table.shape
    n, dev = dst.numel(), dst.device
    fine = (dst >= 0) & (dst < rows) & (src >= 0) & (src < rows) & (want >= 0) & (want <= width * page)
    to, of = dst.clamp(0, rows - 1), src.clamp(0, rows - 1)
    inside = (dst >= 0) & (dst < rows)
    uses = torch.zeros(rows, dtype=torch.int64, device=dev)
    uses.index_add_(0, to, inside.long())
    uses.index_add_(0, of, ((src >= 0) & (src < rows) & (src != dst)).long())
    fine &= uses[to] == 1
    length = c.length.clamp(0, width * page)
    kept = torch.minimum(length[of], want)
    same = src == dst
    column = torch.arange(width, device=dev)
    old, sources = c.table[to].long(), c.table[of].long()
    first = torch.where(same, (want + page - 1) // page, 0)
    _release(c, old, (column >= first[:, None]) & (column < ((length[to] + page - 1) // page)[:, None])
             & fine[:, None])
    # the page in which the kept tokens end, when more will be written into it
    whole, part = kept // page, kept % page
    ends = (part > 0) & (want > kept)
    last = sources.gather(1, whole.clamp(max=width - 1)[:, None])[:, 0]
    copied = ends & (~same | (c.refs[last.clamp_min(0)] > 1))
    reused = whole + (part > 0) - copied.long()
    fresh = torch.where(fine, (want + page - 1) // page - reused, 0)
    total = fresh.cumsum(0)
    empty = c.refs == 0
    ok = fine & ((fresh == 0) | (total <= empty.sum()))
    # the free pages in order, and each row's
    rank = empty.cumsum(0) - 1
    order = torch.zeros(c.refs.numel() + 1, dtype=torch.int64, device=dev)
    order[torch.where(empty, rank, c.refs.numel())] = torch.arange(c.refs.numel(), device=dev)
    new = column >= reused[:, None]
    mine = order[((total - fresh)[:, None] + column - reused[:, None]).clamp(0, c.refs.numel())]
    held = column < ((want + page - 1) // page)[:, None]
    entry = torch.where(new, mine, sources)
    entry = torch.where(held, entry, c.table[to].long())
    shared = held & ~new & ~same[:, None] & ok[:, None]
    c.refs.index_add_(0, torch.where(shared, sources, 0).flatten(), shared.flatten().int())
    taken = held & new & ok[:, None]
    c.refs.index_add_(0, torch.where(taken, mine, 0).flatten(), taken.flatten().int())
    _release(c, last[:, None], (copied & same & ok)[:, None])
    go = copied & ok
    a, b = last[go], entry.gather(1, whole.clamp(max=width - 1)[:, None])[:, 0][go]
    some = (torch.arange(page, device=dev) < part[go][:, None])[None, :, None, :, None]
    for x in (c.k, c.v):
        x[:, b] = torch.where(some, x[:, a], x[:, b])
    c.table[to[ok]] = entry[ok].int()
    c.length[to[fine & ~ok & ~same]] = 0
    c.length[to[ok]] = want[ok]
    _set_free(c)
    return ok


def _plain_branch(s):
    ok = _branched(s["cache"], s["case"]["page"], s["dst"], s["src"], s["want"])
    return _whole(s["cache"], ok)


def _plain_accept(s):
    c, page, keep = s["cache"], s["case"]["page"], s["keep"]
    room = _branched(c, page, s["rows"], s["rows"], s["want"])
    rows, start = s["rows"], s["prefix"]
    width = c.table.shape[1]
    length = c.length[rows]
    step = torch.arange(keep.shape[1], device=keep.device)
    count = (keep >= 0).long().cumprod(1).sum(1)
    taken = step < count[:, None]
    rising = torch.ones_like(taken)
    rising[:, 1:] = keep[:, 1:] > keep[:, :-1]
    ok = (rising | ~taken).all(1) & (start >= 0) & (start <= length)
    ok &= ((start[:, None] + keep < length[:, None]) | ~taken).all(1)
    moved = taken & (keep != step)
    table = c.table[rows].long()
    to = (start[:, None] + step).clamp(0, width * page - 1)
    of = (start[:, None] + keep).clamp(0, width * page - 1)
    to_page, of_page = table.gather(1, to // page), table.gather(1, of // page)
    ok &= ((c.refs[to_page.clamp_min(0)] == 1) | ~moved).all(1)
    go = moved & ok[:, None]
    to_page, to_slot, of_page, of_slot = to_page[go], (to % page)[go], of_page[go], (of % page)[go]
    for x in (c.k, c.v):
        x[:, to_page, :, to_slot] = x[:, of_page, :, of_slot]
    column = torch.arange(width, device=keep.device)
    now = start + count
    _release(c, table, (column >= ((now + page - 1) // page)[:, None])
             & (column < ((length + page - 1) // page)[:, None]) & ok[:, None])
    c.length[rows[ok]] = now[ok]
    _set_free(c)
    return {"room": room, **_whole(c, ok)}


# ------------------------------------------------------------------------------ the work


def work(case):
    e = SIZES[case["dtype"]]
    if case["kind"] == "branch":
        token = 2 * case["layers"] * case["kv_heads"] * case["dh"] * e
        page = case["page"]
        lengths = _spread(case["parents"], (case["context"] + 1) // 2, case["context"])
        own_of = [lengths[i * case["parents"] // case["children"]] for i in range(case["children"])]
        copied = sum(x % page for x in own_of)
        # the parts copied, table entries and references of each page a child holds
        held = sum(-(-(x + case["room"]) // page) for x in own_of)
        return {"bytes": 2 * copied * token + held * 16 + case["children"] * 33, "flops": 0}
    cached, drafts = _lengths(case)
    tokens = sum(drafts)
    token = 2 * case["kv_heads"] * case["dh"] * e
    if case["kind"] == "append":
        return {"bytes": 2 * tokens * token + tokens * 16, "flops": 0}
    if case["kind"] == "accept":
        # about 3 tokens of most rows, nearly all of which move
        moved = case["seqs"] * 0.875 * min(3.0, (case["queries"] + 1) * 0.75 * 3 / case["queries"])
        held = sum(-(-(a + b) // case["page"]) for a, b in zip(cached, drafts))
        return {"bytes": 2 * moved * token * case["layers"] + held * 8
                + case["seqs"] * (case["queries"] * 8 + 34), "flops": 0}
    held = sum(cached) + tokens
    words = -(-case["queries"] // 64) if case["tree"] else 0
    moved = 2 * tokens * case["heads"] * case["dh"] * e + held * token
    moved += 8 * words * tokens + 4 * held / case["page"]
    # drafts see about half of the drafts before them without a tree, a few with one
    mean = sum(cached) / case["seqs"] + (4 if case["tree"] else case["queries"] / 2)
    return {"bytes": moved, "flops": 4 * case["heads"] * case["dh"] * tokens * mean}


# ------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(state)
    if case["kind"] == "append":
        return _exact_append(state)
    if case["kind"] == "branch":
        rows = _Rows(state["cache"])
        ok = rows.branch(state["dst"].tolist(), state["src"].tolist(), state["want"].tolist())
        return rows.whole(ok)
    return _exact_accept(state)


def _exact_attend(s):
    """Sequence by sequence in 64 bits."""
    case, c = s["case"], s["cache"]
    group = case["heads"] // case["kv_heads"]
    rows, prefix, offsets = s["rows"].tolist(), s["prefix"].tolist(), s["offsets"].tolist()
    length, table = c.length.tolist(), c.table.cpu()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, row in enumerate(rows):
        n = length[row]
        held = table[row, :-(-n // case["page"])].long().cuda()
        first, end = offsets[i], offsets[i + 1]
        t = end - first
        allowed = torch.zeros(t, n, dtype=torch.bool, device="cuda")
        allowed[:, :prefix[i]] = True
        d = n - prefix[i]
        if s["mask"] is None:
            allowed[:, prefix[i]:] = torch.ones(t, d, dtype=torch.bool, device="cuda").tril()
        else:
            b = torch.arange(d, device="cuda")
            allowed[:, prefix[i]:] = (s["mask"][first:end][:, b // 64] >> (b % 64)) % 2 == 1
        k, v = (x[0, held].transpose(0, 1).reshape(case["kv_heads"], -1, case["dh"])[:, :n].double()
                for x in (c.k, c.v))
        q = s["q"][first:end].double().view(t, -1, group, case["dh"]).permute(1, 2, 0, 3)
        a = (q / case["dh"] ** 0.5).reshape(case["kv_heads"], group * t, case["dh"]) @ k.mT
        a = a.view(-1, group, t, n).masked_fill(~allowed, -torch.inf).softmax(3)
        a = (a.view(-1, group * t, n) @ v).view(-1, group, t, case["dh"])
        out[first:end] = a.permute(2, 0, 1, 3).reshape(t, -1, case["dh"])
    return out


def _exact_append(s):
    c, page = s["cache"], s["case"]["page"]
    table = c.table.tolist()
    where = [table[r][p // page] for r, p in zip(s["token_rows"].tolist(), s["pos"].tolist())]
    where, slot = torch.tensor(where, device="cuda"), s["pos"] % page
    k, v = c.k.double(), c.v.double()
    k[0].transpose(1, 2)[where, slot] = s["k_new"].double()
    v[0].transpose(1, 2)[where, slot] = s["v_new"].double()
    return k, v


class _Rows:
    """The cache's rows as lists, worked on one entry at a time."""

    def __init__(self, c):
        self.c, self.page = c, c.k.shape[3]
        self.rows, self.width = c.table.shape
        self.table, self.length, self.refs = c.table.tolist(), c.length.tolist(), c.refs.tolist()
        self.k, self.v = c.k.double(), c.v.double()

    def held(self, row):
        return -(-self.length[row] // self.page)

    def branch(self, dst, src, want):
        used = {}
        for d, s in zip(dst, src):
            for r in {d, s}:
                used[r] = used.get(r, 0) + 1
        ok = [used[d] == 1 for d in dst]
        for d, s, n, fine in zip(dst, src, want, ok):
            first = -(-n // self.page) if d == s else 0
            for j in range(first, self.held(d) if fine else 0):
                self.refs[self.table[d][j]] -= 1
        after = list(self.refs)
        empty = iter([p for p, r in enumerate(after) if r == 0])
        pairs = []
        for d, s, n, fine in zip(dst, src, want, ok):
            if not fine:
                continue
            kept = min(self.length[s], n)
            pages = self.table[s][:-(-kept // self.page)]
            if d != s:
                for p in pages:
                    self.refs[p] += 1
            if kept < n and kept % self.page and (d != s or after[pages[-1]] > 1):
                self.refs[pages[-1]] -= 1
                p = next(empty)
                pairs.append((pages[-1], p, kept % self.page))
                self.refs[p] += 1
                pages[-1] = p
            for _ in range(-(-n // self.page) - len(pages)):
                p = next(empty)
                self.refs[p] += 1
                pages.append(p)
            self.table[d][:len(pages)] = pages
            self.length[d] = n
        if pairs:
            a, b, part = torch.tensor(pairs, device="cuda").T
            for slot in range(self.page):
                go = part > slot
                for x in (self.k, self.v):
                    x[:, b[go], :, slot] = x[:, a[go], :, slot]
        return ok

    def whole(self, ok):
        def on(x, dtype):
            return torch.tensor(x, dtype=dtype, device="cuda")

        free = [0] * (-(-len(self.refs) // 64))
        for p, r in enumerate(self.refs):
            free[p // 64] |= (r == 0) << (p % 64)
        free = [f - (1 << 64) if f >> 63 else f for f in free]
        return {"ok": on(ok, torch.bool), "k": self.k, "v": self.v,
                "table": on(self.table, torch.int32), "length": on(self.length, torch.int64),
                "refs": on(self.refs, torch.int32), "free": on(free, torch.int64)}


def _exact_accept(s):
    rows = _Rows(s["cache"])
    names = s["rows"].tolist()
    room = rows.branch(names, names, s["want"].tolist())
    page, a, b = rows.page, [], []
    for r, start, keep in zip(names, s["prefix"].tolist(), s["keep"].tolist()):
        path = [x for x in keep if x >= 0]
        for j, x in enumerate(path):
            a.append(rows.table[r][(start + x) // page] * page + (start + x) % page)
            b.append(rows.table[r][(start + j) // page] * page + (start + j) % page)
        now = start + len(path)
        for j in range(-(-now // page), rows.held(r)):
            rows.refs[rows.table[r][j]] -= 1
        rows.length[r] = now
    if a:
        a, b = torch.tensor(a, device="cuda"), torch.tensor(b, device="cuda")
        for name in ("k", "v"):
            x = getattr(rows, name).transpose(2, 3).flatten(1, 2)
            x[:, b] = x[:, a]
            shape = s["cache"].k.shape
            x = x.view(shape[0], shape[1], page, shape[2], shape[4])
            setattr(rows, name, x.transpose(2, 3).contiguous())
    return {"room": torch.tensor(room, device="cuda"), **rows.whole([True] * len(names))}
