"""Attention and the key/value cache of a served model, as a program calls them.

Between the projections of a decoder layer such a program attends over whole
prompts, then over a paged cache for the tokens a draft proposed, and keeps the
cache's pages: it forks sequences, keeps the accepted path of a verified tree
and moves the pages in use to the front. A case is one such call; ``op`` says
which:

  prompt   causal attention of packed prompts, each with some rows of context
  tree     attention of drafted tokens (a tree a sequence) over a paged cache
  fork     sequences branch off others (full pages shared, the last one copied),
           then get pages for their next tokens
  commit   the accepted path of every verified tree becomes part of the cache
  compact  the pages in use move to the front of the pool

Lengths follow from the case (``mix`` seeds them); values follow from the seed.
``heads``/``kv_heads``/``dim`` 40/8/128 are those of a 14B-class decoder block
(projections of 5120 and 1024 columns).
"""
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCORES = 1 << 30  # scores of one block of query rows that the plain form holds


def listed():
    return [
        # One short prompt of a small model: the launch and its start-up.
        dict(name="prompt_short", op="prompt", seqs=1, low=77, high=77, past=0, heads=16, kv_heads=16, dim=64, dtype="fp16", mix=1),
        # A batch of ragged prompts, some continuing a context, as a server packs them.
        dict(name="prompt_ragged", op="prompt", seqs=12, low=65, high=1999, past=700, heads=40, kv_heads=8, dim=128, dtype="bf16", mix=2),
        # One long document.
        dict(name="prompt_long", op="prompt", seqs=1, low=16384, high=16384, past=0, heads=40, kv_heads=8, dim=128, dtype="bf16", mix=3),
        # Plain token generation of one sequence: latency.
        dict(name="tree_single", op="tree", seqs=1, low=501, high=501, drafts_low=1, drafts=1, heads=40, kv_heads=8, dim=128, page=16, dtype="bf16", mix=4),
        # Verification of draft trees of different sizes for a batch.
        dict(name="tree_verify", op="tree", seqs=8, low=700, high=6000, drafts_low=1, drafts=33, heads=40, kv_heads=8, dim=128, page=64, dtype="bf16", mix=5),
        # The same over long contexts: the cache's bytes decide.
        dict(name="tree_long", op="tree", seqs=16, low=9000, high=65000, drafts_low=4, drafts=16, heads=40, kv_heads=8, dim=128, page=128, dtype="bf16", mix=6),
        # Four branches of one sequence in a small cache.
        dict(name="fork_small", op="fork", seqs=1, branches=4, low=300, high=300, layers=4, kv_heads=8, dim=128, page=16, spare=5, dtype="bf16", mix=7),
        # Many branches of a batch's sequences, eight layers' pages.
        dict(name="fork_wide", op="fork", seqs=8, branches=12, low=400, high=4000, layers=8, kv_heads=8, dim=128, page=64, spare=17, dtype="bf16", mix=8),
        # One sequence's accepted tokens.
        dict(name="commit_small", op="commit", seqs=1, drafts=8, accept=4, low=100, high=100, layers=4, kv_heads=8, dim=128, page=16, dtype="fp16", mix=9),
        # A batch's accepted tokens in all 40 layers.
        dict(name="commit_wide", op="commit", seqs=64, drafts=32, accept=12, low=33, high=190, layers=40, kv_heads=8, dim=128, page=64, dtype="bf16", mix=10),
        # A small pool, half in use.
        dict(name="compact_small", op="compact", pages=64, used=32, layers=2, kv_heads=4, dim=64, page=16, dtype="fp16", mix=11),
        # A large pool after most of its sequences ended.
        dict(name="compact_large", op="compact", pages=1200, used=600, layers=8, kv_heads=8, dim=128, page=64, dtype="bf16", mix=12),
    ]


HEADS = ((40, 8, 128), (40, 8, 128), (32, 8, 128), (16, 16, 64), (12, 4, 64), (8, 1, 128), (16, 8, 96), (8, 4, 256))


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    """One more call: 1 to 16384 rows a prompt, contexts of 16 to 65000, trees
    of 1 to 64 tokens, pools of 24 to 1200 pages; shrunk until it costs no more
    than the largest listed call of its kind."""
    op = rng.choice(("prompt", "prompt", "prompt", "tree", "tree", "tree", "fork", "commit", "compact"))
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(("bf16", "bf16", "fp16")), "mix": rng.randrange(1 << 20)}
    most = {"prompt": 2.7e12, "tree": 2.0e9, "fork": 2.0e9, "commit": 2.0e9, "compact": 2.0e9}[op]
    if op == "prompt":
        high = _log_int(rng, 1, 16384)
        case |= {"seqs": _log_int(rng, 1, 24), "low": max(1, high // rng.choice((1, 3, 16))), "high": high,
                 "past": rng.choice((0, 0, rng.randint(1, 2000))), "heads": heads}
    elif op == "tree":
        high = _log_int(rng, 16, 65000)
        drafts = rng.choice((1, 1, _log_int(rng, 2, 64)))
        case |= {"seqs": _log_int(rng, 1, 64), "low": max(1, high // rng.choice((1, 4, 16))), "high": high, "heads": heads,
                 "drafts_low": rng.randint(1, drafts), "drafts": drafts, "page": rng.choice((16, 16, 32, 64, 128))}
    elif op == "fork":
        high = _log_int(rng, 16, 4000)
        case |= {"seqs": rng.randint(1, 8), "branches": rng.randint(1, 12), "low": max(1, high // 4), "high": high,
                 "layers": rng.randint(1, 8), "page": rng.choice((16, 32, 64)), "spare": rng.randint(1, 40)}
    elif op == "commit":
        drafts = rng.randint(2, 48)
        case |= {"seqs": _log_int(rng, 1, 64), "drafts": drafts, "accept": rng.randint(1, min(12, drafts)), "low": 1,
                 "high": rng.randint(2, 190), "layers": rng.randint(1, 40), "page": rng.choice((16, 32, 64))}
    else:
        pages = _log_int(rng, 24, 1200)
        case |= {"pages": pages, "used": rng.randint(pages // 4, 3 * pages // 4), "layers": rng.randint(1, 8), "page": rng.choice((16, 32, 64))}
    while _cost(case) > most:
        if op == "compact":
            case["pages"], case["used"] = max(24, case["pages"] // 2), max(6, case["used"] // 2)
        elif op in ("fork", "commit"):
            case["layers"] = max(1, case["layers"] // 2)
        elif case["seqs"] > 1:
            case["seqs"] = max(1, case["seqs"] * 2 // 3)
        else:
            case["high"] = max(1, case["high"] * 2 // 3)
            case["low"] = min(case["low"], case["high"])
    return case


def _cost(case):
    if case["op"] == "prompt":  # the rows are padded to the longest in the plain form
        pairs = case["seqs"] * case["high"] * (case["high"] / 2 + case["past"])
        return 4.0 * pairs * case["heads"] * case["dim"]
    return 2.0 * _cache_elements(case)


def _cache_elements(case):
    """Elements of the keys and values that a state of a cache call holds."""
    row = 2 * case["kv_heads"] * case["dim"]
    if case["op"] == "tree":
        return row * case["seqs"] * case["high"]
    return row * case["layers"] * case["page"] * _n_pages(case)


def _pages(tokens, page):
    return -(-tokens // page)


def _n_pages(case):
    if case["op"] == "compact":
        return case["pages"]
    held = sum(_pages(n, case["page"]) for n in _lengths(case, case["seqs"], case["low"], case["high"]))
    if case["op"] == "fork":
        held += 2 * case["seqs"] * case["branches"] * (1 + _pages(case["spare"], case["page"]))
    else:
        held += case["seqs"] * _pages(case["drafts"] + case["page"], case["page"])
    return held + 8


def _lengths(case, n, low, high, salt=0):
    """n lengths from low to high, spread over their logarithm; the longest is high."""
    rng = random.Random(case["mix"] * 16 + salt)
    got = [_log_int(rng, low, high) for _ in range(n)]
    got[rng.randrange(n)] = high
    return got


def _prompt_lengths(case):
    rows = _lengths(case, case["seqs"], case["low"], case["high"])
    rng = random.Random(case["mix"] + 1)
    return rows, [n + rng.randint(0, case["past"]) for n in rows]


def _tree_sizes(case):
    return (_lengths(case, case["seqs"], case["low"], case["high"]),
            _lengths(case, case["seqs"], case["drafts_low"], case["drafts"], salt=1))


# --------------------------------------------------------------------------
# Inputs.
# --------------------------------------------------------------------------

def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype).mul_(scale)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _tree_masks(rng, sizes):
    """Ancestor bits of each drafted token, 64 to a word: a root, then children of earlier tokens."""
    masks = []
    for n in sizes:
        bits = []
        for t in range(n):
            parent = rng.randrange(max(0, t - 6), t) if t else -1
            bits.append((bits[parent] if t else 0) | 1 << t)
        masks += bits
    words = _pages(max(sizes), 64)
    return [[((m >> 64 * w & (1 << 64) - 1) ^ 1 << 63) - (1 << 63) for w in range(words)] for m in masks]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    op, dtype, kv, dim = case["op"], TYPES[case["dtype"]], case["kv_heads"], case["dim"]
    state = {"case": case}
    if op == "prompt":
        rows, keys = _prompt_lengths(case)
        # Queries and keys of the size that normed heads have: scores of a few units.
        state |= {"rows": rows, "keys": keys, "q": _randn(g, sum(rows), case["heads"], dim, dtype=dtype, scale=2.0),
                  "k": _randn(g, sum(keys), kv, dim, dtype=dtype), "v": _randn(g, sum(keys), kv, dim, dtype=dtype),
                  "q_offsets": _ints(_offsets(rows)), "k_offsets": _ints(_offsets(keys))}
        return state
    if op == "compact":
        n_pages, used, page = case["pages"], case["used"], case["page"]
        order = list(range(n_pages))
        rng.shuffle(order)
        live = order[:used]
        seqs = max(1, used // 12)
        held = [used // seqs + (b < used % seqs) for b in range(seqs)]
        at = _offsets(held)
        rows = [live[at[b]:at[b + 1]] for b in range(seqs)]
        refs = [0] * n_pages
        for p in live:
            refs[p] = 1
        # A branch of the first sequence shares all its pages.
        rows.append(rows[0])
        held.append(held[0])
        for p in rows[0]:
            refs[p] += 1
        width = max(held) + 1
        lengths = [h * page - rng.randrange(page) for h in held]
    else:
        page = case["page"]
        lengths = _lengths(case, case["seqs"], case["low"], case["high"])
        more = [0] * len(lengths)
        if op == "tree":
            more = _tree_sizes(case)[1]
        elif op == "commit":
            more = [case["drafts"]] * len(lengths)
        held = [_pages(n + m, page) for n, m in zip(lengths, more)]
        n_pages = sum(held) + 8 if op == "tree" else _n_pages(case)
        order = list(range(n_pages))
        rng.shuffle(order)
        at = _offsets(held)
        rows = [order[at[b]:at[b + 1]] for b in range(len(held))]
        refs = [0] * n_pages
        for p in order[:at[-1]]:
            refs[p] = 1
        width = max(held)
        if op == "fork":
            n = case["seqs"] * case["branches"]
            rows, held, lengths = rows + [[]] * n, held + [0] * n, lengths + [0] * n
            width += 1 + _pages(case["spare"], page)
            state |= {"src": _ints([b % case["seqs"] for b in range(n)]), "dst": _ints([case["seqs"] + b for b in range(n)]),
                      "tokens": _ints([rng.randint(1, case["spare"]) for _ in range(n)])}
    state |= {"page_table": _ints([r + [-1] * (width - len(r)) for r in rows]), "lengths": _ints(lengths), "held": _ints(held),
              "refs": _ints(refs), "status": _ints([0])}
    if op == "tree":
        contexts, sizes = _tree_sizes(case)
        state |= {"k_pages": _randn(g, n_pages, kv, page, dim, dtype=dtype), "v_pages": _randn(g, n_pages, kv, page, dim, dtype=dtype),
                  "q": _randn(g, sum(sizes), case["heads"], dim, dtype=dtype, scale=2.0), "seqs": _ints(list(range(case["seqs"]))),
                  "offsets": _ints(_offsets(sizes)), "masks": _ints(_tree_masks(rng, sizes), torch.int64),
                  "drafts": max(sizes), "context": max(contexts)}
        return state
    state["pool"] = _randn(g, case["layers"], 2, n_pages, kv, page, dim, dtype=dtype)
    if op == "commit":
        counts = [rng.randint(0, case["accept"]) for _ in lengths]
        counts[0] = case["accept"]
        paths = [sorted(rng.sample(range(case["drafts"]), case["accept"])) for _ in lengths]
        state |= {"seqs": _ints(list(range(case["seqs"]))), "accepted": _ints(paths), "counts": _ints(counts),
                  "new_lengths": torch.zeros_like(state["lengths"])}
    elif op == "compact":
        state |= {"new_table": torch.empty_like(state["page_table"]), "new_refs": torch.empty_like(state["refs"])}
    return state


# --------------------------------------------------------------------------
# The plain forms.
# --------------------------------------------------------------------------

def _softmax_product(scores, visible, values):
    """softmax over the visible scores times the values; zeros where nothing is visible."""
    scores = scores.masked_fill_(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p.flatten(2, 3), values).view(*p.shape[:-1], values.shape[-1]).div_(total.clamp_min_(1e-30))


def _plain_prompt(s):
    q, k, v, q_at, k_at = s["q"], s["k"], s["v"], s["q_offsets"].long(), s["k_offsets"].long()
    n, heads, dim = q.shape
    kv = k.shape[1]
    seqs, long_q, long_k = len(s["rows"]), max(s["rows"]), max(s["keys"])
    rows, keys = q_at.diff()[:, None], k_at.diff()[:, None]
    i, j = torch.arange(long_q, device=DEVICE), torch.arange(long_k, device=DEVICE)
    q_of, k_of = (q_at[:-1, None] + i).clamp_max(n - 1), (k_at[:-1, None] + j).clamp_max(k.shape[0] - 1)
    kt = k[k_of].permute(0, 2, 3, 1).float().contiguous()  # [seqs, kv, dim, keys]
    vt = v[k_of].permute(0, 2, 1, 3).float().contiguous()  # [seqs, kv, keys, dim]
    step = max(1, SCORES // (seqs * heads * long_k))
    out = []
    # Blocks of query rows, so that a block's scores fit the memory; each sees the keys up to its last row's.
    for a in range(0, long_q, step):
        b = min(long_q, a + step)
        most = max(1, max(min(kn, b + kn - qn) for qn, kn in zip(s["rows"], s["keys"])))
        block = q[q_of[:, a:b]].view(seqs, b - a, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).float()
        scores = torch.matmul(block.flatten(2, 3), kt[..., :most].contiguous()).mul_(dim ** -0.5).view(seqs, kv, heads // kv, b - a, most)
        visible = (j[:most] <= (i[a:b] + keys - rows)[..., None]) & (j[:most] < keys[..., None])
        o = _softmax_product(scores, visible[:, None, None], vt[:, :, :most].contiguous())
        out.append(o.permute(0, 3, 1, 2, 4).reshape(seqs, b - a, heads, dim))
    at = torch.arange(n, device=DEVICE)
    seq = torch.bucketize(at, q_at[1:], right=True)
    return torch.cat(out, 1).flatten(0, 1)[seq * long_q + at - q_at[seq]].to(q.dtype)


def _plain_tree(s):
    q, at, seqs, lengths = s["q"], s["offsets"].long(), s["seqs"].long(), s["lengths"].long()
    n, heads, dim = q.shape
    kv, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    table = s["page_table"][seqs].clamp_min(0).long()
    count, drafts = len(seqs), s["drafts"]
    long_k = table.shape[1] * page
    kt = s["k_pages"][table].permute(0, 2, 4, 1, 3).reshape(count, kv, dim, long_k).float()
    vt = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(count, kv, long_k, dim).float()
    t = torch.arange(drafts, device=DEVICE)
    q_of = (at[:-1, None] + t).clamp_max(n - 1)
    block = q[q_of].view(count, drafts, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).float()
    scores = torch.matmul(block.flatten(2, 3), kt).mul_(dim ** -0.5).view(count, kv, heads // kv, drafts, long_k)
    # Key j: context below the length, then the drafted tokens by their bits.
    j = torch.arange(long_k, device=DEVICE) - lengths[seqs][:, None]
    bits = s["masks"][q_of]
    word = (j.clamp(0, drafts - 1) >> 6)[:, None].expand(-1, drafts, -1)
    drafted = (torch.gather(bits, 2, word) >> (j & 63)[:, None]) & 1
    visible = (j[:, None] < 0) | ((drafted == 1) & (j < at.diff()[:, None])[:, None])
    o = _softmax_product(scores, visible[:, None, None], vt)
    row = torch.arange(n, device=DEVICE)
    seq = torch.bucketize(row, at[1:], right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(count * drafts, heads, dim)[seq * drafts + row - at[seq]].to(q.dtype)


def _lowest_free(refs, most):
    """The `most` free pages of lowest index."""
    free = refs == 0
    rank = free.long().cumsum(0) - 1
    pick = torch.zeros(most + 1, dtype=torch.long, device=DEVICE)
    pick.scatter_(0, torch.where(free & (rank < most), rank, most), torch.arange(len(refs), device=DEVICE))
    return pick[:most]


def _plain_fork(s):
    table, lengths, held, refs, pool = s["page_table"], s["lengths"], s["held"], s["refs"], s["pool"]
    src, dst, page = s["src"].long(), s["dst"].long(), pool.shape[4]
    n, column = len(src), torch.arange(table.shape[1], device=DEVICE)
    old, new, size = table[dst].long(), table[src].long(), lengths[src].long()
    full, tail = size // page, size % page
    has = (tail > 0).long()
    got = _lowest_free(refs, n)[(has.cumsum(0) - 1).clamp_min(0)]
    last = new.gather(1, (full - 1 + has).clamp_min(0)[:, None])[:, 0].clamp_min(0)
    shared, gone = column < full[:, None], column < held[dst][:, None]
    refs.index_add_(0, new.clamp_min(0).flatten(), shared.flatten().int())
    refs.index_add_(0, old.clamp_min(0).flatten(), -gone.flatten().int())
    refs.index_add_(0, got, has.int())
    table[dst] = torch.where(shared, new, torch.where((column == full[:, None]) & (tail > 0)[:, None], got[:, None], -1)).int()
    lengths[dst], held[dst] = size.int(), (full + has).int()
    keep = torch.arange(page, device=DEVICE) < tail[:, None]
    # A sequence with nothing to copy writes the last page of its source back to itself.
    to = torch.where(has == 1, got, last)
    pool[:, :, to] = torch.where(keep[None, None, :, None, :, None], pool[:, :, last], pool[:, :, to])
    # Pages for the next tokens.
    need = ((size + s["tokens"] + page - 1) // page - held[dst]).clamp_min(0)
    start = need.cumsum(0) - need
    most = n * _pages(s["case"]["spare"], page)
    rank = start[:, None] + column - held[dst][:, None]
    fill = (column >= held[dst][:, None]) & (column < (held[dst] + need)[:, None])
    pages = _lowest_free(refs, most)[rank.clamp(0, most - 1)]
    refs.index_add_(0, pages.flatten(), fill.flatten().int())
    table[dst] = torch.where(fill, pages, table[dst].long()).int()
    held[dst] += need.int()
    return [table, lengths, held, refs, pool, s["status"]]


def _plain_commit(s):
    pool, table, lengths, seqs = s["pool"], s["page_table"].long(), s["lengths"].long(), s["seqs"].long()
    page, counts, paths = pool.shape[4], s["counts"].long(), s["accepted"].long()
    i = torch.minimum(torch.arange(paths.shape[1], device=DEVICE), (counts - 1).clamp_min(0)[:, None])
    a = lengths[seqs][:, None] + torch.where(counts[:, None] > 0, paths.gather(1, i), 0)
    b = lengths[seqs][:, None] + i
    rows = table[seqs]
    pool[:, :, rows.gather(1, b // page), :, b % page] = pool[:, :, rows.gather(1, a // page), :, a % page].clone()
    s["new_lengths"][seqs] = (lengths[seqs] + counts).int()
    return [pool, s["new_lengths"]]


def _plain_compact(s):
    pool, table, refs = s["pool"], s["page_table"].long(), s["refs"]
    used, at = refs > 0, torch.arange(len(refs), device=DEVICE)
    n = used.sum()
    high, low = torch.nonzero(used & (at >= n))[:, 0], torch.nonzero(~used & (at < n))[:, 0]
    pool[:, :, low] = pool[:, :, high]
    to = at.clone()
    to[high] = low
    s["new_table"].copy_(torch.where(table >= 0, to[table.clamp_min(0)], -1))
    s["new_refs"].copy_(refs)
    s["new_refs"][low] = refs[high]
    s["new_refs"][high] = 0
    return [pool, s["new_table"], s["new_refs"], n.to(torch.int32)]


PLAIN = {"prompt": _plain_prompt, "tree": _plain_tree, "fork": _plain_fork, "commit": _plain_commit, "compact": _plain_compact}


# --------------------------------------------------------------------------
# One pass.
# --------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if not own:
        return PLAIN[op](state)
    from afterimage_amd.runtime.attention import prompt_attention, tree_attention
    from afterimage_amd.runtime.kv_cache import PagedKVCache

    if op == "prompt":
        return prompt_attention(state["q"], state["k"], state["v"], state["q_offsets"], state["k_offsets"])
    if op == "tree":
        return tree_attention(state["q"], state["k_pages"], state["v_pages"], state["page_table"], state["lengths"], state["seqs"],
                              state["offsets"], state["masks"], max_drafts=state["drafts"], max_context=state["context"])
    cache = state.get("cache")  # the handle that a program keeps: these same tensors
    if cache is None:
        cache = state["cache"] = PagedKVCache(state["pool"], state["page_table"], state["lengths"], state["held"], state["refs"], state["status"])
    if op == "fork":
        cache.fork(state["src"], state["dst"])
        cache.reserve(state["dst"], state["tokens"])
        return [cache.page_table, cache.lengths, cache.held, cache.refs, cache.pool, cache.status]
    if op == "commit":
        return [cache.pool, cache.commit(state["seqs"], state["accepted"], state["counts"], new_lengths=state["new_lengths"])]
    used = cache.compact(new_table=state["new_table"], new_refs=state["new_refs"])
    return [cache.pool, state["new_table"], state["new_refs"], used]


def work(case):
    op, kv, dim = case["op"], case["kv_heads"], case["dim"]
    row = 2 * 2 * kv * dim  # bytes of a token's key and value in one layer
    if op == "prompt":
        rows, keys = _prompt_lengths(case)
        pairs = sum(q * k - q * (q - 1) / 2 for q, k in zip(rows, keys))
        return {"bytes": 4.0 * sum(rows) * case["heads"] * dim + row * sum(keys), "flops": 4.0 * pairs * case["heads"] * dim}
    if op == "tree":
        contexts, sizes = _tree_sizes(case)
        pairs = sum(n * (c + n / 2) for c, n in zip(contexts, sizes))
        table = sum(4 * _pages(c + n, case["page"]) for c, n in zip(contexts, sizes))
        return {"bytes": 4.0 * sum(sizes) * case["heads"] * dim + row * (sum(contexts) + sum(sizes)) + table, "flops": 4.0 * pairs * case["heads"] * dim}
    if op == "fork":
        lengths = _lengths(case, case["seqs"], case["low"], case["high"])
        tails = sum(n % case["page"] for n in lengths) * case["branches"]
        rows = sum(_pages(n, case["page"]) for n in lengths) * case["branches"]
        return {"bytes": 2.0 * row * case["layers"] * tails + 4 * (3 * rows + 2 * _n_pages(case)), "flops": 0.0}
    if op == "commit":
        return {"bytes": 2.0 * row * case["layers"] * case["seqs"] * (case["accept"] / 2) + 8 * case["seqs"], "flops": 0.0}
    moved = case["used"] * (1 - case["used"] / case["pages"])
    return {"bytes": 2.0 * row * case["layers"] * case["page"] * moved + 16 * case["pages"], "flops": 0.0}


# --------------------------------------------------------------------------
# The definition, in 64 bits.
# --------------------------------------------------------------------------

def _attend_exact(q, k, v, visible):
    """One sequence, one key/value head: rows [n, group, dim] over keys [m, dim]; visible [n, m]."""
    weight = torch.exp(torch.einsum("ngd,md->ngm", q, k).mul_(q.shape[-1] ** -0.5)) * visible[:, None]
    return torch.einsum("ngm,md->ngd", weight, v) / weight.sum(-1, keepdim=True).clamp_min(1e-300)


def exact(case, seed):
    """The attention's rows, one sequence, head and block of rows at a time;
    None for the calls that only move rows and count pages."""
    if case["op"] not in ("prompt", "tree"):
        return None
    s = prepare(case, seed)
    q, group = s["q"].double(), case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    if case["op"] == "prompt":
        spans = list(zip(_offsets(s["rows"]), _offsets(s["keys"]), s["rows"], s["keys"]))
    else:
        contexts, sizes = _tree_sizes(case)
        spans = list(zip(_offsets(sizes), contexts, sizes, [c + n for c, n in zip(contexts, sizes)]))
    for b, (row, at, n, m) in enumerate(spans):
        j = torch.arange(m, device=DEVICE)
        if case["op"] == "prompt":
            k, v = s["k"][at:at + m], s["v"][at:at + m]
        else:
            page = case["page"]
            p = s["page_table"][b, :_pages(m, page)].long()
            k, v = (s[x][p].transpose(1, 2).flatten(0, 1)[:m] for x in ("k_pages", "v_pages"))
        step = max(1, (1 << 27) // (m * group))
        for h in range(case["kv_heads"]):
            kh, vh = k[:, h].double(), v[:, h].double()
            for a in range(0, n, step):
                i = torch.arange(a, min(n, a + step), device=DEVICE)
                if case["op"] == "prompt":
                    visible = j <= i[:, None] + (m - n)
                else:
                    d = (j - at).clamp_min(0)
                    bit = s["masks"][row + i][:, d >> 6] >> (d & 63) & 1
                    visible = (j < at) | (bit == 1)
                heads = slice(h * group, (h + 1) * group)
                out[row + a:row + a + len(i), heads] = _attend_exact(q[row + a:row + a + len(i), heads], kh, vh, visible.double())
    return out
