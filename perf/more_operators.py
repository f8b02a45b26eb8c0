"""A served token's way through an 8-bit cache to its successor, as a program calls it.

Each layer of such a program rotates its queries and keys by their positions,
puts keys and values into a paged cache (in 8 bits, with a scale for each block
of 16 positions and head, or in 16) and attends over it; the last layer's logits
become a token. A case is one such call; ``op`` says which:

  step    drafted tokens (a tree a sequence, or one token) into an 8-bit cache,
          rotated on the way, then their attention over it; the cache, as the
          values of its 8 bits and their scales, comes back too
  piece   the next rows of prompts into a cache, rotated on the way, then the
          whole context back as packed 16-bit rows, for the prompts' attention
  sample  tokens from logits: temperature, top-k, top-p and min-p, with given
          random numbers

Lengths follow from the case (``mix`` seeds them); values follow from the seed.
``heads``/``kv_heads``/``dim`` 40/8/128 are those of a 14B-class decoder block
(projections of 5120 and 1024 columns), 151936 logits those of its head.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 16       # positions that share a scale
MOST = 448.0     # the largest value of 8 bits (4 of exponent, 3 of mantissa)
LOW, HIGH = -100, 119  # exponents of scales


def listed():
    return [
        # Plain token generation of one sequence: latency.
        dict(name="step_single", op="step", seqs=1, low=501, high=501, drafts_low=1, drafts=1, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=16, dtype="bf16", mix=1),
        # A batch that generates a token each over chats of different lengths.
        dict(name="step_batch", op="step", seqs=64, low=1900, high=8100, drafts_low=1, drafts=1, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=64, dtype="bf16", mix=2),
        # Verification of draft trees of different sizes; half of each head is rotated, in neighbouring pairs.
        dict(name="step_verify", op="step", seqs=8, low=700, high=6000, drafts_low=1, drafts=33, heads=32, kv_heads=8, dim=128, rot=64, paired=True, page=32, dtype="fp16", mix=3),
        # Trees over long contexts: the cache's bytes decide.
        dict(name="step_long", op="step", seqs=16, low=9000, high=65000, drafts_low=4, drafts=16, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=128, dtype="bf16", mix=4),
        # One short prompt of a small model in a 16-bit cache.
        dict(name="piece_short", op="piece", seqs=1, low=77, high=77, past=0, heads=16, kv_heads=16, dim=64, rot=64, paired=False, page=16, cache="fp16", dtype="fp16", mix=5),
        # A batch of prompts' pieces of different lengths over different contexts, 8-bit cache.
        dict(name="piece_ragged", op="piece", seqs=12, low=65, high=1999, past=2500, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=64, cache="fp8", dtype="bf16", mix=6),
        # The next piece of one long document.
        dict(name="piece_long", op="piece", seqs=1, low=8192, high=8192, past=24000, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=128, cache="fp8", dtype="bf16", mix=7),
        # One long document at once, 16-bit cache.
        dict(name="piece_whole", op="piece", seqs=1, low=16384, high=16384, past=0, heads=40, kv_heads=8, dim=128, rot=128, paired=False, page=64, cache="bf16", dtype="bf16", mix=8),
        # One sequence's next token: latency.
        dict(name="sample_one", op="sample", rows=1, vocab=151936, dtype="bf16", temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, spread=2.5, mixed=False),
        # The rows of a few draft trees; fp32 logits of an odd vocabulary.
        dict(name="sample_verify", op="sample", rows=37, vocab=50001, dtype="fp32", temperature=0.6, top_k=0, top_p=1.0, min_p=0.05, spread=2.0, mixed=False),
        # A batch where every request brings its own settings (a few of them greedy).
        dict(name="sample_batch", op="sample", rows=64, vocab=151936, dtype="bf16", temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, spread=2.5, mixed=True),
        # A large batch from the distribution as it is.
        dict(name="sample_large", op="sample", rows=256, vocab=151936, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, spread=3.0, mixed=False),
    ]


HEADS = ((40, 8, 128), (40, 8, 128), (32, 8, 128), (16, 16, 64), (12, 4, 64), (8, 1, 128), (16, 8, 96), (8, 4, 256))


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    """One more call: contexts of 16 to 65000, trees of 1 to 64 tokens, pieces of
    1 to 16384 rows, 1 to 256 rows of 500 to 262144 logits; shrunk until it
    costs no more than the largest listed call of its kind."""
    op = rng.choice(("step", "step", "piece", "piece", "sample", "sample"))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    if op == "sample":
        case |= {"rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 500, 262144), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                 "temperature": rng.choice((1.0, 0.0, round(rng.uniform(0.3, 1.5), 3))), "top_k": rng.choice((0, 0, 1, _log_int(rng, 2, 2000))),
                 "top_p": rng.choice((1.0, 1.0, round(rng.uniform(0.05, 0.99), 3))), "min_p": rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 4))),
                 "spread": round(rng.uniform(1.5, 4.0), 2), "mixed": rng.random() < 0.4}
        while case["rows"] * case["vocab"] > 256 * 151936:
            case["rows"] = case["rows"] * 2 // 3
        return case
    heads, kv_heads, dim = rng.choice(HEADS)
    case |= {"heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rng.choice((dim, dim, dim // 2)), "paired": rng.random() < 0.3,
             "page": rng.choice((16, 16, 32, 64, 128)), "mix": rng.randrange(1 << 20)}
    if op == "step":
        high = _log_int(rng, 16, 65000)
        drafts = rng.choice((1, 1, _log_int(rng, 2, 64)))
        case |= {"seqs": _log_int(rng, 1, 64), "low": max(1, high // rng.choice((1, 4, 16))), "high": high,
                 "drafts_low": rng.randint(1, drafts), "drafts": drafts}
        most = 1.0e9
    else:
        high = _log_int(rng, 1, 16384)
        case |= {"seqs": _log_int(rng, 1, 24), "low": max(1, high // rng.choice((1, 3, 16))), "high": high,
                 "past": rng.choice((0, rng.randint(1, 2000), _log_int(rng, 16, 24000))), "cache": rng.choice(("fp8", "fp8", case["dtype"]))}
        most = 6.6e7
    while True:
        each = case["high"] if op == "step" else case["high"] + case["past"]
        if 2.0 * case["kv_heads"] * dim * case["seqs"] * each <= most:
            return case
        if case["seqs"] > 1:
            case["seqs"] = max(1, case["seqs"] * 2 // 3)
        else:
            case["high"] = max(1, case["high"] * 2 // 3)
            case["low"] = min(case["low"], case["high"])
            if op == "piece":
                case["past"] = case["past"] * 2 // 3


def _blocks(tokens, size=BLOCK):
    return -(-tokens // size)


def _lengths(case, low, high, salt=0):
    """A length for each sequence from low to high, spread over their logarithm; the longest is high."""
    rng = random.Random(case["mix"] * 16 + salt)
    got = [_log_int(rng, low, high) for _ in range(case["seqs"])]
    got[rng.randrange(len(got))] = high
    return got


def _sizes(case):
    """Positions that each sequence holds, and its rows of the call."""
    if case["op"] == "step":
        return _lengths(case, case["low"], case["high"]), _lengths(case, case["drafts_low"], case["drafts"], salt=1)
    rng = random.Random(case["mix"] + 1)
    rows = _lengths(case, case["low"], case["high"])
    return [rng.randint(case["past"] // 2, case["past"]) for _ in rows], rows


# --------------------------------------------------------------------------
# Inputs.
# --------------------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _trees(rng, sizes):
    """Ancestor bits of each drafted token, 64 to a word, and its depth: a root, then children of earlier tokens."""
    masks, depths = [], []
    for n in sizes:
        bits, depth = [], []
        for t in range(n):
            parent = rng.randrange(max(0, t - 6), t) if t else -1
            bits.append((bits[parent] if t else 0) | 1 << t)
            depth.append(depth[parent] + 1 if t else 0)
        masks += bits
        depths += depth
    words = _blocks(max(sizes), 64)
    return [[((m >> 64 * w & (1 << 64) - 1) ^ 1 << 63) - (1 << 63) for w in range(words)] for m in masks], depths


def _scale_for(top):
    """The smallest power of two that brings `top` (any floating type) to at most 448."""
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(LOW, HIGH)
    exponent = torch.where(top == 0, torch.full_like(exponent, LOW), exponent)
    return torch.ldexp(torch.ones_like(top), exponent)


def _pool(g, pages, page, kv, dim, dtype, kind):
    """Pages of one layer as a program finds them: keys with a few strong columns, values without."""
    shape = (1, 2, pages, kv, page, dim)
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
    x[:, 0, ..., ::17] *= 4.0
    if kind != "fp8":
        return x, None
    codes = torch.empty(shape, device=DEVICE, dtype=torch.float8_e4m3fn)
    scales = torch.empty((1, 2, pages, kv, page // BLOCK), device=DEVICE)
    step = max(1, (1 << 27) // (kv * page * dim))
    for half in range(2):
        for a in range(0, pages, step):
            part = x[0, half, a:a + step].float().view(-1, kv, page // BLOCK, BLOCK, dim)
            scale = _scale_for(part.abs().amax((-1, -2)))
            scales[0, half, a:a + step] = scale
            codes[0, half, a:a + step] = (part / scale[..., None, None]).to(torch.float8_e4m3fn).view(-1, kv, page, dim)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # A bulk, a few hundred strong candidates, and one id in a hundred that the program ruled out.
        x = torch.randn((rows, vocab), generator=g, device=DEVICE).mul_(case["spread"])
        chance = torch.rand((rows, vocab), generator=g, device=DEVICE)
        x += torch.where(chance < 200 / vocab, 3.0 * case["spread"] * torch.rand((rows, vocab), generator=g, device=DEVICE), 0.0)
        x.masked_fill_(chance > 0.99, float("-inf"))
        settings = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["mixed"]:
            settings = {"temperature": torch.tensor([rng.choice((0.0, 0.5, 0.7, 1.0, 1.2)) for _ in range(rows)], device=DEVICE),
                        "top_k": _ints([rng.choice((0, 0, 20, 50, 400)) for _ in range(rows)]),
                        "top_p": torch.tensor([rng.choice((1.0, 0.9, 0.95, 0.5)) for _ in range(rows)], device=DEVICE),
                        "min_p": torch.tensor([rng.choice((0.0, 0.0, 0.02, 0.1)) for _ in range(rows)], device=DEVICE)}
        return state | settings | {"logits": x.to(dtype), "uniforms": torch.rand(rows, generator=g, device=DEVICE)}
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    held, rows = _sizes(case)
    kind = case.get("cache", "fp8")
    count = [_blocks(h + r, page) for h, r in zip(held, rows)]
    n_pages = sum(count) + 3
    order = list(range(n_pages))
    rng.shuffle(order)
    at = _offsets(count)
    table = [order[at[b]:at[b + 1]] for b in range(len(held))]
    refs = [0] * n_pages
    for p in order[:at[-1]]:
        refs[p] = 1
    pool, scales = _pool(g, n_pages, page, kv, dim, dtype, kind)
    n = sum(rows)
    # Queries of the size that normed heads have: scores of a few units.
    q = torch.randn((n, heads, dim), generator=g, device=DEVICE, dtype=dtype).mul_(1.5)
    k = torch.randn((n, kv, dim), generator=g, device=DEVICE, dtype=dtype)
    k[..., ::17] *= 4.0
    angle = torch.arange(max(h + r for h, r in zip(held, rows)), device=DEVICE, dtype=torch.float64)[:, None] \
        * 1e6 ** (-torch.arange(0, case["rot"], 2, device=DEVICE, dtype=torch.float64) / case["rot"])
    state |= {"q": q, "k": k, "v": torch.randn((n, kv, dim), generator=g, device=DEVICE, dtype=dtype), "cos": angle.cos().float(), "sin": angle.sin().float(),
              "pool": pool, "scales": scales, "page_table": _ints([r + [-1] * (max(count) - len(r)) for r in table]), "lengths": _ints(held),
              "held": _ints(count), "refs": _ints(refs), "status": _ints([0]), "slots": _ints(list(range(len(held)))), "offsets": _ints(_offsets(rows)),
              "most": max(rows), "context": max(held)}
    if case["op"] == "step":
        masks, depths = _trees(rng, rows)
        tokens = [(b, d) for b, d in zip([b for b, r in enumerate(rows) for _ in range(r)], depths)]
        tree = case["drafts"] > 1
        state |= {"masks": _ints(masks, torch.int64) if tree else None, "positions": _ints([held[b] + d for b, d in tokens]) if tree else None}
    else:
        both = [h + r for h, r in zip(held, rows)]
        state |= {"positions": None, "all_offsets": _ints(_offsets(both)), "all_rows": sum(both), "longest": max(both)}
    return state


# --------------------------------------------------------------------------
# The plain forms.
# --------------------------------------------------------------------------

def _rows_of(s):
    """Sequence, index within it and cache position of each row of the call."""
    at = s["offsets"].long()
    row = torch.arange(s["q"].shape[0], device=DEVICE)
    seq = torch.bucketize(row, at[1:], right=True)
    index = row - at[seq]
    return seq, index, s["lengths"].long()[seq] + index


def _rotate(x, cos, sin, paired):
    """x [rows, heads, dim] turned by the angles of cos and sin [rows, half], in x's own precision."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., ::2], turned[..., 1::2]) if paired else (turned[..., :half], turned[..., half:])
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((first, second), -1).flatten(-2) if paired else torch.cat((first, second), -1)
    return torch.cat((turned, rest), -1)


def _store(s, which, x):
    """Rows x (fp32) of the call into the keys (0) or values (1) of the pool."""
    pool, table, page = s["pool"][0, which], s["page_table"].long(), s["case"]["page"]
    seq, index, position = _rows_of(s)
    if s["scales"] is None:
        pool[table[seq, position // page], :, position % page] = x.to(pool.dtype)
        return
    # Whole blocks from that of the first new row on: earlier rows as they stand, new ones, nothing else.
    codes, scales, size = pool.view(torch.uint8), s["scales"][0, which], page // BLOCK
    lengths, rows = s["lengths"].long(), s["offsets"].long().diff()
    start = lengths // BLOCK * BLOCK
    width = _blocks(s["most"] + BLOCK - 1) * BLOCK
    at = start[:, None] + torch.arange(width, device=DEVICE)
    end = (lengths + rows)[:, None]
    inside = at.clamp_max(table.shape[1] * page - 1)
    ids = table.gather(1, inside // page).clamp_min(0)
    old = codes[ids, :, inside % page].view(torch.float8_e4m3fn).float() * scales[ids, :, inside % page // BLOCK][..., None]
    old = torch.where((at < lengths[:, None])[..., None, None], old, 0.0)
    old[seq, position - start[seq]] = x
    block = old.view(len(lengths), -1, BLOCK, *x.shape[1:])
    scale = _scale_for(block.abs().amax((2, 4)))
    new = (block / scale[:, :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(old.shape)
    keep = at < end
    codes[ids[keep], :, (inside % page)[keep]] = new[keep]
    first = keep[:, ::BLOCK]
    scales[ids[:, ::BLOCK][first], :, (inside % page // BLOCK)[:, ::BLOCK][first]] = scale[first]


def _append(s):
    """The rows into the cache; returns the turned queries (fp32)."""
    seq, index, position = _rows_of(s)
    p = position if s["positions"] is None else s["positions"].long()
    cos, sin, paired = s["cos"][p], s["sin"][p], s["case"]["paired"]
    _store(s, 0, _rotate(s["k"].float(), cos, sin, paired))
    _store(s, 1, s["v"].float())
    return _rotate(s["q"].float(), cos, sin, paired)


def _held_rows(s, ids, slots, which):
    """Rows `slots` of pages `ids` in 32 bits, [..., kv_heads, dim]."""
    pool = s["pool"][0, which]
    if s["scales"] is None:
        return pool[ids, :, slots].float()
    codes = pool.view(torch.uint8)[ids, :, slots].view(torch.float8_e4m3fn).float()
    return codes.mul_(s["scales"][0, which][ids, :, slots // BLOCK][..., None])


def _plain_step(s):
    q = _append(s).to(s["q"].dtype).float()
    at, lengths = s["offsets"].long(), s["lengths"].long()
    n, heads, dim = q.shape
    kv, page, count, drafts = s["case"]["kv_heads"], s["case"]["page"], len(lengths), s["most"]
    long_k = s["page_table"].shape[1] * page
    j = torch.arange(long_k, device=DEVICE)
    ids, slots = s["page_table"].long().clamp_min(0)[:, j // page], (j % page).expand(count, -1)
    kt = _held_rows(s, ids, slots, 0).permute(0, 2, 3, 1).contiguous()  # [seqs, kv, dim, keys]
    t = torch.arange(drafts, device=DEVICE)
    q_of = (at[:-1, None] + t).clamp_max(n - 1)
    block = q[q_of].view(count, drafts, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(block.flatten(2, 3), kt).mul_(dim ** -0.5).view(count, kv, heads // kv, drafts, long_k)
    del kt
    # Key j: context below the length, then the drafted tokens by their bits.
    d = j - lengths[:, None]
    if s["masks"] is None:
        drafted = d[:, None] <= t[:, None]
    else:
        bits = s["masks"][q_of]
        word = (d.clamp(0, drafts - 1) >> 6)[:, None].expand(-1, drafts, -1)
        drafted = (torch.gather(bits, 2, word) >> (d & 63)[:, None]) & 1 == 1
    visible = (d[:, None] < 0) | (drafted & (d < at.diff()[:, None])[:, None])
    scores = scores.masked_fill_(~visible[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    vt = _held_rows(s, ids, slots, 1).transpose(1, 2).contiguous()
    o = torch.matmul(p.flatten(2, 3), vt).view(*p.shape[:-1], dim).div_(total.clamp_min_(1e-30))
    seq, index, _ = _rows_of(s)
    return [o.permute(0, 3, 1, 2, 4).reshape(count * drafts, heads, dim)[seq * drafts + index].to(s["q"].dtype), s["pool"], s["scales"]]


def _plain_piece(s):
    q = _append(s).to(s["q"].dtype)
    at = s["all_offsets"].long()
    row = torch.arange(s["all_rows"], device=DEVICE)
    seq = torch.bucketize(row, at[1:], right=True)
    position, page = row - at[seq], s["case"]["page"]
    ids = s["page_table"].long()[seq, position // page]
    return [q] + [_held_rows(s, ids, position % page, which).to(q.dtype) for which in (0, 1)]


def _column(x):
    return x.double()[:, None] if isinstance(x, torch.Tensor) else x


def _plain_sample(s):
    x, order = torch.sort(s["logits"].double(), descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=DEVICE)
    t, k, p, least = (_column(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = torch.as_tensor(t, device=DEVICE) <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, torch.as_tensor(t, device=DEVICE, dtype=torch.float64)))
    w = torch.where(greedy, (rank == 0).double(), w)
    limit = torch.as_tensor(k, device=DEVICE)
    w = w * ((limit <= 0) | (rank < limit))
    before = w.cumsum(1) - w
    w = w * (before < p * w.sum(1, keepdim=True)) * (w >= least)
    total = w.sum(1, keepdim=True)
    at = (w.cumsum(1) <= s["uniforms"].double()[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    return [order.gather(1, at)[:, 0], torch.log(w.gather(1, at) / total)[:, 0].float()]


PLAIN = {"step": _plain_step, "piece": _plain_piece, "sample": _plain_sample}


# --------------------------------------------------------------------------
# One pass.
# --------------------------------------------------------------------------

def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return PLAIN[op](s)
    from afterimage_amd.runtime.kv_cache import PagedKVCache
    from afterimage_amd.runtime.sampling import sample

    if op == "sample":
        return list(sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], logprobs=True))
    cache = s.get("handle")  # what a program keeps: these same tensors
    if cache is None:
        cache = s["handle"] = PagedKVCache(s["pool"], s["page_table"], s["lengths"], s["held"], s["refs"], s["status"], s["scales"])
    q = cache.append_rotated(0, s["q"], s["k"], s["v"], s["slots"], s["offsets"], s["cos"], s["sin"], s["positions"], interleaved=s["case"]["paired"])
    if op == "step":
        return [cache.attend(0, q, s["slots"], s["offsets"], s["masks"], max_drafts=s["most"], max_context=s["context"]), cache.pool, cache.scales]
    return [q, *cache.read(0, s["slots"], s["all_offsets"], s["all_rows"], dtype=s["q"].dtype)]


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": float(case["rows"] * (case["vocab"] * size + 4 + 8 + 4)), "flops": 0.0}
    held, rows = _sizes(case)
    heads, kv, dim, n = case["heads"], case["kv_heads"], case["dim"], sum(rows)
    row = kv * dim * 2  # elements of a position's key and value
    kept = row * 1 + kv * 2 * 4 / BLOCK if case.get("cache", "fp8") == "fp8" else row * 2.0  # bytes of it in the cache
    table = 4 * sum(_blocks(h + r, case["page"]) for h, r in zip(held, rows))
    # Queries in and out, new rows in and into the cache, their angles, the context.
    nbytes = 4.0 * n * heads * dim + 2.0 * n * row + n * kept + 4.0 * n * case["rot"] + sum(held) * kept + table
    if case["op"] == "piece":
        return {"bytes": nbytes + 2.0 * row * (sum(held) + n), "flops": 3.0 * n * (heads + kv) * case["rot"]}
    pairs = sum(r * (h + r / 2) for h, r in zip(held, rows))
    return {"bytes": nbytes, "flops": 4.0 * pairs * heads * dim}


# --------------------------------------------------------------------------
# The definition, in 64 bits.
# --------------------------------------------------------------------------

def _nearest8(x):
    """x to the nearest of the values that 8 bits hold, ties to the even one: steps of 2^-3 of the leading power, 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-300))).clamp_min(-6.0) - 3.0)
    return torch.round(x / step) * step


def _formed(x):
    """What blocks x [..., 16, dim] hold in 8 bits, and their scales: the values they then stand for are the products."""
    top = x.abs().amax((-1, -2), keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -400) / MOST))
    e = torch.where(top > MOST * torch.exp2(e), e + 1, torch.where(top <= MOST * torch.exp2(e - 1), e - 1, e)).clamp(LOW, HIGH)
    return _nearest8(x / torch.exp2(e)), torch.exp2(e)


def _turned(x, cos, sin, paired):
    """Each pair of x [rows, heads, dim] as a complex number, times that of its angle."""
    half = cos.shape[1]
    pair = x[..., :2 * half].unflatten(-1, (half, 2) if paired else (2, half))
    pair = pair if paired else pair.transpose(-1, -2)
    z = torch.view_as_complex(pair.contiguous()) * torch.complex(cos, sin)[:, None]
    back = torch.view_as_real(z)
    back = back if paired else back.transpose(-1, -2)
    return torch.cat((back.flatten(-2), x[..., 2 * half:]), -1)


def _exact_rows(s, b, held, at, n, cos, sin, paired, codes, scales):
    """Sequence b's keys and values with its n new rows, [2, kv_heads, positions, dim] in 64 bits. codes and scales (where not None) take what 8 bits hold."""
    page = s["case"]["page"]
    m = held + n
    ids = s["page_table"][b, :_blocks(m, page)].long()
    pair = []
    for which, new in ((0, _turned(s["k"][at:at + n].double(), cos, sin, paired)), (1, s["v"][at:at + n].double())):
        x = s["pool"][0, which][ids].double() if s["scales"] is None else \
            (s["pool"][0, which].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double().unflatten(2, (-1, BLOCK)) * s["scales"][0, which][ids].double()[..., None, None]).flatten(2, 3)
        x = x.transpose(0, 1).flatten(1, 2).clone()  # [kv, positions, dim]
        x[:, held:m] = new.transpose(0, 1)
        x = x[:, :m]
        if s["scales"] is not None:
            first = held // BLOCK * BLOCK
            tail = torch.nn.functional.pad(x[:, first:], (0, 0, 0, -m % BLOCK))
            new, scale = _formed(tail.unflatten(1, (-1, BLOCK)))
            x[:, first:] = (new * scale).flatten(1, 2)[:, :m - first]
            if codes is not None:
                j, block = torch.arange(first, m, device=DEVICE), torch.arange(first, m, BLOCK, device=DEVICE)
                codes[0, which, ids[j // page], :, j % page] = new.flatten(1, 2)[:, :m - first].transpose(0, 1)
                scales[0, which, ids[block // page], :, block % page // BLOCK] = scale[..., 0, 0].t()
        pair.append(x)
    return torch.stack(pair)


def _exact_sample(s):
    tokens, logs = [], []
    setting = {name: s[name].tolist() if isinstance(s[name], torch.Tensor) else [s[name]] * s["logits"].shape[0] for name in ("temperature", "top_k", "top_p", "min_p")}
    for r, u in enumerate(s["uniforms"].tolist()):
        x = s["logits"][r].double()
        value, count = torch.unique(x[x > float("-inf")], return_counts=True)
        value, count = value.flip(0), count.flip(0)  # distinct values, the largest first, and how often they occur
        t, k, p, least = (setting[name][r] for name in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            k, t = 1, 1.0
        w = torch.exp((value - value[0]) / t)
        before = count.cumsum(0) - count
        if k > 0:
            count = torch.minimum(count, (k - before).clamp_min(0))
        mass = (w * count).cumsum(0)
        # Of a value's equals, those that some of p is still missing before.
        need = torch.ceil((p * mass[-1] - (mass - w * count)) / w.clamp_min(1e-300))
        count = torch.minimum(count, need.clamp(0, 1e9).long()) * (w >= least)
        mass = (w * count).cumsum(0)
        goal = u * mass[-1]
        g = int((mass <= goal).sum())
        j = int(((goal - (mass[g] - w[g] * count[g])) / w[g]).floor().clamp(0, int(count[g]) - 1))
        tokens.append(torch.nonzero(x == value[g])[j, 0])
        logs.append(torch.log(w[g] / mass[-1]))
    return [torch.stack(tokens), torch.stack(logs)]


def exact(case, seed):
    """One sequence at a time (and, of the attention, one key/value head); of a sampled row, its distinct values and their counts."""
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    held, rows = _sizes(case)
    heads, kv, paired = case["heads"], case["kv_heads"], case["paired"]
    group = heads // kv
    out, keys, values = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE), [], []
    codes, scales = (s["pool"].double(), s["scales"].double()) if case["op"] == "step" else (None, None)
    for b, (at, h, n) in enumerate(zip(_offsets(rows), held, rows)):
        p = torch.arange(h, h + n, device=DEVICE) if s["positions"] is None else s["positions"][at:at + n].long()
        cos, sin = s["cos"][p].double(), s["sin"][p].double()
        q = _turned(s["q"][at:at + n].double(), cos, sin, paired)
        k, v = _exact_rows(s, b, h, at, n, cos, sin, paired, codes, scales)
        if case["op"] == "piece":
            out[at:at + n] = q
            keys.append(k.transpose(0, 1))
            values.append(v.transpose(0, 1))
            continue
        j, i = torch.arange(h + n, device=DEVICE), torch.arange(n, device=DEVICE)[:, None]
        d = (j - h).clamp_min(0)
        visible = j <= h + i if s["masks"] is None else (j < h) | (s["masks"][at:at + n][:, d >> 6] >> (d & 63) & 1 == 1)
        for g in range(kv):
            weight = torch.exp(torch.einsum("ngd,md->ngm", q[:, g * group:(g + 1) * group], k[g]) / math.sqrt(case["dim"])) * visible[:, None]
            out[at:at + n, g * group:(g + 1) * group] = torch.einsum("ngm,md->ngd", weight, v[g]) / weight.sum(-1, keepdim=True)
    return [out, codes, scales] if case["op"] == "step" else [out, torch.cat(keys), torch.cat(values)]
