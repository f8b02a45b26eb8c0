"""Decoding, then the same tokens out of one verified draft tree.

A small decoder-only model whose projections stay compressed on the GPU
(decode_linear decodes each as it is used) runs the way a speculative engine
does (afterimage/runtime/streaming_engine.py:2488-2600 drafts step_k tokens and
verifies them in one target pass):

  - the prompts of a batch go through prompt_attention, their keys and values
    into a PagedKVCache;
  - each sequence is forked: the first branch decodes, a token a pass: the
    largest logit's, or one sampled with a random number for each position;
  - the other verifies a tree that holds those tokens among wrong guesses, in
    one pass, and commits the path it accepts: a child is accepted where it is
    its parent's token by the same rule and random number, so that what is
    accepted follows the model's distribution.

Both branches hold the same tokens afterwards where the cache has 16 bits and no
two logits are nearer than the passes' roundings. Queries and keys may be turned
by their positions on their way into the cache, which may hold 16 bits or 8; in 8
its 16 positions share a scale, so rows are rounded with the drafts beside them,
and the branches may part. Run as
``python -m afterimage_amd.examples.verify_tree``: greedily with a cache in 16
bits; with ``--sampled``, with sampling, rotation and a cache in 8.
"""
from __future__ import annotations

import sys

import torch

from ..runtime.attention import prompt_attention, rotary_tables, tree_masks
from ..runtime.compressed_store import compress_layer
from ..runtime.device import DeviceTensor, decode_linear
from ..runtime.kv_cache import PagedKVCache
from ..runtime.sampling import sample


def _ints(values, device) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=device)


class Linear:
    """x @ W.T for a bf16 weight that is kept compressed on the GPU."""

    def __init__(self, rows: int, cols: int, generator: torch.Generator, device):
        weight = (torch.randn(rows, cols, generator=generator) * cols ** -0.5).to(torch.bfloat16)
        layer = compress_layer(weight)
        self.tensor = DeviceTensor.from_encoded(layer.encoded, layer.sign_mantissa, device)
        self.rows, self.cols = rows, cols

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return decode_linear(self.tensor, x, self.rows, self.cols, 0)


class Model:
    """Attention blocks with a residual, an embedding and an output projection, random weights. With positions, so many of
    them have angles that queries and keys turn by."""

    def __init__(self, layers: int = 2, heads: int = 8, kv_heads: int = 2, dim: int = 64, vocab: int = 512, seed: int = 0,
                 device="cuda", positions: int = 0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.device = heads, kv_heads, dim, torch.device(device)
        width = heads * dim
        self.embedding = torch.randn(vocab, width, generator=g).to(torch.bfloat16).to(device)
        self.blocks = [{"q": Linear(width, width, g, device), "k": Linear(kv_heads * dim, width, g, device),
                        "v": Linear(kv_heads * dim, width, g, device), "o": Linear(width, width, g, device)}
                       for _ in range(layers)]
        self.head = Linear(vocab, width, g, device)
        self.rotary = rotary_tables(positions, dim, device=device) if positions else None

    def forward(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """Logits of each token; attend(layer, q, k, v) is the attention of one layer."""
        x = self.embedding[tokens]
        n = x.shape[0]
        for layer, block in enumerate(self.blocks):
            h = torch.nn.functional.rms_norm(x, (x.shape[1],))
            q, k, v = (block[name](h).view(n, -1, self.dim) for name in ("q", "k", "v"))
            x = x + block["o"](attend(layer, q, k, v).view(n, -1))
        return self.head(torch.nn.functional.rms_norm(x, (x.shape[1],)))


class Choice:
    """A token for each row of logits: the largest's, or sampled with the settings and a random number for each (sequence, position)."""

    def __init__(self, sequences: int, positions: int, settings: dict | None, seed: int, device):
        self.settings = settings
        self.uniforms = torch.rand(sequences, positions, generator=torch.Generator().manual_seed(seed)).to(device)

    def __call__(self, logits: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        if self.settings is None:
            return logits.argmax(-1)
        return sample(logits, self.uniforms[sequences, positions], **self.settings)


def prefill(model: Model, cache: PagedKVCache, prompts: list[list[int]], slots: torch.Tensor) -> torch.Tensor:
    """The prompts into their slots; returns the logits after each."""
    lengths = [len(p) for p in prompts]
    offsets = _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)], model.device)
    cache.reserve(slots, _ints(lengths, model.device))

    def attend(layer, q, k, v):
        if model.rotary is None:
            cache.append(layer, k, v, slots, offsets)
        else:  # the cache's rows are the turned ones, of the cache's precision
            q = cache.append_rotated(layer, q, k, v, slots, offsets, *model.rotary)
            k, v = cache.read(layer, slots, offsets, q.shape[0])
        return prompt_attention(q, k, v, offsets)

    logits = model.forward(torch.tensor(sum(prompts, []), device=model.device), attend)
    cache.advance(slots, offsets)
    return logits[offsets[1:].long() - 1]


def verify(model: Model, cache: PagedKVCache, slots: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor,
           masks: torch.Tensor | None, most: int, positions: torch.Tensor | None = None) -> torch.Tensor:
    """Logits of drafted tokens, whose keys and values go past the slots' lengths."""
    cache.reserve(slots, offsets.diff())

    def attend(layer, q, k, v):
        if model.rotary is None:
            cache.append(layer, k, v, slots, offsets)
        else:
            q = cache.append_rotated(layer, q, k, v, slots, offsets, *model.rotary, positions)
        return cache.attend(layer, q, slots, offsets, masks, max_drafts=most)

    return model.forward(tokens, attend)


def decode(model: Model, cache: PagedKVCache, slots: torch.Tensor, tokens: torch.Tensor, steps: int, choose: Choice) -> torch.Tensor:
    """[sequences, steps + 1]: the given tokens and what follows them, a token a pass."""
    n = slots.shape[0]
    offsets = torch.arange(n + 1, dtype=torch.int32, device=model.device)
    out, sequences = [tokens], torch.arange(n, device=model.device)
    for _ in range(steps):
        logits = verify(model, cache, slots, out[-1], offsets, None, 1)
        cache.advance(slots, offsets)
        out.append(choose(logits, sequences, cache.lengths[slots.long()].long()))
    return torch.stack(out, 1)


def accept(tree: list[int], parents: list[int], best: list[int]) -> list[int]:
    """The path from the root (token 0) along children that are the model's choice after their parent."""
    path = [0]
    while True:
        child = next((i for i, p in enumerate(parents) if p == path[-1] and tree[i] == best[path[-1]]), None)
        if child is None:
            return path
        path.append(child)


def run(prompts=(37, 5, 130), steps: int = 5, wrong: int = 2, seed: int = 0, device="cuda", dtype: torch.dtype = torch.bfloat16,
        rotary: bool = False, settings: dict | None = None) -> dict:
    """Both ways of decoding; the tokens of each and the cache. dtype: the cache's; settings: sample's, None for the largest logit."""
    positions = max(prompts) + steps + 2
    model = Model(seed=seed, device=device, positions=positions if rotary else 0)
    rng = torch.Generator().manual_seed(seed + 1)
    vocab, n = model.embedding.shape[0], len(prompts)
    texts = [torch.randint(vocab, (length,), generator=rng).tolist() for length in prompts]
    cache = PagedKVCache.allocate(len(model.blocks), 64, 16, model.kv_heads, model.dim, 2 * n, 16, dtype, device)
    choose = Choice(n, positions + 1, settings, seed + 2, device)
    slots = _ints(list(range(n)), device)
    branches = _ints(list(range(n, 2 * n)), device)
    first = choose(prefill(model, cache, texts, slots), torch.arange(n, device=device), cache.lengths[:n].long())
    cache.fork(slots, branches)
    decoded = decode(model, cache, slots, first, steps, choose)
    # A tree for each sequence: the decoded tokens in a row, wrong ones beside each.
    trees, parents = [], []
    for row in decoded.tolist():
        tree, up, last = [row[0]], [-1], 0
        for token in row[1:]:
            for guess in range(wrong):
                tree.append((token + 1 + guess) % vocab)
                up.append(last)
            tree.append(token)
            up.append(last)
            last = len(tree) - 1
        trees.append(tree)
        parents.append(up)
    most = max(map(len, trees))
    offsets = _ints([sum(map(len, trees[:i])) for i in range(n + 1)], device)
    masks = tree_masks(_ints(sum(parents, []), device), offsets, most)
    # A drafted token's position is that of its place in the tree; what follows it comes after that.
    depths = []
    for up in parents:
        depth = []
        for p in up:
            depth.append(0 if p < 0 else depth[p] + 1)
        depths += depth
    sequences = torch.tensor([b for b, t in enumerate(trees) for _ in t], device=device)
    at = cache.lengths[branches.long()].long()[sequences] + torch.tensor(depths, device=device)
    logits = verify(model, cache, branches, torch.tensor(sum(trees, []), device=device), offsets, masks, most, at.int())
    best = choose(logits, sequences, at + 1).tolist()
    paths = []
    for b in range(n):
        at = int(offsets[b])
        paths.append(accept(trees[b], parents[b], best[at:at + len(trees[b])]))
    longest = max(map(len, paths))
    cache.commit(branches, _ints([p + [0] * (longest - len(p)) for p in paths], device), _ints([len(p) for p in paths], device))
    cache.check()
    return {"model": model, "cache": cache, "decoded": decoded, "accepted": [[t[i] for i in p] for t, p in zip(trees, paths)],
            "following": [best[int(offsets[b]) + p[-1]] for b, p in enumerate(paths)], "slots": slots, "branches": branches}


SAMPLED = {"dtype": torch.float8_e4m3fn, "rotary": True, "settings": {"temperature": 0.8, "top_k": 40, "top_p": 0.95}}


def main(sampled: bool = False) -> None:
    got = run(**SAMPLED) if sampled else run()
    for b, (row, path) in enumerate(zip(got["decoded"].tolist(), got["accepted"])):
        print("sequence %d: decoded %s, accepted from its tree %s" % (b, row, path))
    cache = got["cache"]
    cache.release(got["slots"])
    print("pages in use after the first branches ended: %d of %d" % (int(cache.compact()), cache.n_pages))


if __name__ == "__main__":
    main("--sampled" in sys.argv[1:])
