"""A token's way together: rotation and append, attention over the cache, the
rows back, the tree's accepted path, sampling; as a program calls them, captured
and replayed, on another stream, and beside calls of other sizes."""
import pytest
import torch

from afterimage_amd.examples import verify_tree
from afterimage_amd.runtime.attention import prompt_attention, rotary_tables, tree_masks
from afterimage_amd.runtime.kv_cache import PagedKVCache
from afterimage_amd.runtime.sampling import sample
from tests.attention_oracle import attend, check
from tests.eight_bits import Copy, turn

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KV, DIM = 2, 6, 2, 64


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def heads(g, n, count, dtype=torch.bfloat16):
    return torch.randn(n, count, DIM, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
def test_prompts_trees_and_their_paths(kind):
    """Three pieces of two prompts, a verified tree, and the next tree after its accepted path; every layer's rows
    against the definition, the attention of prompts over what was read back."""
    g = torch.Generator().manual_seed(1)
    cache = PagedKVCache.allocate(LAYERS, 20, 16, KV, DIM, 3, 8, kind)
    cache.pool.view(torch.uint8 if kind is torch.float8_e4m3fn else torch.int16).zero_()
    if cache.scales is not None:
        cache.scales.fill_(1.0)
    cos, sin = rotary_tables(128, DIM, 1e4, "cpu")
    tables = (cos.cuda(), sin.cuda())
    slots, lengths = [2, 0], [0, 0]
    copy = Copy(cache)

    def put(layer, k, v, sizes, at):
        for which, x in ((0, turn(k.cpu().float(), cos[at], sin[at], False)), (1, v.cpu().float())):
            first = 0
            for b, n in enumerate(sizes):
                for head in range(KV):
                    copy.put(layer, which, head, slots[b], lengths[b], list(x[first:first + n, head].double()))
                first += n

    for sizes in ([17, 3], [1, 30], [20, 9]):
        offsets = ints([0, sizes[0], sum(sizes)])
        cache.reserve(ints(slots), ints(sizes))
        copy.table = cache.page_table.cpu().clone()
        at = [lengths[b] + i for b, n in enumerate(sizes) for i in range(n)]
        for layer in range(LAYERS):
            q, k, v = (heads(g, sum(sizes), h) for h in (HEADS, KV, KV))
            q2 = cache.append_rotated(layer, q, k, v, ints(slots), offsets, *tables)
            put(layer, k, v, sizes, at)
            assert torch.equal(q2.cpu(), turn(q.cpu().float(), cos[at], sin[at], False).to(q.dtype))
            both = [a + n for a, n in zip(lengths, sizes)]
            k_at = ints([0, both[0], sum(both)])
            ks, vs = cache.read(layer, ints(slots), k_at, sum(both))
            o = prompt_attention(q2, ks, vs, offsets, k_at)
            first, k_first = 0, 0
            for n, m in zip(sizes, both):
                visible = torch.arange(m, device="cuda") <= torch.arange(n, device="cuda")[:, None] + m - n
                want, bound, _ = attend(q2[first:first + n], ks[k_first:k_first + m], vs[k_first:k_first + m], visible, DIM ** -0.5)
                check(o[first:first + n], want, bound)
                first, k_first = first + n, k_first + m
        cache.advance(ints(slots), offsets)
        for b, n in enumerate(sizes):
            lengths[b] += n
            copy.lengths[slots[b]] += n
        copy.same(cache)
    parents, sizes = [-1, 0, 0, 1, 3, -1, 0, 1], [5, 3]
    depths = [0, 1, 1, 2, 3, 0, 1, 2]
    offsets, masks = ints([0, 5, 8]), None
    for paths in ([[0, 2], [0, 1, 2]], [[0, 1, 3, 4], []]):
        masks = tree_masks(ints(parents), offsets, 5)
        cache.reserve(ints(slots), ints(sizes))
        copy.table = cache.page_table.cpu().clone()
        at = [lengths[0] + d for d in depths[:5]] + [lengths[1] + d for d in depths[5:]]
        for layer in range(LAYERS):
            q, k, v = (heads(g, 8, h) for h in (HEADS, KV, KV))
            q2 = cache.append_rotated(layer, q, k, v, ints(slots), offsets, *tables, ints(at))
            put(layer, k, v, sizes, at)
            o = cache.attend(layer, q2, ints(slots), offsets, masks, max_drafts=5, max_context=max(lengths))
            for b, (first, n) in enumerate(((0, 5), (5, 3))):
                m = lengths[b] + n
                ks, vs = cache.read(layer, ints([slots[b]]), ints([0, m]), m)
                bits = masks[first:first + n, 0]
                j = torch.arange(m, device="cuda")
                visible = (j < lengths[b]) | ((bits[:, None] >> (j - lengths[b]).clamp_min(0)) & 1 == 1)
                want, bound, _ = attend(q2[first:first + n], ks, vs, visible, DIM ** -0.5)
                check(o[first:first + n], want, bound)
        cache.commit(ints(slots), ints([p + [0] * (4 - len(p)) for p in paths]), ints([len(p) for p in paths]))
        for b, p in enumerate(paths):
            copy.commit(slots[b], p)
            lengths[b] += len(p)
        copy.same(cache)
    cache.check()


def test_a_step_in_a_graph_beside_eager_calls():
    """A captured step (reserve, append, attend, sample, advance), replayed with the program's own work of
    other sizes between; every replay against the same steps made eagerly on a cache of its own."""
    g = torch.Generator().manual_seed(2)
    tables = rotary_tables(4096, DIM)
    caches = [PagedKVCache.allocate(1, 300, 16, KV, DIM, 4, 200, torch.float8_e4m3fn) for _ in range(2)]
    slots, one = ints([0, 1]), ints([1, 1])
    offsets = ints([0, 1, 2])
    k0, v0 = heads(g, 2000, KV), heads(g, 2000, KV)
    q0 = heads(g, 2000, HEADS)
    for cache in caches:
        cache.reserve(slots, ints([1500, 500]))
        cache.append_rotated(0, q0, k0, v0, slots, ints([0, 1500, 2000]), *tables)
        cache.advance(slots, ints([0, 1500, 2000]))
    q, k, v = (heads(g, 2, h) for h in (HEADS, KV, KV))
    weight = torch.randn(HEADS * DIM, 50001, generator=g).to(torch.bfloat16).cuda()
    u = torch.rand(2, generator=g).cuda()
    inputs = [torch.empty_like(x) for x in (q, k, v, u)]

    def step(cache, q, k, v, u):
        cache.reserve(slots, one)
        q = cache.append_rotated(0, q, k, v, slots, offsets, *tables)
        o = cache.attend(0, q, slots, offsets, max_drafts=1, max_context=4000)
        cache.advance(slots, offsets)
        return o, sample(o.view(2, -1) @ weight, u, temperature=0.7, top_k=100, top_p=0.9)

    for to, x in zip(inputs, (q, k, v, u)):
        to.copy_(x)
    lengths = [c.lengths.clone() for c in caches]
    step(caches[0], *inputs)  # as a program does once before it captures
    caches[0].lengths.copy_(lengths[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0], *inputs)
    caches[0].lengths.copy_(lengths[0])  # nothing ran while it was captured
    for turn_ in range(6):
        new = [torch.randn(x.shape, generator=g).to(x.dtype).cuda() for x in (q, k, v)] + [torch.rand(2, generator=g).cuda()]
        for to, x in zip(inputs, new):
            to.copy_(x)
        want = step(caches[1], *new)
        # Calls of other sizes, whose workspaces come and go.
        sample(torch.randn(3 + turn_, 60000, device="cuda"), torch.rand(3 + turn_, device="cuda"))
        caches[1].attend(0, q0[:1 + turn_], slots[:1], ints([0, 1 + turn_]), max_drafts=1 + turn_, max_context=1500)
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])
        assert all(bool((x == 7).all()) for x in others)
        assert torch.equal(caches[0].lengths, caches[1].lengths)
        # What no row has been written to holds whatever its memory held.
        a, b = (c.read(0, slots, ints([0, 1501 + turn_, 2002 + 2 * turn_]), 2002 + 2 * turn_) for c in caches)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for cache in caches:
        cache.check()


def test_two_graphs_and_two_streams_at_once():
    """Two captured calls of sampling and two caches' steps, on streams of their own at the same time."""
    x, y = torch.randn(3, 151936, device="cuda"), torch.randn(40, 60000, device="cuda").half()
    u, w = torch.rand(3, device="cuda"), torch.rand(40, device="cuda")
    want = sample(x, u, top_p=0.9), sample(y, w, min_p=0.01)
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for logits, uniforms, rule in ((x, u, {"top_p": 0.9}), (y, w, {"min_p": 0.01})):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(sample(logits, uniforms, **rule))
        graphs.append(graph)
    for _ in range(5):
        for t in got:
            t.fill_(-5)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        a = sample(x, u, top_p=0.9)  # and an eager call beside them
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(a, want[0])


def test_long_rows_sampled_from_a_graph():
    """Rows that several workgroups share: every replay starts from its own inputs, whatever eager calls ran in between."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x, u = torch.empty(3, 100000, device="cuda", dtype=torch.bfloat16), torch.empty(3, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x.normal_(generator=g), u.uniform_(generator=g)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sample(x, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(stream)
    with torch.cuda.graph(graph):
        tokens, logs = sample(x, u, top_p=0.9, logprobs=True)
    for spread in (2.5, 1e-3, 0.0, 4.0, 2.5):
        x.normal_(generator=g).mul_(spread), u.uniform_(generator=g)
        graph.replay()
        want, want_logs = sample(x, u, top_p=0.9, logprobs=True)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want) and torch.equal(logs, want_logs)


def test_calls_on_another_stream():
    g = torch.Generator().manual_seed(5)
    tables = rotary_tables(64, DIM)
    q, k, v = (heads(g, 40, h) for h in (HEADS, KV, KV))
    x, u = torch.randn(2, 50001, generator=g).cuda(), torch.rand(2, generator=g).cuda()
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        cache = PagedKVCache.allocate(1, 8, 16, KV, DIM, 2, 4, torch.float8_e4m3fn)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            cache.reserve(ints([1]), ints([40]))
            q2 = cache.append_rotated(0, q, k, v, ints([1]), ints([0, 40]), *tables)
            o = cache.attend(0, q2, ints([1]), ints([0, 40]), max_drafts=40, max_context=0)
            results.append([q2, o, *cache.read(0, ints([1]), ints([0, 40]), 40), sample(x, u)])
        stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_the_example_samples_with_rotation_and_eight_bits():
    """What a verified tree accepts is the decoded text, as far as both passes draw the same tokens."""
    got = verify_tree.run(**verify_tree.SAMPLED)
    decoded, cache = got["decoded"].tolist(), got["cache"]
    assert cache.scales is not None
    for b, (row, path) in enumerate(zip(decoded, got["accepted"])):
        assert row[:len(path)] == path and len(path) >= 1
        assert int(cache.lengths[len(decoded) + b]) == int(cache.lengths[b]) - (len(row) - 1) + len(path)


def test_the_example_turns_greedily_in_sixteen_bits():
    got = verify_tree.run(rotary=True)
    for row, path in zip(got["decoded"].tolist(), got["accepted"]):
        assert row[:len(path)] == path and len(path) >= 1


def test_the_sampled_example_runs_as_a_command(capsys):
    verify_tree.main(True)
    out = capsys.readouterr().out
    assert out.count("accepted from its tree") == 3 and "pages in use" in out


def test_refusals():
    cache = PagedKVCache.allocate(1, 4, 16, KV, DIM, 1, 2, torch.float8_e4m3fn)
    wide = PagedKVCache.allocate(1, 4, 16, KV, DIM, 1, 2, torch.float16)
    cos, sin = rotary_tables(8, DIM)
    q, k = (torch.zeros(2, h, DIM, dtype=torch.bfloat16, device="cuda") for h in (HEADS, KV))
    slots, offsets = ints([0]), ints([0, 2])

    def turned(c=cache, q=q, k=k, v=k, seqs=slots, offsets=offsets, cos=cos, sin=sin, positions=None, out=None, layer=0):
        return c.append_rotated(layer, q, k, v, seqs, offsets, cos, sin, positions, out=out)

    for options, text in (({"c": wide}, "float16"), ({"q": q.float()}, "bf16 or fp16"), ({"k": k.half()}, "k must be"), ({"v": k[:1]}, "same rows"),
                          ({"q": q[:, :, :32]}, "q must be"), ({"k": k[:, :1]}, "k must be"), ({"cos": cos.double()}, "cos must be"),
                          ({"cos": torch.zeros(8, DIM, device="cuda")}, "cos must be"), ({"sin": sin[:4]}, "sin must"), ({"positions": ints([0])}, "positions"),
                          ({"out": q[:1]}, "out must"), ({"layer": 1}, "layer"), ({"offsets": ints([0])}, "offsets"), ({"cos": cos.cpu()}, "cos must be"),
                          ({"q": q.transpose(0, 1).contiguous().transpose(0, 1)[..., 8:]}, "q must be"), ({"seqs": slots.long()}, "seqs")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            turned(**options)
    for options, text in (({"rows": -1}, "negative"), ({"dtype": torch.float32}, "bf16 or fp16"), ({"out": (k[:1], k)}, "out must hold")):
        with pytest.raises(ValueError, match=text):
            cache.read(**({"layer": 0, "seqs": slots, "offsets": offsets, "rows": 2} | options))
    with pytest.raises(ValueError, match="float16"):
        wide.read(0, slots, offsets, 2, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no backward"):
        turned(q=q.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="sin requires"):
        turned(sin=sin.clone().requires_grad_())
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache(cache.pool, cache.page_table, cache.lengths, cache.held, cache.refs, cache.status)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache(wide.pool, cache.page_table, cache.lengths, cache.held, cache.refs, cache.status, cache.scales)
    for more in ({"page_size": 24}, {"dim": 24}, {"dim": 272}):
        sizes = {"n_layers": 1, "n_pages": 2, "page_size": 16, "kv_heads": 1, "dim": 16, "max_seqs": 1, "max_pages": 1} | more
        with pytest.raises(ValueError, match="8 bits"):
            PagedKVCache.allocate(**sizes, dtype=torch.float8_e4m3fn)
    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for options, text in (({"temperature": -1.0}, "temperature"), ({"temperature": float("nan")}, "temperature"), ({"top_k": -1}, "top_k"), ({"top_p": 1.5}, "top_p"),
                          ({"min_p": -0.1}, "min_p"), ({"top_k": torch.zeros(2, device="cuda")}, "top_k"), ({"temperature": torch.zeros(3, device="cuda")}, "temperature"),
                          ({"out": torch.zeros(2, device="cuda")}, "out")):
        with pytest.raises(ValueError, match=text):
            sample(x, u, **options)
    for logits, text in ((x.double(), "bf16"), (x.t(), "contiguous"), (x[0], "rows"), (torch.zeros(1, (1 << 18) + 1, device="cuda"), "vocab")):
        with pytest.raises(ValueError, match=text):
            sample(logits, u)
    with pytest.raises(RuntimeError, match="no backward"):
        sample(x, u, temperature=torch.ones(2, device="cuda").requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        sample(x.requires_grad_(), u)
