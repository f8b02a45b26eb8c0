"""Causal attention of packed prompts against its definition in 64 bits."""
import pytest
import torch

from afterimage_amd.runtime.attention import prompt_attention
from tests.attention_oracle import attend, check

pytestmark = pytest.mark.gpu


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


def _expected(q, k, v, rows, keys, scale):
    out, bounds, lses = [], [], []
    a = b = 0
    for n, m in zip(rows, keys):
        i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
        o, bound, lse = attend(q[a:a + n], k[b:b + m], v[b:b + m], j <= i[:, None] + (m - n), scale)
        out.append(o), bounds.append(bound), lses.append(lse)
        a, b = a + n, b + m
    return torch.cat(out), torch.cat(bounds), torch.cat(lses)


def _case(rows, keys, heads, kv, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (_randn(g, sum(rows), heads, dim, dtype=dtype) * 2, _randn(g, sum(keys), kv, dim, dtype=dtype),
            _randn(g, sum(keys), kv, dim, dtype=dtype))


SHAPES = [
    # rows, keys, heads, kv_heads, dim
    ([1], [1], 1, 1, 64),
    ([1, 1, 2], [1, 5, 2], 4, 4, 128),
    ([31, 32, 33], [31, 32, 33], 8, 2, 64),
    ([63, 64, 65, 1], [63, 64, 65, 1], 5, 1, 128),
    ([127, 128, 129], [127, 128, 129], 6, 3, 96),
    ([200, 0, 77, 0], [200, 0, 77, 0], 10, 2, 128),
    ([5, 130, 64], [70, 131, 300], 8, 8, 64),
    ([300], [300], 3, 3, 8),
    ([257, 100], [300, 100], 4, 2, 256),
    ([129], [400], 2, 1, 168),
    ([513, 40], [513, 1000], 40, 8, 128),
    # Few rows over many keys: split along the keys.
    ([13], [2900], 8, 1, 128),
    ([1, 30, 7, 2], [1, 3000, 700, 5000], 10, 2, 64),
    ([40, 9], [1400, 2600], 8, 4, 256),
    ([150], [1600], 5, 1, 96),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,keys,heads,kv,dim", SHAPES)
def test_packed_prompts(rows, keys, heads, kv, dim, dtype):
    q, k, v = _case(rows, keys, heads, kv, dim, dtype)
    lse = torch.empty(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), lse=lse)
    o, bound, want = _expected(q, k, v, rows, keys, dim ** -0.5)
    check(out, o, bound)
    # Scores in fp32, then one logarithm.
    assert (lse.double() - want).abs().max().item() <= 2.0 ** -24 * (3 * dim * 8 + 64)


@pytest.mark.parametrize("rows,keys", [([40], [10]), ([70, 200], [0, 100]), ([3], [0])])
def test_rows_that_see_no_key_give_zeros(rows, keys):
    """More rows than keys: the first rows see nothing."""
    q, k, v = _case(rows, keys, 4, 2, 64, torch.bfloat16)
    lse = torch.zeros(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), lse=lse)
    o, bound, want = _expected(q, k, v, rows, keys, 64 ** -0.5)
    check(out, o, bound)
    none = want == float("-inf")
    assert bool(none.any()) and torch.equal(lse == float("-inf"), none)
    assert float(out[none].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_reach_it(bad, dtype):
    """Rows before a bad key (and other sequences) are as if it were not there; rows that see a bad value show it."""
    rows = [50, 150, 60]
    q, k, v = _case(rows, rows, 4, 2, 128, dtype)
    clean = prompt_attention(q, k, v, _offsets(rows), scale=0.1)
    at = 50 + 97
    k2, v2 = k.clone(), v.clone()
    v2[at, 1, 5] = bad
    out = prompt_attention(q, k, v2, _offsets(rows), scale=0.1)
    rest = torch.ones(out.shape, dtype=torch.bool, device="cuda")
    rest[at:200, 2:, 5] = False
    assert torch.equal(out[rest], clean[rest])
    seen = out[at:200, 2:, 5].float()
    assert bool(torch.isnan(seen).all()) if bad != bad else bool((seen == bad).all())
    k2[at] = float("nan")
    out = prompt_attention(q, k2, v, _offsets(rows), scale=0.1)
    rest[at:200] = False
    assert torch.equal(out[rest], clean[rest]) and bool(torch.isnan(out[at:200]).all())


@pytest.mark.parametrize("rows,keys,heads,kv", [([40, 9], [40, 9], 4, 2), ([13], [2900], 8, 1), ([1, 30, 7], [1, 3000, 700], 10, 2)])
def test_a_nan_query_gives_nan_and_no_other_row_does(rows, keys, heads, kv):
    q, k, v = _case(rows, keys, heads, kv, 64, torch.bfloat16)
    clean = prompt_attention(q, k, v, _offsets(rows), _offsets(keys))
    q[5, 2, 30] = float("nan")
    lse = torch.empty(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), lse=lse)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[5, 2] = True
    assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])
    assert torch.equal(torch.isnan(lse), hit[..., 0])


def test_opposite_infinities_meet_in_a_masked_tile():
    q, k, v = _case([20], [20], 1, 1, 64, torch.bfloat16)
    v[3, 0, 7], v[5, 0, 7] = float("inf"), float("-inf")
    out = prompt_attention(q, k, v, _offsets([20]), scale=0.1)[:, 0, 7].float()
    assert bool(torch.isfinite(out[:3]).all()) and bool((out[3:5] == float("inf")).all()) and bool(torch.isnan(out[5:]).all())


def test_large_scores():
    """Scores far apart and large: the running maximum moves by much more than
    the step below which the sums are left as they are."""
    q, k, v = _case([300], [300], 2, 1, 64, torch.bfloat16)
    k = (k.float() * torch.linspace(0.01, 30, 300, device="cuda")[:, None, None]).to(torch.bfloat16)
    out = prompt_attention(q, k, v, _offsets([300]), scale=1.0)
    o, bound, _ = _expected(q, k, v, [300], [300], 1.0)
    check(out, o, bound)


def test_strided_heads_and_output():
    """q, k and v as slices of one projection's output, out as a slice of a wider tensor."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = [90, 33]
    x = _randn(g, 123, 12, 64, dtype=torch.float16)
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    wide = torch.full((123, 9, 64), 7.0, dtype=torch.float16, device="cuda")
    out = prompt_attention(q, k, v, _offsets(rows), out=wide[:, 1:])
    o, bound, _ = _expected(q, k, v, rows, rows, 64 ** -0.5)
    check(out, o, bound)
    assert bool((wide[:, 0] == 7.0).all())
    # Heads outermost in memory.
    y = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(prompt_attention(y, k, v, _offsets(rows)), out)
    # One key and value for all positions (stride 0).
    k1 = k[:1].expand(123, 2, 64)
    o, bound, _ = _expected(q, k1, v, rows, rows, 64 ** -0.5)
    check(prompt_attention(q, k1, v, _offsets(rows)), o, bound)


def test_rows_outside_every_sequence_are_left_alone():
    q, k, v = _case([100], [100], 2, 2, 64, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    at = torch.tensor([10, 40, 60], dtype=torch.int32, device="cuda")
    prompt_attention(q, k, v, at, out=out)
    o, bound, _ = _expected(q[10:60], k[10:60], v[10:60], [30, 20], [30, 20], 64 ** -0.5)
    check(out[10:60], o, bound)
    assert bool((out[:10] == 3.0).all()) and bool((out[60:] == 3.0).all())


def test_offsets_outside_the_rows_are_bounded():
    q, k, v = _case([100], [100], 2, 2, 64, torch.bfloat16)
    at = torch.tensor([-5, 60, 4000], dtype=torch.int32, device="cuda")
    o, bound, _ = _expected(q, k, v, [60, 40], [60, 40], 64 ** -0.5)
    check(prompt_attention(q, k, v, at), o, bound)


def test_another_stream_and_repeated_calls_agree():
    q, k, v = _case([700, 41], [700, 41], 8, 2, 128, torch.bfloat16)
    at = _offsets([700, 41])
    first = prompt_attention(q, k, v, at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [prompt_attention(q, k, v, at) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(x, first) for x in again)


def test_nothing_to_do():
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert prompt_attention(q, k, k, _offsets([])).shape == (0, 4, 64)
    assert prompt_attention(q, k, k, _offsets([0, 0])).shape == (0, 4, 64)


def test_refusals():
    q, k, v = _case([20], [20], 4, 2, 64, torch.bfloat16)
    at = _offsets([20])
    for bad, message in [
        (dict(q=q.float()), "bf16 or fp16"), (dict(k=k.half(), v=v.half()), "must be torch.bfloat16"),
        (dict(k=k[:, :, :56], v=v[:, :, :56]), "q's dim"), (dict(v=v[:10]), "one shape"),
        (dict(k=k[:, :1].expand(20, 3, 64), v=v[:, :1].expand(20, 3, 64)), "multiple of k's"),
        (dict(q=q[..., 4:], k=k[..., 4:], v=v[..., 4:]), "multiple of 8"),
        (dict(q=q.transpose(1, 2)), "multiple of 8|last dimension"), (dict(q_offsets=at.long()), "int32"),
        (dict(k_offsets=_offsets([10, 10])), "one entry more"), (dict(scale=-1.0), "positive"),
        (dict(scale=float("nan")), "positive"), (dict(out=q[:10]), "q's shape"),
        (dict(lse=torch.empty(20, 4, dtype=torch.float64, device="cuda")), "fp32"), (dict(k=k[:10], v=v[:10]), "k_offsets"),
    ]:
        args = dict(q=q, k=k, v=v, q_offsets=at) | bad
        with pytest.raises(ValueError, match=message):
            prompt_attention(**args)
    with pytest.raises(RuntimeError, match="GPU only"):
        prompt_attention(q.cpu(), k, v, at)
