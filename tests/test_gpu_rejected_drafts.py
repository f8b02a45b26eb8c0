"""What rejected drafts leave behind in a cache in 8 bits.

Drafted rows share the scale of their 16 positions with the rows before them.
Where they raise it to S, earlier elements of at least 2^-6 S, which have 4
significant bits already, stay; those below are rounded to multiples of 2^-9 S,
by 2^-10 S at most, and stay so when the drafts are rejected. Drafts that raise
no scale leave nothing. A cache in 16 bits is as it was.
"""
import pytest
import torch

from afterimage_amd.runtime.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("larger", [0.5, 1.0, 8.0, 4096.0])
@pytest.mark.parametrize("length", [5, 16, 27])
@pytest.mark.parametrize("kept", [0, 1])
def test_earlier_rows_after_rejected_drafts(kind, larger, length, kept):
    cache = PagedKVCache.allocate(2, 4, 16, 2, 64, 1, 4, kind)
    g = torch.Generator(device="cuda").manual_seed(length)
    cache.reserve(ints([0]), ints([length + 6]))
    for layer in range(2):
        x = torch.randn(length, 2, 64, generator=g, device="cuda").bfloat16()
        x[0, :, 0] = x[-1, :, 0] = 7.0  # each block's largest, in both of its parts
        x[length // 16 * 16 if length % 16 else 0, :, 0] = 7.0
        cache.append(layer, x, -x, ints([0]), ints([0, length]))
    cache.advance(ints([0]), ints([0, length]))
    before = [cache.read(layer, ints([0]), ints([0, length]), length) for layer in range(2)]
    for layer in range(2):
        x = (torch.randn(6, 2, 64, generator=g, device="cuda").clamp(-4, 4) * larger).bfloat16()
        if larger > 1:
            x[3, :, 5] = 7.0 * larger  # of a draft that is rejected
        else:
            x.clamp_(-6.0, 6.0)
        cache.append(layer, x, -x, ints([0]), ints([0, 6]))
    cache.commit(ints([0]), ints([[0, 1]]), ints([kept]))
    cache.check()
    after = [cache.read(layer, ints([0]), ints([0, length]), length) for layer in range(2)]
    first = length // 16 * 16  # of the block that the drafts came into
    for (old, new), which in ((pair, which) for which in range(2) for pair in zip([b[which] for b in before], [a[which] for a in after])):
        assert torch.equal(old[:first], new[:first])
        if kind is torch.bfloat16 or larger <= 1:
            assert torch.equal(old, new), which
            continue
        scale = 7.0 * larger / 448.0  # 2^-6 * larger, a power of two
        old, new = old[first:].double(), new[first:].double()
        large = old.abs() >= 2.0 ** -6 * scale
        assert torch.equal(old[large], new[large])
        assert bool(((old - new).abs() <= 2.0 ** -10 * scale).all())
        if larger > 1000 and length % 16:
            assert not torch.equal(old, new)
