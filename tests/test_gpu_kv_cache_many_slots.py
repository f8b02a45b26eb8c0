"""Calls of more slots than a workgroup has threads, against the model in Python lists."""
import itertools
import random

import pytest
import torch

from tests.test_gpu_kv_cache import Pair, _ints

pytestmark = pytest.mark.gpu


class Small(Pair):
    LAYERS, HEADS, DIM = 1, 1, 8

    def append(self, seqs, counts):
        """Pair.append's rows, made at once."""
        offsets = [0, *itertools.accumulate(counts)]
        numbers = list(range(self.next, self.next + offsets[-1]))
        self.next += offsets[-1]
        rows = (torch.arange(16, device="cuda") * 7 + torch.tensor(numbers, device="cuda")[:, None] * 31) % 251
        kv = rows.view(-1, 2, 1, 8).to(self.cache.pool.dtype)
        if numbers:
            self.cache.append(0, kv[:, 0], kv[:, 1], _ints(seqs), _ints(offsets))
        return [numbers[offsets[i]:offsets[i + 1]] for i in range(len(counts))], offsets


@pytest.mark.parametrize("slots", [1025, 2048, 3000])
def test_reserve_fork_and_release(slots):
    rng = random.Random(slots)
    p = Small(n_pages=5 * slots, page=4, max_seqs=slots + 7, max_pages=6)
    seqs = list(range(slots))
    rng.shuffle(seqs)
    p.write(seqs, [rng.choice((0, 0, 1, 3, 4, 5, 9)) for _ in seqs])
    _check(p)
    # Every slot a branch of some slot, kept ones among them.
    src = [s if rng.random() < 0.2 else rng.randrange(slots + 7) for s in seqs]
    p.fork(src, seqs)
    _check(p)
    p.write(seqs, [rng.choice((0, 0, 1, 2, 6)) for _ in seqs])
    _check(p)
    p.release(seqs[:slots // 2])
    _check(p)
    p.compact()
    _check(p)


def test_too_few_pages_for_many_slots_change_nothing():
    p = Small(n_pages=1500, page=4, max_seqs=1400, max_pages=6)
    p.write(list(range(1100)), [1] * 1100)
    for step in (lambda: p.cache.reserve(_ints(list(range(1400))), _ints([4] * 1400)), lambda: p.cache.fork(_ints([0] * 401), _ints(list(range(900, 1301))))):
        step()
        with pytest.raises(RuntimeError, match="free pages"):
            p.cache.check()
        _check(p)


def _check(p):
    """Pair.check, with the pool read once."""
    c, m = p.cache, p.model
    assert c.lengths.tolist() == [len(r) for r in m.rows]
    assert c.held.tolist() == [len(x) for x in m.pages]
    assert c.page_table.tolist() == [x + [-1] * (m.max_pages - len(x)) for x in m.pages]
    assert c.refs.tolist() == m.refs()
    c.check()
    at = [(m.pages[s][j // m.page], j % m.page, number) for s, rows in enumerate(m.rows) for j, number in enumerate(rows)]
    page, slot, number = torch.tensor(at).t()
    got = c.pool[0, :, :, 0].cpu()[:, page, slot].transpose(0, 1).flatten(1)  # [rows, keys then values]
    assert torch.equal(got.long(), (torch.arange(16) * 7 + number[:, None] * 31) % 251)
