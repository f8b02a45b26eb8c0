"""The decoding example: one verified tree gives the tokens that greedy decoding
gives a token at a time, and leaves the same rows in the cache."""
import pytest
import torch

from afterimage_amd.examples import verify_tree

pytestmark = pytest.mark.gpu


def _rows(cache, slot, layer):
    n, page = int(cache.lengths[slot]), cache.page_size
    at = torch.arange(n, device="cuda")
    pages = cache.page_table[slot, (at // page)].long()
    return cache.pool[layer][:, pages, :, at % page]


def test_verified_tree_equals_greedy_decoding():
    got = verify_tree.run()
    decoded, cache = got["decoded"], got["cache"]
    # The accepted path is the decoded text, up to its last token (whose own pass greedy decoding left out).
    assert got["accepted"] == decoded.tolist()
    n = decoded.shape[0]
    assert cache.lengths.tolist()[n:] == [x + 1 for x in cache.lengths.tolist()[:n]]
    for b in range(n):
        for layer in range(cache.n_layers):
            a, c = _rows(cache, b, layer), _rows(cache, n + b, layer)[:int(cache.lengths[b])]
            # Two passes of a bf16 model over the same tokens: rows of a few units, a few roundings apart.
            assert (a.float() - c.float()).abs().max().item() <= 0.1
    prefix = int(cache.lengths[0]) // cache.page_size * cache.page_size
    assert prefix > 0 and torch.equal(cache.page_table[0, :1], cache.page_table[n, :1])


def test_the_example_runs_as_a_command(capsys):
    verify_tree.main()
    out = capsys.readouterr().out
    assert out.count("accepted from its tree") == 3 and "pages in use" in out
