"""The serving engine and the operators' plain forms where they can go wrong, on the CPU."""
import math

import pytest
import torch

from tests.test_serving_cpu import _model


@pytest.mark.parametrize("method", ["dense", "gdn_hybrid_swa"])
@pytest.mark.parametrize("fault", ["pool", "limit"])
def test_a_refused_reservation_takes_nothing(method, fault):
    """Rows before the one that cannot be served want a page too; nothing of the cache moves, and after a release the same
    call gives what a cache that never refused gives."""
    from nexttransformer_b200.inference import PagedCache, decode_paged
    c, m = _model(method)
    torch.manual_seed(4)
    ids = torch.randint(0, c.vocab_size, (3, 16))
    new = torch.randint(0, c.vocab_size, (3, 2))
    calm, cache = (PagedCache(m, 3, 48, page=16, pages=n) for n in (9, 4 if fault == "pool" else 9))
    for x in (calm, cache):
        decode_paged(m, ids, x)
    if fault == "limit":                       # row 2 stands at the cache's end
        for x in (calm, cache):
            decode_paged(m, ids, x, [0, 0, 16])
            decode_paged(m, ids, x, [0, 0, 16])

    def books():
        return [list(h) for h in cache.held], list(cache.free), list(cache.lengths), cache.table.clone(), cache.start.clone()
    before = books()
    with pytest.raises((RuntimeError, ValueError), match="no free pages" if fault == "pool" else "pass the cache"):
        decode_paged(m, new, cache)
    for a, b in zip(before, books()):
        assert torch.equal(a, b) if torch.is_tensor(a) else a == b
    cache.release(2)
    calm.release(2)
    counts = [2, 2, 0]
    for _ in range(2):
        assert torch.equal(decode_paged(m, new, cache, counts)[:2], decode_paged(m, new, calm, counts)[:2])
    assert sorted(cache.free + sum(cache.held, [])) == list(range(len(cache.free) + sum(map(len, cache.held))))
