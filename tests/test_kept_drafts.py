"""PagedKVCache.keep on the CPU: paths of drafted tokens moved up in the pages,
against a list of tokens per sequence, and its refusals."""
import ctypes
import random

import pytest
import torch

from santa_amd import paged
from test_paged import _cache, _contents, _write


@pytest.mark.parametrize("seed", range(6))
def test_keep(seed):
    """Random paths of random drafts, among them none and all, sequences with
    shared prefixes: every token's contents, the lengths and the pages in use."""
    r = random.Random(seed)
    cache = _cache(pages=120, page=8, seqs=6, max_len=160, layers=2)
    prompt, = cache.add([r.choice((0, 5, 16, 21))])
    n = cache.lengths([prompt])[0]
    _write(cache, prompt, 0, n, 0.0)
    seqs = [prompt, *cache.fork(prompt, 3)]
    want = {s: [float(i) for i in range(n)] for s in seqs}
    for step in range(1, 12):
        some = r.sample(seqs, r.randint(1, len(seqs)))
        new = [r.choice((0, 1, 3, 8, 9, 20)) for _ in some]
        cache.extend(some, new)
        for s, t in zip(some, new):
            n = len(want[s])
            _write(cache, s, n, n + t, 1000.0 * step)
        kept = [sorted(r.sample(range(t), r.choice((0, t, r.randint(0, t))))) for t in new]
        cache.keep(some, new, kept)
        for s, k in zip(some, kept):
            n = len(want[s])
            want[s] += [1000.0 * step + n + i for i in k]
        assert cache.lengths(seqs) == [len(want[s]) for s in seqs]
        for s in seqs:
            for j, got in enumerate(_contents(cache, s)):
                assert got == [x + 1000.0 * j for x in want[s]], (step, s)
            assert len(cache.pages(s)) == -(-len(want[s]) // 8)
        held = {p for s in seqs for p in cache.pages(s)}
        assert cache.used_pages == len(held)
        if max(map(len, want.values())) > 120:
            break


def test_refusals():
    """A refused call changes nothing."""
    cache = _cache(pages=30, page=8)
    a, b = cache.add([20, 9])
    _write(cache, a, 0, 20, 0.0)
    child, = cache.fork(a)
    before = ([t.clone() for t in cache.k], cache.lengths([a, b, child]), cache.used_pages, cache.pages(a))
    for args, error, text in [
        (([a], 4, [[1, 0]]), RuntimeError, "ascending"), (([a], 4, [[0, 0]]), RuntimeError, "ascending"),
        (([a], 4, [[4]]), RuntimeError, "numbers below 4"), (([a], 4, [[-1]]), RuntimeError, "numbers below 4"),
        (([a], 2, [[0, 1, 1]]), RuntimeError, "cannot stay"), (([a], 21, [[0]]), RuntimeError, "holds 20"),
        (([a], -1, [[]]), RuntimeError, "holds 20"), (([a, a], 1, [[0], [0]]), RuntimeError, "named twice"),
        (([7], 1, [[0]]), RuntimeError, "no sequence 7"), (([b, a], 3, [[1], [1]]), RuntimeError, "other sequences hold"),
        (([a], 1, [[0], [0]]), ValueError, "one entry"), (([a], [1, 1], [[0]]), ValueError, "one entry"),
        (([a], 3, [[0.5]]), ValueError, "whole"), (([a], [0.5], [[]]), ValueError, "whole"),
    ]:
        with pytest.raises(error, match=text):
            cache.keep(*args)
        assert all(torch.equal(x, y) for x, y in zip(cache.k, before[0]))
        assert (cache.lengths([a, b, child]), cache.used_pages, cache.pages(a)) == before[1:]
    cache.keep([a], 4, [[0, 1]])  # in place: nothing that the child holds is written
    assert cache.lengths([a, child]) == [18, 20]
    cache.keep([], 1, [])
    lib, none = paged._lib(), ctypes.POINTER(ctypes.c_int)()
    assert lib.santa_pages_keep(None, none, none, none, none, 0) == 1
    assert lib.santa_pages_keep(cache._pages, none, none, none, none, 1) == 1
    assert lib.santa_pages_apply_moves(None, None, 0, 32, 32, None) == 1
    wide = _cache(page=32)
    c, = wide.add([9])
    wide.keep([c], 8, [[7]])
    pool = (ctypes.c_void_p * 1)(16)
    assert lib.santa_pages_apply_moves(wide._pages, pool, 1, 16 * 9, 16 * 9, None) == 1  # not whole rows
    assert b"is not 32 rows" in lib.santa_last_error()
