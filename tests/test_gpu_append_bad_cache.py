"""GPU: new tokens whose place in the cache cannot be told are not written anywhere: the pools are another
sequence's too, and outlive the call that reports the fault."""
import numpy as np
import pytest

import text_tower_ref as R
from test_gpu_rotary import append, check_append

pytestmark = pytest.mark.gpu
UNTOUCHED = 0x4321


def lost(cache, what):
    """Spoils the cache's description; the tokens that then have no place."""
    start, length = cache.start.astype(np.int64), cache.length
    if what == "page":
        # one page of the second sequence: those of its new tokens that lie in it
        page = (length[1] - 1) // cache.page_rows
        cache.table[1, page] = cache.pages
        rows = length[1] - cache.new[1] + np.arange(cache.new[1])
        return start[1] + np.flatnonzero(rows // cache.page_rows == page)
    if what == "far page":
        cache.table[2, (length[2] - cache.new[2]) // cache.page_rows:] = 0xffffffff
        return np.arange(start[2], start[3])
    if what == "length":
        cache.length = length.copy()
        cache.length[1] = cache.width * cache.page_rows + 5
        return np.arange(start[1], start[2])
    if what == "far length":
        cache.length = length.astype(np.uint32)
        cache.length[1] = 0xffffffff
        return np.arange(start[1], start[2])
    if what == "end":
        cache.start[3] = cache.tokens + 1
        return np.arange(start[2], start[3])
    assert what == "start"  # the first sequence's end and the second's beginning
    cache.start[1] = 0xfffffff0
    return np.arange(start[0], start[2])


@pytest.mark.parametrize("what", ["page", "far page", "length", "far length", "end", "start"])
@pytest.mark.parametrize("new,length", [([1, 1, 1], [20, 30, 40]), ([2, 20, 3], [20, 36, 50]),
                                        ([3, 400, 2], [40, 500, 18])])
def test_tokens_without_a_place_are_not_written(gpu, new, length, what):
    rng = np.random.default_rng(sum(new))
    cache = R.Cache(rng, new, length, 16, 2)
    # Entries past a sequence's last page may name pages, here other sequences' live ones.
    for b in range(3):
        cache.table[b, -(-length[b] // 16):] = cache.table[(b + 1) % 3, 0]
    q = R.random_bf16(rng, cache.tokens, 4, 128)
    k, v = R.random_bf16(rng, cache.tokens, 2, 128), R.random_bf16(rng, cache.tokens, 2, 128)
    freq = np.ones(64, np.float32)
    good = np.ones(cache.tokens, bool)
    true = R.Cache.__new__(R.Cache)
    true.__dict__.update(cache.__dict__, table=cache.table.copy(), start=cache.start.copy())
    good[lost(cache, what)] = False
    ok, error, got = append(gpu, cache, q, k, v, freq, 1.0, 128, True)
    assert not ok and "sequence" in error
    out, keys, values = got
    want_k, want_v = cache.k.copy(), cache.v.copy()
    for b in range(3):
        lo, hi = int(true.start[b]), int(true.start[b + 1])
        tokens = np.arange(lo, hi)
        row = true.length[b] - (hi - lo) + np.arange(hi - lo)
        tokens, row = tokens[good[tokens]], row[good[tokens]]
        at = true.table[b, row // 16], row % 16
        if len(tokens):
            R.check_rotated(out[tokens], *R.rotate(R.wide(q[tokens]), row, freq, 1.0, True))
            R.check_rotated(keys[at], *R.rotate(R.wide(k[tokens]), row, freq, 1.0, True))
        want_k[at], want_v[at] = keys[at], v[tokens]
    assert (keys == want_k).all() and (values == want_v).all()
    assert (out[~good] == UNTOUCHED).all()
    # and the context keeps working
    again = append(gpu, true, q, k, v, freq, 1.0, 128, True)
    assert again[0], again[1]
    check_append(true, again[2], q, k, v, freq, 1.0, True, UNTOUCHED)
