"""GPU: long contexts of few rows, whose units lie in the runs of up to all CTAs: every part counts."""
import numpy as np
import pytest

import text_tower_ref as R
from test_gpu_paged_attention import SCALE, attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,length,heads,kv", [
    ([1], [60000], 1, 1), ([2], [60000], 1, 1), ([3], [40000], 1, 1), ([1], [57000], 5, 1), ([2], [61003], 4, 1),
    ([2], [59990], 8, 1), ([16], [38000], 1, 1), ([1], [30011], 4, 2), ([1, 1], [25000, 31000], 8, 1)])
def test_every_part_counts(gpu, new, length, heads, kv):
    """128 keys in places of their own carry all the weight, in equal parts, and each alone has a value in one
    dimension: an element of the result is that key's weight."""
    rng = np.random.default_rng(length[0])
    cache = R.Cache(rng, new, length, 64, kv)
    base = rng.choice([-1.0, 1.0], 128)
    cache.k[:], cache.v[:] = R.random_bf16(rng, *cache.k.shape, std=0.02), 0
    for b in range(len(new)):
        page, r = cache.rows(b)
        step = (length[b] - new[b]) / 128
        for h in range(kv):
            at = (np.arange(128) * step + rng.integers(0, int(step), 128)).astype(int)
            # (a score of about 22: the other keys together weigh less than 2^-16 of these)
            cache.k[page[at], r[at], h] = R.abi.f32_to_bf16((2 * base).astype(np.float32))
            cache.v[page[at], r[at], h, rng.permutation(128)] = R.abi.f32_to_bf16(np.float32([1.0]))
    q = R.abi.f32_to_bf16(np.broadcast_to(base, (cache.tokens, heads, 128)).astype(np.float32))
    # heads and tokens differ a little
    q = R.abi.f32_to_bf16((R.wide(q) + rng.standard_normal(q.shape) * 0.02).astype(np.float32))
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    exact, size, real = R.attention(cache, q, SCALE)
    assert (exact[real] > 0.002).all()
    R.check_attention(got[real], exact[real], size[real])
    again = attend(gpu, cache, q)
    assert (again[2] == got).all()


@pytest.mark.parametrize("new,length,heads,kv", [([1], [700], 160, 1), ([3, 1], [90, 200], 130, 1), ([20], [150], 258, 2)])
def test_more_heads_than_a_tile_of_rows(gpu, new, length, heads, kv):
    """More than 128 query heads of a kv head: the kernel for few rows takes them all, whatever the tokens."""
    rng = np.random.default_rng(heads)
    cache = R.Cache(rng, new, length, 16, kv)
    q = R.random_bf16(rng, cache.tokens, heads, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    exact, size, real = R.attention(cache, q, SCALE)
    R.check_attention(got[real], exact[real], size[real])
