"""GPU: NaN and infinities in queries and in visible cache rows come out where the definition has them, however
a sequence's keys are divided."""
import numpy as np
import pytest

import text_tower_ref as R
from test_gpu_paged_attention import SCALE, attend

pytestmark = pytest.mark.gpu
NAN, INF, MINUS_INF = 0x7fc0, 0x7f80, 0xff80

# One token: a unit in one CTA, in several, in many; a unit to a warp; several tokens; two tiles of rows; chunks
# whole, in halves, in parts.
SHAPES = [([1], [100], 8, 2), ([1], [150], 8, 2), ([1], [3000], 8, 2), ([1], [9000], 1, 1), ([1] * 40, [60] * 40, 32, 8),
          ([3], [700], 8, 2), ([4], [3000], 16, 2), ([16], [2000], 2, 2), ([1, 30, 1], [500, 200, 900], 8, 2),
          ([60], [900], 8, 2), ([200], [260], 4, 2), ([130], [4000], 2, 1)]


def check(cache, got, q, where):
    """A row is NaN in every dimension whose formula is, and right elsewhere."""
    heads, share = q.shape[1], q.shape[1] // cache.kv_heads
    with np.errstate(invalid="ignore"):
        exact, size, real = R.attention(cache, q, SCALE)
    value = R.wide(got)
    assert where[real].any() and not where[real].all()
    assert (np.isnan(exact) == where).all()
    assert (np.isnan(value[real]) == where[real]).all()
    keep = real[:, None, None] & ~where
    err = np.abs(value[keep] - exact[keep])
    assert (err <= R.HALF_STEP * np.abs(exact[keep]) + (R.HALF_STEP + 2.0 ** -12) * size[keep]).all()
    assert heads == share * cache.kv_heads


def make(new, length, heads, kv):
    rng = np.random.default_rng(sum(length) + heads)
    cache = R.Cache(rng, new, length, 16, kv)
    return rng, cache, R.random_bf16(rng, cache.tokens, heads, 128)


@pytest.mark.parametrize("bits", [NAN, INF])
@pytest.mark.parametrize("new,length,heads,kv", SHAPES)
def test_a_query(gpu, new, length, heads, kv, bits):
    """One element of one head of one token; an infinite one makes scores of both signs."""
    if length[0] == 9000:
        new, heads = [2], 1  # (a row beside it that stays right)
    _, cache, q = make(new, length, heads, kv)
    token, head = cache.tokens - 1, heads - 1
    q[token, head, 77] = bits
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    where = np.zeros(q.shape, bool)
    where[token, head] = True
    check(cache, got, q, where)


@pytest.mark.parametrize("where", [0.0, 0.4, 0.999])
@pytest.mark.parametrize("new,length,heads,kv", [s for s in SHAPES if s[3] > 1])
def test_a_key(gpu, new, length, heads, kv, where):
    """A NaN key makes the rows that see it NaN, the masked ones of the other kv heads not."""
    _, cache, q = make(new, length, heads, kv)
    row = int(where * (length[-1] - new[-1]))
    page, r = cache.rows(len(new) - 1)
    cache.k[page[row], r[row], kv - 1, 5] = NAN
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    expected = np.zeros(q.shape, bool)
    expected[int(cache.start[-2]):int(cache.start[-1]), (kv - 1) * (heads // kv):] = True
    check(cache, got, q, expected)


@pytest.mark.parametrize("new,length,heads,kv", [s for s in SHAPES if s[3] > 1])
def test_a_run_of_keys(gpu, new, length, heads, kv):
    """Many NaN keys in a row: parts of the keys that see nothing else."""
    _, cache, q = make(new, length, heads, kv)
    old = length[-1] - new[-1]
    page, r = cache.rows(len(new) - 1)
    rows = np.arange(old // 3, old)
    cache.k[page[rows], r[rows], 0] = NAN
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    expected = np.zeros(q.shape, bool)
    expected[int(cache.start[-2]):int(cache.start[-1]), :heads // kv] = True
    check(cache, got, q, expected)


@pytest.mark.parametrize("first,count", [(0, 128), (128, 128), (256, 256)])
@pytest.mark.parametrize("new,length,heads,kv", [([1], [700], 8, 2), ([1], [3000], 8, 2), ([3], [700], 4, 1),
                                                 ([60], [3000], 8, 2), ([200], [4000], 2, 1)])
def test_all_keys_of_a_part(gpu, new, length, heads, kv, first, count):
    """A part, or a tile, of nothing but NaN keys has no maximum, and is not left out for that."""
    _, cache, q = make(new, length, heads, kv)
    page, r = cache.rows(0)
    rows = np.arange(first, first + count)
    cache.k[page[rows], r[rows], 0] = NAN
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    value = R.wide(got)
    assert np.isnan(value[:, :heads // kv]).all() and np.isfinite(value[:, heads // kv:]).all()


@pytest.mark.parametrize("where", [0.0, 0.6])
@pytest.mark.parametrize("new,length,heads,kv", SHAPES)
def test_a_value(gpu, new, length, heads, kv, where):
    """A NaN in a value is its dimension's alone."""
    _, cache, q = make(new, length, heads, kv)
    row = int(where * (length[-1] - new[-1]))
    page, r = cache.rows(len(new) - 1)
    cache.v[page[row], r[row], kv - 1, 99] = NAN
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    expected = np.zeros(q.shape, bool)
    expected[int(cache.start[-2]):int(cache.start[-1]), (kv - 1) * (heads // kv):, 99] = True
    check(cache, got, q, expected)


@pytest.mark.parametrize("new,length,heads,kv", SHAPES)
def test_keys_of_minus_infinity(gpu, new, length, heads, kv):
    """Scores of minus infinity have no weight."""
    _, cache, q = make(new, length, heads, kv)
    q[..., 3] = 0x3f80  # 1
    old = length[-1] - new[-1]
    page, r = cache.rows(len(new) - 1)
    rows = np.arange(0, old, 2) if old else np.arange(0)
    cache.k[page[rows], r[rows], 0, 3] = MINUS_INF
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    exact, size, real = R.attention(cache, q, SCALE)
    R.check_attention(got[real], exact[real], size[real])
