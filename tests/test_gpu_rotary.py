"""GPU: rotary positions, alone and into a paged cache, against their 64-bit form."""
import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi

pytestmark = pytest.mark.gpu


def rotary(gpu, q, k, positions, freq, magnitude, rotary_dim, halves, in_place=False):
    tokens, heads, dim = q.shape
    qt, pt, ft = gpu.bf16(q), gpu.u32(positions), gpu.f32(freq)
    qo = qt if in_place else gpu.new_bf16(q.size)
    kt = gpu.bf16(k) if k is not None else None
    ko = kt if in_place or k is None else gpu.new_bf16(k.size)
    kv = k.shape[1] if k is not None else 0
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_rotary_bf16(gpu.handle, qo, ko, qt, kt, pt, ft, tokens, heads, kv, dim, rotary_dim,
                                         int(halves), magnitude), "rotary")
    gpu.submit()
    got = [gpu.read_bf16(qo, q.size).reshape(q.shape)]
    got.append(gpu.read_bf16(ko, k.size).reshape(k.shape) if k is not None else None)
    for t in {qt, pt, ft, qo, kt, ko} - {None}:
        gpu.free(t)
    return got


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,part", [
    (1, 32, 8, 128, 128), (7, 32, 8, 128, 64), (412, 32, 8, 128, 128), (3000, 5, 1, 64, 32),
    (33, 3, 3, 80, 40), (19, 4, 2, 80, 20), (21, 2, 1, 96, 24), (9, 3, 1, 256, 256), (5, 2, 2, 512, 500),
    (6, 1, 1, 2, 2), (4, 3, 2, 10, 6), (13, 28, 4, 128, 2)])
def test_rotary(gpu, tokens, heads, kv, dim, part, halves):
    rng = np.random.default_rng(tokens * dim + part)
    q, k = R.random_bf16(rng, tokens, heads, dim), R.random_bf16(rng, tokens, kv, dim)
    positions = rng.integers(0, 4000, tokens).astype(np.uint32)
    freq = (1e4 ** (-np.arange(part // 2) / (part // 2))).astype(np.float32)
    for in_place in (False, True):
        got = rotary(gpu, q, k, positions, freq, 1.25, part, halves, in_place)
        for bits, x in zip(got, (q, k)):
            R.check_rotated(bits, *R.rotate(R.wide(x), positions, freq, 1.25, halves))
            assert (bits[..., part:] == x[..., part:]).all()
    alone, _ = rotary(gpu, q, None, positions, freq, 1.25, part, halves)
    assert (alone == got[0]).all()


def test_far_positions(gpu):
    """Angles of positions near 2^32 keep their fraction of a turn."""
    rng = np.random.default_rng(1)
    positions = np.array([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31, 2 ** 32 - 1], np.uint32)
    freq = (1e6 ** (-np.arange(64) / 64)).astype(np.float32)
    q = R.random_bf16(rng, 6, 2, 128)
    got, _ = rotary(gpu, q, None, positions, freq, 1.0, 128, True)
    exact, size = R.rotate(R.wide(q), positions, freq, 1.0, True)
    R.check_rotated(got, exact, size)


def append(gpu, cache, q, k, v, freq, magnitude, part, halves, positions=None, in_place=False):
    tokens, heads, dim = q.shape
    kp, vp, table, start, length = cache.upload(gpu)
    qt, kt, vt, ft = gpu.bf16(q), gpu.bf16(k), gpu.bf16(v), gpu.f32(freq)
    pt = gpu.u32(positions) if positions is not None else None
    qo = qt if in_place else gpu.bf16(np.full_like(q, 0x4321))
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_rotary_append_bf16(
        gpu.handle, qo, kp, vp, qt, kt, vt, pt, ft, table, start, length, cache.batch, tokens, cache.width,
        cache.page_rows, heads, cache.kv_heads, dim, part, int(halves), magnitude), "append")
    ok = gpu.lib.h3_gpu_submit(gpu.handle)
    error = gpu.error()
    got = (gpu.read_bf16(qo, q.size).reshape(q.shape), gpu.read_bf16(kp, cache.k.size).reshape(cache.k.shape),
           gpu.read_bf16(vp, cache.v.size).reshape(cache.v.shape))
    for t in {kp, vp, table, start, length, qt, kt, vt, ft, pt, qo} - {None}:
        gpu.free(t)
    return ok, error, got


def check_append(cache, got, q, k, v, freq, magnitude, halves, untouched, positions=None):
    out, keys, values = got
    want_k, want_v, touched = cache.k.copy(), cache.v.copy(), np.zeros(cache.k.shape[:2], bool)
    real = np.zeros(len(q), bool)
    for b in range(cache.batch):
        lo, hi = int(cache.start[b]), int(cache.start[b + 1])
        row = cache.length[b] - (hi - lo) + np.arange(hi - lo)
        tokens, row = np.arange(lo, hi)[row >= 0], row[row >= 0]
        at = cache.table[b, row // cache.page_rows], row % cache.page_rows
        p = row if positions is None else positions[tokens]
        real[tokens] = True
        touched[at] = True
        want_v[at] = v[tokens]
        if len(tokens):
            R.check_rotated(out[tokens], *R.rotate(R.wide(q[tokens]), p, freq, magnitude, halves))
            R.check_rotated(keys[at], *R.rotate(R.wide(k[tokens]), p, freq, magnitude, halves))
    assert (values == want_v).all()
    assert (keys[~touched] == want_k[~touched]).all()
    assert (out[~real] == (untouched if np.isscalar(untouched) else untouched[~real])).all()


@pytest.mark.parametrize("new,length,page,heads,kv,dim,part,halves,tail", [
    ([1], [1], 16, 32, 8, 128, 128, True, 0),
    ([1] * 64, list(range(1, 2 * 64, 2)), 16, 32, 8, 128, 64, True, 3),
    ([17, 0, 1, 300], [17, 0, 40, 333], 32, 8, 1, 128, 128, False, 60),
    ([700], [1000], 64, 6, 2, 64, 64, True, 0),
    ([5, 9], [5, 100], 128, 4, 4, 80, 20, True, 1),
    ([1] * 300, [30] * 300, 16, 3, 1, 16, 16, False, 0),
    ([40, 3], [25, 3], 16, 2, 1, 128, 32, True, 2),  # more new tokens than rows
])
def test_append(gpu, new, length, page, heads, kv, dim, part, halves, tail):
    rng = np.random.default_rng(len(new) + page + dim)
    cache = R.Cache(rng, new, length, page, kv, dim, tail=tail)
    q = R.random_bf16(rng, cache.tokens, heads, dim)
    k, v = R.random_bf16(rng, cache.tokens, kv, dim), R.random_bf16(rng, cache.tokens, kv, dim)
    freq = (1e6 ** (-np.arange(part // 2) / (part // 2))).astype(np.float32)
    ok, error, got = append(gpu, cache, q, k, v, freq, 0.75, part, halves)
    assert ok, error
    check_append(cache, got, q, k, v, freq, 0.75, halves, 0x4321)
    positions = rng.integers(0, 100000, cache.tokens).astype(np.uint32)
    ok, error, got = append(gpu, cache, q, k, v, freq, 0.75, part, halves, positions, in_place=True)
    assert ok, error
    check_append(cache, got, q, k, v, freq, 0.75, halves, q, positions)


@pytest.mark.parametrize("what", ["page", "start", "end", "length"])
def test_append_reports_a_bad_cache(gpu, what):
    """Clamped to what is there, and said at submit; the context keeps working."""
    rng = np.random.default_rng(4)
    cache = R.Cache(rng, [2, 3], [20, 30], 16, 2)
    q = R.random_bf16(rng, cache.tokens, 4, 128)
    k, v = R.random_bf16(rng, cache.tokens, 2, 128), R.random_bf16(rng, cache.tokens, 2, 128)
    freq = np.ones(64, np.float32)
    good = append(gpu, cache, q, k, v, freq, 1.0, 128, True)
    assert good[0]
    table, start, length = cache.table.copy(), cache.start.copy(), cache.length.copy()
    if what == "page":
        cache.table[1, 1] = cache.pages
    elif what == "start":
        cache.start[1] = 9
    elif what == "end":
        cache.start[2] = 6
    else:
        cache.length[0] = cache.width * 16 + 1
    ok, error, _ = append(gpu, cache, q, k, v, freq, 1.0, 128, True)
    assert not ok and "sequence" in error
    cache.table, cache.start, cache.length = table, start, length
    again = append(gpu, cache, q, k, v, freq, 1.0, 128, True)
    assert again[0] and all((a == b).all() for a, b in zip(good[2], again[2]))
