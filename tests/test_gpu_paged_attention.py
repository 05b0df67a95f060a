"""GPU: attention of new tokens over the paged cache against its 64-bit form."""
import ctypes as C
import math

import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128.0)
UNTOUCHED = 0x4321


def enqueue(gpu, cache, out, q, tensors, heads, max_new=None, scale=SCALE):
    kp, vp, table, start, length = tensors
    most = max(1, int(cache.new.max())) if max_new is None else max_new
    gpu.check(gpu.lib.qw_gpu_paged_attention_bf16(
        gpu.handle, out, q, kp, vp, table, start, length, cache.batch, cache.tokens, most, cache.width,
        cache.page_rows, heads, cache.kv_heads, 128, scale), "paged attention")


def attend(gpu, cache, q, max_new=None, scale=SCALE):
    tensors = cache.upload(gpu)
    qt, out = gpu.bf16(q), gpu.bf16(np.full_like(q, UNTOUCHED))
    gpu.begin()
    enqueue(gpu, cache, out, qt, tensors, q.shape[1], max_new, scale)
    ok = gpu.lib.h3_gpu_submit(gpu.handle)
    error = gpu.error()
    got = gpu.read_bf16(out, q.size).reshape(q.shape)
    for t in (*tensors, qt, out):
        gpu.free(t)
    return ok, error, got


def check(cache, got, q, scale=SCALE):
    exact, size, real = R.attention(cache, q, scale)
    R.check_attention(got[real], exact[real], size[real])
    assert (got[~real] == UNTOUCHED).all()


CASES = [
    # one token of each sequence
    ([1], [1], 16, 32, 8), ([1], [16], 16, 32, 8), ([1], [17], 16, 8, 1), ([1], [2000], 64, 32, 8),
    ([1, 1, 1], [5, 1000, 129], 16, 28, 4), ([1] * 9, list(range(1, 400, 45)), 32, 24, 24),
    ([1] * 150, [33 + i % 70 for i in range(150)], 16, 4, 2),
    # many short ones: a warp for a unit
    ([1] * 300, [i % 70 for i in range(300)], 16, 32, 8), ([1] * 400, [90 + i % 40 for i in range(400)], 64, 24, 24),
    ([4] * 200, [4 + 3 * i % 60 for i in range(200)], 16, 32, 8),
    ([1, 2, 3] * 100, [7 * i % 50 for i in range(300)], 32, 24, 24),
    ([16] * 150, [16 + i for i in range(150)], 16, 5, 5),
    # a few
    ([2, 3, 1], [2, 77, 500], 16, 32, 8), ([4, 4], [300, 4], 128, 16, 2), ([5], [999], 256, 8, 8),
    ([7, 0, 2, 9], [40, 33, 2, 9], 16, 6, 2), ([1, 1], [0, 3], 16, 4, 4),
    # chunks: at, before and behind the tiles' borders
    ([16], [16], 16, 8, 2), ([31], [200], 32, 8, 2), ([32], [32], 16, 8, 2), ([33], [161], 64, 8, 2),
    ([64], [128], 128, 4, 1), ([65], [129], 16, 4, 1), ([127], [127], 16, 3, 3), ([128], [500], 256, 2, 2),
    ([129], [130], 32, 2, 1), ([300], [700], 16, 7, 1), ([257], [257], 4096, 5, 1),
    # both in one batch
    ([1, 200, 1, 0, 65], [300, 260, 1, 7, 65], 16, 8, 2), ([90, 1, 1, 140], [90, 513, 128, 1000], 64, 6, 2),
]


@pytest.mark.parametrize("new,length,page,heads,kv", CASES)
def test_attention(gpu, new, length, page, heads, kv):
    rng = np.random.default_rng(sum(length) + page + heads)
    cache = R.Cache(rng, new, length, page, kv, tail=5)
    q = R.random_bf16(rng, cache.tokens, heads, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)


@pytest.mark.parametrize("new,heads,kv", [
    ([5] * 200 + [1] * 300, 32, 8), ([33, 64, 65] * 25, 32, 8), ([20] * 60, 24, 24), ([1, 40] * 130, 8, 8)])
def test_more_units_than_ctas(gpu, new, heads, kv):
    """A CTA of the kernel for chunks takes several units, whole and divided in halves."""
    rng = np.random.default_rng(len(new))
    length = [max(0, n + int(x)) for n, x in zip(new, rng.integers(-40, 300, len(new)))]
    cache = R.Cache(rng, new, length, 16, kv, tail=3)
    q = R.random_bf16(rng, cache.tokens, heads, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)


@pytest.mark.parametrize("max_new", [1, 3, 100, 5000])
def test_max_new_only_chooses_kernels(gpu, max_new):
    rng = np.random.default_rng(2)
    cache = R.Cache(rng, [1, 70, 3, 200], [400, 300, 3, 210], 16, 2, tail=2)
    q = R.random_bf16(rng, cache.tokens, 8, 128)
    ok, error, got = attend(gpu, cache, q, max_new)
    assert ok, error
    check(cache, got, q)


@pytest.mark.parametrize("new,length", [([1, 1], [37, 129]), ([3], [50]), ([100, 1], [333, 20]), ([150], [150])])
@pytest.mark.parametrize("stale", [0x7fc0, 0x7f80, 0xff80, 0xff7f])
def test_rows_past_the_end_may_hold_anything(gpu, new, length, stale):
    """NaN, infinities, the lowest value in pages' unused rows and in unused pages."""
    rng = np.random.default_rng(3)
    cache = R.Cache(rng, new, length, 32, 2, stale=stale)
    q = R.random_bf16(rng, cache.tokens, 8, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)


@pytest.mark.parametrize("new,length", [([40], [25]), ([5, 2], [3, 0]), ([200, 1], [130, 1])])
def test_tokens_without_a_row_store_zeros(gpu, new, length):
    rng = np.random.default_rng(4)
    cache = R.Cache(rng, new, length, 16, 2, tail=1)
    q = R.random_bf16(rng, cache.tokens, 4, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)
    for b, n in enumerate(new):
        lo = int(cache.start[b])
        assert (got[lo:lo + max(0, n - length[b])] == 0).all()


@pytest.mark.parametrize("new,length", [([1], [3000]), ([60], [900]), ([200], [260])])
def test_large_scores(gpu, new, length):
    """Scores in the hundreds: the running maximum moves, weights underflow."""
    rng = np.random.default_rng(5)
    cache = R.Cache(rng, new, length, 64, 2)
    order = cache.rows(0)
    # keys that grow towards the end, so that every tile raises the maximum
    grow = np.linspace(0.05, 6.0, length[0])[:, None, None]
    cache.k[order] = abi.f32_to_bf16((R.wide(cache.k[order]) * grow).astype(np.float32))
    q = R.random_bf16(rng, cache.tokens, 8, 128, std=3.0)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    exact, size, real = R.attention(cache, q, SCALE)
    # scores of up to 400 in fp32: 128 products, each sum within 2^-23 of magnitudes up to 2000
    err = np.abs(R.wide(got) - exact)
    assert (err <= R.HALF_STEP * np.abs(exact) + (R.HALF_STEP + 2.0 ** -8) * size).all(), err.max()


def test_a_page_twice_and_shared_pages(gpu):
    rng = np.random.default_rng(6)
    cache = R.Cache(rng, [1, 1, 40], [64, 64, 100], 16, 2)
    cache.table[1, :3] = cache.table[0, :3]  # a common beginning
    cache.table[2, 2] = cache.table[2, 1]
    q = R.random_bf16(rng, cache.tokens, 8, 128)
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)


@pytest.mark.parametrize("new", [[1, 1, 1], [2, 90, 200]])
def test_twice_the_same_bits_and_other_batches_between(gpu, new):
    rng = np.random.default_rng(7)
    cache = R.Cache(rng, new, [2500, 700, 1200], 16, 8)
    other = R.Cache(rng, [1] * 5, [9, 3000, 40, 2, 800], 32, 4)
    q, q2 = R.random_bf16(rng, cache.tokens, 32, 128), R.random_bf16(rng, other.tokens, 8, 128)
    first = attend(gpu, cache, q)
    attend(gpu, other, q2)
    again = attend(gpu, cache, q)
    assert first[0] and again[0] and (first[2] == again[2]).all()


@pytest.mark.parametrize("what", ["page", "start", "end", "length"])
@pytest.mark.parametrize("new", [[2, 3], [1, 100]])
def test_a_bad_cache_is_reported(gpu, what, new):
    """Clamped to what is there, and said at submit; the context keeps working."""
    rng = np.random.default_rng(8)
    cache = R.Cache(rng, new, [20, 130], 16, 2)
    q = R.random_bf16(rng, cache.tokens, 4, 128)
    good = attend(gpu, cache, q)
    assert good[0]
    table, start, length = cache.table.copy(), cache.start.copy(), cache.length.copy()
    if what == "page":
        cache.table[1, 3] = 0xfffffff0
    elif what == "start":
        cache.start[1] = 1000
    elif what == "end":
        cache.start[2] += 1
    else:
        cache.length[0] = 0xffffffff
        cache.table[0] = 0
    ok, error, _ = attend(gpu, cache, q)
    assert not ok and "sequence" in error
    cache.table, cache.start, cache.length = table, start, length
    again = attend(gpu, cache, q)
    assert again[0] and (good[2] == again[2]).all()


@pytest.mark.parametrize("new", [[1, 1], [70, 1]])
def test_a_captured_step_takes_new_lengths(gpu, new):
    rng = np.random.default_rng(9)
    cache = R.Cache(rng, new, [900, 600], 16, 2)
    q = R.random_bf16(rng, cache.tokens, 8, 128)
    tensors = cache.upload(gpu)
    qt, out = gpu.bf16(q), gpu.new_bf16(q.size)
    gpu.begin()
    enqueue(gpu, cache, out, qt, tensors, 8)
    gpu.submit()
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_graph_begin(gpu.handle))
    enqueue(gpu, cache, out, qt, tensors, 8)
    graph = gpu.lib.qw_gpu_graph_end(gpu.handle)
    gpu.check(graph)
    gpu.submit()
    host = gpu.lib.qw_gpu_host_alloc(8)
    for lengths in ([900, 600], [80, 599], [100, 1]):
        cache.length = np.asarray(lengths)
        C.memmove(host, np.asarray(lengths, np.uint32).ctypes.data, 8)
        gpu.begin()
        gpu.check(gpu.lib.qw_gpu_tensor_write_lane(gpu.handle, tensors[4], host, 2, 0))
        gpu.check(gpu.lib.qw_gpu_graph_launch(gpu.handle, graph))
        gpu.submit()
        got = gpu.read_bf16(out, q.size).reshape(q.shape)
        check(cache, got, q)
    gpu.lib.qw_gpu_host_free(host)
    gpu.lib.qw_gpu_graph_free(graph)
    for t in (*tensors, qt, out):
        gpu.free(t)


def test_a_first_call_inside_a_capture_is_refused():
    with abi.Gpu() as gpu:
        rng = np.random.default_rng(10)
        cache = R.Cache(rng, [1], [20], 16, 1)
        q = R.random_bf16(rng, cache.tokens, 2, 128)
        tensors = cache.upload(gpu)
        qt, out = gpu.bf16(q), gpu.new_bf16(q.size)
        gpu.begin()
        gpu.check(gpu.lib.qw_gpu_graph_begin(gpu.handle))
        with pytest.raises(abi.GpuError, match="before capturing"):
            enqueue(gpu, cache, out, qt, tensors, 2)
        gpu.lib.qw_gpu_graph_free(gpu.lib.qw_gpu_graph_end(gpu.handle))
        assert not gpu.lib.h3_gpu_submit(gpu.handle)
        ok, error, got = attend(gpu, cache, q)
        assert ok, error
        check(cache, got, q)


def test_agrees_with_the_whole_prompt(gpu):
    """A prompt in one causal call, and in chunks over the cache: the same attention."""
    rng = np.random.default_rng(11)
    total, heads, kv = 300, 8, 2
    whole = R.Cache(rng, [total], [total], 16, kv)
    q = R.random_bf16(rng, total, heads, 128)
    k, v = whole.k[whole.rows(0)], whole.v[whole.rows(0)]
    ts = [gpu.new_bf16(q.size), gpu.bf16(q), gpu.bf16(k), gpu.bf16(v)]
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_gqa_causal_bf16(gpu.handle, *ts, total, heads, kv, 128, SCALE))
    gpu.submit()
    want = gpu.read_bf16(ts[0], q.size).reshape(q.shape)
    for t in ts:
        gpu.free(t)
    at = 0
    for n in (150, 1, 1, 20, 128):
        part = R.Cache.__new__(R.Cache)
        part.__dict__.update(whole.__dict__, new=np.array([n]), length=np.array([at + n]), tokens=n,
                             start=np.array([0, n], np.uint32))
        ok, error, got = attend(gpu, part, q[at:at + n])
        assert ok, error
        # each is within half a step and the weights' half steps of the definition
        size = R.attention(part, q[at:at + n], SCALE)[1]
        d = np.abs(R.wide(got) - R.wide(want[at:at + n]))
        assert (d <= 2 * (R.HALF_STEP * np.abs(R.wide(got)) + (R.HALF_STEP + 2.0 ** -11) * size)).all()
        at += n


@pytest.mark.parametrize("new,length", [(300, 1500), (40, 1500), (100, 6000)])
def test_bounded_waits_run_out_cleanly(gpu, new, length):
    """Key tiles from the second on stay away (nothing is in flight): the waits behind them run out, the
    submit says so and the next call is right."""
    rng = np.random.default_rng(12)
    cache = R.Cache(rng, [new], [length], 32, 2)
    q = R.random_bf16(rng, cache.tokens, 8, 128)
    gpu.check(gpu.lib.qw_gpu_debug_attention_waits(gpu.handle, 2_000_000, 1))
    try:
        ok, error, _ = attend(gpu, cache, q)
    finally:
        gpu.lib.qw_gpu_debug_attention_waits(gpu.handle, 0, 0)
    assert not ok and "wait ran out" in error
    ok, error, got = attend(gpu, cache, q)
    assert ok, error
    check(cache, got, q)
