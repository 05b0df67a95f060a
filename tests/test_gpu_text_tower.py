"""GPU: a text tower's attention half as it is served, the ops together: 4-bit projections, rotation into the
paged cache, attention over it, 4-bit output projection; prompts in chunks, then tokens one by one, a step
captured once and replayed.  Every stage is held to its 64-bit form on the inputs that it was given."""
import ctypes as C
import math

import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDTH, GROUP, PAGE = 8, 2, 128, 512, 64, 16
SCALE = 1.0 / math.sqrt(DIM)


class Weight:
    def __init__(self, gpu, rng, outputs, inputs):
        w = R.random_bf16(rng, outputs, inputs, std=1.0 / math.sqrt(inputs))
        self.words = np.zeros((outputs, inputs // 8), np.uint32)
        self.scales = np.zeros((outputs, inputs // GROUP), np.uint16)
        assert gpu.lib.qw_w4_quantize_host(abi._ptr(w), outputs, inputs, GROUP, abi._ptr(self.words),
                                           abi._ptr(self.scales))
        self.on = gpu.u32(self.words), gpu.bf16(self.scales)
        self.outputs, self.inputs = outputs, inputs

    def check(self, x, got):
        R.check_linear(got, *R.linear_w4(x, self.words, self.scales, None, None, GROUP))


class Layer:
    """One layer of a batch of sequences over one cache."""

    def __init__(self, gpu, rng, batch, most_tokens, width):
        self.gpu, self.batch, self.width, self.most = gpu, batch, width, most_tokens
        self.wq, self.wk, self.wv = (Weight(gpu, rng, n * DIM, WIDTH) for n in (HEADS, KV, KV))
        self.wo = Weight(gpu, rng, WIDTH, HEADS * DIM)
        self.freq = np.zeros(DIM // 2, np.float32)
        magnitude = C.c_float()
        assert gpu.lib.qw_rotary_frequencies_host(DIM, 1e6, 3, 4.0, 64, abi._ptr(self.freq), C.byref(magnitude))
        self.magnitude = magnitude.value
        pages = batch * width
        self.table = rng.permutation(pages).astype(np.uint32).reshape(batch, width)
        shape = pages * PAGE * KV * DIM
        self.keys, self.values = (gpu.bf16(np.full(shape, 0x7fc0, np.uint16)) for _ in range(2))  # NaN
        self.table_t, self.freq_t = gpu.u32(self.table), gpu.f32(self.freq)
        self.start_t, self.len_t = gpu.u32(np.zeros(batch + 1)), gpu.u32(np.zeros(batch))
        self.x, self.y = gpu.new_bf16(most_tokens * WIDTH), gpu.new_bf16(most_tokens * WIDTH)
        self.q, self.turned, self.o = (gpu.new_bf16(most_tokens * HEADS * DIM) for _ in range(3))
        self.k, self.v = (gpu.new_bf16(most_tokens * KV * DIM) for _ in range(2))
        self.length = np.zeros(batch, np.int64)
        # What the cache should hold, from the stages' own outputs.
        self.host_k = np.zeros((batch, width * PAGE, KV, DIM), np.uint16)
        self.host_v = np.zeros_like(self.host_k)
        self.pinned = gpu.lib.qw_gpu_host_alloc(4 * (2 * batch + 1))

    def lengths(self, new):
        """The step's token ranges and cache lengths, in stream order."""
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        length = (self.length + new).astype(np.uint32)
        C.memmove(self.pinned, start.ctypes.data, start.nbytes)
        C.memmove(self.pinned + start.nbytes, length.ctypes.data, length.nbytes)
        lib, g = self.gpu.lib, self.gpu.handle
        self.gpu.check(lib.qw_gpu_tensor_write_lane(g, self.start_t, self.pinned, self.batch + 1, 0))
        self.gpu.check(lib.qw_gpu_tensor_write_lane(g, self.len_t, self.pinned + start.nbytes, self.batch, 0))

    def enqueue(self, tokens, max_new):
        lib, g = self.gpu.lib, self.gpu.handle
        for out, w in ((self.q, self.wq), (self.k, self.wk), (self.v, self.wv)):
            self.gpu.check(lib.qw_gpu_linear_w4_bf16(g, out, self.x, *w.on, None, None, tokens, WIDTH, w.outputs, GROUP))
        self.gpu.check(lib.qw_gpu_rotary_append_bf16(
            g, self.turned, self.keys, self.values, self.q, self.k, self.v, None, self.freq_t, self.table_t,
            self.start_t, self.len_t, self.batch, tokens, self.width, PAGE, HEADS, KV, DIM, DIM, 1, self.magnitude))
        self.gpu.check(lib.qw_gpu_paged_attention_bf16(
            g, self.o, self.turned, self.keys, self.values, self.table_t, self.start_t, self.len_t, self.batch, tokens,
            max_new, self.width, PAGE, HEADS, KV, DIM, SCALE))
        self.gpu.check(lib.qw_gpu_linear_w4_bf16(g, self.y, self.o, *self.wo.on, None, None, tokens, HEADS * DIM, WIDTH,
                                                 GROUP))

    def check(self, x, new):
        n = int(new.sum())
        read = lambda t, heads: self.gpu.read_bf16(t, n * heads * DIM).reshape(n, heads, DIM)  # noqa: E731
        q, turned, o = (read(t, HEADS) for t in (self.q, self.turned, self.o))
        k, v = read(self.k, KV), read(self.v, KV)
        self.wq.check(x, q.reshape(n, -1))
        self.wk.check(x, k.reshape(n, -1))
        self.wv.check(x, v.reshape(n, -1))
        pool_k = self.gpu.read_bf16(self.keys, self.batch * self.width * PAGE * KV * DIM).reshape(-1, PAGE, KV, DIM)
        pool_v = self.gpu.read_bf16(self.values, pool_k.size).reshape(pool_k.shape)
        at = 0
        for b, count in enumerate(new):
            rows = self.length[b] + np.arange(count)
            mine = slice(at, at + count)
            R.check_rotated(turned[mine], *R.rotate(R.wide(q[mine]), rows, self.freq, self.magnitude, True))
            new_k = pool_k[self.table[b, rows // PAGE], rows % PAGE]
            R.check_rotated(new_k, *R.rotate(R.wide(k[mine]), rows, self.freq, self.magnitude, True))
            self.host_k[b, rows], self.host_v[b, rows] = new_k, v[mine]
            every = np.arange(self.length[b] + count)
            assert (pool_k[self.table[b, every // PAGE], every % PAGE] == self.host_k[b, every]).all()
            assert (pool_v[self.table[b, every // PAGE], every % PAGE] == self.host_v[b, every]).all()
            at += count
        self.length += new
        cache = R.Cache.__new__(R.Cache)
        cache.__dict__.update(new=new, length=self.length, batch=self.batch, page_rows=PAGE, kv_heads=KV, table=self.table,
                              start=np.concatenate([[0], np.cumsum(new)]), k=pool_k, v=pool_v)
        exact, size, _ = R.attention(cache, turned, SCALE)
        R.check_attention(o, exact, size)
        self.wo.check(o.reshape(n, -1), self.gpu.read_bf16(self.y, n * WIDTH).reshape(n, WIDTH))

    def free(self):
        self.gpu.lib.qw_gpu_host_free(self.pinned)


def test_prompts_in_chunks_then_tokens_one_by_one():
    rng = np.random.default_rng(0)
    with abi.Gpu() as gpu:
        layer = Layer(gpu, rng, 3, 256, 20)
        steps = [[100, 37, 1], [90, 0, 60], [1, 1, 1], [1, 20, 1], [5, 2, 3]]
        for new in steps:
            new = np.array(new)
            x = R.random_bf16(rng, int(new.sum()), WIDTH)
            gpu.write_bf16(layer.x, x)
            gpu.begin()
            layer.lengths(new)
            layer.enqueue(len(x), int(new.max()))
            gpu.submit()
            layer.check(x, new)
        # Generation: one step captured, replayed with the lengths written before each.
        new = np.ones(3, np.int64)
        gpu.begin()
        gpu.check(gpu.lib.qw_gpu_graph_begin(gpu.handle))
        layer.enqueue(3, 1)
        graph = gpu.lib.qw_gpu_graph_end(gpu.handle)
        gpu.check(graph)
        gpu.submit()
        for _ in range(18):
            x = R.random_bf16(rng, 3, WIDTH)
            gpu.write_bf16(layer.x, x)
            gpu.begin()
            layer.lengths(new)
            gpu.check(gpu.lib.qw_gpu_graph_launch(gpu.handle, graph))
            gpu.submit()
            layer.check(x, new)
        gpu.lib.qw_gpu_graph_free(graph)
        layer.free()


def test_two_contexts_at_once():
    """Each context has its stream and its workspace: chains of two, open at the same time, do not meet."""
    rng = np.random.default_rng(1)
    with abi.Gpu() as one, abi.Gpu() as two:
        layers = [Layer(g, rng, 2, 128, 40) for g in (one, two)]
        for new in ([60, 64], [1, 1], [1, 1], [50, 1]):
            new = np.array(new)
            xs = [R.random_bf16(rng, int(new.sum()), WIDTH) for _ in layers]
            for layer, x in zip(layers, xs):
                layer.gpu.write_bf16(layer.x, x)
                layer.gpu.begin()
                layer.lengths(new)
            for _ in range(4):
                for layer, x in zip(layers, xs):
                    layer.enqueue(len(x), int(new.max()))
            for layer in layers:
                layer.gpu.submit()
            for layer, x in zip(layers, xs):
                layer.check(x, new)
        for layer in layers:
            layer.free()


def test_two_graphs_share_the_workspace():
    """Two captured steps of one context, replayed in turn within a chain."""
    rng = np.random.default_rng(2)
    with abi.Gpu() as gpu:
        tensors, graphs, wants = [], [], []
        for new, length, kv in (([1, 1], [3000, 40], 2), ([70], [500], 4)):
            cache = R.Cache(rng, new, length, 16, kv)
            q = R.random_bf16(rng, cache.tokens, 8, 128)
            on = (*cache.upload(gpu), gpu.bf16(q), gpu.new_bf16(q.size))
            call = lambda: gpu.check(gpu.lib.qw_gpu_paged_attention_bf16(  # noqa: E731
                gpu.handle, on[6], on[5], *on[:5], cache.batch, cache.tokens, int(max(new)), cache.width, 16, 8, kv,
                128, SCALE))
            gpu.begin()
            call()
            gpu.submit()
            gpu.begin()
            gpu.check(gpu.lib.qw_gpu_graph_begin(gpu.handle))
            call()
            graphs.append(gpu.lib.qw_gpu_graph_end(gpu.handle))
            gpu.submit()
            wants.append((q.size, gpu.read_bf16(on[6], q.size)))
            R.check_attention(wants[-1][1].reshape(q.shape), *R.attention(cache, q, SCALE)[:2])
            tensors.append(on)
        for on, (n, _) in zip(tensors, wants):
            gpu.write_bf16(on[6], np.zeros(n, np.uint16))
        gpu.begin()
        for _ in range(5):
            for graph in graphs:
                gpu.check(gpu.lib.qw_gpu_graph_launch(gpu.handle, graph))
        gpu.submit()
        for on, (n, want) in zip(tensors, wants):
            assert (gpu.read_bf16(on[6], n) == want).all()
        for graph in graphs:
            gpu.lib.qw_gpu_graph_free(graph)
