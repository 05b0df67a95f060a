"""GPU: linear layers with 4-bit weights against their 64-bit form."""
import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi

pytestmark = pytest.mark.gpu


def make(rng, rows, inputs, outputs, group, with_zeros, with_bias):
    words = rng.integers(0, 2 ** 32, (outputs, inputs // 8), dtype=np.uint64).astype(np.uint32)
    scales = R.random_bf16(rng, outputs, inputs // group, std=0.02)
    zeros = R.random_bf16(rng, outputs, inputs // group, std=4.0) if with_zeros else None
    if with_zeros == "whole":
        zeros = abi.f32_to_bf16(rng.integers(0, 16, (outputs, inputs // group)).astype(np.float32))
    bias = R.random_bf16(rng, outputs) if with_bias else None
    return R.random_bf16(rng, rows, inputs), words, scales, zeros, bias


def linear(gpu, x, words, scales, zeros, bias, group, guard=64):
    rows, inputs = x.shape
    outputs = len(words)
    ts = [gpu.bf16(x), gpu.u32(words), gpu.bf16(scales)]
    ts += [gpu.bf16(a) if a is not None else None for a in (zeros, bias)]
    y = gpu.bf16(np.full(rows * outputs + guard, 0x4321, np.uint16))
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_linear_w4_bf16(gpu.handle, y, *ts, rows, inputs, outputs, group), "linear")
    gpu.submit()
    got = gpu.read_bf16(y, rows * outputs + guard)
    for t in [t for t in ts if t] + [y]:
        gpu.free(t)
    assert (got[rows * outputs:] == 0x4321).all()
    return got[:rows * outputs].reshape(rows, outputs)


SIZES = [(1, 32, 1, 32), (1, 128, 16, 128), (1, 4096, 6144, 128), (2, 192, 33, 64), (3, 2208, 100, 32),
         (5, 1024, 47, 256), (8, 384, 64, 128), (9, 160, 31, 32), (13, 4096, 513, 32), (16, 640, 129, 64),
         (17, 512, 95, 128), (32, 320, 65, 64), (33, 96, 40, 32), (64, 1408, 257, 128), (100, 2048, 130, 64),
         (412, 1024, 384, 128), (300, 224, 77, 32), (17, 4096, 128, 128), (48, 8192, 260, 512), (130, 4096, 200, 64),
         (20, 2080, 1000, 32), (700, 512, 1290, 256),
         # each number of outputs for an SM that has a shape of its own
         *[(rows, 640, outputs, group) for rows in (1, 8, 11) for outputs in (2001, 3100, 6000, 9001, 10100)
           for group in (32, 64, 128)],
         # tiles of more than 128 rows
         (200, 512, 9600, 128), (140, 288, 12000, 32), (256, 192, 9600, 64), (1000, 640, 4100, 128), (257, 160, 18900, 32),
         (17, 2176, 1500, 128), (20, 2080, 1300, 32), (32, 320, 1200, 64), (30, 1024, 1184, 128)]


@pytest.mark.parametrize("with_zeros,with_bias", [(False, False), (True, True), ("whole", False)])
@pytest.mark.parametrize("rows,inputs,outputs,group", SIZES)
def test_linear(gpu, rows, inputs, outputs, group, with_zeros, with_bias):
    rng = np.random.default_rng(rows * inputs + outputs)
    x, words, scales, zeros, bias = make(rng, rows, inputs, outputs, group, with_zeros, with_bias)
    got = linear(gpu, x, words, scales, zeros, bias, group)
    R.check_linear(got, *R.linear_w4(x, words, scales, zeros, bias, group))


@pytest.mark.parametrize("rows,group", [(1, 128), (12, 32), (40, 64), (200, 128)])
def test_every_column_has_its_place(gpu, rows, group):
    """One column of x at a time: the weight's own value comes out, exactly."""
    rng = np.random.default_rng(rows)
    inputs, outputs = 256, 24
    x, words, scales, zeros, _ = make(rng, rows, inputs, outputs, group, False, False)
    scales[:] = abi.f32_to_bf16(np.float32([0.5]))
    q = R.unpack(words).astype(np.float64) - 8
    for column in list(range(0, 40)) + [127, 128, 191, 255]:
        x[:] = 0
        x[:, column] = abi.f32_to_bf16(np.float32([2.0]))
        got = R.wide(linear(gpu, x, words, scales, None, None, group))
        assert (got == q[None, :, column]).all(), column


def test_rows_do_not_mix_and_infinities_stay_in_theirs(gpu):
    rng = np.random.default_rng(7)
    for rows in (3, 15, 70):
        x, words, scales, zeros, bias = make(rng, rows, 256, 50, 64, True, False)
        clean = linear(gpu, x, words, scales, zeros, None, 64)
        x[1, 5], x[2, 200] = 0x7f80, 0x7fc0
        got = linear(gpu, x, words, scales, zeros, None, 64)
        keep = np.ones(rows, bool)
        keep[1:3] = False
        assert (got[keep] == clean[keep]).all()
        assert not np.isfinite(R.wide(got[2])).any()


def test_quantized_weights_of_the_host(gpu):
    rng = np.random.default_rng(8)
    w = R.random_bf16(rng, 70, 512, std=0.05)
    words, scales = np.zeros((70, 64), np.uint32), np.zeros((70, 4), np.uint16)
    assert abi.load().qw_w4_quantize_host(abi._ptr(w), 70, 512, 128, abi._ptr(words), abi._ptr(scales))
    x = R.random_bf16(rng, 6, 512)
    got = linear(gpu, x, words, scales, None, None, 128)
    R.check_linear(got, *R.linear_w4(x, words, scales, None, None, 128))
    # half a step of the grid for every weight
    off = np.abs(R.wide(got) - R.wide(x) @ R.wide(w).T)
    step = np.repeat(R.wide(scales), 128, 1)
    assert (off <= np.abs(R.wide(x)) @ (0.51 * step + 0.01 * np.abs(R.wide(w))).T + 0.1).all()


@pytest.mark.parametrize("rows", [1, 20, 150])
def test_captured_and_twice_the_same(gpu, rows):
    rng = np.random.default_rng(9)
    x, words, scales, zeros, bias = make(rng, rows, 1024, 200, 128, True, True)
    ts = [gpu.bf16(x), gpu.u32(words), gpu.bf16(scales), gpu.bf16(zeros), gpu.bf16(bias)]
    y = gpu.new_bf16(rows * 200)
    call = lambda: gpu.check(gpu.lib.qw_gpu_linear_w4_bf16(gpu.handle, y, *ts, rows, 1024, 200, 128))  # noqa: E731
    gpu.begin()
    call()
    gpu.submit()
    first = gpu.read_bf16(y, rows * 200)
    gpu.begin()
    gpu.check(gpu.lib.qw_gpu_graph_begin(gpu.handle))
    call()
    graph = gpu.lib.qw_gpu_graph_end(gpu.handle)
    gpu.check(graph)
    gpu.submit()
    x2 = R.random_bf16(rng, rows, 1024)
    for values in (x2, x):
        gpu.write_bf16(ts[0], values)
        gpu.begin()
        gpu.check(gpu.lib.qw_gpu_graph_launch(gpu.handle, graph))
        gpu.submit()
        got = gpu.read_bf16(y, rows * 200)
        R.check_linear(got.reshape(rows, 200), *R.linear_w4(values, words, scales, zeros, bias, 128))
    assert (got == first).all()
    gpu.lib.qw_gpu_graph_free(graph)
    for t in ts + [y]:
        gpu.free(t)


@pytest.mark.parametrize("rows,inputs", [(100, 4096), (40, 512)])
def test_bounded_waits_run_out_cleanly(gpu, rows, inputs):
    """Steps from the second on stay away (nothing is in flight): the waits behind them run out, the submit
    says so and the next call is right."""
    rng = np.random.default_rng(10)
    x, words, scales, _, _ = make(rng, rows, inputs, 300, 128, False, False)
    gpu.check(gpu.lib.qw_gpu_debug_linear_waits(gpu.handle, 2_000_000, 1, 0))
    try:
        with pytest.raises(abi.GpuError, match="wait ran out"):
            linear(gpu, x, words, scales, None, None, 128)
    finally:
        gpu.lib.qw_gpu_debug_linear_waits(gpu.handle, 0, 0, 0)
    got = linear(gpu, x, words, scales, None, None, 128)
    R.check_linear(got, *R.linear_w4(x, words, scales, None, None, 128))
