"""GPU: 4-bit weights are not rounded, whatever the number of rows."""
import numpy as np
import pytest

import text_tower_ref as R
from qwen_metal_b200 import abi
from test_gpu_linear_w4 import linear, make

pytestmark = pytest.mark.gpu

SHAPES = [(1, 256, 48, 128), (13, 256, 130, 32), (16, 320, 65, 64), (17, 256, 130, 128), (17, 320, 64, 32),
          (24, 1024, 4800, 64), (33, 384, 200, 64), (100, 2048, 130, 128), (130, 256, 9600, 32), (200, 640, 9600, 128),
          (300, 512, 260, 256)]


def weights(words, scales, zeros, group):
    q = R.unpack(words).astype(np.float64)
    z = 8.0 if zeros is None else np.repeat(R.wide(zeros), group, 1)
    return np.repeat(R.wide(scales), group, 1) * (q - z)


def differences(rng, rows, inputs):
    """Rows of x with a one and a minus one, and their places."""
    first = rng.integers(0, inputs, rows)
    second = (first + 1 + rng.integers(0, inputs - 1, rows)) % inputs
    x = np.zeros((rows, inputs), np.float32)
    x[np.arange(rows), first], x[np.arange(rows), second] = 1.0, -1.0
    return abi.f32_to_bf16(x), first, second


@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES)
def test_differences_of_two_weights(gpu, rows, inputs, outputs, group):
    """s (q - 8) has at most 12 bits; with scales of one binade the difference of two is exact in fp32, and all
    that is rounded is the result.  (Up to 16 rows 136 s x is taken from a sum: 2^-24 of it for every addition.)"""
    rng = np.random.default_rng(rows + outputs)
    _, words, _, _, _ = make(rng, rows, inputs, outputs, group, False, False)
    scales = abi.f32_to_bf16(rng.uniform(1.0, 2.0, (outputs, inputs // group)).astype(np.float32))
    x, first, second = differences(rng, rows, inputs)
    got = linear(gpu, x, words, scales, None, None, group)
    w = weights(words, scales, None, group).T
    exact = w[first] - w[second]
    slack = 2.0 ** -24 * 8 * 136 * 2 * 2 if rows <= 32 else 0.0
    assert (np.abs(R.wide(got) - exact) <= R.HALF_STEP * np.abs(exact) + slack).all()
    if rows > 32:
        assert (got == abi.f32_to_bf16(exact.astype(np.float32))).all()


@pytest.mark.parametrize("zeros", ["whole", "far", "any", "wild"])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES)
def test_differences_with_zero_points(gpu, rows, inputs, outputs, group, zeros):
    """Two bf16 numbers hold s (q - z): what rounding the first leaves is within 2^-8 of the weight, and at most
    2^-7 with the rest of the zero point; that is rounded once or twice, 2^-16 and 2^-15 of the weight.  (Up to 16
    rows as above, with 128 + z for 136.)"""
    rng = np.random.default_rng(rows * 3 + outputs)
    _, words, _, z, _ = make(rng, rows, inputs, outputs, group, True, False)
    scales = abi.f32_to_bf16(rng.uniform(1.0, 2.0, (outputs, inputs // group)).astype(np.float32))
    if zeros == "whole":
        z = abi.f32_to_bf16(rng.integers(0, 16, z.shape).astype(np.float32))
    elif zeros == "far":
        z = abi.f32_to_bf16(rng.integers(-120, 120, z.shape).astype(np.float32))
    elif zeros == "wild":  # of any size, two outputs of three like whole ones
        z = abi.f32_to_bf16((rng.standard_normal(z.shape) * 10.0 ** rng.integers(-6, 5, z.shape)).astype(np.float32))
        z[np.arange(outputs) % 3 > 0] = 0x4100
    x, first, second = differences(rng, rows, inputs)
    got = linear(gpu, x, words, scales, z, None, group)
    w = weights(words, scales, z, group).T
    a, b = w[first], w[second]
    exact = a - b
    bound = R.HALF_STEP * np.abs(exact) + (2.0 ** -16 + 2.0 ** -15 + 2.0 ** -23) * (np.abs(a) + np.abs(b))
    if rows <= 32:
        size = (16 + 128 + np.abs(R.wide(z)).max()) * 2
        bound = bound + 2.0 ** -24 * 8 * size * 2
    assert (np.abs(R.wide(got) - exact) <= bound).all()


@pytest.mark.parametrize("with_zeros,with_bias", [(False, False), (True, True)])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES + [(412, 1024, 384, 128), (64, 4096, 260, 32)])
def test_many_products(gpu, rows, inputs, outputs, group, with_zeros, with_bias):
    """The bound of few rows for every number of them: sums in fp32 within 2^-14 of the magnitudes, a result
    rounded once."""
    rng = np.random.default_rng(rows * inputs)
    x, words, scales, zeros, bias = make(rng, rows, inputs, outputs, group, with_zeros, with_bias)
    got = linear(gpu, x, words, scales, zeros, bias, group)
    y, size, _ = R.linear_w4(x, words, scales, zeros, bias, group)
    assert (np.abs(R.wide(got) - y) <= R.HALF_STEP * np.abs(y) + 2.0 ** -14 * size).all()


@pytest.mark.parametrize("rows,group", [(1, 128), (40, 32), (40, 64), (150, 128)])
def test_scales_of_any_size(gpu, rows, group):
    """s (q - 8) x is in range wherever it is, also where 24 s or what is left of s (q - 8) is not, or hardly."""
    rng = np.random.default_rng(rows)
    _, words, _, _, _ = make(rng, rows, 256, 200, group, False, False)
    power = rng.integers(-100, 124, (200, 256 // group)).astype(np.float64)
    power[:40] = 120 + rng.integers(0, 4, power[:40].shape)
    scales = abi.f32_to_bf16((2.0 ** power * rng.uniform(1.0, 2.0, power.shape)).astype(np.float32))
    w = weights(words, scales, None, group)
    for column in (0, 33, 100, 255):
        x = np.zeros((rows, 256), np.float32)
        x[:, column] = 2.0 ** -8
        got = linear(gpu, abi.f32_to_bf16(x), words, scales, None, None, group)
        assert (got == abi.f32_to_bf16((w[None, :, column] * 2.0 ** -8).astype(np.float32))).all()
