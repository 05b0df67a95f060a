"""GPU: a long wait budget of the 4-bit linear layers is long."""
import numpy as np
import pytest

import text_tower_ref as R
from test_gpu_linear_w4 import linear, make

pytestmark = pytest.mark.gpu


def test_a_budget_of_more_probes_than_an_int_holds(gpu):
    """10000 cycles a probe: 2^31 of them were none at all."""
    rng = np.random.default_rng(0)
    x, words, scales, zeros, bias = make(rng, 40, 512, 200, 128, True, True)
    gpu.check(gpu.lib.qw_gpu_debug_linear_waits(gpu.handle, 10000 << 31, 0, 0))
    try:
        got = linear(gpu, x, words, scales, zeros, bias, 128)
    finally:
        gpu.lib.qw_gpu_debug_linear_waits(gpu.handle, 0, 0, 0)
    R.check_linear(got, *R.linear_w4(x, words, scales, zeros, bias, 128))
