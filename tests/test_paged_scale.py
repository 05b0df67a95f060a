"""CPU: the paged attention refuses a scale that its exponents in powers of two cannot take."""
import numpy as np
import pytest

from test_text_tower_host import PASSED, attend_args, fake  # noqa: F401 (a fixture)

LOG2E = 1.4426950408889634


@pytest.mark.parametrize("scale,fine", [(3.4e38, False), (2.5e38, False), (2.3e38, True), (1e-30, True), (1.0, True)])
def test_scale_times_log2e_is_finite(fake, scale, fine):  # noqa: F811
    assert (np.float64(scale) * LOG2E < 3.4028235e38) == fine
    said = fake.says("qw_gpu_paged_attention_bf16", dict(attend_args(fake), scale=scale))
    assert said == PASSED if fine else "scale" in said
