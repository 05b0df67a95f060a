"""CPU: the paged attention's merge of a unit's parts has room for every CTA that a launch can have."""
import ctypes as C

import pytest

from qwen_metal_b200 import abi

PART = 16 * (128 + 2) * 4  # bytes of 16 rows, their maxima and sums
ROOM = 4 * 132             # weights of a row that the merge holds: what four warps' rows leave


@pytest.mark.parametrize("sms", [1, 100, 148, 160, 176, 177, 200, 1000])
def test_no_more_parts_than_the_merge_holds(sms):
    fn = abi.load().qwcu_paged_few_workspace_bytes
    fn.restype, fn.argtypes = C.c_size_t, [C.c_int]
    ctas, rest = divmod(fn(sms), 2 * PART + 4)
    assert rest == 0 and ctas == min(3 * sms, ROOM)
