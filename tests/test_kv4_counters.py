"""The arrival counters of the split-K scratch (64 KiB) hold those of every divided attention call, on devices of any
number of compute units."""
import ctypes

import pytest

COUNTERS = 64 * 1024 // 4


@pytest.mark.parametrize("sms", [1, 8, 256, 300, 2048, 2049, 5000, 100000, 2 ** 31 - 1])
@pytest.mark.parametrize("D,g", [(128, -1), (64, 32)])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (32, 32), (64, 8), (7, 7)])
def test_counters_hold_a_divided_call(built_lib, sms, D, g, heads, kv_heads):
    """The kernel of few rows has a counter a workgroup, that of prompts one a part and wave of eight."""
    out = (ctypes.c_int * 3)()
    for q, kv in ((1, 1 << 30), (300, 1 << 30), (300, 100000)):
        assert built_lib.marlin_hip_kv4_plan(1, heads, kv_heads, D, g, q, kv, sms, out) == 0
        prompts, workgroups, split = out
        assert workgroups > 0
        if split:
            assert workgroups * (8 if prompts else 1) <= COUNTERS, (q, kv, list(out))
