"""Row ranges of the few-token kernels at the largest sizes that their entry points take, on the CPU: nothing is counted beyond 32 bits."""
import ctypes

import pytest

from tensor_parallel_b200 import build

pytestmark = pytest.mark.skipif(not build.LIB_PATH.exists(), reason="native library not built")


def _rows(features, sms, cta):
    from tensor_parallel_b200.ops import native

    capacity = features // (128 * sms) + 8
    shape, starts = (ctypes.c_int * 5)(), (ctypes.c_int * capacity)()
    code = native.LIB.tpb_gemm_stream_rows(features, sms, cta, shape, starts, capacity)
    return code, list(shape), starts[0:shape[2] + 1]


@pytest.mark.parametrize("sms", [148, 132, 20])
@pytest.mark.parametrize("features", [22016, 151936, 40_000_000, 270_000_000, "most"])
def test_passes_follow_one_another(features, sms):
    most = 32 * 4 * 2 ** 14 * sms  # what a launch counts
    features, last = most if features == "most" else min(features, most), 0
    for cta in (0, 1, sms // 2, sms - 1):
        code, (units, grid, passes, longest, box), mine = _rows(features, sms, cta)
        assert code == 0 and units == -(-features // 32) and grid == sms and 1 <= box <= longest <= 4
        assert mine[0] == cta * units // grid and mine[-1] == (cta + 1) * units // grid and mine[0] >= last
        assert all(box <= b - a <= longest for a, b in zip(mine, mine[1:]))
        last = mine[-1]
    assert last == units


@pytest.mark.parametrize("sms", [148, 132, 20])
@pytest.mark.parametrize("features", ["most", 500_000_000, 2 ** 31 - 512])
def test_longer_ranges_are_not_for_one_launch(features, sms):
    from tensor_parallel_b200.ops import native

    features = 32 * 4 * 2 ** 14 * sms + 1 if features == "most" else features
    assert _rows(features, sms, 0)[0] == 7  # (too large)
    plan = native.GemmPlan()
    if sms == 148:
        native.check(native.LIB.tpb_gemm_plan_ex(1, features, 64, 1, 0, 0, 0, ctypes.byref(plan)), "gemm_plan")
        assert not plan.stream
