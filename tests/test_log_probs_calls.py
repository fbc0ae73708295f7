"""What the log-probabilities refuse before anything runs, beside
tests/test_experts.py."""

import pytest

from wpt_amd import _lib


@pytest.mark.parametrize("B, T, V, top", [(1 << 24, 1, 16, 0), (1 << 13, 1 << 11, 3, 2), (1 << 11, 1 << 13, 513, 1),
                                          (1 << 24, 1, 5, 0), (1 << 23, 1, 20000, 4), ((1 << 31) - 1, 1, 100, 0)])
@pytest.mark.parametrize("dtype", [_lib.WPTV_F32, _lib.WPTV_BF16])
def test_more_rows_than_a_launch_has_threads_for_are_refused(B, T, V, top, dtype):
    status = _lib.lib().wptv_log_probs(16, V, V, dtype, 16, 1.0, B, T, V, top, 16, 16, 16, 16, 16, 1 << 50, None)
    assert status == -3 and b"rows" in _lib.lib().wptv_last_error()
