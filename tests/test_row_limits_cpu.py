"""Rows longer than the row quantiser's 32-bit column counters reach are refused on the host (a thread steps 1024 columns at a time)."""
import pytest

import adcdiff  # noqa: F401
from adcdiff import _lib

LONGEST = 1 << 30


@pytest.mark.parametrize("K", [LONGEST + 1, (1 << 31) - 1025, (1 << 31) - 1024, (1 << 31) - 17, (1 << 31) - 1])
@pytest.mark.parametrize("dtype", [0, 1])
def test_rows_past_the_counters(K, dtype):
    pitch = (K + 15) // 16 * 16
    assert _lib.load().adcdiff_quantize_rows(4096, K, dtype, 1, K, 4096, pitch, 4096, None) == -1
    assert "columns" in _lib.load().adcdiff_last_error().decode()


def test_counters_hold_the_longest_row():
    for c in range(1024):                                      # the last turn's counter of every thread, and the codes rounded up to 16
        assert (LONGEST - 1 - c) // 1024 * 1024 + c + 1024 < 1 << 31
    assert (LONGEST + 15) // 16 * 16 + 1024 < 1 << 31
