"""CPU tests of what the 8-bit activation path refuses, beyond those of test_int8_path.py."""
import pytest

from mixed_gemv_b200 import _lib
from mixed_gemv_b200.enums import Status
from tests.test_int8_path import _gemm


@pytest.mark.parametrize("hints", [32, 64, 128, 1 << 13, 1 << 30, -(1 << 31), _lib.GEMM_HINT_PAIR | 32])
@pytest.mark.parametrize("M", [0, 4])
def test_unknown_hints_are_refused(hints, M):
    assert _gemm(M=M, hints=hints) == Status.INVALID_ARGUMENT
    assert b"hints" in _lib.load().mgv_last_error()
