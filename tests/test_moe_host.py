"""The host side of the mixture-of-experts layer.  CPU only."""
import ctypes

import pytest

from test_ffn_refusals import _desc


@pytest.mark.parametrize("T", [-1, 65])
def test_work_bytes_says_why(lk_host, T):
    """A count of tokens out of range leaves its own error, not that of an earlier call."""
    lib = lk_host.load()
    assert lib.lk_gemm_i8(None, 0, None, None, 0, None, -1, 0, 1, 0, None, 0, None, 0, None) == 1
    assert b"lk_gemm_i8" in lib.lk_last_error()
    assert lib.lk_moe_work_bytes(ctypes.byref(_desc(lk_host)), T) == 0
    assert b"lk_moe_work_bytes" in lib.lk_last_error() and str(T).encode() in lib.lk_last_error()
