"""pl_capture_id without a capture."""

import ctypes

from pagelora_amd import _lib


def test_refusals():
    lib, number = _lib.load(), ctypes.c_ulonglong(7)
    assert lib.pl_capture_id(None, None) == _lib.PL_ERR_INVALID
    assert lib.pl_capture_id(None, ctypes.byref(number)) in (_lib.PL_ERR_INVALID, _lib.PL_ERR_HIP)  # (no device, or no capture)
    assert number.value == 0 and lib.pl_last_error()
