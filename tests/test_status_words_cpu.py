"""CPU: the host checks of the status words' calls."""

import ctypes

from pa_b200 import _lib


def test_null_pointers_are_refused():
    L = _lib.lib()
    assert L.pa_device_status(None) == _lib.PA_ERR_INVALID_ARG
    out = ctypes.c_int(0)
    assert L.pa_read_status(None, ctypes.byref(out), None) == _lib.PA_ERR_INVALID_ARG
    assert L.pa_read_status(1 << 20, None, None) == _lib.PA_ERR_INVALID_ARG
