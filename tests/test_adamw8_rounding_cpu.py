"""Type bits of odw_adamw8, without a GPU: refused, or nothing to launch."""
import ctypes

from od_wscl_amd import _lib


def test_the_library_takes_the_form_and_no_other():
    lib = _lib.lib()
    arr = lambda t, x: (t * 1)(x)               # noqa: E731
    some, one = arr(ctypes.c_void_p, 4096), arr(ctypes.c_float, 1e-3)

    def call(types, n):
        return lib.odw_adamw8(1, some, some, some, some, some, None, arr(ctypes.c_int64, n), arr(ctypes.c_int, types), one, one, 0.9, 0.999, 1e-8, 1,
                              None, None, 1.0, 0, 0, 0, None)
    assert call(7, 0) == 0 and call(8, 0) == -1 and call(8, 8) == -1
