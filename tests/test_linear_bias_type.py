"""The bias's type in the C interface, refused before anything reaches a device."""
import ctypes

from sparseconv import _native

P = ctypes.c_void_p(256)


def test_refusals():
    lib = _native.load_library()
    f = lib.spconv_linear_forward_ex
    for dtype, bias_dtype in ((0, 1), (0, 2), (1, 2), (2, 1), (2, 7), (1, -1)):
        assert f(P, dtype, 10, 8, P, P, bias_dtype, None, 8, 0, P, None, None, 0, 0, None, None) == 1
        assert b"bias" in lib.spconv_last_error()
        # no bias: its type is not looked at
        assert f(None, dtype, 0, 8, None, None, bias_dtype, None, 8, 0, None, None, None, 0, 0, None, None) == 0
    for dtype, bias_dtype in ((0, 0), (1, 0), (2, 0), (1, 1), (2, 2)):
        assert f(P, dtype, 0, 8, P, P, bias_dtype, None, 8, 0, P, None, None, 0, 0, None, None) == 0
    assert f(P, 2, 50000, 257, P, P, 0, None, 131, 0, P, None, P, 8, 0, None, None) == 1          # workspace
