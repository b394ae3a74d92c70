"""Refusals of the 4-bit entry points that need no GPU (include/ipx.h): a status and a message, nothing is touched."""
import ctypes as C

import numpy as np
import pytest

from mural_amd import _lib, mx4

ARG = 1


def refused(rc, words):
    msg = _lib.lib().ipx_last_error().decode()
    assert rc == ARG and words in msg, (rc, msg)


def test_quantize_and_dequantize_refuse_bad_arguments(ipx):
    x = np.zeros((4, 64), np.float32)
    c, s = np.zeros((4, 2, 16), np.uint8), np.zeros((4, 2), np.uint8)
    px, pc, ps = (C.c_void_p(a.ctypes.data) for a in (x, c, s))
    q = lambda *a: ipx.ipx_mx4_quantize(*a)
    refused(q(px, -1, 64, 64, 0, pc, ps, 0, 0, None), "n < 0")
    refused(q(px, 4, 0, 64, 0, pc, ps, 0, 0, None), "dimension")
    refused(q(px, 4, 65537, 65537, 0, pc, ps, 0, 0, None), "dimension")
    refused(q(px, 4, 64, 64, 3, pc, ps, 0, 0, None), "dtype")
    refused(q(px, 4, 64, 63, 0, pc, ps, 0, 0, None), "stride")
    refused(q(None, 4, 64, 64, 0, pc, ps, 0, 0, None), "null")
    refused(q(px, 4, 64, 64, 0, None, ps, 0, 0, None), "null")
    refused(q(px, 4, 64, 64, 0, pc, None, 0, 0, None), "null")
    refused(q(px, 4, 64, 64, 0, C.c_void_p(c.ctypes.data + 1), ps, 0, 0, None), "multiple of 4")
    assert q(None, 0, 64, 64, 0, None, None, 0, 0, None) == 0
    d = lambda *a: ipx.ipx_mx4_dequantize(*a)
    refused(d(pc, ps, -1, 64, px, 0, 0, 0, None), "n < 0")
    refused(d(pc, ps, 4, 0, px, 0, 0, 0, None), "dimension")
    refused(d(pc, ps, 4, 64, px, 7, 0, 0, None), "dtype")
    refused(d(pc, None, 4, 64, px, 0, 0, 0, None), "null")
    assert d(None, None, 0, 64, None, 0, 0, 0, None) == 0


def test_index_calls_refuse_a_null_index(ipx):
    z = C.c_void_p(np.zeros(64).ctypes.data)
    refused(ipx.ipx_add_mx4(None, z, z, 1, 0, None), "null index")
    refused(ipx.ipx_scores(None, z, 0, 1, 0, 1, z, 0, None), "null index")
    refused(ipx.ipx_scores_mx4(None, z, z, 1, 0, 1, z, 0, None), "null index")
    refused(ipx.ipx_lookup(None, z, 1, None, z, 0, 0, None), "null index")


def test_python_checks_shapes_before_any_call():
    c, s = np.zeros((4, 2, 16), np.uint8), np.zeros((4, 2), np.uint8)
    for bad in ((c, s, 65), (c, s, 32), (c[:3], s, 64), (c.astype(np.int8), s, 64), (c, s.astype(np.int32), 64), (c[:, :, :8], s, 64)):
        with pytest.raises(AssertionError):
            mx4.dequantize(*bad)
    with pytest.raises(KeyError):
        mx4.dequantize(c, s, 64, dtype=np.int32)
    with pytest.raises(ValueError):
        mx4.quantize(np.zeros(64, np.float32))
    assert mx4.n_blocks(1) == 1 and mx4.n_blocks(32) == 1 and mx4.n_blocks(33) == 2


def test_the_oracle_rounds_as_the_format_says():
    """the test oracle itself, on values whose codes are known"""
    import mx4_oracle as M
    x = np.array([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, 7.0, 0.26]])
    want = [[6, 0, 1, 1, 2, 2, 4, 4, 0, -1, 6, 0.5]]
    assert M.rounded(x).tolist() == want
    assert M.rounded(x * 2.0 ** 50).tolist() == (np.array(want) * 2.0 ** 50).tolist()
    assert np.isnan(M.rounded(np.array([[1.0, np.inf]]))).all()
