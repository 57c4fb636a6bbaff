"""FlatI4's numpy statement holds its own bounds, and the entry points refuse
bad calls before they touch a device. CPU only."""
import ctypes as C

import numpy as np
import pytest

from aikit_b200 import _ffi
from aikit_b200.ann import B200Backend, I4Index
from aikit_b200._ffi import Fi8Error

import i4_util


@pytest.mark.parametrize("dim", [1, 31, 32, 33, 100, 768])
def test_quantizer_error_is_half_a_step(dim):
    """Every value is within half a step of its group, and the step is at most
    1/m above a separate scale's (its group's maximum over 7)."""
    rng = np.random.default_rng(dim)
    v = (rng.standard_normal((50, dim)) * np.exp(rng.standard_normal((50, 1)))).astype(np.float32)
    codes, mults, scales = i4_util.quantize(v)
    back = i4_util.numbers(codes, mults)[:, :dim] * scales[:, None].astype(np.float64)
    step = (mults.astype(np.float64) * scales[:, None]).repeat(32, 1)[:, :dim]
    # the float32 steps of the quantizer move a value by a few 2^-24 of its size (at most 7 steps): 1e-5 of a step
    assert (np.abs(back - v) <= step * (0.5 + 1e-5)).all()
    x = np.zeros((50, codes.shape[1] * 32))
    x[:, :dim] = np.abs(v)
    gmax = x.reshape(50, -1, 32).max(2)
    own = gmax / 7
    assert (mults * scales[:, None].astype(np.float64) <= own + scales[:, None] * (1 + 1e-4)).all()


def test_quantizer_odd_values():
    v = np.zeros((7, 40), np.float32)
    v[1, 3] = 2.0
    v[2, :] = np.nan
    v[3, 5], v[3, 39] = np.inf, 1.0
    v[4, 0], v[4, 35] = 1e-44, -1e-44
    v[5, 0], v[5, 33] = 3e38, 1e-30
    v[6, :] = np.where(np.arange(40) % 2, np.nan, 1.0)
    codes, mults, scales = i4_util.quantize(v)
    w = i4_util.numbers(codes, mults)
    assert (w[0] == 0).all() and scales[0] == 1
    assert w[1, 3] == 7 * 255 and (np.delete(w[1], 3) == 0).all()
    assert (w[2] == 0).all() and scales[2] == 1
    assert np.isinf(scales[3]) and (w[3] == 0).all()
    assert w[5, 0] == 7 * 255 and w[5, 33] <= 7
    assert w[6, 0] == 7 * 255 and w[6, 1] == 0


def test_dot_stays_in_32_bits():
    """The largest dot of 4096 values, whatever the nibbles, is below 2^31."""
    assert 8 * 255 * 127 * 4096 < 2**31


def test_null_handles_are_refused():
    L = _ffi.lib()
    out, p = C.c_void_p(), C.c_void_p(16)
    assert L.fi8_i4_create(None, p, p, p, 4, 32, 0, C.byref(out)) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_create_f32(None, p, 4, 32, 0, C.byref(out)) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_create_empty(None, 4, 32, 0, C.byref(out)) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_create_empty(None, 4, 32, 0, None) == _ffi.FI8_ERR_ARG
    assert b"null ctx" in L.fi8_last_error() or b"null out" in L.fi8_last_error()
    assert L.fi8_i4_set_rows_async(None, 0, p, 1, None) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_read_rows(None, p, p, p) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_info(None, None, None) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_score_batch(None, p, 1, p) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_score_async(None, p, 1, p, None) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_topk_batch(None, p, 1, 1, None, 0, p, p) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_topk_async(None, p, 1, 1, None, 0, p, None) == _ffi.FI8_ERR_ARG
    assert L.fi8_i4_destroy(None) == _ffi.FI8_OK


class _NoContext:
    handle = None


def test_python_shape_checks():
    be = B200Backend.__new__(B200Backend)
    be.ctx = _NoContext()
    with pytest.raises(Fi8Error, match="shape mismatch"):
        be.NewI4Index(np.zeros(15, np.uint8), np.zeros(1, np.uint8), np.zeros(1), 1, 32)
    with pytest.raises(Fi8Error, match="empty"):
        be.NewI4Index([], [], [], 0, 32)
    with pytest.raises(Fi8Error, match="empty"):
        be.NewI4IndexFromFloats(np.zeros((0, 4)))
    with pytest.raises(Fi8Error, match="null ctx"):
        be.NewI4IndexEmpty(4, 32)
    ix = I4Index(be.ctx, None, 4, 32, 0)
    with pytest.raises(Fi8Error, match="query dim"):
        ix.ScoreBatch(np.zeros((1, 31)), np.zeros(4, np.float32))
    with pytest.raises(Fi8Error, match="dst len"):
        ix.ScoreBatch(np.zeros((1, 32)), np.zeros(5, np.float32))
