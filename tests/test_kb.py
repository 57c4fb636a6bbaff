"""KeyBlocks refuses bad calls before they touch a device, and its numpy
statement chooses what it says. CPU only."""
import ctypes as C

import numpy as np
import pytest

from aikit_b200 import _ffi
from aikit_b200._ffi import Fi8Error
from aikit_b200.ann import B200Backend

import kb_util


def test_null_handles_are_refused():
    L = _ffi.lib()
    p, out = C.c_void_p(16), C.c_void_p()
    bad = _ffi.FI8_ERR_ARG
    assert L.fi8_kb_create(None, C.byref(_ffi.KbDesc()), C.byref(out)) == bad
    assert L.fi8_kb_create(p, None, C.byref(out)) == bad
    assert L.fi8_kb_create(p, C.byref(_ffi.KbDesc()), None) == bad
    assert L.fi8_kb_update_async(None, p, p, p, 1, 1, None) == bad
    assert L.fi8_kb_select_async(None, p, 8, p, p, 1, 1, 0, 1, p, None) == bad
    assert L.fi8_kb_attend_async(None, p, 8, p, p, 1, p, 1, 1.0, p, None, None) == bad
    assert L.fi8_kb_query_async(None, p, 8, p, p, 1, 1, 0, 1, 1.0, p, p, None, None) == bad
    assert L.fi8_kb_read_rows(None, 0, p, p, p) == bad
    assert L.fi8_kb_sync(None) == bad
    assert L.fi8_kb_destroy(None) == _ffi.FI8_OK


def test_dtype_is_checked_first():
    be = B200Backend.__new__(B200Backend)
    with pytest.raises(Fi8Error, match="bf16 or f16"):
        be.NewKeyBlocks(16, 16, dtype="f32", slots=1, kv_heads=1, q_heads=1, head_dim=16, capacity=16, block=16, max_rows=1,
                        max_select=1, slot_stride=256, head_stride=256, token_stride=16)


def test_select_by_hand():
    """Blocks along one axis: the best inner blocks, ties by number, first and last kept."""
    D, block = 32, 2
    keys = np.zeros((1, 14, D))
    for b, x in enumerate([0.0, 5.0, 3.0, 5.0, 1.0, 5.0, -9.0]):
        keys[0, 2 * b : 2 * b + 2, 0] = x
    rows = kb_util.block_rows(keys, block)
    q = np.zeros((1, D), np.float32)
    q[0, 0] = 2
    assert kb_util.select(rows, q, 14, block, 4, 1, 1)[0].tolist() == [0, 1, 3, 6]
    assert kb_util.select(rows, q, 13, block, 3, 0, 1)[0].tolist() == [1, 3, 6]
    assert kb_util.select(rows, q, 5, block, 4, 1, 1)[0].tolist() == [0, 1, 2, -1]
    assert kb_util.select(rows, q, 0, block, 2, 1, 1)[0].tolist() == [-1, -1]
    assert kb_util.select(rows, -q, 14, block, 2, 0, 1)[0].tolist() == [0, 6]
