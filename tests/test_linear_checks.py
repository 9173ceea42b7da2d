"""Forward operators: checks that need no GPU."""
import numpy as np
import pytest

import zkml_b200 as Z
from test_linear import _bare

RECORD = np.dtype([("s", "<i2"), ("w", "<i4"), ("t", "<i2")])  # 8 bytes, the word at 2
PACKED = np.dtype([("w", "<i4"), ("s", "<i2")])                # 6 bytes


def test_wait_self_test_refuses_null_arguments():
    assert Z.lib().zkml_selftest_linear_wait(None, None, 1, 20) == 1


def test_checked_call_refuses_null_arguments():
    assert Z.lib().zkml_linear_forward_checked(None, None) == 1


def awkward_words(w):
    """The words of w in arrays whose addresses or strides are no whole words, or run downwards."""
    views = []
    for dtype in (RECORD, PACKED):
        r = np.zeros(w.shape, dtype)
        r["w"] = w.view(np.int32)
        views.append(r["w"])
        r = np.zeros(w.T.shape, dtype)
        r["w"] = w.view(np.int32).T
        views.append(r["w"].T)
    odd = np.zeros(4 * w.size + 1, np.uint8)
    odd[1:] = np.ascontiguousarray(w).view(np.uint8).reshape(-1)
    views.append(odd[1:].view(np.uint32).reshape(w.shape))
    views.append(np.ascontiguousarray(w[::-1, ::-1])[::-1, ::-1])
    for v in views:
        np.testing.assert_array_equal(v.view(np.uint32) if v.flags.c_contiguous else v.astype(np.uint32), w)
    return views


def test_words_of_arrays_in_whole_words():
    w = np.arange(5 * 7, dtype=np.uint32).reshape(5, 7)
    for v in awkward_words(w):
        got = _bare()._words(v, "weight")
        assert got.ctypes.data % 4 == 0 and all(s >= 0 and s % 4 == 0 for s in got.strides)
        np.testing.assert_array_equal(got.astype(np.uint32), w)
    for v in (w, w.T, w[::2, 1:], np.broadcast_to(w[0], (5, 7))):  # read in place
        assert _bare()._words(v, "weight") is v


def test_an_array_beside_a_tensor_is_refused():
    w = _bare()
    for rows in (np.zeros((3, 6), np.uint32), np.zeros(6, np.int32), [[0] * 6]):
        with pytest.raises(Z.InvalidArgument, match="tensors on cuda:0"):
            w._rows(rows, 6, "residual")
