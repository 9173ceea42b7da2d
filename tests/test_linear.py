"""Forward operators: plain forms, argument checks that need no GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import linear_plain as L
import zkml_b200 as Z
from helpers import uniform_m31


def test_plain_product_is_the_definition():
    x, w = uniform_m31(5 * 40, 1).reshape(5, 40), uniform_m31(40 * 7, 2).reshape(40, 7)
    want = (x.astype(object) @ w.astype(object)) % L.P
    np.testing.assert_array_equal(L.product(x, w), want.astype(np.int64))


@pytest.mark.parametrize("tag", [1, 2, 3, 4, 5])
def test_plain_activation_is_the_framework_table(tag):
    """The tables hold f of the words from 0 on."""
    t = Z.activation_table(tag).astype(np.int64)
    y, unsure = L.activation(np.arange(t.size), tag)
    assert unsure.sum() <= 4
    np.testing.assert_array_equal(np.where(unsure, t, y), t % L.P)


def test_plain_activation_of_negative_words():
    z = L.words([-1, -65536, -(1 << 20), -(1 << 30) + 1])
    assert (L.activation(z, 1)[0] == 0).all() and (L.activation(z, 3)[0] == 0).all()
    np.testing.assert_array_equal(L.activation(z, 4)[0], [65536, 65536, 2, 1])
    silu = L.signed(L.activation(z, 5)[0])
    # -1/65536 sigmoid(-1/65536) is just above -1/2 in fixed point; the last two underflow
    np.testing.assert_array_equal(silu, [0, round(-65536 / (1 + np.e)), 0, 0])


def _bare(k=6, n=4, gated=False):
    w = (Z.GatedLinearM31 if gated else Z.LinearM31).__new__(Z.GatedLinearM31 if gated else Z.LinearM31)
    w.k, w.n, w.device, w._handle = k, n, 0, None
    return w


def test_rows_of_a_matrix():
    w = _bare()
    words = torch.zeros(5, 3, 8, dtype=torch.int32)
    for bad, match in ((torch.zeros(3, 6), "uint32"), (torch.zeros(3, 5, dtype=torch.int32), "rows of 6"),
                       (torch.zeros(6, 3, dtype=torch.int32).t(), "contiguous"),
                       (torch.zeros((), dtype=torch.int32), "rows of 6"),
                       (words.transpose(0, 1)[:, :, :6], "one stride"),
                       (torch.zeros(3, 6, dtype=torch.int32), "not on cuda"),
                       (words[:, :, :6], "not on cuda")):
        with pytest.raises(Z.InvalidArgument, match=match):
            w._rows(bad, 6, "x")


def test_activation_names():
    from zkml_b200.forward import _tag
    assert [_tag(a) for a in (None, "none", "ReLU", "gelu", "sigmoid", "softmax", "SiLU", 3)] == [0, 0, 1, 2, 3, 4, 5, 3]
    with pytest.raises(Z.InvalidArgument):
        _tag("tanh")


def test_closed_handle_is_refused():
    with pytest.raises(Z.InvalidArgument, match="closed"):
        _bare()._call(torch.zeros(1, 6, dtype=torch.int32), None, None, None, None, None, False, 31, False)


def test_null_arguments_are_refused():
    lib = Z.lib()
    out, size = C.c_void_p(), C.c_size_t()
    assert lib.zkml_linear_create(None, 16, 1, 1, 1, 1, None, None, C.byref(out)) == 1
    assert lib.zkml_linear_create_gated(None, 16, 16, 1, 1, 1, 1, None, None, None, C.byref(out)) == 1
    assert lib.zkml_linear_create(None, 16, 1, 1, 1, 1, None, None, None) == 1
    assert lib.zkml_linear_workspace(None, 1, 31, C.byref(size)) == 1
    assert lib.zkml_linear_forward(None, None) == 1
    assert lib.zkml_linear_check(None, None) == 1
    assert lib.zkml_linear_destroy(None) == 0
