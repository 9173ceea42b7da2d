"""Forward operators on the GPU where something goes wrong: waits that run out, words that do not belong,
several callers of one handle, and the ends of the accumulators' range."""
import ctypes as C

import numpy as np
import pytest
import torch

import linear_plain as L
import zkml_b200 as Z
from test_linear_gpu import LinearCall, TAGS, dev, host, ints

pytestmark = pytest.mark.gpu
P = L.P
TIMEOUT = 5  # ZKML_ERR_TIMEOUT
MARK = -7    # no word of a result


def selftest(lin, x, out, act, withhold, limit_ms=20):
    """zkml_selftest_linear_wait of lin(x, activation=act, out=out)."""
    m, k = x.shape
    need = C.c_size_t()
    assert Z.lib().zkml_linear_workspace(lin._handle, m, 31, C.byref(need)) == 0
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device="cuda")
    c = LinearCall(x=x.data_ptr(), m=m, ldx=k, x_bits=31, activation=TAGS[act], out=out.data_ptr(), ld_out=out.shape[1],
                   workspace=ws.data_ptr() if need.value else None, workspace_bytes=need.value, stream=1)
    rc = Z.lib().zkml_selftest_linear_wait(lin._handle, C.addressof(c), withhold, limit_ms)
    torch.cuda.synchronize()
    return rc


# 1: the accumulators' completion, 2: a copy of weights, 3: the activation table, 4: a tile of activations
@pytest.mark.parametrize("m,k,withhold,act", [(16, 256, 1, "none"), (16, 256, 2, "none"), (16, 256, 3, "silu"),
                                              (16, 2000, 1, "gelu"), (16, 2000, 2, "gelu"),
                                              (1, 256, 1, "none"), (1, 256, 2, "none"), (1, 256, 4, "silu"),
                                              (7, 700, 1, "none"), (7, 700, 2, "none"), (7, 700, 4, "none")])
def test_a_wait_that_runs_out_is_reported_and_its_tile_is_left_alone(m, k, withhold, act):
    """One whole tile of 128 outputs to a block, so what block 0 gives up is the first 128 columns."""
    n = 128 * torch.cuda.get_device_properties(0).multi_processor_count
    x, w = ints((m, k), 31, m), ints((k, n), 8, k)
    y, _, unsure = L.linear(x, w, None, TAGS[act])
    lin, tx = Z.LinearM31(dev(w)), dev(x)
    out = torch.full((m, n), MARK, dtype=torch.int32, device="cuda")
    assert selftest(lin, tx, out, act, withhold) == 0
    assert (out[:, :128] == MARK).all()
    L.same(host(out[:, 128:].contiguous()), y[:, 128:], unsure[:, 128:])
    with pytest.raises(Z.ZkmlError) as e:
        lin.check()
    assert e.value.status == TIMEOUT
    lin.check()  # reported once
    L.same(host(lin(tx, activation=act, out=out)), y, unsure)


@pytest.mark.parametrize("m,k,n,withhold", [(1, 2000, 1280, 1), (1, 2000, 1280, 2), (5, 2000, 1280, 4), (8, 1024, 200, 1),
                                            (5, 13824, 130, 2)])
def test_a_block_of_a_cluster_that_gives_up(m, k, n, withhold):
    """K is shared by a cluster: the rows of its tile are not finished from the parts that did arrive."""
    x, w = ints((m, k), 31, m), ints((k, n), 8, k)
    lin, tx, want = Z.LinearM31(dev(w)), dev(x), L.product(x, w)
    out = torch.full((m, n), MARK, dtype=torch.int32, device="cuda")
    assert selftest(lin, tx, out, "none", withhold) == 0
    assert (out[:, :128] == MARK).all()
    L.same(host(out[:, 128:].contiguous()), want[:, 128:])
    with pytest.raises(Z.ZkmlError) as e:
        lin.check()
    assert e.value.status == TIMEOUT
    L.same(host(lin(tx, out=out)), want)


@pytest.mark.parametrize("m,k,n", [(40, 2000, 300), (200, 1000, 130)])
@pytest.mark.parametrize("withhold", [1, 2])
def test_a_share_of_a_cut_tile_that_never_comes(m, k, n, withhold):
    """Tiles cut over several blocks: a tile that lacks a part is left alone, every written word is right."""
    x, w = ints((m, k), 31, m), ints((k, n), 8, k)
    lin, tx, want = Z.LinearM31(dev(w)), dev(x), L.product(x, w)
    out = torch.full((m, n), MARK, dtype=torch.int32, device="cuda")
    assert selftest(lin, tx, out, "none", withhold) == 0
    left = (out == MARK).cpu().numpy()
    assert left.any() and (left | (host(out) == want)).all()
    with pytest.raises(Z.ZkmlError) as e:
        lin.check()
    assert e.value.status == TIMEOUT
    L.same(host(lin(tx, out=out)), want)


def test_refusals_of_the_wait_self_test():
    w = dev(ints((40, 30), 8, 1))
    lin, gat = Z.LinearM31(w), Z.GatedLinearM31(w, w)
    x, few = (torch.zeros(m, 40, dtype=torch.int32, device="cuda") for m in (40, 1))
    out = torch.zeros(40, 30, dtype=torch.int32, device="cuda")
    for args in ((lin, x, out, "none", 0), (lin, x, out, "none", 5), (lin, x, out, "none", 1, 0), (lin, x, out, "none", 1, 1001),
                 (lin, x, out, "relu", 3), (lin, x, out, "none", 4), (lin, few, out[:1], "silu", 3), (gat, x, out, "none", 1)):
        assert selftest(*args) == 1, args[3:]
    lin.check()
