"""Forward operators on the GPU against their plain 64-bit forms: every output word is equal."""
import ctypes as C

import numpy as np
import pytest
import torch

import linear_plain as L
import zkml_b200 as Z
from helpers import uniform_m31

pytestmark = pytest.mark.gpu
P = L.P
TAGS = {"none": 0, "relu": 1, "gelu": 2, "sigmoid": 3, "softmax": 4, "silu": 5}


def ints(shape, bits, stream):
    """Seeded words of `bits`-bit signed integers (31: any word below P), the ends of the range among them."""
    rng = np.random.default_rng(1000 * bits + stream)
    if bits == 31:
        v = rng.integers(0, P, shape)
        v.flat[0] = HALF_UP if v.size < 3 else P - 1
    else:
        v = rng.integers(-(1 << (bits - 1)), 1 << (bits - 1), shape)
        v.flat[0], v.flat[-1] = -(1 << (bits - 1)), (1 << (bits - 1)) - 1
    return L.words(v)


HALF_UP = (P + 1) // 2


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint32)


@pytest.mark.parametrize("x_bits", [8, 16, 31])
@pytest.mark.parametrize("w_bits", [8, 16, 24, 31])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 576, 130), (2, 33, 17), (5, 127, 129), (17, 128, 128), (64, 300, 257),
                                   (65, 129, 64), (130, 257, 33), (300, 1000, 40)])
def test_linear_shapes_and_widths(m, k, n, x_bits, w_bits):
    x, w = ints((m, k), x_bits, m), ints((k, n), w_bits, n)
    lin = Z.LinearM31(dev(w))
    L.same(host(lin(dev(x), x_bits=x_bits)), L.product(x, w))


@pytest.mark.parametrize("k", [100, 512, 1000, 1024, 1500, 2047, 2600, 3100, 3600, 4096, 9000])
@pytest.mark.parametrize("m,x_bits", [(1, 31), (3, 31), (4, 31), (5, 31), (8, 31), (9, 31), (1, 16), (8, 16), (13, 16),
                                      (16, 16), (1, 8), (16, 8), (29, 8), (32, 8), (33, 8)])
def test_a_few_tokens(k, m, x_bits):
    """One to eight blocks share K; both digit widths, and the sizes around where the kernels change."""
    n = 200
    x, w, w2, r = ints((m, k), x_bits, 1), ints((k, n), 8, 2), ints((k, n), 8, 3), ints((m, n), 31, 4)
    y, z, unsure = L.linear(x, w, None, 5, r)
    got = Z.LinearM31(dev(w))(dev(x), activation="silu", residual=dev(r), keep=True, x_bits=x_bits)
    L.same(host(got[1]), z)
    L.same(host(got[0]), y, unsure)
    h, g, u, unsure = L.gated(x, w, w2)
    got = Z.GatedLinearM31(dev(w), dev(w2))(dev(x), keep=True, x_bits=x_bits)
    L.same(host(got[1]), g)
    L.same(host(got[2]), u)
    L.same(host(got[0]), h, unsure)


@pytest.mark.parametrize("act", list(TAGS))
@pytest.mark.parametrize("bias,residual,keep", [(0, 0, 0), (1, 0, 1), (0, 1, 0), (1, 1, 1)])
def test_linear_epilogues(act, bias, residual, keep):
    """8-bit inputs over k = 300: |z| < 300 2^14 = 75 in fixed point, where the functions bend."""
    m, k, n = 37, 300, 259
    x, w = ints((m, k), 8, 1), ints((k, n), 8, 2)
    b = ints((n,), 16, 3) if bias else None
    r = ints((m, n), 31, 4) if residual else None
    lin = Z.LinearM31(dev(w), bias=None if b is None else dev(b))
    got = lin(dev(x), activation=act, residual=None if r is None else dev(r), keep=bool(keep), x_bits=8)
    y, z, unsure = L.linear(x, w, b, TAGS[act], r)
    if keep:
        L.same(host(got[1]), z)
        got = got[0]
    L.same(host(got), y, unsure)


@pytest.mark.parametrize("act", list(TAGS))
@pytest.mark.parametrize("bits", [8, 31])
def test_activations_at_their_bends(act, bits):
    """k = 1, x = 1: z is the weight itself, so the epilogue sees chosen words: zero, the sign's border, the
    places where SiLU, GELU and their roundings saturate, the segments of Softmax-exp."""
    near = np.array([0, 1, 2, 65535, 65536, 65537, 1 << 19, 1 << 20, (1 << 20) + 1, 12 * 65536, 16 * 65536, 20 * 65536,
                     30 * 65536, 36 * 65536, 37 * 65536, 38 * 65536, 40 * 65536, 11 << 16, (1 << 30) - 1])
    v = np.unique(np.concatenate([near + d for d in range(-3, 4)]))
    v = np.concatenate([v, -v, np.random.default_rng(5).integers(-40 * 65536, 40 * 65536, 4000)])
    v = v[np.abs(v) < 1 << 30]
    z = L.words(v)
    if bits == 8:
        x, w = np.ones((1, 1), np.uint32), z.reshape(1, -1)
    else:  # the chosen words come from x, one to a token
        x, w = z.reshape(-1, 1), np.ones((1, 1), np.uint32)
    y, zz, unsure = L.linear(x, w, None, TAGS[act])
    assert unsure.sum() <= 4
    L.same(host(Z.LinearM31(dev(w))(dev(x), activation=act)), y, unsure)


@pytest.mark.parametrize("act,first", [("silu", i << 20) for i in range(-2, 3)] + [("gelu", -(1 << 20)), ("gelu", 0)])
def test_every_word_where_the_function_bends(act, first):
    """2^20 consecutive words at a time: SiLU bends for reals in (-16, 37), GELU in (-8.5, 8.5).  Left out
    are the words whose binary64 value lies within 2^-19 of a half-integer: 2^-18 of them, 4 expected."""
    z = L.words(first + np.arange(1 << 20))
    y, unsure = L.activation(z, TAGS[act])
    assert unsure.sum() < 40
    got = host(Z.LinearM31(dev(z.reshape(1, -1)))(torch.ones(1, 1, dtype=torch.int32, device="cuda"),
                                                  activation=act)).reshape(-1).astype(np.int64)
    assert ((got == y) | unsure).all()


@pytest.mark.parametrize("x_bits,w_bits,keep,bias", [(31, 8, True, False), (8, 8, True, True), (16, 8, False, True),
                                                     (31, 31, True, True)])
@pytest.mark.parametrize("m,k,n", [(1, 64, 1), (1, 576, 200), (3, 130, 63), (33, 257, 65), (70, 128, 129), (140, 96, 64)])
def test_gated(m, k, n, x_bits, w_bits, keep, bias):
    x, wg, wu = ints((m, k), x_bits, 1), ints((k, n), w_bits, 2), ints((k, n), w_bits, 3)
    bg, bu = (ints((n,), 31, 4), ints((n,), 31, 5)) if bias else (None, None)
    op = Z.GatedLinearM31(dev(wg), dev(wu), *(None if b is None else dev(b) for b in (bg, bu)))
    got = op(dev(x), activation="silu", x_bits=x_bits, keep=keep)
    h, g, u, unsure = L.gated(x, wg, wu, bg, bu)
    if keep:
        L.same(host(got[1]), g)
        L.same(host(got[2]), u)
        got = got[0]
    L.same(host(got), h, unsure)


@pytest.mark.parametrize("act", list(TAGS))
def test_gated_activations(act):
    x, wg, wu = ints((9, 200), 8, 1), ints((200, 70), 8, 2), ints((200, 70), 8, 3)
    h, _, _, unsure = L.gated(x, wg, wu, tag=TAGS[act])
    L.same(host(Z.GatedLinearM31(dev(wg), dev(wu))(dev(x), activation=act, x_bits=8)), h, unsure)


def test_one_bias_of_two():
    x, wg, wu, b = ints((3, 40), 31, 1), ints((40, 9), 8, 2), ints((40, 9), 8, 3), ints((9,), 31, 4)
    for bg, bu in ((b, None), (None, b)):
        op = Z.GatedLinearM31(dev(wg), dev(wu), None if bg is None else dev(bg), None if bu is None else dev(bu))
        h, _, _, unsure = L.gated(x, wg, wu, bg, bu)
        L.same(host(op(dev(x))), h, unsure)


@pytest.mark.parametrize("x_bits,xv", [(8, -128), (8, 127), (16, -32768), (16, 32767), (31, HALF_UP), (31, HALF_UP - 1)])
@pytest.mark.parametrize("wv", [-128, 127])
def test_largest_sums(x_bits, xv, wv):
    """Every product at the end of its range, over the longest sums of the layers here."""
    k = 13824
    x, w = L.words(np.full((2, k), xv)), L.words(np.full((k, 3), wv))
    want = int(L.signed(xv)) * wv * k % P
    assert (host(Z.LinearM31(dev(w))(dev(x), x_bits=x_bits)) == want).all()


@pytest.mark.parametrize("wv", [-128, 127, HALF_UP])
def test_sums_longer_than_a_32_bit_accumulator(wv):
    k = 300001
    x, w = L.words(np.full((1, k), HALF_UP)), L.words(np.full((k, 2), wv))
    want = HALF_UP * (wv % P) * k % P
    assert (host(Z.LinearM31(dev(w))(dev(x))) == want).all()


def test_one_wide_weight_among_narrow_ones():
    x, w = ints((4, 700), 31, 1), ints((700, 300), 8, 2)
    for v in (128, -129, 40000, 1 << 23, HALF_UP, HALF_UP - 1):
        w[699, 299] = L.words(v)
        L.same(host(Z.LinearM31(dev(w))(dev(x))), L.product(x, w))


def test_word_p_is_zero():
    x, w, b, r = (np.full(s, P, np.uint32) for s in ((2, 5), (5, 3), (3,), (2, 3)))
    lin = Z.LinearM31(dev(w), bias=dev(b))
    for act, want in (("none", 0), ("sigmoid", 32768), ("softmax", 65536), ("silu", 0), ("gelu", 0)):
        assert (host(lin(dev(x), activation=act, residual=dev(r))) == want).all()


def test_strided_arguments_and_untouched_words():
    """x, residual and outputs as column ranges of wider buffers; nothing beside or below them changes."""
    m, k, n = 19, 100, 77
    x, w, r = ints((m, k), 31, 1), ints((k, n), 8, 2), ints((m, n), 31, 3)
    xb = torch.full((m, k + 13), -5, dtype=torch.int32, device="cuda")
    rb = torch.full((m, n + 1), -5, dtype=torch.int32, device="cuda")
    ob = torch.full((m + 40, 2 * n + 9), -7, dtype=torch.int32, device="cuda")
    xb[:, 3:3 + k], rb[:, :n] = dev(x), dev(r)
    y, z = ob[:m, 1:1 + n], ob[:m, n + 4:2 * n + 4]  # interleaved rows of one buffer
    got = Z.LinearM31(dev(w))(xb[:, 3:3 + k], activation="silu", residual=rb[:, :n], out=y, pre=z)
    wy, wz, unsure = L.linear(x, w, None, 5, r)
    assert got[0] is y and got[1] is z
    L.same(host(y.contiguous()), wy, unsure)
    L.same(host(z.contiguous()), wz)
    rest = torch.ones_like(ob, dtype=torch.bool)
    rest[:m, 1:1 + n] = False
    rest[:m, n + 4:2 * n + 4] = False
    assert (ob[rest] == -7).all() and (xb[:, :3] == -5).all()


def test_residual_in_place_and_repeated_rows():
    m, k, n = 70, 64, 65
    x, w, r = ints((m, k), 31, 1), ints((k, n), 8, 2), ints((m, n), 31, 3)
    lin = Z.LinearM31(dev(w))
    acc = dev(r)
    lin(dev(x), residual=acc, out=acc)
    L.same(host(acc), L.linear(x, w, None, 0, r)[0])
    L.same(host(lin(dev(x), residual=dev(r[5]))), L.linear(x, w, None, 0, r[5])[0])
    rows = dev(x[7:8]).expand(m, k)
    L.same(host(lin(rows)), np.repeat(L.product(x[7:8], w), m, 0))


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_unaligned_rows(offset):
    m, k, n = 5, 97, 35
    x, w = ints((m, k), 31, 1), ints((k, n), 8, 2)
    buf = torch.zeros(m * k + 8, dtype=torch.int32, device="cuda")
    buf[offset:offset + m * k] = dev(x).reshape(-1)
    L.same(host(Z.LinearM31(dev(w))(buf[offset:offset + m * k].view(m, k))), L.product(x, w))


def test_transposed_host_and_strided_weights():
    x, w = ints((6, 90), 31, 1), ints((90, 50), 8, 2)
    wide = torch.zeros(90, 64, dtype=torch.int32, device="cuda")
    wide[:, 7:57] = dev(w)
    want = L.product(x, w)
    for weight in (dev(w.T).t(), w, np.ascontiguousarray(w.T).T, wide[:, 7:57], torch.from_numpy(w.view(np.int32))):
        L.same(host(Z.LinearM31(weight)(dev(x))), want)
    h, _, _, unsure = L.gated(x, w, w[:, ::-1])
    up = np.ascontiguousarray(w[:, ::-1])
    for gate_up in ((dev(w), dev(up.T).t()), (w, np.asfortranarray(up)), (w, np.flip(np.ascontiguousarray(np.flip(up)))), (dev(w), up), (w, dev(up))):
        L.same(host(Z.GatedLinearM31(*gate_up)(dev(x))), h, unsure)


def test_shapes_of_more_dimensions_and_arrays():
    x, w = ints((12, 40), 31, 1), ints((40, 30), 8, 2)
    lin, want = Z.LinearM31(dev(w)), L.product(x, w)
    assert lin(dev(x).view(3, 4, 40)).shape == (3, 4, 30)
    L.same(host(lin(dev(x).view(3, 4, 40))).reshape(12, 30), want)
    L.same(host(lin(dev(x)[0])), want[0])
    y, z = lin(x, activation="relu", keep=True)
    L.same(y, L.linear(x, w, None, 1)[0])
    L.same(z, want)
    out = torch.zeros(30, dtype=torch.int32, device="cuda")
    lin(dev(x)[3], out=out)
    L.same(host(out), want[3])
    got = lin(dev(x).view(torch.uint32))
    assert got.dtype == torch.int32
    L.same(host(got), want)


def test_bad_words_are_reported_once():
    x, w, r = ints((4, 40), 31, 1), ints((40, 30), 8, 2), ints((4, 30), 31, 3)
    lin, want = Z.LinearM31(dev(w)), L.linear(x, w, None, 0, r)[0]
    bx, br = x.copy(), r.copy()
    bx[3, 39], br[0, 0] = 0x80000001, 0xffffffff
    for args in ((bx, r), (x, br)):
        with pytest.raises(Z.InvalidArgument, match="2\\^31"):
            lin(dev(args[0]), residual=dev(args[1]))
        L.same(host(lin(dev(x), residual=dev(r))), want)
    lin(dev(bx), check=False)
    lin(dev(x), check=False)
    with pytest.raises(Z.InvalidArgument, match="2\\^31"):
        lin.check()
    lin.check()
    bw = w.copy()
    bw[39, 29] = 0x80000000
    with pytest.raises(Z.InvalidArgument, match="2\\^31"):
        Z.LinearM31(dev(bw))
    with pytest.raises(Z.InvalidArgument, match="2\\^31"):
        Z.LinearM31(dev(w), bias=dev(bw[39]))


@pytest.mark.parametrize("bits", [8, 16])
def test_activations_wider_than_declared_are_reported(bits):
    w = ints((40, 30), 8, 2)
    lin = Z.LinearM31(dev(w))
    top = 1 << (bits - 1)
    for v in (top, -top - 1):
        x = L.words(np.zeros((2, 40)))
        x[1, 17] = L.words(v)
        with pytest.raises(Z.InvalidArgument, match="x_bits"):
            lin(dev(x), x_bits=bits)
    for v in (top - 1, -top):
        x[1, 17] = L.words(v)
        L.same(host(lin(dev(x), x_bits=bits)), L.product(x, w))


def test_refused_calls():
    w = ints((40, 30), 8, 2)
    lin, gat = Z.LinearM31(dev(w)), Z.GatedLinearM31(dev(w), dev(w))
    x = torch.zeros(4, 40, dtype=torch.int32, device="cuda")
    o = torch.zeros(4, 30, dtype=torch.int32, device="cuda")
    buf = torch.zeros(4, 100, dtype=torch.int32, device="cuda")
    for call in (lambda: lin(x, x_bits=9), lambda: lin(x, activation=6), lambda: lin(x, activation=-1),
                 lambda: lin(x[:, :39]), lambda: lin(x.t()), lambda: lin(x.float()), lambda: lin(x.cpu()),
                 lambda: lin(x[:0]), lambda: lin(x, residual=o[:3]), lambda: lin(x, out=o[:3]),
                 lambda: lin(x, out=o[0].expand(4, 30)), lambda: lin(x, out=o, pre=o),
                 lambda: lin(buf[:, :40], out=buf[:, 39:69]), lambda: lin(buf[:, :40], out=buf[:, 80:110]),
                 lambda: lin(x, residual=buf[:, :30], out=buf[:, 1:31]),
                 lambda: lin(x, residual=buf[:, :30], pre=buf[:, 10:40]),
                 lambda: gat(x, out=o, up=o), lambda: gat(x, gate=o, up=o),
                 lambda: Z.LinearM31(dev(w), bias=dev(w[0, :29])), lambda: Z.LinearM31(dev(w)[0]),
                 lambda: Z.LinearM31(torch.zeros(0, 4, dtype=torch.int32, device="cuda")),
                 lambda: Z.GatedLinearM31(dev(w), dev(w[:, :29])), lambda: Z.LinearM31(dev(w).float())):
        with pytest.raises((Z.InvalidArgument, TypeError)):
            call()
    lin(buf[:, :40], out=buf[:, 40:70])  # interleaved rows that share no word
    with pytest.raises(Z.InvalidArgument):
        lin.close()
        lin(x)


class LinearCall(C.Structure):
    """zkml_linear_call."""
    _fields_ = [("x", C.c_void_p), ("m", C.c_size_t), ("ldx", C.c_size_t), ("x_bits", C.c_int), ("activation", C.c_int),
                ("residual", C.c_void_p), ("ld_residual", C.c_size_t), ("out", C.c_void_p), ("ld_out", C.c_size_t),
                ("pre", C.c_void_p), ("ld_pre", C.c_size_t), ("up", C.c_void_p), ("ld_up", C.c_size_t),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("stream", C.c_void_p),
                ("pointers_checked", C.c_int)]


def _c_call(lin, **kw):
    c = LinearCall()
    for key, v in kw.items():
        setattr(c, key, v.data_ptr() if hasattr(v, "data_ptr") else v)
    return Z.lib().zkml_linear_forward(lin._handle, C.addressof(c))


def test_refused_at_the_c_boundary():
    w = ints((40, 30), 8, 2)
    lin, gat = Z.LinearM31(dev(w)), Z.GatedLinearM31(dev(w), dev(w))
    x = torch.zeros(40, 40, dtype=torch.int32, device="cuda")
    o, q = (torch.zeros(40, 30, dtype=torch.int32, device="cuda") for _ in range(2))
    need = C.c_size_t()
    assert Z.lib().zkml_linear_workspace(lin._handle, 40, 31, C.byref(need)) == 0
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device="cuda")
    good = dict(x=x, m=40, ldx=40, x_bits=31, out=o, ld_out=30, workspace=ws, workspace_bytes=need.value, stream=1)
    assert _c_call(lin, **good) == 0
    for change in (dict(x=None), dict(out=None), dict(m=0), dict(m=1 << 40), dict(ld_out=29), dict(x_bits=32),
                   dict(activation=6), dict(x=x.data_ptr() + 2), dict(x=x.cpu()), dict(out=o.cpu()), dict(up=q, ld_up=30),
                   dict(pre=q, ld_pre=29), dict(ldx=1 << 40)):
        assert _c_call(lin, **{**good, **change}) == 1, change
    assert _c_call(lin, **good, pointers_checked=1) == 0
    assert _c_call(lin, **{**good, "x": x.data_ptr() + 2}, pointers_checked=1) == 1
    if need.value:
        assert _c_call(lin, **{**good, "workspace": None}) == 1
        assert _c_call(lin, **{**good, "workspace_bytes": need.value - 1}) == 1
        assert _c_call(lin, **{**good, "workspace": ws.data_ptr() + 4}) == 1
    assert _c_call(gat, **{**good, "residual": q, "ld_residual": 30}) == 1
    torch.cuda.synchronize()


def test_another_stream_and_two_streams_at_once():
    m, k, n = 130, 700, 300
    x, w = ints((m, k), 31, 1), ints((k, n), 8, 2)
    lin, want = Z.LinearM31(dev(w)), L.product(x, w)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    tx = dev(x)
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(s1 if i % 2 else s2):
            outs.append(lin(tx + 0, check=False))
    torch.cuda.synchronize()
    for o in outs:
        L.same(host(o), want)
    with torch.cuda.stream(s1):
        lin.check()
        fresh = Z.LinearM31(dev(w) + 0)  # laid out in this stream's order
        got = fresh(tx)
    torch.cuda.synchronize()
    L.same(host(got), want)


def test_captured_and_replayed():
    """Two graphs of the same handles, replayed in turn with new inputs; checks while capturing are refused."""
    k, n = 256, 192
    wg, wu, wd = ints((k, n), 8, 1), ints((k, n), 8, 2), ints((n, k), 8, 3)
    gat, down = Z.GatedLinearM31(dev(wg), dev(wu)), Z.LinearM31(dev(wd))
    graphs = []
    for m in (1, 70):
        tx = torch.zeros(m, k, dtype=torch.int32, device="cuda")
        Z.gated_ffn_m31(tx, gat, down, residual=tx)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(Z.InvalidArgument):
                down(torch.zeros(1, n, dtype=torch.int32, device="cuda"))
            y = Z.gated_ffn_m31(tx, gat, down, residual=tx, check=False)
        graphs.append((m, tx, g, y))
    for i in range(3):
        runs = []
        for m, tx, g, y in graphs:
            x = ints((m, k), 31, 10 + i)
            tx.copy_(dev(x))
            g.replay()
            runs.append((x, y))
        torch.cuda.synchronize()
        for x, y in runs:
            h, _, _, unsure = L.gated(x, wg, wu)
            assert not unsure.any()
            L.same(host(y), L.linear(h, wd, None, 0, x)[0])
    gat.check()
    down.check()


def test_gated_block_in_a_row():
    m, k, n = 33, 160, 420
    x, r = ints((m, k), 8, 1), ints((m, k), 31, 2)
    wg, wu, wd = ints((k, n), 8, 3), ints((k, n), 8, 4), ints((n, k), 8, 5)
    bg, bu, bd = ints((n,), 16, 6), ints((n,), 16, 7), ints((k,), 31, 8)
    gat, down = Z.GatedLinearM31(dev(wg), dev(wu), dev(bg), dev(bu)), Z.LinearM31(dev(wd), dev(bd))
    h, _, _, unsure = L.gated(x, wg, wu, bg, bu)
    assert not unsure.any()
    want = L.linear(h, wd, bd, 0, r)[0]
    L.same(host(Z.gated_ffn_m31(dev(x), gat, down, residual=dev(r), x_bits=8)), want)
    L.same(Z.gated_ffn_m31(x, gat, down, residual=r, x_bits=8), want)
    small = Z.gated_ffn_m31(dev(x[:1]), gat, down, residual=dev(r[:1]), x_bits=8)
    L.same(host(small), want[:1])


def test_equal_results_on_every_run():
    x, w = dev(ints((200, 3000), 31, 1)), dev(ints((3000, 130), 8, 2))
    lin = Z.LinearM31(w)
    first = lin(x)
    for _ in range(20):
        assert torch.equal(lin(x), first)


def test_handles_closed_while_work_is_queued_and_while_capturing():
    """Closing waits for the calls that read the weights, and is no part of another handle's capture."""
    x, w = ints((300, 2000), 31, 1), ints((2000, 500), 8, 2)
    tx, tw, want = dev(x), dev(w), L.product(x, w)
    outs = []
    for _ in range(5):
        lin = Z.LinearM31(tw)
        outs += [lin(tx, check=False) for _ in range(3)]
        lin.close()
    torch.cuda.synchronize()
    for o in outs:
        L.same(host(o), want)
    lin, other = Z.LinearM31(tw), Z.LinearM31(tw)
    lin(tx)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(tx, check=False)
        other.close()
    g.replay()
    torch.cuda.synchronize()
    L.same(host(y), want)
    lin.check()


def test_a_call_behind_long_and_mixed_work():
    """Calls of every size in one stream, each reading the one before: nothing is read too early."""
    d = 640
    ws = [ints((d, d), 8, i) for i in range(3)]
    ops = [Z.LinearM31(dev(w)) for w in ws]
    x = ints((200, d), 31, 9)
    tx, y = dev(x), x
    torch.cuda._sleep(20_000_000)
    cur = tx
    for i, m in enumerate((200, 200, 40, 40, 8, 8, 1, 1)):
        cur = ops[i % 3](cur[:m], residual=cur[:m], check=False)
        y = L.linear(y[:m], ws[i % 3], None, 0, y[:m])[0]
    torch.cuda.synchronize()
    L.same(host(cur), y)


def test_two_threads_share_a_handle():
    import threading
    x, w = ints((50, 700), 31, 1), ints((700, 300), 8, 2)
    lin, want, tx = Z.LinearM31(dev(w)), L.product(x, w), dev(x)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [lin(tx[:1 + 7 * i], check=False) for _ in range(30)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i, outs in got.items():
        for o in outs:
            L.same(host(o), want[:1 + 7 * i])


@pytest.mark.parametrize("m,k,n", [(270001, 20, 8001), (600001, 4099, 3)])
def test_offsets_past_32_bits(m, k, n):
    """More than 2^31 words of output, of input and of digits: the first and last rows are right."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(0, P, (m, k), generator=g, device="cuda", dtype=torch.int32)
    w = ints((k, n), 8, 2)
    y = Z.LinearM31(dev(w))(x)
    for rows in (slice(0, 70), slice(m // 2, m // 2 + 70), slice(m - 70, m)):
        L.same(host(y[rows].contiguous()), L.product(host(x[rows].contiguous()), w))


def test_many_drawn_calls():
    """Sizes, widths, epilogues and strides drawn at random."""
    rng = np.random.default_rng(11)
    for i in range(60):
        m, k, n = (int(round(2 ** rng.uniform(0, top))) for top in (8, 10, 9))
        xb, wb = int(rng.choice([8, 16, 31])), int(rng.choice([8, 8, 16, 24, 31]))
        act = str(rng.choice(list(TAGS)))
        x, w, w2 = ints((m, k), xb, i), ints((k, n), wb, i + 1), ints((k, n), wb, i + 2)
        b, r = ints((n,), 31, i + 3), ints((m, n), 31, i + 4)
        px = torch.zeros(m, k + int(rng.integers(0, 5)), dtype=torch.int32, device="cuda")[:, :k]
        px.copy_(dev(x))
        y, z, unsure = L.linear(x, w, b, TAGS[act], r)
        got = Z.LinearM31(dev(w), bias=dev(b))(px, activation=act, residual=dev(r), keep=True, x_bits=xb)
        L.same(host(got[0]), y, unsure)
        L.same(host(got[1]), z)
        h, g, u, unsure = L.gated(x, w, w2, b, None, TAGS[act])
        got = Z.GatedLinearM31(dev(w), dev(w2), bias_gate=dev(b))(px, activation=act, keep=True, x_bits=xb)
        for a, want in zip(got, (h, g, u)):
            L.same(host(a), want, unsure if want is h else None)
