"""Forward operators on the GPU where something goes wrong: waits that run out, words that do not belong,
several callers of one handle, and the ends of the accumulators' range."""
import ctypes as C

import numpy as np
import pytest
import torch

import linear_plain as L
import zkml_b200 as Z
from test_linear_checks import awkward_words
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


def test_a_call_answers_for_itself():
    """What another call of the handle met is neither raised by a checked call nor lost with it."""
    x, w = ints((4, 40), 31, 1), ints((40, 30), 8, 2)
    bx = x.copy()
    bx[3, 39] = 0x80000001
    for m in (4, 1):  # the bad word is in the last row
        lin, tx, bad, want = Z.LinearM31(dev(w)), dev(x[-m:]), dev(bx[-m:]), L.product(x[-m:], w)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            lin(bad, check=False)
        s1.synchronize()
        with torch.cuda.stream(s2):
            L.same(host(lin(tx)), want)  # checked, and right
            with pytest.raises(Z.InvalidArgument, match="2\\^31"):
                lin(bad)
            with pytest.raises(Z.InvalidArgument, match="2\\^31"):
                lin.check()  # the first call's, on s1
            lin.check()
            L.same(host(lin(tx)), want)


def run_threads(n, work):
    import threading
    errors = []

    def guarded(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                work(i)
        except BaseException as e:  # noqa: B902 -- reported below
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=guarded, args=(i,)) for i in range(n)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors[:3]


@pytest.mark.parametrize("n_threads,calls", [(8, 100), (80, 10)])
def test_checked_calls_of_many_threads(n_threads, calls):
    """Exactly the calls with a bad word raise, also with more callers than the handle has status words."""
    x, w = ints((9, 200), 8, 1), ints((200, 130), 8, 2)
    lin, tx, want = Z.LinearM31(dev(w)), dev(x), L.product(x, w)
    bad = tx.clone()
    bad[:, 7] = 1 << 20  # beyond 8 bits
    torch.cuda.synchronize()

    def work(i):
        for j in range(calls):
            m = 1 + (i + j) % 9
            if (i + j) % 2:
                with pytest.raises(Z.InvalidArgument, match="x_bits"):
                    lin(bad[:m], x_bits=8)
            else:
                L.same(host(lin(tx[:m], x_bits=8)), want[:m])

    run_threads(n_threads, work)
    lin.check()


def test_checks_of_several_threads_lose_nothing():
    """Every finding is raised by one of the checks that run at the same time."""
    w = ints((40, 30), 8, 2)
    lin = Z.LinearM31(dev(w))
    bad = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    raised, done = [0, 0, 0], []

    def check(i):
        try:
            lin.check()
        except Z.InvalidArgument:
            raised[i] += 1

    def work(i):
        import time
        if i:
            while not done:
                check(i)
            return
        try:
            for _ in range(300):
                before = sum(raised)
                lin(bad, check=False)
                torch.cuda.current_stream().synchronize()
                check(0)
                end = time.monotonic() + 5
                while sum(raised) == before:
                    assert time.monotonic() < end, "a finding was lost"
                    time.sleep(0)
        finally:
            done.append(1)

    run_threads(3, work)


def test_a_checked_call_is_refused_in_a_capture():
    """Before anything of it is launched, and the capture goes on."""
    x, w = ints((9, 200), 31, 1), ints((200, 130), 8, 2)
    lin, tx = Z.LinearM31(dev(w)), dev(x)
    lin(tx)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(Z.InvalidArgument, match="captured"):
            lin(tx)
        with pytest.raises(Z.InvalidArgument, match="captured"):
            lin.check()
        y = lin(tx, check=False)
    g.replay()
    torch.cuda.synchronize()
    L.same(host(y), L.product(x, w))
    lin.check()


HAMMER = """
#include <atomic>
#include <thread>
#include <vector>
extern "C" int hammer(int (*forward)(void*, const void*), void* lin, void* const* calls, int threads, int times) {
    std::atomic<int> failed{0}, ready{0};
    std::vector<std::thread> all;
    for (int t = 0; t < threads; t++)
        all.emplace_back([&, t] {
            ready++;
            while (ready < threads) {}
            for (int i = 0; i < times; i++) failed += forward(lin, calls[t]) != 0;
        });
    for (std::thread& t : all) t.join();
    return failed;
}
"""


def test_launches_of_several_threads_are_all_counted(tmp_path):
    """Native threads, which no interpreter lock keeps apart."""
    import subprocess
    (tmp_path / "hammer.cpp").write_text(HAMMER)
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-pthread", "-o", str(tmp_path / "hammer.so"),
                    str(tmp_path / "hammer.cpp")], check=True)
    w = ints((40, 30), 8, 2)
    lin, tx, threads, times = Z.LinearM31(dev(w)), dev(ints((1, 40), 31, 1)), 8, 5000
    out = torch.empty(threads, 30, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(threads)]
    calls = [LinearCall(x=tx.data_ptr(), m=1, ldx=40, x_bits=31, out=out[t].data_ptr(), ld_out=30,
                        stream=streams[t].cuda_stream, pointers_checked=1) for t in range(threads)]
    torch.cuda.synchronize()
    before = Z.context(0).kernel_launches()
    failed = C.CDLL(str(tmp_path / "hammer.so")).hammer(
        C.cast(Z.lib().zkml_linear_forward, C.c_void_p), lin._handle,
        (C.c_void_p * threads)(*(C.addressof(c) for c in calls)), threads, times)
    torch.cuda.synchronize()
    assert failed == 0
    assert Z.context(0).kernel_launches() - before == threads * times  # one launch a call for a single token
    assert torch.equal(out, lin(tx).expand(threads, 30))
    lin.check()


def test_host_weights_of_any_byte_stride():
    """Fields of records, odd addresses, both alone and beside a plain matrix in a gated block."""
    x, w, up, b = ints((3, 90), 31, 1), ints((90, 50), 8, 2), ints((90, 50), 8, 3), ints((50,), 31, 4)
    want = L.linear(x, w, b)[0]
    h, _, _, unsure = L.gated(x, w, up)
    wide = np.zeros((90, 100), np.uint32)[:, ::2]  # as many whole words from one to the next as a record's field
    wide[...] = up
    for weight, bias in zip(awkward_words(w), awkward_words(np.repeat(b[None], 2, 0))):
        L.same(host(Z.LinearM31(weight, bias[1])(dev(x))), want)
        for other in (up, wide, dev(up), np.asfortranarray(up)):
            L.same(host(Z.GatedLinearM31(weight, other)(dev(x))), h, unsure)


FIRST_HANDLE = """
import ctypes as C
import sys
sys.path[:0] = {path!r}
import numpy as np
import torch
import linear_plain as L
import zkml_b200 as Z
from test_linear_gpu import dev, host, ints

Z.context(0)
x, w = ints((9, 300), 8, 1), ints((300, 130), 8, 2)
tx, side, handle = dev(x), torch.cuda.Stream(), C.c_uint64()
assert int(torch.cuda.cudart().cudaStreamCreate(C.addressof(handle))) == 0  # a stream that orders with the legacy one
blocking, g = torch.cuda.ExternalStream(handle.value), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=blocking, capture_error_mode="relaxed"):
    twice = tx + tx
    with torch.cuda.stream(side):
        lin = Z.LinearM31(w)
with torch.cuda.stream(side):
    for m in (9, 1):  # both kernels read the tables
        y, _, unsure = L.linear(x[:m], w, None, 5)
        L.same(host(lin(tx[:m], activation="silu", x_bits=8)), y, unsure)
g.replay()
torch.cuda.synchronize()
assert torch.equal(twice, tx + tx)
print("ok")
"""


def test_the_first_handle_uses_its_own_stream_alone():
    """A process's first handle uploads the activation tables; made beside the capture of a stream that orders
    with the legacy stream, it neither fails nor ends the capture."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    path = [str(root), str(root / "tests"), str(root / "stwo-ml_b200")]
    r = subprocess.run([sys.executable, "-c", FIRST_HANDLE.format(path=path)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-4000:]


def test_a_forward_pass_gives_large_scratch_back():
    """Weights of any field element (four bytes each when laid out, 64 MiB and more) leave no more of the
    memory taken than signed bytes of the same shape do."""
    d = 4096
    x = L.words(np.random.default_rng(1).integers(-50, 50, (2, d)))

    def free_after(w):
        p = Z.prove_gkr_chain(x, [("linear", w)], n_queries=2)
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0], p.io_commitment

    narrow, wide = ints((d, d), 8, 1), ints((d, d), 31, 2)
    free_after(narrow)
    before, io = free_after(narrow)
    after, wide_io = free_after(wide)
    assert after >= before
    assert free_after(narrow)[1] == io and free_after(wide)[1] == wide_io


def test_arrays_and_tensors_in_one_call():
    x, w, r = ints((4, 40), 31, 1), ints((40, 30), 8, 2), ints((4, 30), 31, 3)
    lin, tx = Z.LinearM31(dev(w)), dev(x)
    for args in (dict(residual=r), dict(residual=r[0]), dict(out=np.zeros((4, 30), np.uint32)), dict(pre=r)):
        with pytest.raises(Z.InvalidArgument):
            lin(tx, **args)
    with pytest.raises(Z.InvalidArgument):
        lin(x, out=torch.zeros(4, 30, dtype=torch.int32, device="cuda"))
    L.same(lin(x, residual=dev(r)), L.linear(x, w, None, 0, r)[0])


SEGMENT = 1023 * 128  # K of one 32-bit accumulation


def extreme_rows(m, k, x_bits, rng):
    """Rows of two constants each (at the ends of the digits' range in most), and where the second begins."""
    ends = {8: [-128, 127], 16: [-32768, 32767, -32640, 128 - 128 * 257],
            31: [-(1 << 30) + 1, (1 << 30) - 1, 128 - 128 * 65793, 128 + 127 * 65793]}[x_bits]
    first = np.array([ends[i % len(ends)] for i in range(m)], np.int64)
    second = np.array([ends[(i // len(ends)) % len(ends)] for i in range(m)], np.int64)
    at = rng.integers(0, k, m)
    at[0] = k
    x = torch.empty(m, k, dtype=torch.int32, device="cuda")
    for i in range(m):
        x[i, :at[i]], x[i, at[i]:] = int(L.words(first[i])), int(L.words(second[i]))
    return x, first, second, at


def sliding_weights(k, n, top, rng):
    """w[t][j] = v[t + j], v at one end of the signed bytes but for a few: its column sums come from prefix sums."""
    v = np.full(k + n - 1, top, np.int64)
    v[rng.integers(0, v.size, 64)] = rng.integers(-128, 128, 64)
    d = dev(L.words(v))
    return torch.as_strided(d, (k, n), (1, 1)), np.concatenate([[0], np.cumsum(v)])


def sliding_product(rows, sums, k, n):
    _, first, second, at = rows
    j = np.arange(n)
    head = sums[at[:, None] + j] - sums[j]             # sum of w[t][j] over t < at
    tail = sums[k + j] - sums[at[:, None] + j]
    assert np.abs(sums).max() < 1 << 32                # times a first or second below 2^31: 63 bits
    return (first[:, None] * head % P + second[:, None] * tail % P) % P


@pytest.mark.parametrize("top", [-128, 127])
@pytest.mark.parametrize("m,x_bits,extra", [(16, 31, 0), (16, 31, 2), (16, 8, 0), (16, 8, 2), (16, 16, 2), (40, 31, 2), (1, 31, 0)])
def test_accumulations_are_cut_where_32_bits_end(m, x_bits, extra, top):
    """Whole tiles of K past one accumulation, and (extra tiles) shares of cut tiles as long as that."""
    k, n = 1100 * 128, 128 * (torch.cuda.get_device_properties(0).multi_processor_count + extra)
    assert k > SEGMENT and 128 * 128 * (k - 64) > 1 << 31  # digits and weights of -128: past 32 bits without a cut
    rng = np.random.default_rng(500 + m + x_bits + extra + top)
    rows, (w, sums) = extreme_rows(m, k, x_bits, rng), sliding_weights(k, n, top, rng)
    L.same(host(Z.LinearM31(w)(rows[0], x_bits=x_bits)), sliding_product(rows, sums, k, n))


@pytest.mark.parametrize("extra", [0, 2])
def test_gated_accumulations_are_cut_where_32_bits_end(extra):
    m, k, n = 16, 1100 * 128, 64 * (torch.cuda.get_device_properties(0).multi_processor_count + extra)
    rng = np.random.default_rng(extra)
    rows, (wg, sg), (wu, su) = extreme_rows(m, k, 31, rng), sliding_weights(k, n, -128, rng), sliding_weights(k, n, 127, rng)
    g, u = sliding_product(rows, sg, k, n), sliding_product(rows, su, k, n)
    got = Z.GatedLinearM31(wg, wu)(rows[0], activation="relu", keep=True)
    for a, want in zip(got, (L.activation(g, 1)[0] * u % P, g, u)):
        L.same(host(a), want)


@pytest.mark.parametrize("m,x_bits", [(1, 31), (8, 31), (3, 8), (8, 16)])
@pytest.mark.parametrize("top", [-128, 127])
def test_shares_of_a_cluster_up_to_one_accumulation(m, x_bits, top):
    """A few tokens, K over six blocks: each share is the longest that the kernel for few tokens takes."""
    k, n = 6137 * 128, 100
    assert SEGMENT - 256 < k // 6 <= SEGMENT
    rng = np.random.default_rng(500 + m + x_bits + top)
    rows, (w, sums) = extreme_rows(m, k, x_bits, rng), sliding_weights(k, n, top, rng)
    L.same(host(Z.LinearM31(w)(rows[0], x_bits=x_bits)), sliding_product(rows, sums, k, n))


@pytest.mark.parametrize("m,x_bits", [(1, 31), (4, 31), (8, 31), (2, 16), (8, 8)])
@pytest.mark.parametrize("w_bits", [16, 24, 31])
@pytest.mark.parametrize("k", [1024, 2600])
def test_wide_weights_over_a_cluster(k, w_bits, m, x_bits):
    """Several planes of weights where K is shared by the blocks of a cluster."""
    n = 200
    x, w, w2, r = ints((m, k), x_bits, 1), ints((k, n), w_bits, 2), ints((k, n), w_bits, 3), ints((m, n), 31, 4)
    y, z, unsure = L.linear(x, w, None, 5, r)
    got = Z.LinearM31(dev(w))(dev(x), activation="silu", residual=dev(r), keep=True, x_bits=x_bits)
    L.same(host(got[1]), z)
    L.same(host(got[0]), y, unsure)
    h, g, u, unsure = L.gated(x, w, w2)
    got = Z.GatedLinearM31(dev(w), dev(w2))(dev(x), keep=True, x_bits=x_bits)
    for a, want in zip(got, (h, g, u)):
        L.same(host(a), want, unsure if want is h else None)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("m", [1, 40])
def test_inputs_written_late_on_another_stream(m, captured):
    """A call behind another call of its stream and an event of a second stream: it starts early for the first,
    and still waits for the second."""
    k, n = 600, 300
    x, w = ints((m, k), 31, 1), ints((k, n), 8, 2)
    lin, other, want = Z.LinearM31(dev(w)), Z.LinearM31(dev(w)), L.product(x, w)
    source, tx = dev(x), torch.zeros(m, k, dtype=torch.int32, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()

    def step():
        s1.wait_stream(s2)
        with torch.cuda.stream(s1):
            torch.cuda._sleep(2_000_000)
            tx.copy_(source)
        with torch.cuda.stream(s2):
            other(source, check=False)
            s2.wait_stream(s1)
            y = lin(tx, check=False)
            z = other(tx, residual=y, check=False)
            tx.zero_()  # the calls have read it by then
        return y, z

    torch.cuda.synchronize()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s2):
            y, z = step()
    for _ in range(4):
        if captured:
            g.replay()
        else:
            y, z = step()
        torch.cuda.synchronize()
        L.same(host(y), want)
        L.same(host(z), 2 * want % P)
    lin.check()
    other.check()


@pytest.mark.parametrize("m", [9, 1])
def test_rows_further_apart_than_32_bits(m):
    """x, residual, input of the activation and result as column ranges of one buffer whose rows are 2^29 words
    apart: the ninth row begins 2^32 words in."""
    k, n, ld = 300, 130, 1 << 29
    x, w, r = ints((10, k), 8, 1), ints((k, n), 8, 2), ints((10, n), 31, 3)
    buf = torch.empty(9 * ld + 4096, dtype=torch.int32, device="cuda")
    first = 10 - m  # one token: the last row alone, at its own offset
    rows = torch.as_strided(buf, (m, 4096), (ld, 1), first * ld if m == 1 else 0)
    rows.fill_(MARK)
    at = {"x": (7, k), "r": (400, n), "z": (700, n), "y": (1001, n)}
    part = {name: rows[:, a:a + width] for name, (a, width) in at.items()}
    part["x"].copy_(dev(x[first:]))
    part["r"].copy_(dev(r[first:]))
    y, z, unsure = L.linear(x[first:], w, None, 5, r[first:])
    Z.LinearM31(dev(w))(part["x"], activation="silu", residual=part["r"], out=part["y"], pre=part["z"], x_bits=8)
    L.same(host(part["y"].contiguous()), y, unsure)
    L.same(host(part["z"].contiguous()), z)
    rest = torch.ones(m, 4096, dtype=torch.bool, device="cuda")
    for a, width in at.values():
        rest[:, a:a + width] = False
    assert (rows[rest] == MARK).all()


@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("m", [1, 7, 24, 200])
def test_calls_that_read_what_the_call_before_wrote_beside_its_input(m, gap):
    """Two column ranges of one buffer in turn, input and result of one call sharing sectors: what is kept of a
    range from an earlier read never stands for what has been written since."""
    d = 137
    w, x = ints((d, d), 31, 1), ints((m, d), 31, 2)
    lin = Z.LinearM31(dev(w))
    buf = torch.zeros(m, 2 * d + gap + 5, dtype=torch.int32, device="cuda")
    parts = [buf[:, 1:1 + d], buf[:, 1 + d + gap:1 + 2 * d + gap]]
    parts[0].copy_(dev(x))
    torch.cuda._sleep(5_000_000)  # the calls queue up and start early
    want = x
    for i in range(40):
        lin(parts[i % 2], out=parts[1 - i % 2], check=False)
        want = L.product(want, w)
    L.same(host(parts[0].contiguous()), want)
    lin.check()
