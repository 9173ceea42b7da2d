"""Plain 64-bit forms of the forward operators (numpy), for the tests."""
import numpy as np

P = (1 << 31) - 1
HALF = (P - 1) // 2


def words(v):
    """Signed integers as M31 words."""
    return (np.asarray(v, np.int64) % P).astype(np.uint32)


def signed(v):
    v = np.asarray(v, np.int64) % P
    return np.where(v > HALF, v - P, v)


def product(x, w):
    """x w mod P: 16-bit halves of x, so every 64-bit sum stays below 2^16 2^31 k < 2^62 (k < 2^15)."""
    x, w = np.asarray(x, np.int64) % P, np.asarray(w, np.int64) % P
    assert x.shape[1] < 1 << 15
    hi = ((x >> 16) @ w) % P
    lo = ((x & 0xffff) @ w) % P
    return (hi * 65536 + lo) % P


def activation(z, tag):
    """ActivationType::as_fn on full field elements, and where it may be off by one: a binary64 evaluation
    is within 2^-50 of a value below 2^31 in units of 2^-16, so only where it lies within 2^-19 of a
    half-integer can two correct evaluations round to different sides."""
    z = np.asarray(z, np.int64) % P
    unsure = np.zeros(z.shape, bool)
    if tag == 0:
        return z, unsure
    neg = z > HALF
    if tag == 1:
        return np.where(neg, 0, z), unsure
    if tag == 3:
        return np.where(neg, 0, np.where(z == 0, 32768, 65536)), unsure
    if tag == 4:
        down = np.maximum(65536 >> np.minimum((P - 1 - z) // 65536, 20), 1)
        up = 65536 << np.minimum(z // 65536, 10)
        return np.where(neg, down, np.minimum(up, P - 1)), unsure
    x = signed(z) / 65536.0
    with np.errstate(over="ignore"):
        if tag == 2:
            r = 0.5 * x * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (x + 0.044715 * x * x * x)))
        else:
            r = x / (1.0 + np.exp(-x))
    y = np.abs(r) * 65536.0
    q = np.floor(y)
    q = np.minimum(q + (y - q >= 0.5), P - 1).astype(np.int64)
    unsure = np.abs(y - np.floor(y) - 0.5) < 2.0 ** -19
    return np.where(r < 0, -q, q) % P, unsure


def linear(x, w, b=None, tag=0, r=None):
    """(y, z, unsure) of y = f(z) + r, z = x w + b."""
    z = product(x, w)
    if b is not None:
        z = (z + np.asarray(b, np.int64)) % P
    y, unsure = activation(z, tag)
    if r is not None:
        y = (y + np.asarray(r, np.int64)) % P
    return y, z, unsure


def gated(x, wg, wu, bg=None, bu=None, tag=5):
    """(h, g, u, unsure) of h = f(g) u."""
    f, g, unsure = linear(x, wg, bg, tag)
    u = linear(x, wu, bu)[0]
    return f * u % P, g, u, unsure


def same(got, want, unsure=None):
    """Equal words; an output that hangs on an unsure rounding is left out (a handful at most)."""
    got = np.asarray(got).astype(np.int64)
    assert got.shape == want.shape and got.min() >= 0 and got.max() < P
    ok = got == want
    if unsure is not None:
        assert unsure.sum() <= 4
        ok |= unsure
    assert ok.all(), f"{(~ok).sum()} of {ok.size} words differ, first at {np.argwhere(~ok)[0]}"
