"""Measured calls of the forward operators over the Mersenne field P = 2^31 - 1.

* linear: y = f(x W + b) + r mod P, a matrix product with bias, activation and residual in its
  epilogue, with the pre-activation x W + b beside y where the activation is proved afterwards;
* gated: h = f(x Wg + bg) * (x Wu + bu) mod P, the up side of a gated feed-forward block, with both
  projections beside h where they are proved;
* ffn: gated, then linear with the residual, as a decoder layer runs them.

Values are field elements as int32 words in [0, P); v stands for v (v <= (P - 1) / 2) or v - P.  Weights
are quantised signed bytes, or any field element (w_bits 31).  x_bits is the width the activations
are quantised to: 8, 16, or 31 for any field element, which is what every layer behind the first
product sees, since products are not requantised.
"""
import torch

own = False

P = (1 << 31) - 1
HALF = (P - 1) // 2


def _case(name, op, m, k, n, act="none", x_bits=31, w_bits=8, bias=False, residual=False, keep=False):
    c = {"op": op, "m": m, "k": k, "n": n, "act": act, "x_bits": x_bits, "w_bits": w_bits, "bias": bias,
         "residual": residual, "keep": keep}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token through the small model's gate projection: a call of a few microseconds
        _case("linear_token_small", "linear", 1, 576, 1536, act="silu"),
        # one new token through the large model's down projection, added to the residual stream
        _case("linear_token_down", "linear", 1, 13824, 5120, residual=True),
        # the 64-token layer that is proved: int16 activations, SiLU, its input kept for the proof
        _case("linear_64_silu_kept", "linear", 64, 5120, 13824, act="silu", x_bits=16, keep=True),
        # ragged sizes, weights that are not quantised (any field element), every epilogue at once
        _case("linear_ragged_wide", "linear", 37, 1001, 579, act="gelu", w_bits=31, bias=True, residual=True,
              keep=True),
        # int8 activations of a model's first layer over a prompt
        _case("linear_prompt_int8", "linear", 512, 5120, 13824, x_bits=8, bias=True, act="relu"),
        # a long prompt through the output projection of attention, added to the residual stream
        _case("linear_prompt", "linear", 2048, 5120, 5120, residual=True),
        # one new token through the small model's gated block
        _case("gated_token_small", "gated", 1, 576, 1536, act="silu"),
        # one new token through the large model's gated block: two weights of 5120 x 13824
        _case("gated_token", "gated", 1, 5120, 13824, act="silu"),
        # the same layer for 64 tokens, both projections kept for the proof
        _case("gated_64_kept", "gated", 64, 5120, 13824, act="silu", keep=True),
        # odd sizes, biases, int8 activations: most SiLU inputs lie where the function bends
        _case("gated_odd", "gated", 131, 577, 1535, act="silu", x_bits=8, bias=True),
        # a long prompt through the gated block
        _case("gated_prompt", "gated", 2048, 5120, 13824, act="silu"),
        # a whole feed-forward block for a batch of 16 tokens: gated, down projection, residual
        _case("ffn_batch", "ffn", 16, 5120, 13824, act="silu", residual=True),
    ]


def _cost(c):
    products = {"linear": 1, "gated": 2, "ffn": 3}[c["op"]]
    return products * c["m"] * c["k"] * c["n"] * (4 if c["w_bits"] == 31 else 1)


def draw(rng):
    def size(lo, hi):
        return round(lo * (hi / lo) ** rng.random())  # spread over the logarithm

    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["linear", "linear", "gated", "gated", "ffn"])
        m, k, n = size(1, 2048), size(16, 13824), size(8, 13824)
        c = _case(None, op, m, k, n, act=rng.choice(["none", "relu", "gelu", "sigmoid", "softmax", "silu", "silu"]),
                  x_bits=rng.choice([8, 16, 31, 31]), w_bits=rng.choice([8, 8, 8, 31]), bias=rng.random() < 0.5,
                  residual=op != "gated" and rng.random() < 0.5, keep=op != "ffn" and rng.random() < 0.5)
        if _cost(c) <= most:
            return c


# ---- inputs -----------------------------------------------------------------------------------------


def _values(shape, bits, gen):
    """Uniform signed values of `bits` bits (31: any field element) as field elements."""
    if bits == 31:
        return torch.randint(0, P, shape, generator=gen, device="cuda", dtype=torch.int32)
    top = (1 << (bits - 1)) - 1
    v = torch.randint(-top, top + 1, shape, generator=gen, device="cuda", dtype=torch.int32)
    return torch.where(v < 0, v + P, v)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, n, op, wb = case["m"], case["k"], case["n"], case["op"], case["w_bits"]
    s = dict(case)
    s["x"] = _values((m, k), case["x_bits"], gen)
    s["w"] = _values((k, n), wb, gen)
    s["b"] = _values((n,), 31, gen) if case["bias"] else None
    if op != "linear":
        s["w_up"] = _values((k, n), wb, gen)
        s["b_up"] = _values((n,), 31, gen) if case["bias"] else None
    if op == "ffn":
        s["w_down"] = _values((n, k), wb, gen)
        s["b_down"] = _values((k,), 31, gen) if case["bias"] else None
    # the residual stream: as wide as the output of the linear product
    s["r"] = _values((m, k if op == "ffn" else n), 31, gen) if case["residual"] else None
    if own:
        Z = _framework()
        if op == "linear":
            s["linear"] = Z.LinearM31(s["w"], bias=s["b"])
        else:
            s["gated"] = Z.GatedLinearM31(s["w"], s["w_up"], bias_gate=s["b"], bias_up=s["b_up"])
        if op == "ffn":
            s["down"] = Z.LinearM31(s["w_down"], bias=s["b_down"])
    return s


def _framework():
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parents[1] / "stwo-ml_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import zkml_b200

    return zkml_b200


# ---- the plain form ---------------------------------------------------------------------------------


def _signed(v):
    v = v.to(torch.float64)
    return torch.where(v > HALF, v - P, v)


def _mod(v):
    """A whole float64 (below 2^53 in magnitude) as an int64 in [0, P)."""
    return torch.remainder(v, P).to(torch.int64)


def _product(x, x_bits, w, w_bits):
    """x W mod P by float64 products whose sums stay below 2^53, so that each is exact."""
    xs, ws = _signed(x), _signed(w)
    if x_bits + w_bits - 2 + x.shape[1].bit_length() <= 53:
        return _mod(xs @ ws)
    x1, w1 = torch.floor(xs / 65536), torch.floor(ws / 65536)
    x0, w0 = xs - 65536 * x1, ws - 65536 * w1
    high, mid, low = _mod(x1 @ w1), _mod(x1 @ w0 + x0 @ w1), _mod(x0 @ w0)
    return (2 * high + 65536 * mid + low) % P  # 2^32 = 2 mod P


def _fixed(r):
    """A real value in fixed point with 16 fraction bits, halves away from zero, as a field element."""
    y = torch.abs(r) * 65536.0
    whole = torch.floor(y)
    q = torch.clamp((whole + (y - whole >= 0.5)), max=float(P - 1)).to(torch.int64)
    return torch.where(r >= 0, q, (P - q) % P)


def _activation(z, act):
    """The activation of field elements read in fixed point with 16 fraction bits."""
    negative = z > HALF
    real = _signed(z) / 65536.0
    if act == "relu":
        return torch.where(negative, 0, z)
    if act == "gelu":
        inner = (2.0 / torch.pi) ** 0.5 * (real + 0.044715 * real * real * real)
        return _fixed(0.5 * real * (1.0 + torch.tanh(inner)))
    if act == "sigmoid":
        return torch.where(negative, 0, torch.where(z == 0, 32768, 65536))
    if act == "softmax":
        decay = torch.clamp(((P - 1) - z) // 65536, max=20)
        growth = torch.clamp(z // 65536, max=10)
        down = torch.clamp(65536 >> decay, min=1)
        up = torch.clamp(65536 << growth, max=P - 1)
        return torch.where(negative, down, up)
    if act == "silu":
        return _fixed(real / (1.0 + torch.exp(-real)))
    return z


def _plain_linear(x, x_bits, w, w_bits, b, act, r):
    z = _product(x, x_bits, w, w_bits)
    if b is not None:
        z = (z + b) % P
    y = _activation(z, act)
    if r is not None:
        y = (y + r) % P
    return y.to(torch.int32), z.to(torch.int32)


def _plain_gated(s):
    _, g = _plain_linear(s["x"], s["x_bits"], s["w"], s["w_bits"], s["b"], "none", None)
    _, u = _plain_linear(s["x"], s["x_bits"], s["w_up"], s["w_bits"], s["b_up"], "none", None)
    h = _activation(g.to(torch.int64), s["act"]) * u % P
    return h.to(torch.int32), g, u


def run(s):
    act = None if s["act"] == "none" else s["act"]
    if own and s["op"] == "linear":
        return s["linear"](s["x"], activation=act, residual=s["r"], x_bits=s["x_bits"], keep=s["keep"], check=False)
    if own and s["op"] == "gated":
        return s["gated"](s["x"], activation=act, x_bits=s["x_bits"], keep=s["keep"], check=False)
    if own:
        return _framework().gated_ffn_m31(s["x"], s["gated"], s["down"], activation=act, residual=s["r"],
                                          x_bits=s["x_bits"], check=False)
    if s["op"] == "linear":
        y, z = _plain_linear(s["x"], s["x_bits"], s["w"], s["w_bits"], s["b"], s["act"], s["r"])
        return (y, z) if s["keep"] else y
    h, g, u = _plain_gated(s)
    if s["op"] == "gated":
        return (h, g, u) if s["keep"] else h
    return _plain_linear(h, 31, s["w_down"], s["w_bits"], s["b_down"], "none", s["r"])[0]


# ---- work and the 64-bit definition -----------------------------------------------------------------


def work(case):
    m, k, n = case["m"], case["k"], case["n"]
    wide = 1 if case["w_bits"] == 8 else 4  # bytes a weight cannot do without
    weights = {"linear": 1, "gated": 2, "ffn": 3}[case["op"]]
    words_out = {"linear": m * n * (2 if case["keep"] else 1), "gated": m * n * (3 if case["keep"] else 1),
                 "ffn": m * k}[case["op"]]
    x_bytes = {8: 1, 16: 2, 31: 4}[case["x_bits"]]
    bias = {"linear": n, "gated": 2 * n, "ffn": 2 * n + k}[case["op"]] if case["bias"] else 0
    res = (m * (k if case["op"] == "ffn" else n)) if case["residual"] else 0
    return {"bytes": weights * wide * k * n + x_bytes * m * k + 4 * (words_out + bias + res),
            "flops": 2 * weights * m * k * n}


def _exact_product(x, w):
    """sum_t x[i][t] w[t][j] mod P in 64-bit integers, a few terms t at a time."""
    x, w = x.to(torch.int64), w.to(torch.int64)
    z = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.int64, device=x.device)
    step = max(1, (1 << 27) // max(1, x.shape[0] * w.shape[1]))
    for t in range(0, x.shape[1], step):
        z += ((x[:, t:t + step, None] * w[None, t:t + step, :]) % P).sum(1)
        z %= P
    return z


def _exact_real(v, f):
    """f of the fixed-point field elements v, rounded half away from zero to fixed point."""
    s = torch.where(v * 2 > P, v - P, v).double()
    r = f(s * 2.0 ** -16)
    q = torch.trunc(r.abs() * 2.0 ** 16)
    q = (q + (r.abs() * 2.0 ** 16 - q).ge(0.5).double()).clamp(max=P - 1).long()
    return torch.where(r < 0, -q, q) % P


def _exact_act(v, act):
    below = v * 2 > P
    if act == "relu":
        return v.masked_fill(below, 0)
    if act == "gelu":
        c = (2.0 / 3.14159265358979311599796346854) ** 0.5
        return _exact_real(v, lambda t: 0.5 * t * (1.0 + torch.tanh(c * (t + 0.044715 * t * t * t))))
    if act == "sigmoid":
        return (1 << 16) * (~below).long() - (1 << 15) * (v == 0).long()
    if act == "softmax":
        halvings = ((P - 1 - v) >> 16).clamp(0, 20)
        doublings = (v >> 16).clamp(0, 10)
        one = torch.full_like(v, 1 << 16)
        return torch.where(below, (one >> halvings).clamp(min=1), (one << doublings).clamp(max=P - 1))
    if act == "silu":
        return _exact_real(v, lambda t: t / (1.0 + torch.exp(-t)))
    return v


def exact(case, seed):
    if _cost(case) > 1 << 38:
        return None
    s = prepare(case, seed)

    def affine(x, w, b):
        z = _exact_product(x, w)
        return z if b is None else (z + b.long()) % P

    z = affine(s["x"], s["w"], s["b"])
    y = _exact_act(z, s["act"])
    if s["op"] == "linear":
        y = y if s["r"] is None else (y + s["r"].long()) % P
        return (y.int(), z.int()) if s["keep"] else y.int()
    u = affine(s["x"], s["w_up"], s["b_up"])
    h = y * u % P
    if s["op"] == "gated":
        return (h.int(), z.int(), u.int()) if s["keep"] else h.int()
    y = affine(h, s["w_down"], s["b_down"])
    return (y if s["r"] is None else (y + s["r"].long()) % P).int()
