// Device code and launch helper shared by the forward kernels (linear_kernels.cu, linear_token.cu).
#pragma once
#include <cuda_runtime.h>

#include "activation_device.cuh"
#include "imma.cuh"
#include "linear.cuh"
#include "round_arith.cuh"
#include "tcgen05.cuh"

namespace zk {

constexpr uint32_t KSEG = 1023;  // K tiles per 32-bit accumulation: 1023 * 128 * 2^14 < 2^31

// The four balanced byte digits of v (|v| < 2^31 - 2^23), byte i holding the digit of 256^i in
// [-128, 127]: adding 128 to every digit makes them the plain base-256 digits of v + 0x80808080.
__device__ __forceinline__ uint32_t balanced_digits(int v) { return ((uint32_t)v + 0x80808080u) ^ 0x80808080u; }

// The words of four activations -> D words, word b holding the four digits of 256^b (D as in
// linear_kernels.cu); sets the status bits that apply.
template <int D>
__device__ __forceinline__ void activation_digits(const uint4& x, uint32_t (&d)[D], uint32_t& bad) {
    constexpr int OFFSET = D > 1 ? 128 : 0;
    const int v[4] = {m31_signed(x.x) - OFFSET, m31_signed(x.y) - OFFSET, m31_signed(x.z) - OFFSET,
                      m31_signed(x.w) - OFFSET};
    if ((x.x | x.y | x.z | x.w) >> 31) bad |= LIN_BAD_VALUE;
    if (D < 4) {
        constexpr uint32_t LOW = D == 1 ? 128u : 32896u, SPAN = D == 1 ? 256u : 65536u;  // D digits: [-LOW, SPAN - LOW)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if ((uint32_t)v[i] + LOW >= SPAN) bad |= LIN_BAD_RANGE;
    }
    uint32_t p[4];
    byte_planes(make_uint4(balanced_digits(v[0]), balanced_digits(v[1]), balanced_digits(v[2]), balanced_digits(v[3])),
                p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int b = 0; b < D; b++) d[b] = p[b];
}

// SiLU or GELU of the M31 word v with |real| below the saturation bound, canonical.
// Both are mag * w / (1 + e) in units of 2^-16, with mag = |v|, w = 1 for positive and e for
// negative v, and e = exp(-a), a = |x| for SiLU and 2 |u| for GELU's inner term u
// (1 + tanh u = 2 / (1 + exp(-2u))).  e = 2^-k exp(r), |r| <= ln(2) / 2, by the Taylor polynomial
// of degree 9 (remainder below 2^-37), 1 / (1 + e) by one Newton step from a single-precision
// estimate (below 2^-43): the result, below 2^21.3, is off by less than 2^-15.  Where it lies
// within 2^-12 of a half-integer the defining binary64 form decides the rounding.  About 25
// double-precision operations instead of the 150 and more of exp, tanh and a division.
// Out of line: copies at every call site made the kernels miss the instruction cache.
static __device__ __noinline__ uint32_t bent_activation(int tag, uint32_t v, uint32_t mag, bool neg) {
    const double x = (double)mag * (1.0 / 65536.0);
    double a = x;
    if (tag == 2) a = 2.0 * 0.79788456080286535588 * fma(0.044715 * x * x, x, x);  // 2 sqrt(2 / pi) (x + 0.044715 x^3)
    const int k = __double2int_rn(a * 1.44269504088896340736);  // a / ln 2
    const double r = fma((double)k, 0.69314718055994530942, -a);
    double e = 1.0 / 362880.0;
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    e *= __hiloint2double((1023 - k) << 20, 0);  // k < 90
    const double d = 1.0 + e;
    const double q0 = (double)__fdividef(1.0f, (float)d);
    const double q = q0 * fma(-d, q0, 2.0);
    const double y = (double)mag * (neg ? e * q : q);
    const double whole = floor(y), rest = y - whole;
    if (fabs(rest - 0.5) < 1.0 / 4096.0) return red32(act_value(tag, v));
    const uint32_t n = (uint32_t)whole + (rest >= 0.5 ? 1u : 0u);
    return neg && n ? P - n : n;
}

// f(v), canonical.  Where SiLU and GELU equal their argument or round to zero in binary64 the
// result is taken without evaluating them: for real x >= 37, exp(-x) < 2^-53 and 1 + exp(-x) is
// 1; for x <= -16, |x| exp(x) 2^16 < 1/2; for |x| >= 8.5, |tanh| of GELU's inner term (above 28)
// is 1.
__device__ __forceinline__ uint32_t activate(int tag, uint32_t v) {
    if (tag == 0) return v;
    if (tag == 1) return v <= (P - 1) / 2 ? v : 0u;
    if (tag == 5 || tag == 2) {
        const bool neg = v > (P - 1) / 2;
        const uint32_t mag = neg ? P - v : v;
        const uint32_t sat = tag == 2 ? (17u << 15) : neg ? (16u << 16) : (37u << 16);
        if (mag >= sat) return neg ? 0u : v;
        return bent_activation(tag, v, mag, neg);
    }
    return red32(act_value(tag, v));
}

// Tokens handled together: their digits are 16 accumulator columns.
template <int D>
constexpr int GROUP = 16 / D;

// sum_i 256^i acc_i mod P of one token's accumulators.
template <int D>
__device__ __forceinline__ uint32_t join_digits(const uint32_t (&r)[16], int t) {
    if (D == 1) {
        const int v = (int)r[t];
        return red32(v < 0 ? (uint32_t)(v + 0x7fffffff) : (uint32_t)v);
    }
    int64_t s = 0;
#pragma unroll
    for (int i = D - 1; i >= 0; i--) s = s * 256 + (int)r[i * GROUP<D> + t];
    return canon64((uint64_t)s + ((uint64_t)P << 26));  // |s| < 2^56
}

// f(v) as an output word: canonical, or as the reference's forward pass leaves it (LinearIO::as_reference).
__device__ __forceinline__ uint32_t activated(const LinearIO& io, uint32_t v) {
    if (io.as_reference && io.activation) return act_value(io.activation, v);
    return activate(io.activation, v);
}

// Finishes GROUP tokens of this lane's row: z (without the bias) -> outputs.
template <int D, bool GATED>
__device__ __forceinline__ void finish_tokens(const LinearIO& io, uint32_t n, uint32_t nt, uint32_t row, uint32_t tok0,
                                              uint32_t base, uint32_t (&z)[GROUP<D>]) {
    constexpr int G = GROUP<D>;
#pragma unroll
    for (int t = 0; t < G; t++) z[t] = madd(z[t], base);
    if (GATED) {
        // lane l < 16: gate, lane l + 16: up of the same output; of each token pair one lane
        // finishes the first token and the other the second
        const bool up_lane = (row & 16) != 0;
        const uint32_t f = nt * 64 + (row >> 5) * 16 + (row & 15);
#pragma unroll
        for (int t = 0; t < G; t += 2) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up_lane ? z[t] : z[t + 1], 16);
            const uint32_t g = up_lane ? got : z[t], u = up_lane ? z[t + 1] : got;
            const uint32_t tok = tok0 + t + (up_lane ? 1 : 0);
            if (f < n && tok < io.m) {
                if (io.pre) io.pre[(size_t)tok * io.ld_pre + f] = g;
                if (io.up) io.up[(size_t)tok * io.ld_up + f] = u;
                io.out[(size_t)tok * io.ld_out + f] = mmul(activated(io, g), u);
            }
        }
    } else {
        const uint32_t f = nt * LIN_ROWS + row;
        if (f >= n) return;
        uint32_t res[G], bad = 0;
#pragma unroll
        for (int t = 0; t < G; t++)
            res[t] = io.residual && tok0 + t < io.m ? __ldcg(io.residual + (size_t)(tok0 + t) * io.ld_res + f) : 0u;
#pragma unroll
        for (int t = 0; t < G; t++) {
            if (tok0 + t >= io.m) continue;
            if (io.pre) io.pre[(size_t)(tok0 + t) * io.ld_pre + f] = z[t];
            bad |= res[t] >> 31;
            const uint32_t y = activated(io, z[t]);
            io.out[(size_t)(tok0 + t) * io.ld_out + f] = io.residual ? madd(y, red32(res[t])) : y;
        }
        if (bad) atomicOr(io.status, LIN_BAD_VALUE);
    }
}

// Both kernels of a call are programmatic dependents: a block of the product kernel starts, and
// loads weights, as soon as an SM is free, before the digits are made and before the last blocks
// of the previous call are done; what depends on earlier work comes after grid_dependency_wait.
struct Launch {
    cudaLaunchAttribute attr{};
    cudaLaunchConfig_t cfg{};
    Launch(dim3 grid, unsigned block, size_t smem, cudaStream_t s, bool overlap) {
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid;
        cfg.blockDim = dim3(block);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        cfg.attrs = &attr;
        cfg.numAttrs = overlap ? 1 : 0;
    }
};

}  // namespace zk
