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

// Activations are read by these: cached in L1 (neighbouring lanes and loads share sectors), but not as
// data that stays constant while the kernel runs, since a programmatic dependent starts before the
// work that writes them is done.
__device__ __forceinline__ uint32_t load_word(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint4 load_words(const uint32_t* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

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

// SiLU or GELU of M31 words, canonical, with mag = |v|.  Both functions fall short
// of max(x, 0) by the same amount on either side of zero: f(x) = x - delta(x) and f(-x) = -delta(x) for
// x > 0.  delta 2^16 comes from a table of segments, c0 + c1 d + c2 d^2 + c3 d^3 with d the offset from
// the segment's middle: c0 and c1 d are added as integers in 2^-30 units, the rest, below 4, in single
// precision.  Over every word below the limit that is off by at most 2^-16.1 (checked against
// extended precision); where it lies within 2^-14 of a half-integer, 174 words in all, the
// defining binary64 form decides the rounding.  One 16-byte read and about 25 instructions of full
// rate a value (512 int8 tokens x 5120 x 13824, whose inputs all bend: 65 us a call, 46 us with ReLU;
// 110 us with a double-precision exponential).
// Several values a call, so that their reads and sums overlap; from act_limit on, delta 2^16 is below
// 0.12 and f rounds to max(x, 0).  Out of line: copies at every call site made the kernels miss the
// instruction cache.
template <int N>
struct Words {
    uint32_t v[N];
};
template <int N>
static __device__ __noinline__ Words<N> bent_activation(const uint8_t* table, int tag, Words<N> x) {
    const uint32_t bits = act_segment_bits(tag), half = 1u << (bits - 1), limit = act_limit(tag);
    uint32_t mag[N], n[N];
    uint4 s[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        mag[i] = min(x.v[i], P - x.v[i]);
        s[i] = reinterpret_cast<const uint4*>(table)[min(mag[i], limit - 1) >> bits];
    }
    bool unsure = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int d = (int)(mag[i] & (2 * half - 1)) - (int)half;
        const float e = (float)d, g = fmaf(__uint_as_float(s[i].w), e, __uint_as_float(s[i].z)) * (e * e);
        const int64_t t =
            (int64_t)((uint64_t)s[i].x << 13) + (int64_t)(int)s[i].y * d + ((int64_t)__float2int_rn(g) << 10);
        const int off = (int)((uint32_t)t & 0x3fffffffu) - 0x20000000;
        n[i] = mag[i] < limit ? (uint32_t)((t + 0x20000000) >> 30) : 0u;
        unsure |= abs(off) < 65536 && mag[i] < limit;
    }
    Words<N> y;
#pragma unroll
    for (int i = 0; i < N; i++) {  // delta: off a positive value, and what a negative one comes to below zero
        const uint32_t r = (x.v[i] > (P - 1) / 2 ? 0u : x.v[i]) + P - n[i];
        y.v[i] = r >= P ? r - P : r;
    }
    if (unsure) {
#pragma unroll
        for (int i = 0; i < N; i++) y.v[i] = red32(act_value(tag, x.v[i]));
    }
    return y;
}

// Tokens handled together: their digits are 16 accumulator columns.
template <int D>
constexpr int GROUP = 16 / D;

// x + y mod P for x <= P, y < P.
__device__ __forceinline__ uint32_t add_mod(uint32_t x, uint32_t y) { return min(x + y, x + y - P); }

// sum_i 256^i acc_i mod P of one token's accumulators.
template <int D>
__device__ __forceinline__ uint32_t join_digits(const uint32_t (&r)[16], int t) {
    if (D == 1) {
        const int v = (int)r[t];  // |v| <= 1023 * 2^21 < P
        return (uint32_t)(v + ((v >> 31) & 0x7fffffff));
    }
    int64_t s = 0;
#pragma unroll
    for (int i = D - 1; i >= 0; i--) s = s * 256 + (int)r[i * GROUP<D> + t];
    return canon64((uint64_t)s + ((uint64_t)P << 26));  // |s| < 2^56
}

__host__ __device__ inline bool io_bends(const LinearIO& io) {
    return (io.activation == 2 || io.activation == 5) && !io.as_reference;
}

// y = f(y): canonical, or as the reference's forward pass leaves it (LinearIO::as_reference).
template <int N>  // 1 or a multiple of 4
__device__ __forceinline__ void activate(const LinearIO& io, const uint8_t* table, uint32_t (&y)[N]) {
    constexpr int CHUNK = N < 4 ? N : 4;
    if (io.activation == 0) return;
    if (io.activation == 1) {
#pragma unroll
        for (int t = 0; t < N; t++) y[t] = y[t] > (P - 1) / 2 ? 0u : y[t];
    } else if (io_bends(io)) {
#pragma unroll
        for (int t = 0; t < N; t += CHUNK) {
            uint32_t least = P;
#pragma unroll
            for (int i = 0; i < CHUNK; i++) least = min(least, min(y[t + i], P - y[t + i]));
            if (least < act_limit(io.activation)) {
                Words<CHUNK> q;
#pragma unroll
                for (int i = 0; i < CHUNK; i++) q.v[i] = y[t + i];
                q = bent_activation(table, io.activation, q);
#pragma unroll
                for (int i = 0; i < CHUNK; i++) y[t + i] = q.v[i];
            } else {
#pragma unroll
                for (int i = 0; i < CHUNK; i++) y[t + i] = y[t + i] > (P - 1) / 2 ? 0u : y[t + i];
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < N; t++) {
            const uint32_t v = act_value(io.activation, y[t]);
            y[t] = io.as_reference ? v : red32(v);
        }
    }
}

// Finishes GROUP tokens of this lane's row: z (without the bias) -> outputs.
template <int D, bool GATED>
__device__ __forceinline__ void finish_tokens(const LinearIO& io, const uint8_t* table, uint32_t n, uint32_t nt,
                                              uint32_t row, uint32_t tok0, uint32_t base, uint32_t (&z)[GROUP<D>]) {
    constexpr int G = GROUP<D>;
#pragma unroll
    for (int t = 0; t < G; t++) z[t] = add_mod(z[t], base);
    if (GATED) {
        // lane l < 16: gate, lane l + 16: up of the same output; of each token pair one lane
        // finishes the first token and the other the second
        const bool up_lane = (row & 16) != 0;
        const uint32_t f = nt * 64 + (row >> 5) * 16 + (row & 15);
        // pairs by four where a group has as many, so that their activations overlap
        constexpr int PAIRS = G >= 8 ? 4 : 1;
#pragma unroll
        for (int t = 0; t < G; t += 2 * PAIRS) {
            uint32_t y[PAIRS], u[PAIRS];
#pragma unroll
            for (int i = 0; i < PAIRS; i++) {
                const uint32_t a = z[t + 2 * i], b = z[t + 2 * i + 1];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up_lane ? a : b, 16);
                y[i] = up_lane ? got : a;
                u[i] = up_lane ? b : got;
            }
            const uint32_t tok = tok0 + t + (up_lane ? 1 : 0);
            if (f < n && tok < io.m) {
                if (io.pre) {
#pragma unroll
                    for (int i = 0; i < PAIRS; i++)
                        if (tok + 2 * i < io.m) io.pre[(size_t)(tok + 2 * i) * io.ld_pre + f] = y[i];
                }
                if (io.up) {
#pragma unroll
                    for (int i = 0; i < PAIRS; i++)
                        if (tok + 2 * i < io.m) io.up[(size_t)(tok + 2 * i) * io.ld_up + f] = u[i];
                }
                activate(io, table, y);
#pragma unroll
                for (int i = 0; i < PAIRS; i++)
                    if (tok + 2 * i < io.m) io.out[(size_t)(tok + 2 * i) * io.ld_out + f] = mmul(y[i], u[i]);
            }
        }
    } else {
        const uint32_t f = nt * LIN_ROWS + row;
        if (f >= n) return;
        if (io.pre) {
            uint32_t* pre = io.pre + (size_t)tok0 * io.ld_pre + f;
#pragma unroll
            for (int t = 0; t < G; t++, pre += io.ld_pre)
                if (tok0 + t < io.m) *pre = z[t];
        }
        activate(io, table, z);
        if (io.residual) {
            uint32_t res[G], bad = 0;
            const uint32_t* r = io.residual + (size_t)tok0 * io.ld_res + f;
#pragma unroll
            for (int t = 0; t < G; t++, r += io.ld_res) res[t] = tok0 + t < io.m ? __ldcg(r) : 0u;
#pragma unroll
            for (int t = 0; t < G; t++) {
                bad |= res[t] >> 31;
                z[t] = add_mod(z[t], red32(res[t]));
            }
            if (bad) atomicOr(io.status, LIN_BAD_VALUE);
        }
        uint32_t* out = io.out + (size_t)tok0 * io.ld_out + f;
#pragma unroll
        for (int t = 0; t < G; t++, out += io.ld_out)
            if (tok0 + t < io.m) *out = z[t];
    }
}

// What a block whose waits ran out does before it gives up its tensor memory and ends: it says so, and lets
// the copies (the last `issued` of a ring of stages, and the one behind bar2 if that is not 0) and products
// in flight end.  Out of line: no ordinary block comes here.
static __device__ __noinline__ void report_timeout(uint32_t* status, uint32_t full, uint32_t stages, uint32_t issued,
                                                   uint32_t bar2, uint64_t wait_ns) {
    volatile uint32_t never = 0;
    atomicOr(status, LIN_TIMEOUT);
    for (uint32_t i = 0; i < min(issued, stages); i++) {  // a barrier may also lack an arrival: then the limit ends it
        const uint32_t u = issued - 1 - i;
        mbar_wait(full + 8 * (u % stages), (u / stages) & 1, &never, wait_ns);
    }
    if (bar2) mbar_wait(bar2, 0, &never, wait_ns);
}
static __device__ __noinline__ void drain_products(uint32_t drained, uint64_t wait_ns) {
    volatile uint32_t never = 0;
    tc_commit(drained);
    mbar_wait(drained, 0, &never, wait_ns);
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
