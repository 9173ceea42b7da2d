// ActivationType::as_fn (gadgets/lookup_table.rs:193-345) applied to full M31 values, as the
// reference's forward pass does (compiler/prove.rs:1893-1899): fixed point with scale 2^16,
// values above (P - 1) / 2 read as negative; GELU (tanh form) and SiLU in binary64, rounded
// half away from zero and clamped to [0, P - 1] / [-(P - 1), 0]; Sigmoid a step; Softmax-exp a
// shift.  The binary64 evaluation uses the device exp / tanh; they round to nearest within an
// ulp of the host libm's, which decides a result only when x * 2^16 lands within ~1e-9 of a
// half-integer.
#pragma once
#include "qm31.cuh"

namespace zk {

__device__ __forceinline__ double act_real(uint32_t v) {
    return v <= 0x3FFFFFFFu ? (double)v / 65536.0 : -((double)((uint64_t)P - v)) / 65536.0;
}
__device__ __forceinline__ uint32_t act_from_real(double r) {
    const uint64_t pm1 = (uint64_t)P - 1;
    if (r >= 0.0) {
        const uint64_t u = (uint64_t)round(r * 65536.0);
        return (uint32_t)(u < pm1 ? u : pm1);
    }
    uint64_t neg = (uint64_t)round(-r * 65536.0);
    if (neg > pm1) neg = pm1;
    return (uint32_t)((uint64_t)P - neg);
}
// v canonical.  A negative real that rounds to zero comes out as P, as in the reference.
static __device__ __noinline__ uint32_t act_value(int tag, uint32_t v) {
    switch (tag) {
        case 1:  // ReLU
            return v <= (P - 1) / 2 ? v : 0u;
        case 2: {  // GELU
            if (v == 0) return 0;
            const double x = act_real(v);
            const double c = sqrt(2.0 / 3.14159265358979311599796346854);
            const double inner = __dmul_rn(c, __dadd_rn(x, __dmul_rn(__dmul_rn(__dmul_rn(0.044715, x), x), x)));
            return act_from_real(__dmul_rn(__dmul_rn(0.5, x), __dadd_rn(1.0, tanh(inner))));
        }
        case 3:  // Sigmoid step
            if (v > 0x3FFFFFFFu) return 0;
            return v == 0 ? 32768u : 65536u;
        case 4: {  // Softmax exp
            if (v > 0x3FFFFFFFu) {
                uint32_t decay = (((1u << 31) - 2) - v) / 65536u;
                if (decay > 20) decay = 20;
                const uint32_t r = 65536u >> decay;
                return r > 1 ? r : 1;
            }
            if (v == 0) return 65536u;
            uint32_t growth = v / 65536u;
            if (growth > 10) growth = 10;
            const uint64_t r = (uint64_t)65536u << growth, cap = (1ull << 31) - 2;
            return (uint32_t)(r < cap ? r : cap);
        }
        default: {  // SiLU
            if (v == 0) return 0;
            const double x = act_real(v);
            return act_from_real(__ddiv_rn(x, __dadd_rn(1.0, exp(-x))));
        }
    }
}

}  // namespace zk
