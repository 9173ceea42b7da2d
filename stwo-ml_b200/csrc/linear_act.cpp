// Segment tables of SiLU and GELU for the forward kernels (linear.cuh): per segment the cubic through
// the function at the four Chebyshev nodes around its middle, in extended precision.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <vector>

#include "linear.cuh"

namespace zk {

namespace {

typedef long double real;

// x - f(x) for x >= 0.
real silu_delta(real x) { return x / (1.0L + expl(x)); }
real gelu_delta(real x) {  // tanh form
    const real c = sqrtl(2.0L / 3.14159265358979323846264338327950288L);
    return 0.5L * x * (1.0L - tanhl(c * (x + 0.044715L * x * x * x)));
}

std::vector<uint8_t> build(real (*delta)(real), int tag) {
    std::vector<uint8_t> t(act_table_bytes(tag));
    const real half = ldexpl(1.0L, (int)act_segment_bits(tag) - 1);
    real node[4];
    for (int i = 0; i < 4; i++) node[i] = cosl(3.14159265358979323846264338327950288L * (2 * i + 1) / 8);
    for (size_t s = 0; s < t.size() / 16; s++) {
        // Newton's divided differences over the nodes, then the monomial coefficients
        real v[4], c[4] = {0, 0, 0, 0};
        for (int i = 0; i < 4; i++) v[i] = 65536 * delta(((2 * (real)s + 1) * half + half * node[i]) / 65536);
        for (int j = 1; j < 4; j++)
            for (int i = 3; i >= j; i--) v[i] = (v[i] - v[i - 1]) / (node[i] - node[i - j]);
        for (int i = 3; i >= 0; i--) {
            for (int j = 3; j > 0; j--) c[j] = c[j - 1] - node[i] * c[j];
            c[0] = v[i] - node[i] * c[0];
        }
        real scale = 1;
        for (int j = 0; j < 4; j++, scale *= half) c[j] /= scale;
        const uint32_t c0 = (uint32_t)llroundl(ldexpl(fmaxl(c[0], 0), 17));  // delta 2^16 < 18250
        const int32_t c1 = (int32_t)llroundl(ldexpl(c[1], 30));              // slopes within 1/2
        const float c2 = (float)ldexpl(c[2], 20), c3 = (float)ldexpl(c[3], 20);
        memcpy(&t[16 * s], &c0, 4);
        memcpy(&t[16 * s + 4], &c1, 4);
        memcpy(&t[16 * s + 8], &c2, 4);
        memcpy(&t[16 * s + 12], &c3, 4);
    }
    return t;
}

}  // namespace

const uint8_t* act_segment_table(int tag) {
    static std::once_flag once;
    static std::vector<uint8_t> gelu, silu;
    std::call_once(once, [] {
        gelu = build(gelu_delta, 2);
        silu = build(silu_delta, 5);
    });
    return (tag == 5 ? silu : gelu).data();
}

}  // namespace zk
