// Forward operators: y = f(x W + b) + r and h = f(x Wg + bg) * (x Wu + bu), mod P.
#include <cuda_runtime.h>

#include <algorithm>

#include "activation_device.cuh"
#include "linear.cuh"
#include "qm31.cuh"

namespace zk {

namespace {

// Canonical f(v); tag 0 is the identity.
__device__ __forceinline__ uint32_t activate(int tag, uint32_t v) {
    return tag == 0 ? v : red32(act_value(tag, v));
}

__global__ void lay_out_kernel(const uint32_t* __restrict__ src, uint32_t k, uint32_t n, size_t rs, size_t cs,
                               uint32_t* __restrict__ dst, size_t ld, size_t off, uint32_t* __restrict__ status) {
    uint32_t bad = 0;
    const size_t total = (size_t)k * n;
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const size_t r = i / n, c = i % n;
        const uint32_t v = src[r * rs + c * cs];
        bad |= v >> 31;
        dst[r * ld + off + c] = red32(v);
    }
    if (bad) atomicOr(status, LIN_BAD_VALUE);
}

// 64 x 64 outputs per 256-thread block, 4 x 4 per thread, K in steps of 16 through shared memory;
// 64-bit sums reduced every four products (4 P^2 + 2^34 < 2^64).  G = 2: both projections of the
// gated block in one pass over x.
template <int G>
__global__ void __launch_bounds__(256) linear_simple_kernel(LinearArgs a) {
    __shared__ uint32_t As[16][65];
    __shared__ uint32_t Bs[G][16][64];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint32_t row0 = blockIdx.y * 64, col0 = blockIdx.x * 64;
    const size_t ldw = (size_t)G * a.n;
    unsigned long long acc[G][4][4] = {};
    uint32_t bad = 0;
    const uint32_t half = a.x_bits == 31 ? 0x40000000u : 1u << (a.x_bits - 1);
    for (uint32_t l0 = 0; l0 < a.k; l0 += 16) {
        for (int e = threadIdx.x; e < 16 * 64; e += 256) {
            const int rr = e / 16, ll = e % 16;
            const uint32_t gi = row0 + rr, gl = l0 + ll;
            uint32_t v = 0;
            if (gi < a.m && gl < a.k) {
                v = a.x[(size_t)gi * a.ldx + gl];
                bad |= (v >> 31) ? LIN_BAD_VALUE : 0u;
                v = red32(v);
                // signed value in [-half, half)
                if (a.x_bits != 31 && !(v < half || v >= P - half)) bad |= LIN_BAD_RANGE;
            }
            As[ll][rr] = v;
            const int bl = e / 64, bc = e % 64;
            const uint32_t gbl = l0 + bl, gbc = col0 + bc;
#pragma unroll
            for (int g = 0; g < G; g++)
                Bs[g][bl][bc] = (gbl < a.k && gbc < a.n) ? a.w[gbl * ldw + (size_t)g * a.n + gbc] : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int ll = 0; ll < 16; ll++) {
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[g][i][j] += (unsigned long long)As[ll][ty * 4 + i] * Bs[g][ll][tx * 4 + j];
            if ((ll & 3) == 3) {
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[g][i][j] = (acc[g][i][j] & P) + (acc[g][i][j] >> 31);
            }
        }
        __syncthreads();
    }
    if (bad) atomicOr(a.status, bad);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t r = row0 + ty * 4 + i, c = col0 + tx * 4 + j;
            if (r >= a.m || c >= a.n) continue;
            uint32_t z[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                z[g] = red64(acc[g][i][j]);
                if (a.bias) z[g] = madd(z[g], a.bias[(size_t)g * a.n + c]);
            }
            if (a.pre) a.pre[(size_t)r * a.ld_pre + c] = z[0];
            uint32_t y = activate(a.activation, z[0]);
            if (G == 2) {
                if (a.up) a.up[(size_t)r * a.ld_up + c] = z[G - 1];
                y = mmul(y, z[G - 1]);
            } else if (a.residual) {
                const uint32_t v = a.residual[(size_t)r * a.ld_res + c];
                if (v >> 31) atomicOr(a.status, LIN_BAD_VALUE);
                y = madd(y, red32(v));
            }
            a.out[(size_t)r * a.ld_out + c] = y;
        }
}

}  // namespace

void launch_linear_lay_out(const uint32_t* src, uint32_t k, uint32_t n, size_t rs, size_t cs, uint32_t* dst,
                           size_t ld, size_t off, uint32_t* status, cudaStream_t s) {
    const size_t total = (size_t)k * n;
    const unsigned g = (unsigned)std::min<size_t>((total + 255) / 256, 8192);
    lay_out_kernel<<<g, 256, 0, s>>>(src, k, n, rs, cs, dst, ld, off, status);
}

void launch_linear_simple(const LinearArgs& a, cudaStream_t s) {
    const dim3 grid((a.n + 63) / 64, (a.m + 63) / 64);
    if (a.gated)
        linear_simple_kernel<2><<<grid, 256, 0, s>>>(a);
    else
        linear_simple_kernel<1><<<grid, 256, 0, s>>>(a);
}

}  // namespace zk
