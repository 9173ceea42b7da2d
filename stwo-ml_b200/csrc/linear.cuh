// Forward operators with weights laid out once: internal interface of linear_kernels.cu.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace zk {

// Bits of a handle's status word.
constexpr uint32_t LIN_BAD_VALUE = 1u;   // an input word >= 2^31
constexpr uint32_t LIN_BAD_RANGE = 2u;   // an activation that does not fit the declared width

// What one launch reads and writes.  Strides are in words; a row of x / residual may repeat
// (stride 0).  n is the output width (per projection for gated weights).
struct LinearArgs {
    const uint32_t* x;
    const uint32_t* w;        // k x n, row major (gated: k x 2n, gate then up in each row)
    const uint32_t* bias;     // n words (gated: 2n) or NULL
    const uint32_t* residual;
    uint32_t *out, *pre, *up;
    uint32_t* status;
    size_t ldx, ld_res, ld_out, ld_pre, ld_up;
    uint32_t m, k, n;
    int x_bits, activation;
    bool gated;
};

void launch_linear_simple(const LinearArgs& a, cudaStream_t s);
// dst[i][off + j] = src[i * rs + j * cs] mod P, row pitch ld; sets LIN_BAD_VALUE in *status.
void launch_linear_lay_out(const uint32_t* src, uint32_t k, uint32_t n, size_t rs, size_t cs, uint32_t* dst,
                           size_t ld, size_t off, uint32_t* status, cudaStream_t s);

}  // namespace zk
