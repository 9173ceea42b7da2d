// Forward operators with weights laid out once: interface of linear_kernels.cu.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct zkml_ctx;

namespace zk {

// Bits of a handle's status word.
constexpr uint32_t LIN_BAD_VALUE = 1u;  // an input word >= 2^31
constexpr uint32_t LIN_BAD_RANGE = 2u;  // an activation that does not fit the declared width
constexpr uint32_t LIN_TIMEOUT = 4u;    // a bounded wait ran out

// Tiles: 128 rows (outputs) x 128 bytes (K) of weights.
constexpr uint32_t LIN_ROWS = 128;
constexpr uint32_t LIN_KB = 128;
constexpr uint32_t LIN_TILE_BYTES = LIN_ROWS * LIN_KB;

// Weights in the kernels' layout: per plane, row tile and K tile 16 KiB, row r of a tile at
// 128 r with its 16-byte chunk c at c ^ (r & 7) (the 128-byte swizzle).  Plane p holds the signed
// byte digit of 256^p.  Row r of tile t is output 128 t + r, or for gated weights, in every 32
// rows, 16 gate rows and then the 16 up rows of the same outputs (64 outputs a tile), so both
// projections of an output meet in one warp's lanes l and l + 16.
struct PackedWeights {
    const uint8_t* tiles = nullptr;
    const uint32_t* base = nullptr;  // 2 x row slots: bias, and bias + 128 (column sum of the weights), mod P
    uint32_t k = 0, n = 0, k_tiles = 0, n_tiles = 0, planes = 0;
    bool gated = false;
};
inline uint32_t lin_outputs_per_tile(bool gated) { return gated ? LIN_ROWS / 2 : LIN_ROWS; }

// Packs w (and w2 for gated weights); columns' sums are added into sums (one u64 per row slot,
// zeroed by the caller).  status[0] collects LIN_BAD_VALUE, status[1] the planes the values need.
void launch_linear_pack(const uint32_t* w, const uint32_t* w2, size_t rs, size_t cs, const PackedWeights& p,
                        uint8_t* tiles, unsigned long long* sums, uint32_t* status, cudaStream_t s);
// base[] from the sums and the bias (NULL: zero).
void launch_linear_base(const unsigned long long* sums, const uint32_t* bias, const uint32_t* bias2,
                        const PackedWeights& p, uint32_t* base, uint32_t* status, cudaStream_t s);

#ifdef __CUDACC__
#define LIN_HD __host__ __device__
#else
#define LIN_HD
#endif
// Segment tables of SiLU and GELU (linear_act.cpp): by how much f falls short of max(x, 0) for the words
// below act_limit (real x = 16 and 5), in segments of 2^act_segment_bits words, a record of 16 bytes
// {c0, c1, c2, c3} each.
LIN_HD constexpr uint32_t act_limit(int tag) { return tag == 2 ? 5u << 16 : 16u << 16; }
LIN_HD constexpr uint32_t act_segment_bits(int tag) { return tag == 2 ? 10 : 11; }
LIN_HD constexpr uint32_t act_table_bytes(int tag) { return 16 * (act_limit(tag) >> act_segment_bits(tag)); }
constexpr uint32_t ACT_TABLE_MAX = 8192;
static_assert(act_table_bytes(2) <= ACT_TABLE_MAX && act_table_bytes(5) <= ACT_TABLE_MAX, "reserved in the kernels");
const uint8_t* act_segment_table(int tag);  // host; tag 2 or 5

// One call.  Strides are in words.
struct LinearIO {
    const uint32_t* x;
    const uint32_t* residual;
    uint32_t *out, *pre, *up;
    uint32_t* status;
    size_t ldx, ld_res, ld_out, ld_pre, ld_up;
    uint32_t m;
    int activation;
    const uint8_t* act_table = nullptr;  // SiLU, GELU: the segment table in device memory
    bool as_reference = false;  // an activation that rounds a negative value to zero gives the word P, not 0
    // The self-test's alone: LIN_WITHHOLD_*, what block 0 of linear_kernel, or the last block of cluster 0 of
    // linear_token_kernel, leaves undone so that a wait runs out, and the waits' limit.
    int withhold = 0;
    uint64_t wait_ns = 0;
};
constexpr int LIN_WITHHOLD_DONE = 1;    // the commit of its (first) accumulators: the finishing warps wait
constexpr int LIN_WITHHOLD_COPY = 2;    // the copies from a weight tile on: the products' issuer waits
constexpr int LIN_WITHHOLD_TABLE = 3;   // linear_kernel: the activation table's copy
constexpr int LIN_WITHHOLD_DIGITS = 4;  // linear_token_kernel: the arrival of its last digit tile

// How a call is split: fixed by the sizes alone.
struct LinearPlan {
    uint32_t digits;    // byte digits per activation: 1, 2 or 4
    uint32_t tokens;    // tokens per tile
    uint32_t m_tiles;
    uint32_t tiles;     // m_tiles x n_tiles
    uint32_t sk_tiles;  // the first tiles are cut at even shares of their units, the others are whole
    uint32_t ctas;
    uint32_t stages;
    uint32_t slots;     // partial-sum slots per block
    size_t digits_off, slots_off, bytes;  // workspace: counters, digit tiles, slots
};
LinearPlan linear_plan(const PackedWeights& w, uint32_t m, int x_bits, int num_sms);
// The few-token kernel's split, when it takes the call: one launch, no workspace.
struct TokenPlan {
    uint32_t digits, tokens;
    uint32_t parts;   // blocks of a cluster, each with a share of K
    uint32_t stages;
    uint32_t smem;
};
bool linear_token_plan(const PackedWeights& w, uint32_t m, int x_bits, int num_sms, TokenPlan* out);
cudaError_t launch_linear_token(const PackedWeights& w, const TokenPlan& p, const LinearIO& io, cudaStream_t s,
                                bool overlap);
cudaError_t linear_token_configure();
cudaError_t linear_configure(cudaStream_t s);  // per device, before the first launch; uploads tables on s
// The current device's copy of the segment table, NULL for other activations.
cudaError_t linear_act_table(int tag, const uint8_t** out);
// overlap: the weights were in place before the work now queued on s, so they may be read while
// that work still runs.
cudaError_t launch_linear(const PackedWeights& w, const LinearPlan& p, const LinearIO& io, void* workspace,
                          cudaStream_t s, bool overlap);

// One product with weights that are used once (the chain prover's forward pass): lays w (k x n,
// row major, host or device memory) out in the context's scratch and runs the call on its stream.
// x, residual, pre and out are dense device matrices; pre may be NULL.  ZKML_ERR_OOM leaves
// nothing done and no scratch held.  A run of calls is opened by _begin and closed by _end, which waits
// for the stream and reports what the calls met.  The weights' layout is in op.bmle until then.
int linear_once_begin(::zkml_ctx* ctx);
int linear_once_end(::zkml_ctx* ctx);
int linear_once(::zkml_ctx* ctx, const uint32_t* x, size_t m, size_t k, const uint32_t* w, size_t n, int activation,
                const uint32_t* residual, uint32_t* pre, uint32_t* out);

}  // namespace zk
