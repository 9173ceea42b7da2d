// Forward operators for a few tokens (decoding): one launch that is bound by the weights' bytes.
//
// The product of linear_kernels.cu with the activations' digits made inside the block that uses
// them, and K split over the blocks of a cluster instead of over the grid: block r of a cluster
// takes the r-th share of K of one 128-row weight tile, its warps turn the tokens' words into
// digit tiles beside the weight tiles that bulk copies bring in, and the partial sums meet in the
// blocks' shared memory.  So a call has no digit kernel before it, no partial sums in global
// memory, no counters and no workspace; a single token through 13824 x 5120 is a chain of one
// launch, the stream of 71 MB of weights, and one cluster barrier.  Two blocks fit an SM, so the
// next call's blocks (programmatic dependents) load weights while this call's finish.
#include <cuda_runtime.h>

#include <algorithm>

#include "linear_device.cuh"

namespace zk {

namespace {

constexpr uint32_t MAKERS = 8;  // warps that make digit tiles; four of them finish the rows
constexpr uint32_t TOKEN_THREADS = 64 + 32 * MAKERS;
constexpr uint32_t TOKEN_SMEM = 110 * 1024;  // two blocks an SM
constexpr uint32_t MAX_STAGES = 6;
constexpr uint32_t MAX_TOKENS = 8;
constexpr uint32_t MAX_COLS = 32;                // digit columns
constexpr uint32_t GROUPS = MAX_COLS / 16;       // token groups a thread finishes, at most

struct TokenArgs {
    PackedWeights w;
    LinearIO io;
    const uint32_t* base;
    uint32_t tokens, parts, stages;
    uint32_t slices;  // warps that share a unit's tokens: 1, 2 or 4
};

// SELFTEST: with LinearIO::withhold (the instantiation of zkml_selftest_linear_wait alone).
template <int D, bool GATED, bool SELFTEST = false>
__global__ void __launch_bounds__(TOKEN_THREADS, 2) linear_token_kernel(const __grid_constant__ TokenArgs a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 2];
    __shared__ uint32_t tmem_base_s, issued_s;
    __shared__ volatile uint32_t quit_s;
    __shared__ volatile uint32_t missing_s;  // a block of the cluster gave up: its partial sums are not here
    constexpr int G = GROUP<D>;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t nt = blockIdx.x / a.parts, rank = blockIdx.x % a.parts;  // cluster dimension: parts
    const uint64_t wait_ns = SELFTEST ? a.io.wait_ns : WAIT_NS;
    const int withhold = SELFTEST && nt == 0 && rank + 1 == a.parts ? a.io.withhold : 0;
    const uint32_t n_cols = D * a.tokens, stage_bytes = LIN_TILE_BYTES + n_cols * LIN_KB;
    const uint32_t smem0 = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = smem_addr(bars), empty = full + 8 * MAX_STAGES, acc_full = empty + 8 * MAX_STAGES;
    const uint32_t drained = acc_full + 8;
    // partial sums received from the cluster: [source block][quarter held here][token][lane]
    const uint32_t part_base = smem0 + a.stages * stage_bytes;
    const uint32_t k_begin = (uint32_t)((uint64_t)a.w.k_tiles * rank / a.parts);
    const uint32_t k_len = (uint32_t)((uint64_t)a.w.k_tiles * (rank + 1) / a.parts) - k_begin;
    const uint32_t units = k_len * a.w.planes;
    uint32_t cols = 32;
    while (cols < a.w.planes * n_cols) cols <<= 1;
    if (threadIdx.x == 0) {
        quit_s = missing_s = 0;
        for (uint32_t i = 0; i < a.stages; i++) {
            mbar_init(full + 8 * i, 1 + a.slices);  // the copy's issuer and the digit makers
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 2) tmem_alloc(smem_addr(&tmem_base_s), cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    // only now, with its tensor memory in hand: a dependent's block must not take what this grid still needs
    grid_dependents_launch();
    if (a.parts > 1) cluster_arrive();  // this block runs: others may store into it once all have said so

    // K tile and plane of unit u: planes outermost
    const auto tile_of = [&](uint32_t u, uint32_t& plane, uint32_t& kt) {
        plane = u / k_len;
        kt = k_begin + u - plane * k_len;
    };
    // accumulators of this thread's row, joined over digits and planes, group by group
    uint32_t z[GROUPS][G];
    const uint32_t quad = warp & 3, row = quad * 32 + lane;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t st = 0, phase = 1, issued = 0;
            for (uint32_t u = 0; u < units; u++) {
                if (u == a.stages) grid_dependency_wait();  // so that the waits' limit counts this grid's own time alone
                if (!(ok = mbar_wait(empty + 8 * st, phase, &quit_s, wait_ns))) break;
                if (SELFTEST && withhold == LIN_WITHHOLD_COPY && u + 1 == units) break;
                uint32_t plane, kt;
                tile_of(u, plane, kt);
                mbar_expect_tx(full + 8 * st, LIN_TILE_BYTES);
                bulk_load(smem0 + st * stage_bytes,
                          a.w.tiles + (((size_t)plane * a.w.n_tiles + nt) * a.w.k_tiles + kt) * LIN_TILE_BYTES,
                          LIN_TILE_BYTES, full + 8 * st);
                issued++;
                if (++st == a.stages) st = 0, phase ^= 1;
            }
            issued_s = issued;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            grid_dependency_wait();
            const uint32_t idesc = tc_idesc_s8(n_cols);
            uint32_t st = 0, phase = 0, kt_done = 0, plane = 0;
            for (uint32_t u = 0; u < units; u++) {
                if (!(ok = mbar_wait(full + 8 * st, phase, &quit_s, wait_ns))) break;
                tc_fence_after();
                const uint64_t da = tc_desc_k128(smem0 + st * stage_bytes);
                const uint64_t db = tc_desc_k128(smem0 + st * stage_bytes + LIN_TILE_BYTES);
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
                    tc_mma_s8(tmem + plane * n_cols, da + 2 * i, db + 2 * i, idesc, (kt_done | i) != 0);
                tc_commit(empty + 8 * st);
                if (++st == a.stages) st = 0, phase ^= 1;
                if (++kt_done == k_len) kt_done = 0, plane++;
            }
            if (ok && !(SELFTEST && withhold == LIN_WITHHOLD_DONE)) tc_commit(acc_full);
        }
    } else {
        // ---- digit tiles: a lane takes 4 K of a token
        grid_dependency_wait();
        // A unit's tokens are dealt to `slices` warps, at most two to each, and the units to the
        // 8 / slices groups of warps; no more groups than stages, so that a group is never two uses of a
        // stage ahead of its barrier.
        const uint32_t maker = warp - 2, slice = maker % a.slices, groups = min(MAKERS / a.slices, a.stages);
        const bool vec = (a.io.ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(a.io.x) & 15) == 0);
        uint32_t bad = 0;
        const auto load = [&](uint4(&v)[2], uint32_t u) {
            uint32_t plane, kt;
            tile_of(u, plane, kt);
            const uint32_t k0 = kt * LIN_KB + 4 * lane;
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t t = slice + i * a.slices;
                v[i] = make_uint4(0, 0, 0, 0);
                if (t >= a.io.m) continue;
                const uint32_t* src = a.io.x + (size_t)t * a.io.ldx + k0;
                if (vec && k0 + 4 <= a.w.k) {
                    v[i] = load_words(src);
                } else {
                    if (k0 < a.w.k) v[i].x = load_word(src);
                    if (k0 + 1 < a.w.k) v[i].y = load_word(src + 1);
                    if (k0 + 2 < a.w.k) v[i].z = load_word(src + 2);
                    if (k0 + 3 < a.w.k) v[i].w = load_word(src + 3);
                }
            }
        };
        uint32_t u = maker / a.slices < groups ? maker / a.slices : units;
        uint4 v[2], ahead[2];
        if (u < units) load(v, u);
        while (u < units) {
            const uint32_t u_next = u + groups;
            if (u_next < units) load(ahead, u_next);  // on its way while this one becomes digits
            const uint32_t st = u % a.stages, tile = smem0 + st * stage_bytes + LIN_TILE_BYTES;
            // the stage's last product is done
            ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * st, ((u / a.stages) & 1) ^ 1, &quit_s, wait_ns));
            if (!ok) break;
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t t = slice + i * a.slices;
                if (t >= a.io.m) continue;
                uint32_t d[D];
                activation_digits<D>(v[i], d, bad);
#pragma unroll
                for (int b = 0; b < D; b++) {
                    const uint32_t r = b * a.tokens + t;
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(tile + r * LIN_KB + (((lane >> 2) ^ (r & 7)) << 4) +
                                                                4 * (lane & 3)),
                                 "r"(d[b])
                                 : "memory");
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && !(SELFTEST && withhold == LIN_WITHHOLD_DIGITS && u + 1 == units)) mbar_arrive(full + 8 * st);
            u = u_next;
#pragma unroll
            for (int i = 0; i < 2; i++) v[i] = ahead[i];
        }
        if (bad) atomicOr(a.io.status, bad);
        // ---- this warp's quarter of the rows (warps 2 to 5): TMEM lanes 32 (warp % 4) and up
        if (maker < 4 && __all_sync(0xffffffffu, ok)) {
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, &quit_s, wait_ns));
            tc_fence_after();
            if (ok) {
#pragma unroll
                for (uint32_t h = 0; h < GROUPS; h++) {
                    if (h * G >= a.tokens) break;
                    for (uint32_t plane = 0; plane < a.w.planes; plane++) {
                        const uint32_t acc = tmem + plane * n_cols + h * G + ((quad * 32) << 16);
                        uint32_t r[16];
                        if (D == 1) tmem_ld16(r, acc);
#pragma unroll
                        for (int i = 0; i < D; i++) {
                            if (D == 2) tmem_ld8(r, 8 * i, acc + i * a.tokens);
                            if (D == 4) tmem_ld4(r, 4 * i, acc + i * a.tokens);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int t = 0; t < G; t++) {
                            const uint32_t v = join_digits<D>(r, t);
                            z[h][t] = plane ? madd(z[h][t], mmul(v, pow256(plane))) : v;
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    // ---- quarter q of the rows is finished by block q % holders of the cluster
    const uint32_t base = a.base[(size_t)nt * LIN_ROWS + row];
    const bool finisher = warp >= 2 && warp < 6;
    if (a.parts > 1) {
        const uint32_t holders = min(a.parts, 4u), held = (4 + holders - 1) / holders;
        const uint32_t missing_at = smem_addr(const_cast<const uint32_t*>(&missing_s));
        cluster_wait();
        if (finisher && ok) {
            const uint32_t at = part_base + ((rank * held + quad / holders) * a.tokens * 32 + lane) * 4;
#pragma unroll
            for (uint32_t h = 0; h < GROUPS; h++)
#pragma unroll
                for (uint32_t t = 0; t < G; t++)
                    if (h * G + t < a.io.m) cluster_store(at + (h * G + t) * 128, quad % holders, z[h][t]);
        } else if (finisher && lane == 0) {  // this warp gave up: the rows' holder must not finish without it
            cluster_store(missing_at, quad % holders, 1);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (finisher && ok && quad % holders == rank && !missing_s) {
#pragma unroll
            for (uint32_t h = 0; h < GROUPS; h++) {
                if (h * G >= a.io.m) break;
                uint64_t sum[G];
#pragma unroll
                for (int t = 0; t < G; t++) sum[t] = 0;
                for (uint32_t src = 0; src < a.parts; src++) {
                    const uint32_t at = part_base + ((src * held + quad / holders) * a.tokens * 32 + lane) * 4;
#pragma unroll
                    for (uint32_t t = 0; t < G; t++) {
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + (h * G + t) * 128) : "memory");
                        sum[t] += v;
                    }
                }
#pragma unroll
                for (int t = 0; t < G; t++) z[h][t] = canon64(sum[t]);
                finish_tokens<D, GATED>(a.io, a.io.act_table, a.w.n, nt, row, h * G, base, z[h]);
            }
        }
    } else if (finisher && ok) {
#pragma unroll
        for (uint32_t h = 0; h < GROUPS; h++) {
            if (h * G >= a.io.m) break;
            finish_tokens<D, GATED>(a.io, a.io.act_table, a.w.n, nt, row, h * G, base, z[h]);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (quit_s) {  // some role's wait ran out (all roles are done now)
        if (threadIdx.x == 0) report_timeout(a.io.status, full, a.stages, issued_s, 0, wait_ns);
        if (threadIdx.x == 32) drain_products(drained, wait_ns);  // by their issuer
        __syncwarp();
        __syncthreads();
    }
    if (warp == 2) tmem_free(tmem, cols);
}

template <int D>
cudaError_t launch(const TokenArgs& a, const TokenPlan& p, cudaStream_t s, bool overlap) {
    Launch l(dim3(a.w.n_tiles * p.parts), TOKEN_THREADS, p.smem, s, overlap);
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = p.parts;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1] = l.attr;
    l.cfg.attrs = attrs;
    l.cfg.numAttrs = overlap ? 2 : 1;
    if (D == 4 && !a.w.gated && a.io.withhold) return cudaLaunchKernelEx(&l.cfg, linear_token_kernel<4, false, true>, a);
    return a.w.gated ? cudaLaunchKernelEx(&l.cfg, linear_token_kernel<D, true>, a)
                     : cudaLaunchKernelEx(&l.cfg, linear_token_kernel<D, false>, a);
}

}  // namespace

cudaError_t linear_token_configure() {
    const void* kernels[] = {(const void*)linear_token_kernel<1, false>, (const void*)linear_token_kernel<2, false>,
                             (const void*)linear_token_kernel<4, false>, (const void*)linear_token_kernel<1, true>,
                             (const void*)linear_token_kernel<2, true>,  (const void*)linear_token_kernel<4, true>,
                             (const void*)linear_token_kernel<4, false, true>};
    for (const void* k : kernels) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, TOKEN_SMEM);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Taken for up to 8 tokens: beyond, making the digits once for all weight tiles is cheaper than in
// every block (31-bit tokens x 5120 x 13824: 8 tokens 17.8 us here, 17.9 us with a digit kernel; 12
// tokens 23.5 against 17.8 us; x 5120 x 5120: 10.6 against 13.4, 13.8 against 13.6 us).
bool linear_token_plan(const PackedWeights& w, uint32_t m, int x_bits, int num_sms, TokenPlan* out) {
    TokenPlan p{};
    p.digits = x_bits == 8 ? 1 : x_bits == 16 ? 2 : 4;
    const uint32_t n_cols = m * p.digits <= 16 ? 16 : 32;
    if (m > MAX_TOKENS) return false;
    p.tokens = n_cols / p.digits;
    // As many blocks to a cluster as stay resident at once, two an SM less a tenth that clusters cannot
    // fill, up to 6 (one token, 5120 x 5120: 15.8 us with 1, 11.1 with 2, 8.3 with 4, 8.1 with 5, 8.2 with 6;
    // 7 and 8 leave SMs of a GPC idle: 19 us), each with at least 2 K tiles; one block below 8 K tiles,
    // where the cluster's barriers cost more than the shorter K saves (576 x 1536: 5.0 against 5.5 us).
    p.parts = w.k_tiles < 8 ? 1u : std::min(6u, w.k_tiles / 2);
    p.parts = std::min(p.parts, std::max(1u, 9u * num_sms / 5 / w.n_tiles));
    if (w.k_tiles / p.parts + 1 > KSEG) return false;
    const uint32_t holders = std::min(p.parts, 4u), held = (4 + holders - 1) / holders;
    const uint32_t part_bytes = p.parts > 1 ? p.parts * held * p.tokens * 32 * 4 : 0;
    const uint32_t stage = LIN_TILE_BYTES + n_cols * LIN_KB;
    p.stages = std::min(MAX_STAGES, (TOKEN_SMEM - 1024 - part_bytes) / stage);
    p.smem = p.stages * stage + part_bytes + 1024;
    *out = p;
    return true;
}

cudaError_t launch_linear_token(const PackedWeights& w, const TokenPlan& p, const LinearIO& io, cudaStream_t s,
                                bool overlap) {
    TokenArgs a{};
    a.w = w;
    a.io = io;
    a.base = w.base + (p.digits > 1 ? (size_t)w.n_tiles * LIN_ROWS : 0);
    a.tokens = p.tokens;
    a.parts = p.parts;
    a.stages = p.stages;
    a.slices = io.m <= 2 ? 1 : io.m <= 4 ? 2 : 4;
    return p.digits == 1   ? launch<1>(a, p, s, overlap)
           : p.digits == 2 ? launch<2>(a, p, s, overlap)
                           : launch<4>(a, p, s, overlap);
}

}  // namespace zk
