// Forward operators: y = f(x W + b) + r and h = f(x Wg + bg) * (x Wu + bu), mod P.
//
// The product is an exact signed-byte product on the tensor pipe.  An activation, read as a signed
// integer, is split into D balanced byte digits (D = 1, 2, 4 for 8-, 16- and 31-bit activations),
// x = o + sum_i 256^i x_i with x_i in [-128, 127] and o = 128 for D > 1 (the shift makes two digits
// cover exactly the 16-bit integers; o's share of the product is 128 times the weights' column
// sum, laid out beside the bias).  A weight is one balanced byte, or up to four of them (planes).
// So z = sum_{i,p} 256^(i+p) sum_t x_i[t] w_p[t] + 128 sum_t w[t] + b, every inner sum an exact
// s8 x s8 -> s32 product: below 2^14 K, which stays in 32 bits for K <= 1023 tiles of 128; longer
// sums are cut there and joined mod P.
//
// The weights are the 128-row operand and the tokens' digits the N operand (N = D x tokens), so a
// single token fills a 16-column product and costs the weights' bytes, nothing more, and the D
// digits of a token meet in one thread's registers when the accumulators are read back.  Work is
// counted in units of one 128 x 128-byte weight tile; the tiles that do not make a whole wave are
// cut into even shares of units, one per block, and a tile's last block to finish joins its parts.
#include <cuda_runtime.h>

#include <algorithm>

#include "linear_device.cuh"

namespace zk {

namespace {

__device__ __align__(16) uint8_t act_tables[act_table_bytes(2) + act_table_bytes(5)];  // GELU, SiLU

// Epilogue warps: four to each quarter of the accumulators' rows, taking every fourth token group.
// One warp a quarter left each scheduler a single chain of dependent instructions and bound most
// calls by it (64 tokens x 5120 x 13824: 58 us with 4 warps).
constexpr uint32_t EPI_WARPS = 16, EPI_THREADS = 32 * EPI_WARPS, EPI_SUBS = EPI_WARPS / 4;
constexpr uint32_t THREADS = 64 + EPI_THREADS;

// ---------------------------------------------------------------------------
// Weights
// ---------------------------------------------------------------------------

__device__ __forceinline__ int planes_needed(int v) {
    if (v >= -128 && v <= 127) return 1;
    if (v >= -32896 && v <= 32639) return 2;          // 127 * 257 and -128 * 257
    if (v >= -8421504 && v <= 8355711) return 3;      // times 65793
    return 4;
}

// One block per weight tile.  A thread makes four 16-byte chunks of one row (16 consecutive K each;
// reads along the rows of a row-major matrix are coalesced over the lanes), which pass through
// shared memory so that a plane's tile is stored as one run of bytes: stored where they are made,
// 16 bytes to each 128-byte row, 71 M weights took 159 us.
__global__ void __launch_bounds__(256) linear_pack_kernel(const uint32_t* __restrict__ w, const uint32_t* __restrict__ w2,
                                                          size_t rs, size_t cs, PackedWeights p,
                                                          uint8_t* __restrict__ tiles,
                                                          unsigned long long* __restrict__ sums,
                                                          uint32_t* __restrict__ status) {
    __shared__ __align__(16) uint4 stage[LIN_TILE_BYTES / 16];
    const uint32_t nt = blockIdx.x / p.k_tiles, kt = blockIdx.x % p.k_tiles;
    const uint32_t r = threadIdx.x % LIN_ROWS, c0 = threadIdx.x / LIN_ROWS;  // chunks c0, c0 + 2, c0 + 4, c0 + 6
    const uint32_t part = p.gated ? (r >> 4) & 1 : 0;
    const uint32_t f = p.gated ? nt * 64 + (r >> 5) * 16 + (r & 15) : nt * LIN_ROWS + r;
    const uint32_t* src = part ? w2 : w;
    uint32_t bad = 0;
    int need = 1;
    unsigned long long sum = 0;
    uint32_t d[4][4][4];  // [chunk][plane][word]
#pragma unroll
    for (int h = 0; h < 4; h++) {
        const uint32_t k0 = kt * LIN_KB + 16 * (c0 + 2 * h);
        uint32_t v[16];
#pragma unroll
        for (uint32_t j = 0; j < 16; j++)
            v[j] = f < p.n && k0 + j < p.k ? __ldg(src + (size_t)(k0 + j) * rs + (size_t)f * cs) : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bad |= v[4 * i + j] >> 31;
                const int s = m31_signed(v[4 * i + j]);
                sum += (unsigned long long)(s < 0 ? s + (int)P : s);
                need = max(need, planes_needed(s));
                q[j] = balanced_digits(s);
            }
            byte_planes(make_uint4(q[0], q[1], q[2], q[3]), d[h][0][i], d[h][1][i], d[h][2][i], d[h][3][i]);
        }
    }
    const size_t plane = (size_t)p.n_tiles * p.k_tiles * LIN_TILE_BYTES;
    uint4* dst = reinterpret_cast<uint4*>(tiles + ((size_t)nt * p.k_tiles + kt) * LIN_TILE_BYTES);
#pragma unroll
    for (int b = 0; b < 4; b++) {
        if (b >= (int)p.planes) break;
        if (b) __syncthreads();
#pragma unroll
        for (int h = 0; h < 4; h++)
            stage[r * 8 + ((c0 + 2 * h) ^ (r & 7))] = make_uint4(d[h][b][0], d[h][b][1], d[h][b][2], d[h][b][3]);
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 4; h++) dst[b * (plane / 16) + threadIdx.x + 256 * h] = stage[threadIdx.x + 256 * h];
    }
    if (sum) atomicAdd(sums + (size_t)nt * LIN_ROWS + r, sum);
    if (bad) atomicOr(status, LIN_BAD_VALUE);
    if (need > 1) atomicMax(status + 1, (uint32_t)need);
}

__global__ void linear_base_kernel(const unsigned long long* __restrict__ sums, const uint32_t* __restrict__ bias,
                                   const uint32_t* __restrict__ bias2, PackedWeights p, uint32_t* __restrict__ base,
                                   uint32_t* __restrict__ status) {
    const uint32_t slots = p.n_tiles * LIN_ROWS, i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= slots) return;
    const uint32_t nt = i / LIN_ROWS, r = i % LIN_ROWS, part = p.gated ? (r >> 4) & 1 : 0;
    const uint32_t f = p.gated ? nt * 64 + (r >> 5) * 16 + (r & 15) : i;
    const uint32_t* src = part ? bias2 : bias;
    const uint32_t b = src && f < p.n ? src[f] : 0u;
    if (b >> 31) atomicOr(status, LIN_BAD_VALUE);
    base[i] = red32(b);
    base[slots + i] = madd(red32(b), mmul(128, red64(sums[i])));
}

// ---------------------------------------------------------------------------
// Activations -> digit tiles
// ---------------------------------------------------------------------------

// Digit tile of (m tile, K tile): N = D x tokens rows of 128 bytes in the weights' swizzle, row
// i x tokens + t the digit i of token t.  A block takes 32 tokens of a tile (all, if fewer), a
// thread 16 K of one token.  Block 0 also zeroes the counters of the cut tiles.
template <int D>
__global__ void __launch_bounds__(256) linear_digits_kernel(const uint32_t* x, size_t ldx, uint32_t m,
                                                            uint32_t k, uint32_t k_tiles, uint32_t tokens,
                                                            uint8_t* __restrict__ out, uint32_t* __restrict__ counters,
                                                            uint32_t n_counters, uint32_t* __restrict__ status) {
    grid_dependents_launch();  // the product kernel sets up and loads weights meanwhile
    grid_dependency_wait();    // x, and the workspace's last use
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (uint32_t i = threadIdx.x; i < n_counters; i += blockDim.x) counters[i] = 0;
    const uint32_t mt = blockIdx.x / k_tiles, kt = blockIdx.x % k_tiles;
    uint8_t* tile = out + (size_t)blockIdx.x * (D * tokens * LIN_KB);
    const bool vec = (ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(x) & 15) == 0);
    uint32_t bad = 0;
    const uint32_t t = blockIdx.y * 32 + threadIdx.x / 8, c = threadIdx.x % 8;
    if (t < tokens) {
        const uint32_t row = mt * tokens + t, k0 = kt * LIN_KB + 16 * c;
        uint4 v[4];
        const uint32_t* src = x + (size_t)row * ldx + k0;
        if (row < m && vec && k0 + 16 <= k) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = load_words(src + 4 * i);
        } else {
            const auto at = [&](uint32_t i) { return row < m && k0 + i < k ? load_word(src + i) : 0u; };
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) v[i] = make_uint4(at(4 * i), at(4 * i + 1), at(4 * i + 2), at(4 * i + 3));
        }
        uint32_t d[D][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t q[D];
            activation_digits<D>(v[i], q, bad);
#pragma unroll
            for (int b = 0; b < D; b++) d[b][i] = q[b];
        }
#pragma unroll
        for (int b = 0; b < D; b++) {
            const uint32_t r = b * tokens + t;
            *reinterpret_cast<uint4*>(tile + r * LIN_KB + ((c ^ (r & 7)) << 4)) =
                make_uint4(d[b][0], d[b][1], d[b][2], d[b][3]);
        }
    }
    if (bad) atomicOr(status, bad);
}

// ---------------------------------------------------------------------------
// Product and epilogue
// ---------------------------------------------------------------------------

struct KernelArgs {
    PackedWeights w;
    LinearIO io;
    const uint8_t* digits;
    uint32_t* counters;
    uint32_t* slots;
    const uint32_t* base;  // bias with the digits' offset share
    uint32_t tokens, m_tiles, tiles, sk_tiles, stages, slots_per_cta;
};

// A run of units of one tile and plane: one 32-bit accumulation.
struct Segment {
    uint32_t tile, plane, kt, len;
    bool first, last, whole, head;  // of its piece (a block's share of a tile); head: the piece begins inside the tile
    uint32_t piece_units;
};

// The segments of one block, in order: its even share of the cut tiles, then whole tiles.  All
// roles walk the same sequence.
struct Schedule {
    uint32_t k_tiles, per_tile, tiles, dp;
    uint64_t pos, sk_end;
    uint32_t tile, at, piece_begin, piece_end;

    __device__ __forceinline__ void init(const KernelArgs& a) {
        k_tiles = a.w.k_tiles;
        per_tile = a.w.planes * k_tiles;
        tiles = a.tiles;
        const uint64_t units = (uint64_t)a.sk_tiles * per_tile;
        pos = units * blockIdx.x / gridDim.x;
        sk_end = units * (blockIdx.x + 1) / gridDim.x;
        dp = a.sk_tiles + blockIdx.x;
        at = piece_begin = piece_end = 0;
    }
    __device__ __forceinline__ bool next(Segment& s) {
        if (at == piece_end) {
            if (pos < sk_end) {
                tile = (uint32_t)(pos / per_tile);
                const uint64_t begin = (uint64_t)tile * per_tile;
                piece_begin = (uint32_t)(pos - begin);
                piece_end = (uint32_t)min((uint64_t)per_tile, sk_end - begin);
                pos = begin + piece_end;
            } else if (dp < tiles) {
                tile = dp;
                piece_begin = 0;
                piece_end = per_tile;
                dp += gridDim.x;
            } else {
                return false;
            }
            at = piece_begin;
        }
        s.tile = tile;
        s.plane = at / k_tiles;
        s.kt = at - s.plane * k_tiles;
        s.len = min(min(piece_end - at, k_tiles - s.kt), KSEG);
        s.first = at == piece_begin;
        at += s.len;
        s.last = at == piece_end;
        s.whole = piece_begin == 0 && piece_end == per_tile;
        s.head = piece_begin != 0;
        s.piece_units = piece_end - piece_begin;
        return true;
    }
};

// Tiles in groups of up to 8 m tiles, the m tiles of a group innermost, so that blocks running at
// the same time share weight and digit tiles in L2.
__device__ __forceinline__ void tile_at(const KernelArgs& a, uint32_t tile, uint32_t& mt, uint32_t& nt) {
    const uint32_t per_group = 8 * a.w.n_tiles, group = tile / per_group, i = tile - group * per_group;
    const uint32_t high = min(8u, a.m_tiles - 8 * group);
    nt = i / high;
    mt = 8 * group + i - nt * high;
}

// Whether `ok` holds in all epilogue threads: they go on, or give up, together.
__device__ __forceinline__ bool all_of_epilogue(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)ok), "n"(EPI_THREADS)
        : "memory");
    return r != 0;
}

// SELFTEST: with LinearIO::withhold (the instantiation of zkml_selftest_linear_wait alone).
template <int D, bool GATED, bool SELFTEST = false>
__global__ void __launch_bounds__(THREADS, 1) linear_kernel(const __grid_constant__ KernelArgs a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * 16 + 6];
    __shared__ uint32_t tmem_base_s, last_s, issued_s;
    __shared__ volatile uint32_t quit_s;
    constexpr int G = GROUP<D>;
    const uint64_t wait_ns = SELFTEST ? a.io.wait_ns : WAIT_NS;
    const int withhold = SELFTEST && blockIdx.x == 0 ? a.io.withhold : 0;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t n_cols = D * a.tokens, b_bytes = n_cols * LIN_KB, stage_bytes = LIN_TILE_BYTES + b_bytes;
    const uint32_t smem0 = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = smem_addr(bars), empty = full + 8 * 16, acc_full = empty + 8 * 16, acc_empty = acc_full + 16;
    const uint32_t drained = acc_empty + 16, table_full = drained + 8;
    const bool bends = io_bends(a.io);  // the activation takes its table, kept behind the stages
    const uint32_t table_at = smem0 + a.stages * stage_bytes, table_bytes = act_table_bytes(a.io.activation);
    uint32_t cols = 32;
    while (cols < 2 * n_cols) cols <<= 1;
    if (threadIdx.x == 0) {
        quit_s = 0;
        for (uint32_t i = 0; i < a.stages; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, EPI_THREADS);
        }
        mbar_init(drained, 1);
        mbar_init(table_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();  // the block barriers want whole warps
    if (warp == 2) tmem_alloc(smem_addr(&tmem_base_s), cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    // only now, with its tensor memory in hand: a dependent's block must not take what this grid still needs
    grid_dependents_launch();

    if (warp == 0) {
        if (lane == 0) {
            // ---- loads: the weight tiles of the first stages do not wait for the digit kernel
            Schedule sch;
            sch.init(a);
            Segment s{};
            const uint8_t* wp = nullptr;
            const uint8_t* xp = nullptr;
            uint32_t left = 0;
            auto advance = [&]() {  // next unit's pointers
                if (left == 0) {
                    if (!sch.next(s)) return false;
                    uint32_t mt, nt;
                    tile_at(a, s.tile, mt, nt);
                    wp = a.w.tiles + (((size_t)s.plane * a.w.n_tiles + nt) * a.w.k_tiles + s.kt) * LIN_TILE_BYTES;
                    xp = a.digits + ((size_t)mt * a.w.k_tiles + s.kt) * b_bytes;
                    left = s.len;
                } else {
                    wp += LIN_TILE_BYTES;
                    xp += b_bytes;
                }
                left--;
                return true;
            };
            const uint8_t* first_x[16];
            uint32_t issued = 0;
            bool more = true;
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) {
                if (i >= a.stages || !(more = advance())) break;
                if (SELFTEST && withhold == LIN_WITHHOLD_COPY && i == 0) break;
                first_x[i] = xp;
                mbar_expect_tx(full + 8 * i, stage_bytes);
                bulk_load(smem0 + i * stage_bytes, wp, LIN_TILE_BYTES, full + 8 * i);
                issued++;
            }
            if (bends && !(SELFTEST && withhold == LIN_WITHHOLD_TABLE)) {
                mbar_expect_tx(table_full, table_bytes);
                bulk_load(table_at, a.io.act_table, table_bytes, table_full);
            }
            grid_dependency_wait();
#pragma unroll
            for (uint32_t i = 0; i < 16; i++)
                if (i < issued)
                    bulk_load(smem0 + i * stage_bytes + LIN_TILE_BYTES, first_x[i], b_bytes, full + 8 * i);
            uint32_t st = 0, phase = 0;
            while (more && issued >= a.stages && advance()) {
                if (!mbar_wait(empty + 8 * st, phase, &quit_s, wait_ns)) break;
                mbar_expect_tx(full + 8 * st, stage_bytes);
                bulk_load(smem0 + st * stage_bytes, wp, LIN_TILE_BYTES, full + 8 * st);
                bulk_load(smem0 + st * stage_bytes + LIN_TILE_BYTES, xp, b_bytes, full + 8 * st);
                issued++;
                if (++st == a.stages) st = 0, phase ^= 1;
            }
            issued_s = issued;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---- products
            Schedule sch;
            sch.init(a);
            Segment s{};
            grid_dependency_wait();  // so that the waits' limit counts this grid's own time alone
            const uint32_t idesc = tc_idesc_s8(n_cols);
            uint32_t st = 0, phase = 0, seg = 0;
            bool ok = true;
            while (ok && sch.next(s)) {
                const uint32_t buf = seg & 1, use = seg >> 1;
                ok = mbar_wait(acc_empty + 8 * buf, (use & 1) ^ 1, &quit_s, wait_ns);
                tc_fence_after();
                const uint32_t d = tmem + buf * (cols / 2);
                for (uint32_t u = 0; ok && u < s.len; u++) {
                    if (!(ok = mbar_wait(full + 8 * st, phase, &quit_s, wait_ns))) break;
                    tc_fence_after();
                    const uint64_t da = tc_desc_k128(smem0 + st * stage_bytes);
                    const uint64_t db = tc_desc_k128(smem0 + st * stage_bytes + LIN_TILE_BYTES);
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) tc_mma_s8(d, da + 2 * i, db + 2 * i, idesc, (u | i) != 0);
                    tc_commit(empty + 8 * st);
                    if (++st == a.stages) st = 0, phase ^= 1;
                }
                if (ok && !(SELFTEST && withhold == LIN_WITHHOLD_DONE && seg == 0)) tc_commit(acc_full + 8 * buf);
                seg++;
            }
        }
    } else {
        // ---- accumulators -> outputs; this warp's TMEM lanes are 32 (warp % 4) and up
        grid_dependency_wait();  // the counters are zeroed by the kernel before
        const uint32_t quad = warp & 3, row = quad * 32 + lane, sub = (warp - 2) >> 2;
        Schedule sch;
        sch.init(a);
        Segment s{};
        uint32_t seg = 0;
        const bool have_table = !bends || mbar_wait(table_full, 0, &quit_s, wait_ns);
        const uint8_t* table = smem_raw + (table_at - smem_addr(smem_raw));
        uint32_t* const my_slots = a.slots + (size_t)blockIdx.x * a.slots_per_cta * a.tokens * LIN_ROWS;
        while (sch.next(s)) {
            const uint32_t buf = seg & 1, use = seg >> 1;
            seg++;
            if (!all_of_epilogue(have_table && mbar_wait(acc_full + 8 * buf, use & 1, &quit_s, wait_ns))) break;
            tc_fence_after();
            uint32_t mt, nt;
            tile_at(a, s.tile, mt, nt);
            const uint32_t acc = tmem + buf * (cols / 2) + ((quad * 32) << 16);
            const uint32_t base = a.base[(size_t)nt * LIN_ROWS + row];
            const bool direct = s.whole && s.last;
            // slot: 0 a piece that begins inside its tile, 1 one that ends inside it, 2 a whole tile of several segments
            uint32_t* slot = my_slots + (size_t)(s.whole ? 2 : s.head ? 0 : 1) * a.tokens * LIN_ROWS + row;
            const uint32_t scale = pow256(s.plane);
            const uint32_t live = min(a.tokens, a.io.m - mt * a.tokens);  // tokens of this tile
            for (uint32_t t0 = sub * G; t0 < live; t0 += EPI_SUBS * G) {
                uint32_t r[16], z[G];
                if (D == 1) tmem_ld16(r, acc + t0);
#pragma unroll
                for (int i = 0; i < D; i++) {
                    if (D == 2) tmem_ld8(r, 8 * i, acc + i * a.tokens + t0);
                    if (D == 4) tmem_ld4(r, 4 * i, acc + i * a.tokens + t0);
                }
                tmem_wait_ld();
#pragma unroll
                for (int t = 0; t < G; t++) {
                    z[t] = join_digits<D>(r, t);
                    if (s.plane) z[t] = mmul(z[t], scale);
                }
                if (!s.first) {
#pragma unroll
                    for (int t = 0; t < G; t++) z[t] = madd(z[t], slot[(size_t)(t0 + t) * LIN_ROWS]);
                }
                if (direct) {
                    finish_tokens<D, GATED>(a.io, table, a.w.n, nt, row, mt * a.tokens + t0, base, z);
                } else {
#pragma unroll
                    for (int t = 0; t < G; t++) slot[(size_t)(t0 + t) * LIN_ROWS] = z[t];
                }
            }
            tc_fence_before();
            mbar_arrive(acc_empty + 8 * buf);
            if (direct || !s.last) continue;
            // a part of a cut tile: the block that completes the tile's units joins the parts
            __threadfence();
            asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");
            if (threadIdx.x == 64) {
                const uint32_t before = atomicAdd(a.counters + s.tile, s.piece_units);
                __threadfence();
                last_s = before + s.piece_units == sch.per_tile;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");
            if (last_s) {
                __threadfence();
                const uint64_t units = (uint64_t)a.sk_tiles * sch.per_tile, begin = (uint64_t)s.tile * sch.per_tile;
                // block b holds the units from units * b / blocks on
                const uint32_t b0 = (uint32_t)(((begin + 1) * gridDim.x - 1) / units);
                const uint32_t b1 = (uint32_t)(((begin + sch.per_tile) * gridDim.x - 1) / units);
                const size_t pitch = (size_t)a.slots_per_cta * a.tokens * LIN_ROWS;
                constexpr int PARTS = D == 1 ? 1 : D == 2 ? 2 : 4;
                for (uint32_t t0 = sub * G; t0 < live; t0 += EPI_SUBS * G) {
                    uint64_t sum[G];
                    uint32_t z[G];
#pragma unroll
                    for (int t = 0; t < G; t++) sum[t] = 0;
                    for (uint32_t b = b0; b <= b1; b += PARTS) {  // PARTS parts' loads in flight together
                        uint32_t v[PARTS][G];
#pragma unroll
                        for (int i = 0; i < PARTS; i++) {
                            const uint32_t* q = a.slots + (b + i) * pitch +
                                                (size_t)(b + i == b0 ? 1 : 0) * a.tokens * LIN_ROWS +
                                                (size_t)t0 * LIN_ROWS + row;
#pragma unroll
                            for (int t = 0; t < G; t++) v[i][t] = b + i <= b1 ? __ldcg(q + t * LIN_ROWS) : 0u;
                        }
#pragma unroll
                        for (int i = 0; i < PARTS; i++)
#pragma unroll
                            for (int t = 0; t < G; t++) sum[t] += v[i][t];
                    }
#pragma unroll
                    for (int t = 0; t < G; t++) z[t] = canon64(sum[t]);
                    finish_tokens<D, GATED>(a.io, table, a.w.n, nt, row, mt * a.tokens + t0, base, z);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(EPI_THREADS) : "memory");  // last_s is read before it is written again
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (quit_s) {  // some role's wait ran out (all roles are done now)
        if (threadIdx.x == 0) report_timeout(a.io.status, full, a.stages, issued_s, bends ? table_full : 0, wait_ns);
        if (threadIdx.x == 32) drain_products(drained, wait_ns);  // by their issuer
        __syncwarp();
        __syncthreads();
    }
    if (warp == 2) tmem_free(tmem, cols);
}

constexpr uint32_t SMEM_MAX = 225 * 1024;
constexpr uint32_t STAGES_MAX = SMEM_MAX - 1024 - ACT_TABLE_MAX;  // bytes of all stages

template <int D, bool GATED, bool SELFTEST = false>
cudaError_t configure_one() {
    return cudaFuncSetAttribute(linear_kernel<D, GATED, SELFTEST>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
}

template <int D>
cudaError_t launch_all(const KernelArgs& a, const LinearPlan& p, uint8_t* digits, cudaStream_t s, bool overlap) {
    const PackedWeights& w = a.w;
    const unsigned threads = std::min(256u, (p.tokens * 8 + 31) / 32 * 32);
    const Launch d(dim3(p.m_tiles * w.k_tiles, (p.tokens + 31) / 32), threads, 0, s, overlap);
    cudaError_t e = cudaLaunchKernelEx(&d.cfg, linear_digits_kernel<D>, a.io.x, a.io.ldx, a.io.m, w.k, w.k_tiles,
                                       p.tokens, digits, a.counters, p.sk_tiles, a.io.status);
    if (e != cudaSuccess) return e;
    const uint32_t smem = 1024 + p.stages * (LIN_TILE_BYTES + p.digits * p.tokens * LIN_KB) +
                          (io_bends(a.io) ? ACT_TABLE_MAX : 0);
    const Launch l(dim3(p.ctas), THREADS, smem, s, overlap);
    if (D == 4 && !w.gated && a.io.withhold) return cudaLaunchKernelEx(&l.cfg, linear_kernel<4, false, true>, a);
    return w.gated ? cudaLaunchKernelEx(&l.cfg, linear_kernel<D, true>, a)
                   : cudaLaunchKernelEx(&l.cfg, linear_kernel<D, false>, a);
}

}  // namespace

void launch_linear_pack(const uint32_t* w, const uint32_t* w2, size_t rs, size_t cs, const PackedWeights& p,
                        uint8_t* tiles, unsigned long long* sums, uint32_t* status, cudaStream_t s) {
    linear_pack_kernel<<<p.k_tiles * p.n_tiles, 256, 0, s>>>(w, w2, rs, cs, p, tiles, sums, status);
}

void launch_linear_base(const unsigned long long* sums, const uint32_t* bias, const uint32_t* bias2,
                        const PackedWeights& p, uint32_t* base, uint32_t* status, cudaStream_t s) {
    linear_base_kernel<<<p.n_tiles, LIN_ROWS, 0, s>>>(sums, bias, bias2, p, base, status);
}

// Clocks of a split: a model with rates fitted to 916 measured splits of 33 calls (m 9 to 2048, K 300
// to 13824; the split it picks takes 4 % longer than the fastest on average, 16 % at worst).  A block
// multiplies 128 rows x N columns x 128 K in 2 N clocks and takes in 46 bytes a clock, all blocks
// together 5500; a token of a tile costs 30 clocks to finish, under the next tile's products
// except for the last tile; cutting tiles costs a round through memory for the parts, 5200 clocks
// where every tile has the same number of parts and 9300 where shares straddle tiles.
static double plan_clocks(const LinearPlan& p, uint64_t per_tile, uint32_t m, bool straddles) {
    const double n_cols = (double)p.digits * p.tokens, live = std::min(m, p.tokens);
    const double bytes = LIN_TILE_BYTES + n_cols * LIN_KB, unit = std::max(2.0 * n_cols, bytes / 46.0);
    const double finish = 1800 + 30.0 * live, tile = unit * per_tile;
    const uint32_t whole = (p.tiles - p.sk_tiles + p.ctas - 1) / p.ctas;
    double t = whole ? whole * std::max(tile, finish) + finish : 0;
    if (p.sk_tiles) {
        const double tiles = (double)p.sk_tiles / p.ctas, share = tiles * per_tile;
        const double parts = per_tile / share + (straddles ? 1 : 0), pieces = straddles ? tiles + 1 : 1;
        t += share * unit + (straddles ? 9300 : 5200) + pieces * live * 76 + std::max(1.0, tiles) * live * (30 + 19 * parts);
    }
    return std::max(t, (double)p.tiles * per_tile * bytes / 5500 + finish);
}

LinearPlan linear_plan(const PackedWeights& w, uint32_t m, int x_bits, int num_sms) {
    LinearPlan best{};
    const uint32_t digits = x_bits == 8 ? 1 : x_bits == 16 ? 2 : 4;
    const uint32_t unit = 16 / digits, most = 256 / digits;  // N = digits x tokens: a multiple of 16, at most 256
    const uint64_t per_tile = (uint64_t)w.planes * w.k_tiles;
    double best_clocks = 0;
    const uint32_t fewest = (m + most - 1) / most;
    uint32_t last_tokens = 0;
    for (uint32_t want = fewest; want <= 16 * fewest; want += std::max(1u, want / 4)) {
        LinearPlan p{};
        p.digits = digits;
        p.tokens = ((m + want - 1) / want + unit - 1) / unit * unit;
        if (p.tokens == last_tokens) continue;
        last_tokens = p.tokens;
        p.m_tiles = (m + p.tokens - 1) / p.tokens;
        if (want > fewest && (uint64_t)p.m_tiles * w.n_tiles > 16u * num_sms) break;
        p.tiles = p.m_tiles * w.n_tiles;
        const uint32_t waves = p.tiles / num_sms;
        // whole tiles only; the tiles beyond the last full wave but one cut over all blocks; with fewer
        // tiles than blocks, each cut into the same number of parts
        for (uint32_t parts = 0; parts <= 16; parts++) {  // 0: whole tiles, 1: straddling shares, else parts of a tile
            if (parts == 0) {
                p.ctas = std::min(p.tiles, (uint32_t)num_sms);
                p.sk_tiles = 0;
            } else if (parts == 1) {
                p.ctas = (uint32_t)std::min<uint64_t>((uint64_t)num_sms, per_tile * p.tiles);
                if (p.tiles % p.ctas == 0) continue;
                p.sk_tiles = waves ? p.tiles - (waves - 1) * p.ctas : p.tiles;
            } else {
                if (parts > per_tile || (uint64_t)p.tiles * parts > (uint64_t)num_sms) break;
                p.ctas = p.tiles * parts;
                p.sk_tiles = p.tiles;
            }
            const double c = plan_clocks(p, per_tile, m, parts == 1);
            if (!best.tiles || c < best_clocks) best = p, best_clocks = c;
        }
    }
    LinearPlan& p = best;
    const uint32_t stage = LIN_TILE_BYTES + p.digits * p.tokens * LIN_KB;
    p.stages = std::min(16u, STAGES_MAX / stage);
    p.slots = w.planes > 1 || w.k_tiles > KSEG ? 3 : p.sk_tiles ? 2 : 0;
    auto up = [](size_t v) { return (v + 1023) / 1024 * 1024; };
    p.digits_off = up((size_t)p.sk_tiles * 4);
    p.slots_off = p.digits_off + up((size_t)p.m_tiles * w.k_tiles * p.digits * p.tokens * LIN_KB);
    p.bytes = p.slots_off + (size_t)p.ctas * p.slots * p.tokens * LIN_ROWS * 4;
    return p;
}

cudaError_t linear_act_table(int tag, const uint8_t** out) {
    *out = nullptr;
    if (tag != 2 && tag != 5) return cudaSuccess;
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, act_tables);
    if (e == cudaSuccess) *out = static_cast<const uint8_t*>(p) + (tag == 5 ? act_table_bytes(2) : 0);
    return e;
}

cudaError_t linear_configure(cudaStream_t s) {
    cudaError_t e = cudaMemcpyToSymbolAsync(act_tables, act_segment_table(2), act_table_bytes(2), 0,
                                            cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess)
        e = cudaMemcpyToSymbolAsync(act_tables, act_segment_table(5), act_table_bytes(5), act_table_bytes(2),
                                    cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = configure_one<1, false>();
    if (e == cudaSuccess) e = configure_one<2, false>();
    if (e == cudaSuccess) e = configure_one<4, false>();
    if (e == cudaSuccess) e = configure_one<1, true>();
    if (e == cudaSuccess) e = configure_one<2, true>();
    if (e == cudaSuccess) e = configure_one<4, true>();
    if (e == cudaSuccess) e = configure_one<4, false, true>();
    return e;
}

cudaError_t launch_linear(const PackedWeights& w, const LinearPlan& p, const LinearIO& io, void* workspace,
                          cudaStream_t s, bool overlap) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    KernelArgs a{};
    a.w = w;
    a.io = io;
    a.counters = reinterpret_cast<uint32_t*>(ws);
    a.digits = ws + p.digits_off;
    a.slots = reinterpret_cast<uint32_t*>(ws + p.slots_off);
    a.base = w.base + (p.digits > 1 ? (size_t)w.n_tiles * LIN_ROWS : 0);
    a.tokens = p.tokens;
    a.m_tiles = p.m_tiles;
    a.tiles = p.tiles;
    a.sk_tiles = p.sk_tiles;
    a.stages = p.stages;
    a.slots_per_cta = p.slots;
    uint8_t* digits = ws + p.digits_off;
    return p.digits == 1   ? launch_all<1>(a, p, digits, s, overlap)
           : p.digits == 2 ? launch_all<2>(a, p, digits, s, overlap)
                           : launch_all<4>(a, p, digits, s, overlap);
}

}  // namespace zk
