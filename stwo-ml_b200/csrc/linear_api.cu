// C-ABI: forward operators with weights laid out once (zkml_linear_*).
#include <algorithm>
#include <atomic>
#include <condition_variable>
#include <mutex>
#include <new>
#include <string>

#include "context.hpp"
#include "linear.cuh"
#include "qm31.cuh"

struct zkml_linear {
    zkml_ctx* ctx = nullptr;
    int device = 0;
    zk::PackedWeights w;
    const uint8_t* act_table[2] = {nullptr, nullptr};  // GELU, SiLU: on the device
    zk::DevBuf tiles;
    zk::DevBuf small;  // status words, column sums, per-row constants
    // Status words: 0 collects what calls without a report of their own met; each call that reports by
    // itself borrows one of the words from FIRST_SLOT on, all zero while nobody holds them.
    static constexpr int FIRST_SLOT = 2, SLOTS = 62;
    std::mutex slots_mutex;
    std::condition_variable slot_free;
    uint64_t slots_held = 0;
    uint32_t* status(int word) const { return small.as<uint32_t>() + word; }
    void release() {
        tiles.release();
        small.release();
    }
};

namespace zk {
namespace {

// Makes `device` current and puts the calling thread's device back when a call returns.
struct DeviceGuard {
    int prev = -1;
    cudaError_t error;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            cudaGetLastError();
            prev = -1;
        }
        error = prev == device ? cudaSuccess : cudaSetDevice(device);
        if (prev == device) prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

int want_device_words(const zkml_ctx* ctx, const void* p, const char* name) {
    if ((reinterpret_cast<uintptr_t>(p) & 3) != 0)
        return set_error(ZKML_ERR_INVALID_ARG, std::string(name) + " is not aligned to words");
    cudaPointerAttributes attr;
    if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) {
        cudaGetLastError();
        attr.type = cudaMemoryTypeUnregistered;
    }
    if (attr.type == cudaMemoryTypeManaged) return ZKML_OK;
    if (attr.type != cudaMemoryTypeDevice || attr.device != ctx->device)
        return set_error(ZKML_ERR_INVALID_ARG, std::string(name) + " is not memory of the context's GPU");
    return ZKML_OK;
}

// A rows x cols block of words with a row stride.
struct Block {
    const uint32_t* p;
    size_t rows, cols, ld;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t end() const { return begin() + 4 * ((rows - 1) * ld + cols); }
};

// Whether two blocks share a word.  Blocks of the same row stride may interleave (two column
// ranges of one buffer); other interleavings count as sharing.
bool share(const Block& a, const Block& b) {
    if (!a.p || !b.p || a.end() <= b.begin() || b.end() <= a.begin()) return false;
    if (a.ld != b.ld || a.ld == 0) return true;
    const Block &lo = a.begin() <= b.begin() ? a : b, &hi = a.begin() <= b.begin() ? b : a;
    const size_t d = ((hi.begin() - lo.begin()) / 4) % lo.ld;
    return d < lo.cols || d + hi.cols > lo.ld;
}

// The kernel of a call and its split, by sizes alone.
struct Choice {
    bool few;
    TokenPlan token;
    LinearPlan linear;
    size_t bytes() const { return few ? 0 : linear.bytes; }
};
// Planning weighs dozens of splits (microseconds); a thread keeps the last ones it made.
const Choice& choose(const PackedWeights& w, uint32_t m, int x_bits, int num_sms) {
    struct Entry {
        uint32_t k = 0, n = 0, planes = 0, gated = 0, m = 0;
        int x_bits = 0, num_sms = 0;
        Choice c;
    };
    static thread_local Entry kept[64];
    Entry& e = kept[(w.k * 31 + w.n * 17 + m * 7 + w.planes + 2 * w.gated + (uint32_t)x_bits) % 64];
    if (e.k == w.k && e.n == w.n && e.planes == w.planes && e.gated == (uint32_t)w.gated && e.m == m &&
        e.x_bits == x_bits && e.num_sms == num_sms)
        return e.c;
    e.c.few = linear_token_plan(w, m, x_bits, num_sms, &e.c.token);
    if (!e.c.few) e.c.linear = linear_plan(w, m, x_bits, num_sms);
    e.k = w.k, e.n = w.n, e.planes = w.planes, e.gated = w.gated, e.m = m, e.x_bits = x_bits, e.num_sms = num_sms;
    return e.c;
}

int status_error(uint32_t st) {
    if (st & LIN_BAD_VALUE)
        return set_error(ZKML_ERR_INVALID_ARG, "linear: input value >= 2^31 is not an M31 element");
    if (st & LIN_TIMEOUT) return set_error(ZKML_ERR_TIMEOUT, "linear: a wait inside the product kernel ran out");
    if (st) return set_error(ZKML_ERR_INVALID_ARG, "linear: an activation does not fit the declared x_bits");
    return ZKML_OK;
}

constexpr size_t STATUS_BYTES = 256;
static_assert(4 * (zkml_linear::FIRST_SLOT + zkml_linear::SLOTS) <= STATUS_BYTES, "status words");

// A status word of one call for its time; waits while all are in use.
struct StatusSlot {
    zkml_linear* lin;
    int i = 0;
    bool clean = true;  // zero again, or never written
    explicit StatusSlot(zkml_linear* l) : lin(l) {
        std::unique_lock<std::mutex> lock(l->slots_mutex);
        const auto none = (uint64_t(1) << zkml_linear::SLOTS) - 1;
        l->slot_free.wait(lock, [&] { return l->slots_held != none; });
        while (l->slots_held >> i & 1) i++;
        l->slots_held |= uint64_t(1) << i;
    }
    ~StatusSlot() {
        if (!clean) return;  // a CUDA error left it unknown: it is not lent again
        {
            std::lock_guard<std::mutex> lock(lin->slots_mutex);
            lin->slots_held &= ~(uint64_t(1) << i);
        }
        lin->slot_free.notify_one();
    }
    uint32_t* word() const { return lin->status(zkml_linear::FIRST_SLOT + i); }
    // Waits for s and reports what was left in the word by then.
    int report(cudaStream_t s) {
        uint32_t st = 0;
        clean = false;
        ZK_CUDA(cudaMemcpyAsync(&st, word(), 4, cudaMemcpyDeviceToHost, s));
        ZK_CUDA(cudaStreamSynchronize(s));
        if (st) {
            ZK_CUDA(cudaMemsetAsync(word(), 0, 4, s));
            ZK_CUDA(cudaStreamSynchronize(s));
        }
        clean = true;
        return status_error(st);
    }
};

__global__ void take_status_kernel(uint32_t* status, uint32_t* out) { *out = atomicExch(status, 0u); }

int refuse_capture(cudaStream_t s, const char* why) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    ZK_CUDA(cudaStreamIsCapturing(s, &cap));
    return cap == cudaStreamCaptureStatusNone ? (int)ZKML_OK : set_error(ZKML_ERR_INVALID_ARG, why);
}

void set_shape(PackedWeights& w, size_t k, size_t n, bool gated) {
    w.k = (uint32_t)k;
    w.n = (uint32_t)n;
    w.gated = gated;
    w.k_tiles = (uint32_t)((k + LIN_KB - 1) / LIN_KB);
    w.n_tiles = (uint32_t)((n + lin_outputs_per_tile(gated) - 1) / lin_outputs_per_tile(gated));
}

// What the kernels need once per device, in place when this returns: readers of the tables run on any stream.
int configure(int device, cudaStream_t s) {
    static std::mutex one;
    static std::atomic<bool> done[64];
    if (device < 64 && done[device].load(std::memory_order_acquire)) return ZKML_OK;
    std::lock_guard<std::mutex> lock(one);
    if (device < 64 && done[device].load(std::memory_order_acquire)) return ZKML_OK;
    ZK_CUDA(linear_configure(s));
    ZK_CUDA(linear_token_configure());
    ZK_CUDA(cudaStreamSynchronize(s));
    if (device < 64) done[device].store(true, std::memory_order_release);
    return ZKML_OK;
}

// Lays out weights of shape w from device memory (src: the weights, then the biases) and waits;
// *bad: a word >= 2^31 was among them.  Signed bytes in most models: one plane is packed, and again
// with more where a value needs them.
int lay_out(zkml_ctx* ctx, PackedWeights& w, const uint32_t* const src[4], size_t rs, size_t cs, DevBuf& tiles,
            DevBuf& small, cudaStream_t s, uint32_t* bad) {
    const size_t slots = (size_t)w.n_tiles * LIN_ROWS, plane = (size_t)w.n_tiles * w.k_tiles * LIN_TILE_BYTES;
    int rc;
    if ((rc = configure(ctx->device, s))) return rc;
    if ((rc = small.ensure(STATUS_BYTES + slots * 16))) return rc;
    uint32_t* const status = small.as<uint32_t>();
    unsigned long long* const sums = reinterpret_cast<unsigned long long*>(small.as<uint8_t>() + STATUS_BYTES);
    uint32_t* const base = reinterpret_cast<uint32_t*>(sums + slots);
    uint32_t st[2] = {0, 1};
    for (w.planes = 1;; w.planes = st[1]) {
        if ((rc = tiles.ensure(plane * w.planes))) return rc;
        ZK_CUDA(cudaMemsetAsync(status, 0, STATUS_BYTES + slots * 8, s));
        launch_linear_pack(src[0], src[1], rs, cs, w, tiles.as<uint8_t>(), sums, status, s);
        ZK_CUDA(cudaGetLastError());
        launch_linear_base(sums, src[2], src[3], w, base, status, s);
        ZK_CUDA(cudaGetLastError());
        ctx->launches += 2;
        ZK_CUDA(cudaMemcpyAsync(st, status, 8, cudaMemcpyDeviceToHost, s));
        ZK_CUDA(cudaStreamSynchronize(s));
        if (st[0] || st[1] <= w.planes) break;
    }
    *bad = st[0];
    w.tiles = tiles.as<uint8_t>();
    w.base = base;
    return ZKML_OK;
}

cudaError_t launch_choice(const Choice& p, const PackedWeights& w, const LinearIO& io, void* workspace, cudaStream_t s,
                          bool overlap) {
    return p.few ? launch_linear_token(w, p.token, io, s, overlap)
                 : launch_linear(w, p.linear, io, workspace, s, overlap);
}

int create(zkml_ctx* ctx, const uint32_t* const* ws, const uint32_t* const* biases, int parts, size_t k, size_t n,
           size_t rs, size_t cs, void* stream, zkml_linear** out) {
    if (!out) return set_error(ZKML_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!ctx) return set_error(ZKML_ERR_INVALID_ARG, "ctx is NULL");
    for (int g = 0; g < parts; g++)
        if (!ws[g]) return set_error(ZKML_ERR_INVALID_ARG, "NULL weight");
    if (k == 0 || n == 0) return set_error(ZKML_ERR_INVALID_ARG, "empty matrix");
    if (k > (1u << 30) || n > (1u << 30) || k * n > ((size_t)1 << 34))
        return set_error(ZKML_ERR_INVALID_ARG, "matrix too large");
    if (rs > ((size_t)1 << 34) || cs > ((size_t)1 << 34) || (k - 1) * rs + (n - 1) * cs > ((size_t)1 << 36))
        return set_error(ZKML_ERR_INVALID_ARG, "weight stride too large");
    DeviceGuard guard(ctx->device);
    ZK_CUDA(guard.error);
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    int rc = refuse_capture(s, "weights cannot be laid out while the stream is captured");
    if (rc) return rc;
    zkml_linear* lin = new (std::nothrow) zkml_linear();
    if (!lin) return set_error(ZKML_ERR_OOM, "no host memory for the handle");
    struct Drop {
        zkml_linear*& l;
        DevBuf stage[4];
        ~Drop() {  // cudaFree waits for the kernels that use these
            for (DevBuf& b : stage) b.release();
            if (l) {
                l->release();
                delete l;
            }
        }
    } drop{lin, {}};
    lin->ctx = ctx;
    lin->device = ctx->device;
    PackedWeights& w = lin->w;
    set_shape(w, k, n, parts == 2);
    const uint32_t* dev[4] = {};  // weights, then biases
    for (int g = 0; g < 2 * parts; g++) {
        const bool is_bias = g >= parts;
        const uint32_t* src = is_bias ? biases[g - parts] : ws[g];
        if (!src) continue;
        if (reinterpret_cast<uintptr_t>(src) & 3)
            return set_error(ZKML_ERR_INVALID_ARG, "weight or bias is not aligned to words");
        cudaPointerAttributes attr;
        if (cudaPointerGetAttributes(&attr, src) != cudaSuccess) {
            cudaGetLastError();
            attr.type = cudaMemoryTypeUnregistered;
        }
        if (attr.type == cudaMemoryTypeDevice && attr.device != ctx->device)
            return set_error(ZKML_ERR_INVALID_ARG, "input pointer is device memory of another GPU");
        uint32_t** to = const_cast<uint32_t**>(&dev[is_bias ? 2 + g - parts : g]);
        if (attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged) {
            *to = const_cast<uint32_t*>(src);
            continue;
        }
        const size_t bytes = is_bias ? n * 4 : ((k - 1) * rs + (n - 1) * cs + 1) * 4;
        if ((rc = drop.stage[g].ensure(bytes))) return rc;
        ZK_CUDA(cudaMemcpyAsync(drop.stage[g].ptr, src, bytes, cudaMemcpyHostToDevice, s));
        ctx->h2d_bytes += bytes;
        *to = drop.stage[g].as<uint32_t>();
    }
    uint32_t bad = 0;
    if ((rc = lay_out(ctx, w, dev, rs, cs, lin->tiles, lin->small, s, &bad))) return rc;
    if (bad) return set_error(ZKML_ERR_INVALID_ARG, "linear: weight or bias value >= 2^31 is not an M31 element");
    ZK_CUDA(linear_act_table(2, &lin->act_table[0]));
    ZK_CUDA(linear_act_table(5, &lin->act_table[1]));
    *out = lin;
    lin = nullptr;
    return ZKML_OK;
}

}  // namespace

int linear_once_begin(zkml_ctx* ctx) {
    const int rc = ctx->lin.met.ensure(4);
    if (rc) return rc;
    ZK_CUDA(cudaMemsetAsync(ctx->lin.met.ptr, 0, 4, ctx->stream));
    return ZKML_OK;
}

int linear_once_end(zkml_ctx* ctx) {
    uint32_t st = 0;
    ZK_CUDA(cudaMemcpyAsync(&st, ctx->lin.met.ptr, 4, cudaMemcpyDeviceToHost, ctx->stream));
    ZK_CUDA(cudaStreamSynchronize(ctx->stream));
    return status_error(st);
}

static int once(zkml_ctx* ctx, const uint32_t* x, size_t m, size_t k, const uint32_t* w, size_t n, int activation,
                const uint32_t* residual, uint32_t* pre, uint32_t* out);

int linear_once(zkml_ctx* ctx, const uint32_t* x, size_t m, size_t k, const uint32_t* w, size_t n, int activation,
                const uint32_t* residual, uint32_t* pre, uint32_t* out) {
    const int rc = once(ctx, x, m, k, w, n, activation, residual, pre, out);
    if (rc) {  // the caller may need the memory for another way (cudaFree waits for queued work); met stays
        ctx->op.bmle.release();
        ctx->lin.small.release();
        ctx->lin.workspace.release();
    }
    return rc;
}

static int once(zkml_ctx* ctx, const uint32_t* x, size_t m, size_t k, const uint32_t* w, size_t n, int activation,
                const uint32_t* residual, uint32_t* pre, uint32_t* out) {
    if (m > (1u << 30) || k > (1u << 30) || n > (1u << 30) || m * k > ((size_t)1 << 34) || k * n > ((size_t)1 << 34))
        return set_error(ZKML_ERR_INVALID_ARG, "matrix too large");
    if (m * n > ((size_t)1 << 34)) return set_error(ZKML_ERR_OOM, "output too large to be tiled");
    LinearScratch& b = ctx->lin;
    // Weights are laid out where the proof later writes the same weight's evaluations (16 bytes an entry) to
    // open it: no memory of their own is held beside what the proof needs anyway.
    DevBuf& tiles = ctx->op.bmle;
    cudaStream_t s = ctx->stream;
    const void* dev = nullptr;
    PackedWeights p;
    set_shape(p, k, n, false);
    uint32_t bad = 0;
    int rc = device_view(ctx, w, k * n * 4, ctx->b_in, &dev);
    const uint32_t* src[4] = {static_cast<const uint32_t*>(dev), nullptr, nullptr, nullptr};
    if (!rc) rc = lay_out(ctx, p, src, n, 1, tiles, b.small, s, &bad);
    if (rc) return rc;
    if (bad) return set_error(ZKML_ERR_INVALID_ARG, "matmul_m31: input value >= 2^31 is not an M31 element");
    const Choice& c = choose(p, (uint32_t)m, 31, ctx->num_sms);
    if ((rc = b.workspace.ensure(c.bytes()))) return rc;
    LinearIO io{};
    io.x = x;
    io.residual = residual;
    io.out = out;
    io.pre = pre;
    io.status = b.met.as<uint32_t>();
    io.ldx = k;
    io.ld_res = io.ld_out = io.ld_pre = n;
    io.m = (uint32_t)m;
    io.activation = activation;
    io.as_reference = true;
    ZK_CUDA(launch_choice(c, p, io, b.workspace.ptr, s, false));
    ctx->launches += c.few ? 1 : 2;
    return ZKML_OK;
}

}  // namespace zk

using namespace zk;

extern "C" {

int zkml_linear_create(zkml_ctx* ctx, const uint32_t* w, size_t k, size_t n, size_t row_stride, size_t col_stride,
                       const uint32_t* bias, void* stream, zkml_linear** out) {
    return create(ctx, &w, &bias, 1, k, n, row_stride, col_stride, stream, out);
}

int zkml_linear_create_gated(zkml_ctx* ctx, const uint32_t* w_gate, const uint32_t* w_up, size_t k, size_t n,
                             size_t row_stride, size_t col_stride, const uint32_t* bias_gate, const uint32_t* bias_up,
                             void* stream, zkml_linear** out) {
    const uint32_t *ws[2] = {w_gate, w_up}, *bs[2] = {bias_gate, bias_up};
    return create(ctx, ws, bs, 2, k, n, row_stride, col_stride, stream, out);
}

int zkml_linear_destroy(zkml_linear* lin) {
    if (!lin) return ZKML_OK;
    DeviceGuard guard(lin->device);
    // a destructor may run while some stream of the program is captured: freeing is no part of that capture
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    lin->release();  // cudaFree waits for the work that reads the weights
    cudaThreadExchangeStreamCaptureMode(&mode);
    delete lin;
    return ZKML_OK;
}

int zkml_linear_workspace(const zkml_linear* lin, size_t m, int x_bits, size_t* out_bytes) {
    if (!lin || !out_bytes) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    if (x_bits != 8 && x_bits != 16 && x_bits != 31)
        return set_error(ZKML_ERR_INVALID_ARG, "x_bits must be 8, 16 or 31");
    if (m == 0) return set_error(ZKML_ERR_INVALID_ARG, "empty matrix");
    if (m > (1u << 30) || m * lin->w.k > ((size_t)1 << 34) || m * lin->w.n > ((size_t)1 << 34))
        return set_error(ZKML_ERR_INVALID_ARG, "matrix too large");
    *out_bytes = choose(lin->w, (uint32_t)m, x_bits, lin->ctx->num_sms).bytes();
    return ZKML_OK;
}

// The call of zkml_linear_forward with its status bits in `status`; withhold and wait_ns as in LinearIO.
static int forward(zkml_linear* lin, const zkml_linear_call* c, uint32_t* status, int withhold = 0,
                   uint64_t wait_ns = 0) {
    if (!lin || !c || !c->x || !c->out) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    size_t need = 0;
    int rc = zkml_linear_workspace(lin, c->m, c->x_bits, &need);
    if (rc) return rc;
    const size_t m = c->m, k = lin->w.k, n = lin->w.n;
    if (c->activation < 0 || c->activation > 5)
        return set_error(ZKML_ERR_INVALID_ARG, "activation must be 0 (none) or a type tag 1 to 5");
    if (lin->w.gated && c->residual)
        return set_error(ZKML_ERR_INVALID_ARG, "gated weights take no residual");
    if (!lin->w.gated && c->up) return set_error(ZKML_ERR_INVALID_ARG, "up is an output of gated weights only");
    const size_t most = (size_t)1 << 34;
    if (c->ldx > most || c->ld_residual > most || c->ld_out > most || c->ld_pre > most || c->ld_up > most)
        return set_error(ZKML_ERR_INVALID_ARG, "row stride too large");
    if (c->ld_out < n || (c->pre && c->ld_pre < n) || (c->up && c->ld_up < n))
        return set_error(ZKML_ERR_INVALID_ARG, "the row stride of an output is below its width");
    if (c->workspace_bytes < need || (need && !c->workspace))
        return set_error(ZKML_ERR_INVALID_ARG, "workspace of " + std::to_string(need) + " bytes wanted");
    if (need && (reinterpret_cast<uintptr_t>(c->workspace) & 255))
        return set_error(ZKML_ERR_INVALID_ARG, "workspace is not aligned to 256 bytes");
    zkml_ctx* ctx = lin->ctx;
    DeviceGuard guard(ctx->device);
    ZK_CUDA(guard.error);
    if (c->pointers_checked) {
        const uintptr_t all = reinterpret_cast<uintptr_t>(c->x) | reinterpret_cast<uintptr_t>(c->out) |
                              reinterpret_cast<uintptr_t>(c->residual) | reinterpret_cast<uintptr_t>(c->pre) |
                              reinterpret_cast<uintptr_t>(c->up);
        if (all & 3) return set_error(ZKML_ERR_INVALID_ARG, "an argument is not aligned to words");
    } else if ((rc = want_device_words(ctx, c->x, "x")) || (rc = want_device_words(ctx, c->out, "out")) ||
               (need && (rc = want_device_words(ctx, c->workspace, "workspace"))) ||
               (c->residual && (rc = want_device_words(ctx, c->residual, "residual"))) ||
               (c->pre && (rc = want_device_words(ctx, c->pre, "pre"))) ||
               (c->up && (rc = want_device_words(ctx, c->up, "up"))))
        return rc;
    const Block x{c->x, m, k, c->ldx}, res{c->residual, m, n, c->ld_residual}, out{c->out, m, n, c->ld_out};
    const Block pre{c->pre, m, n, c->ld_pre}, up{c->up, m, n, c->ld_up};
    const Block wsp{need ? static_cast<const uint32_t*>(c->workspace) : nullptr, 1, need / 4, 0};
    const bool in_place = c->residual == c->out && c->ld_residual == c->ld_out;
    const bool with_inputs = share(out, x) || share(pre, x) || share(up, x) || share(pre, res) ||
                             (!in_place && share(out, res));
    const bool with_outputs = share(out, pre) || share(out, up) || share(pre, up);
    const bool with_workspace =
        share(wsp, x) || share(wsp, res) || share(wsp, out) || share(wsp, pre) || share(wsp, up);
    if (with_inputs || with_outputs || with_workspace)
        return set_error(ZKML_ERR_INVALID_ARG, "an output overlaps another argument");
    cudaStream_t s = c->stream ? static_cast<cudaStream_t>(c->stream) : ctx->stream;
    LinearIO io{};
    io.x = c->x;
    io.residual = c->residual;
    io.out = c->out;
    io.pre = c->pre;
    io.up = c->up;
    io.status = status;
    io.ldx = c->ldx;
    io.ld_res = c->ld_residual;
    io.ld_out = c->ld_out;
    io.ld_pre = c->ld_pre;
    io.ld_up = c->ld_up;
    io.m = (uint32_t)m;
    io.activation = c->activation;
    io.act_table = c->activation == 2 ? lin->act_table[0] : c->activation == 5 ? lin->act_table[1] : nullptr;
    io.withhold = withhold;
    io.wait_ns = wait_ns;
    const Choice& p = choose(lin->w, io.m, c->x_bits, ctx->num_sms);
    if ((withhold == LIN_WITHHOLD_TABLE && (p.few || !io.act_table)) || (withhold == LIN_WITHHOLD_DIGITS && !p.few))
        return set_error(ZKML_ERR_INVALID_ARG, "the kernel of this call has no such wait");
    ZK_CUDA(launch_choice(p, lin->w, io, c->workspace, s, true));
    ctx->launches += p.few ? 1 : 2;
    return ZKML_OK;
}

int zkml_linear_forward(zkml_linear* lin, const zkml_linear_call* call) {
    return forward(lin, call, lin ? lin->status(0) : nullptr);
}

int zkml_linear_forward_checked(zkml_linear* lin, const zkml_linear_call* call) {
    if (!lin || !call) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    DeviceGuard guard(lin->ctx->device);
    ZK_CUDA(guard.error);
    cudaStream_t s = call->stream ? static_cast<cudaStream_t>(call->stream) : lin->ctx->stream;
    int rc = refuse_capture(s, "a checked call waits for its stream, which is being captured");
    if (rc) return rc;
    StatusSlot slot(lin);
    if ((rc = forward(lin, call, slot.word()))) {
        slot.clean = rc == ZKML_ERR_INVALID_ARG;  // refused before any launch
        return rc;
    }
    return slot.report(s);
}

int zkml_selftest_linear_wait(zkml_linear* lin, const zkml_linear_call* call, int withhold, uint32_t limit_ms) {
    if (!lin || !call) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    if (withhold < LIN_WITHHOLD_DONE || withhold > LIN_WITHHOLD_DIGITS || limit_ms == 0 || limit_ms > 1000 ||
        lin->w.gated || call->x_bits != 31)
        return set_error(ZKML_ERR_INVALID_ARG, "self-test: withhold 1 to 4, 1 to 1000 ms, plain weights, x_bits 31");
    return forward(lin, call, lin->status(0), withhold, limit_ms * 1000000ull);
}

int zkml_linear_check(zkml_linear* lin, void* stream) {
    if (!lin) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    DeviceGuard guard(lin->ctx->device);
    ZK_CUDA(guard.error);
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : lin->ctx->stream;
    const int rc = refuse_capture(s, "the check waits for the stream, which is being captured");
    if (rc) return rc;
    StatusSlot slot(lin);
    // read and cleared in one step: what calls on other streams set meanwhile is reported now or by the next check
    take_status_kernel<<<1, 1, 0, s>>>(lin->status(0), slot.word());
    ZK_CUDA(cudaGetLastError());
    lin->ctx->launches++;
    return slot.report(s);
}

}  // extern "C"
