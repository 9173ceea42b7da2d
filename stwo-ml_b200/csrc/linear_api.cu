// C-ABI: forward operators with weights laid out once (zkml_linear_*).
#include <algorithm>
#include <string>

#include "context.hpp"
#include "linear.cuh"
#include "qm31.cuh"

struct zkml_linear {
    zkml_ctx* ctx = nullptr;
    uint32_t k = 0, n = 0;
    bool gated = false;
    zk::DevBuf w, bias, status;
    void release() {
        w.release();
        bias.release();
        status.release();
    }
};

namespace zk {
namespace {

// The calling thread's current device, put back when a call returns.
struct DeviceGuard {
    int prev = -1;
    DeviceGuard() {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            cudaGetLastError();
            prev = -1;
        }
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
    if (rs > ((size_t)1 << 34) || cs > ((size_t)1 << 34))
        return set_error(ZKML_ERR_INVALID_ARG, "weight stride too large");
    DeviceGuard guard;
    ZK_CUDA(cudaSetDevice(ctx->device));
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    ZK_CUDA(cudaStreamIsCapturing(s, &cap));
    if (cap != cudaStreamCaptureStatusNone)
        return set_error(ZKML_ERR_INVALID_ARG, "weights cannot be laid out while the stream is captured");
    const size_t span = ((k - 1) * rs + (n - 1) * cs + 1) * 4;
    zkml_linear* lin = new zkml_linear();
    struct Drop {
        zkml_linear*& l;
        DevBuf stage;
        ~Drop() {
            stage.release();
            if (l) {
                l->release();
                delete l;
            }
        }
    } drop{lin, {}};
    lin->ctx = ctx;
    lin->k = (uint32_t)k;
    lin->n = (uint32_t)n;
    lin->gated = parts == 2;
    int rc;
    if ((rc = lin->status.ensure(16)) || (rc = lin->w.ensure((size_t)parts * k * n * 4))) return rc;
    const bool any_bias = biases[0] || (parts == 2 && biases[1]);
    if (any_bias && (rc = lin->bias.ensure((size_t)parts * n * 4))) return rc;
    ZK_CUDA(cudaMemsetAsync(lin->status.ptr, 0, 16, s));
    for (int g = 0; g < 2 * parts; g++) {
        const bool is_bias = g >= parts;
        const uint32_t* src = is_bias ? biases[g - parts] : ws[g];
        if (is_bias && !any_bias) continue;
        if (is_bias && !src) {
            ZK_CUDA(cudaMemsetAsync(lin->bias.as<uint32_t>() + (size_t)(g - parts) * n, 0, n * 4, s));
            continue;
        }
        const size_t bytes = is_bias ? n * 4 : span;
        if (reinterpret_cast<uintptr_t>(src) & 3)
            return set_error(ZKML_ERR_INVALID_ARG, "weight or bias is not aligned to words");
        cudaPointerAttributes attr;
        if (cudaPointerGetAttributes(&attr, src) != cudaSuccess) {
            cudaGetLastError();
            attr.type = cudaMemoryTypeUnregistered;
        }
        if (attr.type == cudaMemoryTypeDevice && attr.device != ctx->device)
            return set_error(ZKML_ERR_INVALID_ARG, "input pointer is device memory of another GPU");
        const uint32_t* dev = src;
        if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged) {
            if (drop.stage.ptr) ZK_CUDA(cudaStreamSynchronize(s));
            if ((rc = drop.stage.ensure(bytes))) return rc;
            ZK_CUDA(cudaMemcpyAsync(drop.stage.ptr, src, bytes, cudaMemcpyHostToDevice, s));
            ctx->h2d_bytes += bytes;
            dev = drop.stage.as<uint32_t>();
        }
        if (is_bias)
            launch_linear_lay_out(dev, 1, (uint32_t)n, n, 1, lin->bias.as<uint32_t>(), (size_t)parts * n,
                                  (size_t)(g - parts) * n, lin->status.as<uint32_t>(), s);
        else
            launch_linear_lay_out(dev, (uint32_t)k, (uint32_t)n, rs, cs, lin->w.as<uint32_t>(), (size_t)parts * n,
                                  (size_t)g * n, lin->status.as<uint32_t>(), s);
        ctx->launches++;
    }
    ZK_CUDA(cudaGetLastError());
    uint32_t st = 0;
    ZK_CUDA(cudaMemcpyAsync(&st, lin->status.ptr, 4, cudaMemcpyDeviceToHost, s));
    ZK_CUDA(cudaStreamSynchronize(s));
    if (st) return set_error(ZKML_ERR_INVALID_ARG, "linear: weight or bias value >= 2^31 is not an M31 element");
    *out = lin;
    lin = nullptr;
    return ZKML_OK;
}

}  // namespace
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
    DeviceGuard guard;
    cudaSetDevice(lin->ctx->device);
    lin->release();  // cudaFree waits for the work that reads the weights
    delete lin;
    return ZKML_OK;
}

int zkml_linear_workspace(const zkml_linear* lin, size_t m, int x_bits, size_t* out_bytes) {
    if (!lin || !out_bytes) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    if (x_bits != 8 && x_bits != 16 && x_bits != 31)
        return set_error(ZKML_ERR_INVALID_ARG, "x_bits must be 8, 16 or 31");
    if (m == 0) return set_error(ZKML_ERR_INVALID_ARG, "empty matrix");
    if (m > (1u << 30) || m * lin->k > ((size_t)1 << 34) || m * lin->n > ((size_t)1 << 34))
        return set_error(ZKML_ERR_INVALID_ARG, "matrix too large");
    *out_bytes = 0;
    return ZKML_OK;
}

int zkml_linear_forward(zkml_linear* lin, const zkml_linear_call* c) {
    if (!lin || !c || !c->x || !c->out) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    size_t need = 0;
    int rc = zkml_linear_workspace(lin, c->m, c->x_bits, &need);
    if (rc) return rc;
    const size_t m = c->m, k = lin->k, n = lin->n;
    if (c->activation < 0 || c->activation > 5)
        return set_error(ZKML_ERR_INVALID_ARG, "activation must be 0 (none) or a type tag 1 to 5");
    if (lin->gated && c->residual)
        return set_error(ZKML_ERR_INVALID_ARG, "gated weights take no residual");
    if (!lin->gated && c->up) return set_error(ZKML_ERR_INVALID_ARG, "up is an output of gated weights only");
    const size_t most = (size_t)1 << 34;
    if (c->ldx > most || c->ld_residual > most || c->ld_out > most || c->ld_pre > most || c->ld_up > most)
        return set_error(ZKML_ERR_INVALID_ARG, "row stride too large");
    if (c->ld_out < n || (c->pre && c->ld_pre < n) || (c->up && c->ld_up < n))
        return set_error(ZKML_ERR_INVALID_ARG, "the row stride of an output is below its width");
    if (c->workspace_bytes < need || (need && !c->workspace))
        return set_error(ZKML_ERR_INVALID_ARG, "workspace of " + std::to_string(need) + " bytes wanted");
    zkml_ctx* ctx = lin->ctx;
    DeviceGuard guard;
    ZK_CUDA(cudaSetDevice(ctx->device));
    if ((rc = want_device_words(ctx, c->x, "x")) || (rc = want_device_words(ctx, c->out, "out")) ||
        (c->residual && (rc = want_device_words(ctx, c->residual, "residual"))) ||
        (c->pre && (rc = want_device_words(ctx, c->pre, "pre"))) ||
        (c->up && (rc = want_device_words(ctx, c->up, "up"))))
        return rc;
    const Block x{c->x, m, k, c->ldx}, res{c->residual, m, n, c->ld_residual}, out{c->out, m, n, c->ld_out};
    const Block pre{c->pre, m, n, c->ld_pre}, up{c->up, m, n, c->ld_up};
    const bool in_place = c->residual == c->out && c->ld_residual == c->ld_out;
    if (share(out, x) || share(pre, x) || share(up, x) || share(out, pre) || share(out, up) || share(pre, up) ||
        (!in_place && share(out, res)) || share(pre, res))
        return set_error(ZKML_ERR_INVALID_ARG, "an output overlaps another argument");
    cudaStream_t s = c->stream ? static_cast<cudaStream_t>(c->stream) : ctx->stream;
    LinearArgs a{};
    a.x = c->x;
    a.w = lin->w.as<uint32_t>();
    a.bias = lin->bias.as<uint32_t>();
    a.residual = c->residual;
    a.out = c->out;
    a.pre = c->pre;
    a.up = c->up;
    a.status = lin->status.as<uint32_t>();
    a.ldx = c->ldx;
    a.ld_res = c->ld_residual;
    a.ld_out = c->ld_out;
    a.ld_pre = c->ld_pre;
    a.ld_up = c->ld_up;
    a.m = (uint32_t)m;
    a.k = (uint32_t)k;
    a.n = (uint32_t)n;
    a.x_bits = c->x_bits;
    a.activation = c->activation;
    a.gated = lin->gated;
    launch_linear_simple(a, s);
    ctx->launches++;
    ZK_CUDA(cudaGetLastError());
    return ZKML_OK;
}

int zkml_linear_check(zkml_linear* lin, void* stream) {
    if (!lin) return set_error(ZKML_ERR_INVALID_ARG, "NULL argument");
    DeviceGuard guard;
    ZK_CUDA(cudaSetDevice(lin->ctx->device));
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : lin->ctx->stream;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    ZK_CUDA(cudaStreamIsCapturing(s, &cap));
    if (cap != cudaStreamCaptureStatusNone)
        return set_error(ZKML_ERR_INVALID_ARG, "the check waits for the stream, which is being captured");
    uint32_t st = 0;
    ZK_CUDA(cudaMemcpyAsync(&st, lin->status.ptr, 4, cudaMemcpyDeviceToHost, s));
    ZK_CUDA(cudaStreamSynchronize(s));
    if (!st) return ZKML_OK;
    ZK_CUDA(cudaMemsetAsync(lin->status.ptr, 0, 4, s));
    if (st & LIN_BAD_VALUE)
        return set_error(ZKML_ERR_INVALID_ARG, "linear: input value >= 2^31 is not an M31 element");
    return set_error(ZKML_ERR_INVALID_ARG, "linear: an activation does not fit the declared x_bits");
}

}  // extern "C"
