// operators.cpp -- C entry points of the operators on device tensors: argument checks, the device
// guard and the launches.  Nothing here allocates device memory or keeps state between calls.
#include "operators.hpp"

#include <cuda_fp16.h>
#include <string.h>

#include <cmath>
#include <mutex>
#include <string>

#include "gemma_embed.h"
#include "model.hpp"

namespace {

int fail(int code, const std::string& msg) { return ge::set_thread_error(code, msg); }
int invalid(const std::string& msg) { return fail(GE_ERR_INVALID_OPTIONS, "invalid options: " + msg); }

// Puts the calling thread's current device back on every return path, where it was changed.
struct DeviceGuard {
    int saved = -1, used = -1;
    DeviceGuard() {
        if (cudaGetDevice(&saved) != cudaSuccess) saved = -1;
    }
    ~DeviceGuard() {
        if (saved >= 0 && used >= 0 && used != saved) cudaSetDevice(saved);
    }
};

constexpr int kMaxDevices = 64;
std::mutex g_mu;
int g_sms[kMaxDevices] = {};  // per device: its SM count, once it is known to be an sm_100 device

// Makes `device` current and returns its SM count; 0 with the status in *rc when it cannot be used.
int use_device(DeviceGuard& keep, int device, int* rc) {
    const auto failed = [&](cudaError_t e) {
        *rc = fail(GE_ERR_NO_DEVICE, std::string("cannot use CUDA device: ") + cudaGetErrorString(e));
        return 0;
    };
    if (device < 0 || device >= kMaxDevices) return failed(cudaErrorInvalidDevice);
    cudaError_t e = device == keep.saved ? cudaSuccess : cudaSetDevice(device);
    if (e != cudaSuccess) return failed(e);
    keep.used = device;
    std::lock_guard<std::mutex> g(g_mu);
    if (g_sms[device]) return g_sms[device];
    int major = 0, sms = 0;
    if ((e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess)
        return failed(e);
    if (major != 10) {
        *rc = fail(GE_ERR_NO_DEVICE, "device " + std::to_string(device) + " is not an sm_100 (B200-class) GPU");
        return 0;
    }
    return g_sms[device] = sms;
}

int launched(cudaError_t e) {
    if (e == cudaSuccess) return GE_OK;
    cudaGetLastError();
    return fail(GE_ERR_GPU_FAILURE, std::string("GPU execution failed: ") + cudaGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int32_t kMaxRows = 1 << 30;

int check_shape(const ge_attention_shape* s, bool prefix) {
    if (!s) return invalid("NULL shape");
    if (s->dtype != GE_F16 && s->dtype != GE_BF16) return invalid("dtype must be GE_F16 or GE_BF16");
    if (s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256) return invalid("head_dim must be 64, 128 or 256");
    if (s->heads < 1 || s->kv_heads < 1 || s->heads > 65535 || s->heads % s->kv_heads)
        return invalid("heads must be a multiple of kv_heads, both from 1 to 65535");
    if (s->heads / s->kv_heads > 128) return invalid("at most 128 heads may share a KV head");
    // The kernels take scores times scale log2 e, which has to be finite itself (0 times it is the score of a zero query).
    if (!(s->scale > 0.0f) || !std::isfinite(s->scale * 1.4426950408889634f))
        return invalid("scale must be positive, and finite times log2 e");
    if (s->window < 0) return invalid("window must not be negative");
    if (prefix && s->window > 0) return invalid("a window does not go with a shared prefix");
    return GE_OK;
}

int check_tensor(const char* name, const void* p, int32_t rows, int64_t stride, int64_t width) {
    if (rows == 0) return GE_OK;
    if (!p) return invalid(std::string(name) + " is NULL");
    if (!aligned16(p)) return invalid(std::string(name) + " must be 16-byte aligned");
    if (stride < width || stride % 8 || stride > (int64_t(1) << 38))
        return invalid(std::string(name) + "'s row stride must be a multiple of 8 elements and at least its " +
                       std::to_string(width) + " columns");
    return GE_OK;
}

// Rows of `width` bytes, `stride` bytes apart.
struct Rows {
    const void* p;
    int64_t rows, stride, width;
};
// Whether two arrays share a byte.  Columns of the same wide rows do not; arrays of different strides whose spans
// meet count as sharing one.
bool overlap(const Rows& a, const Rows& b) {
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
    const uint64_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
    const auto end = [](uint64_t at, const Rows& r) { return __int128(at) + __int128(r.rows - 1) * r.stride + r.width; };
    if (end(a0, a) <= __int128(b0) || end(b0, b) <= __int128(a0)) return false;
    if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return true;
    const uint64_t s = uint64_t(a.rows > 1 ? a.stride : b.rows > 1 ? b.stride : 0);
    if (s == 0) return true;
    const uint64_t d = (b0 % s + s - a0 % s) % s;  // b's columns behind a's in a row
    return d < uint64_t(a.width) || d + uint64_t(b.width) > s;
}

void fill_shape(ge::CausalLaunch& a, const ge_attention_shape* s) {
    a.bf16 = s->dtype == GE_BF16;
    a.heads = s->heads;
    a.kv_heads = s->kv_heads;
    a.hd = s->head_dim;
    a.scale = s->scale;
    a.window = s->window;
    a.q_stride = s->q_stride;
    a.k_stride = s->k_stride;
    a.v_stride = s->v_stride;
    a.pk_stride = s->prefix_k_stride;
    a.pv_stride = s->prefix_v_stride;
    a.out_stride = s->out_stride;
}

int run_attention(int device, const ge_attention_shape* s, ge::CausalLaunch& a, int64_t workspace_bytes, void* stream,
                  bool prefix) {
    int rc = check_shape(s, prefix);
    if (rc) return rc;
    if (a.ntok < 0 || a.nkv < 0 || a.prefix < 0 || a.nseq < 0 || a.ntok > kMaxRows || a.nkv > kMaxRows || a.prefix > kMaxRows ||
        a.nseq > kMaxRows)
        return invalid("row and sequence counts must be from 0 to 2^30");
    fill_shape(a, s);
    if (a.ntok == 0 || a.nseq == 0) return GE_OK;
    const int64_t qw = int64_t(a.heads) * a.hd, kw = int64_t(a.kv_heads) * a.hd;
    if ((rc = check_tensor("q", a.q, a.ntok, a.q_stride, qw)) || (rc = check_tensor("out", a.out, a.ntok, a.out_stride, qw)) ||
        (rc = check_tensor("k", a.k, a.nkv, a.k_stride, kw)) || (rc = check_tensor("v", a.v, a.nkv, a.v_stride, kw)) ||
        (rc = check_tensor("prefix_k", a.pk, a.prefix, a.pk_stride, kw)) ||
        (rc = check_tensor("prefix_v", a.pv, a.prefix, a.pv_stride, kw)))
        return rc;
    if (!a.q_seqs || !a.kv_seqs || (reinterpret_cast<uintptr_t>(a.q_seqs) & 3) || (reinterpret_cast<uintptr_t>(a.kv_seqs) & 3))
        return invalid("sequence ranges are NULL or not 4-byte aligned");
    const Rows out{a.out, a.ntok, 2 * a.out_stride, 2 * qw};
    if (overlap(out, {a.q, a.ntok, 2 * a.q_stride, 2 * qw}) || overlap(out, {a.k, a.nkv, 2 * a.k_stride, 2 * kw}) ||
        overlap(out, {a.v, a.nkv, 2 * a.v_stride, 2 * kw}) || overlap(out, {a.pk, a.prefix, 2 * a.pk_stride, 2 * kw}) ||
        overlap(out, {a.pv, a.prefix, 2 * a.pv_stride, 2 * kw}))
        return invalid("out must not overlap q, k, v or the prefix");
    DeviceGuard keep;
    a.num_sms = use_device(keep, device, &rc);
    if (!a.num_sms) return rc;
    const size_t need = ge::causal_workspace(a);
    if (!a.workspace || workspace_bytes < 0 || size_t(workspace_bytes) < need ||
        (reinterpret_cast<uintptr_t>(a.workspace) & 255))
        return invalid("workspace must be 256-byte aligned and hold " + std::to_string(need) + " bytes");
    return launched(ge::launch_causal(a, stream ? static_cast<cudaStream_t>(stream) : cudaStreamLegacy));
}

}  // namespace

extern "C" {

int ge_attention_workspace(int32_t device_ordinal, const ge_attention_shape* shape, int32_t ntok, int32_t prefix_len,
                           int64_t* bytes) {
    int rc = check_shape(shape, false);
    if (rc) return rc;
    if (ntok < 0 || prefix_len < 0 || ntok > kMaxRows || prefix_len > kMaxRows || !bytes)
        return invalid("row counts must be from 0 to 2^30, and bytes not NULL");
    DeviceGuard keep;
    ge::CausalLaunch a;
    fill_shape(a, shape);
    a.ntok = ntok;
    a.nkv = kMaxRows;  // however many keys the call has
    a.prefix = prefix_len;
    a.num_sms = use_device(keep, device_ordinal, &rc);
    if (!a.num_sms) return rc;
    *bytes = int64_t(ge::causal_workspace(a));
    return GE_OK;
}

int ge_attention_causal(int32_t device_ordinal, const ge_attention_shape* shape, const void* d_q, const void* d_k,
                        const void* d_v, int32_t ntok, const uint32_t* d_seqs, int32_t nseq, void* d_out, void* workspace,
                        int64_t workspace_bytes, void* stream) {
    ge::CausalLaunch a;
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.out = d_out;
    a.ntok = a.nkv = ntok;
    a.q_seqs = a.kv_seqs = d_seqs;
    a.nseq = nseq;
    a.workspace = workspace;
    return run_attention(device_ordinal, shape, a, workspace_bytes, stream, false);
}

int ge_attention_prefix(int32_t device_ordinal, const ge_attention_shape* shape, const void* d_q, int32_t ntok,
                        const void* d_k, const void* d_v, int32_t nkv, const void* d_prefix_k, const void* d_prefix_v,
                        int32_t prefix_len, const uint32_t* d_q_seqs, const uint32_t* d_kv_seqs, int32_t nseq, void* d_out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
    ge::CausalLaunch a;
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.pk = d_prefix_k;
    a.pv = d_prefix_v;
    a.out = d_out;
    a.ntok = ntok;
    a.nkv = nkv;
    a.prefix = prefix_len;
    a.q_seqs = d_q_seqs;
    a.kv_seqs = d_kv_seqs;
    a.nseq = nseq;
    a.workspace = workspace;
    return run_attention(device_ordinal, shape, a, workspace_bytes, stream, true);
}

int ge_q4_repack(const uint8_t* blocks, int32_t type, int64_t n, int64_t k, uint8_t* values, uint16_t* scales, uint16_t* mins) {
    if (type != GE_Q4_0 && type != GE_Q4_1)
        return fail(GE_ERR_UNSUPPORTED_TENSOR_TYPE, "unsupported tensor type " + std::to_string(type) + ": Q4_0 and Q4_1 are repacked");
    if (n < 0 || k < 0 || k % 32 || (k > 0 && n > (int64_t(1) << 46) / k)) return invalid("n and k must not be negative, k a multiple of 32");
    if (n == 0 || k == 0) return GE_OK;
    if (!blocks || !values || !scales || (type == GE_Q4_1 && !mins)) return invalid("NULL array");
    const int64_t per = type == GE_Q4_1 ? 20 : 18, count = n * (k / 32);
    for (int64_t b = 0; b < count; b++) {
        const uint8_t* src = blocks + b * per;
        memcpy(&scales[b], src, 2);
        if (type == GE_Q4_1) memcpy(&mins[b], src + 2, 2);
        // GGUF: byte j of a block holds elements j (low half) and j + 16 (high half).
        const uint8_t* q = src + (per - 16);
        uint8_t* dst = values + b * 16;
        for (int i = 0; i < 8; i++) {
            dst[i] = uint8_t((q[2 * i] & 15) | (q[2 * i + 1] << 4));
            dst[8 + i] = uint8_t((q[2 * i] >> 4) | (q[2 * i + 1] & 0xf0));
        }
    }
    return GE_OK;
}

int ge_linear_q4(int32_t device_ordinal, int32_t dtype, const void* d_x, int64_t x_stride, int32_t rows, int32_t k,
                 const uint8_t* d_values, const uint16_t* d_scales, const uint16_t* d_mins, int32_t group, int32_t n,
                 void* d_out, int64_t out_stride, void* stream) {
    if (dtype != GE_F16 && dtype != GE_BF16) return invalid("dtype must be GE_F16 or GE_BF16");
    if (rows < 0 || rows > ge::kQ4MaxRows) return invalid("ge_linear_q4 takes 0.." + std::to_string(ge::kQ4MaxRows) + " rows");
    if (group != 32 && group != 64 && group != 128) return invalid("group must be 32, 64 or 128");
    if (n < 0 || n > kMaxRows || k < group || k % group || k > 65536) return invalid("k must be a multiple of the group, at most 65536");
    if (rows == 0 || n == 0) return GE_OK;
    if (!d_x || !d_values || !d_scales || !d_out) return invalid("NULL device array");
    if (!aligned16(d_x) || !aligned16(d_values) || (reinterpret_cast<uintptr_t>(d_scales) & 1) ||
        (reinterpret_cast<uintptr_t>(d_mins) & 1) || (reinterpret_cast<uintptr_t>(d_out) & 1))
        return invalid("x and values must be 16-byte aligned");
    constexpr int64_t kMaxStride = int64_t(1) << 38;
    if (x_stride < k || x_stride % 8 || out_stride < n || x_stride > kMaxStride || out_stride > kMaxStride)
        return invalid("x's row stride must be a multiple of 8 elements and at least k, out's at least n, both at most 2^38");
    const Rows out{d_out, rows, 2 * out_stride, 2 * int64_t(n)};
    const int64_t groups = int64_t(n) * (k / group);
    if (overlap(out, {d_x, rows, 2 * x_stride, 2 * int64_t(k)}) || overlap(out, {d_values, 1, 0, int64_t(n) * (k / 2)}) ||
        overlap(out, {d_scales, 1, 0, 2 * groups}) || overlap(out, {d_mins, 1, 0, 2 * groups}))
        return invalid("out must not overlap x or the weights");
    DeviceGuard keep;
    int rc = GE_OK;
    ge::Q4Launch a;
    a.num_sms = use_device(keep, device_ordinal, &rc);
    if (!a.num_sms) return rc;
    a.bf16 = dtype == GE_BF16;
    a.x = d_x;
    a.x_stride = x_stride;
    a.rows = rows;
    a.n = n;
    a.k = k;
    a.group = group;
    a.values = d_values;
    a.scales = reinterpret_cast<const __half*>(d_scales);
    a.mins = reinterpret_cast<const __half*>(d_mins);
    a.out = d_out;
    a.out_stride = out_stride;
    return launched(ge::launch_linear_q4(a, stream ? static_cast<cudaStream_t>(stream) : cudaStreamLegacy));
}

}  // extern "C"
