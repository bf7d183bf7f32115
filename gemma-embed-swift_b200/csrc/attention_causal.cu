// attention_causal.cu -- ge_attention_causal and ge_attention_prefix: attention of query rows over a
// shared prefix and over their own sequences' keys up to their own place.
//
// Every query row r reduces to a pair of key ranges: the prefix rows [0, P), the same for every row,
// and its own key rows [lo(r), hi(r)):
//   query i of n in a sequence whose own keys are rows [s, s + m):  hi = s + m - n + i + 1 (cut to
//   [s, s + m]), lo = s, or max(s, hi - window) under a window.
// A causal prompt is the case P = 0, m = n.  k_causal_ranges writes (lo, hi) per query row to the
// workspace, (0, -1) for rows of no sequence, which are never stored.
#include <algorithm>

#include "attention_rows.cuh"
#include "operators.hpp"

namespace ge {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct RangeParams {
    const uint32_t* q_seqs;
    const uint32_t* kv_seqs;
    int nseq, ntok, nkv, window;
    int2* rng;
};

__global__ void __launch_bounds__(1024) k_causal_ranges(RangeParams p) {
    pdl_wait();
    for (int r = threadIdx.x; r < p.ntok; r += blockDim.x) p.rng[r] = make_int2(0, -1);
    __syncthreads();
    for (int s = threadIdx.x >> 5; s < p.nseq; s += int(blockDim.x >> 5)) {
        const int64_t q0 = p.q_seqs[2 * s], n = p.q_seqs[2 * s + 1];
        const int64_t k0 = p.kv_seqs[2 * s], m = p.kv_seqs[2 * s + 1];
        // Ranges past the tensors are cut; a key range that starts outside holds no key.
        const int64_t q1 = min(q0 + n, int64_t(p.ntok));
        const int64_t ks = min(k0, int64_t(p.nkv)), ke = min(k0 + m, int64_t(p.nkv));
        for (int64_t r = q0 + (threadIdx.x & 31); r < q1; r += 32) {
            const int64_t see = k0 + m - n + (r - q0) + 1;
            const int64_t hi = max(ks, min(see, ke));
            const int64_t lo = p.window > 0 ? min(hi, max(ks, see - p.window)) : ks;
            p.rng[r] = make_int2(int(lo), int(hi));
        }
    }
}

struct RowParams {
    const void *q, *k, *v, *pk, *pv;
    void* out;
    int64_t q_stride, k_stride, v_stride, pk_stride, pv_stride, out_stride;
    int heads, group, ntok, prefix;
    float scale_log2e;
    const int2* rng;
};

// One warp per (row, head).
template <typename T, int D>
__global__ void __launch_bounds__(256) k_causal_rows(RowParams p) {
    pdl_wait();
    const int64_t id = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (id >= int64_t(p.ntok) * p.heads) return;
    const int64_t r = id / p.heads;
    const int h = int(id - r * p.heads), kh = h / p.group;
    const int2 rng = p.rng[r];
    if (rng.y < 0) return;
    RowState<D> s;
    row_begin<T, D>(s, static_cast<const T*>(p.q) + r * p.q_stride + int64_t(h) * D, lane);
    if (p.prefix > 0)
        row_keys<T, D>(s, static_cast<const T*>(p.pk) + int64_t(kh) * D, static_cast<const T*>(p.pv) + int64_t(kh) * D,
                       p.pk_stride, p.pv_stride, p.prefix, p.scale_log2e, lane);
    row_keys<T, D>(s, static_cast<const T*>(p.k) + rng.x * p.k_stride + int64_t(kh) * D,
                   static_cast<const T*>(p.v) + rng.x * p.v_stride + int64_t(kh) * D, p.k_stride, p.v_stride,
                   rng.y - rng.x, p.scale_log2e, lane);
    const float inv = s.l == 0.f ? 0.f : 1.0f / s.l;
    uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + r * p.out_stride + int64_t(h) * D + lane * (D / 32));
#pragma unroll
    for (int i = 0; i < D / 64; i++) o[i] = float_to_pair<T>(s.o[2 * i] * inv, s.o[2 * i + 1] * inv);
}

template <typename T, int D>
cudaError_t launch_rows(const CausalLaunch& a, const RowParams& p, cudaStream_t stream) {
    const int64_t blocks = (int64_t(a.ntok) * a.heads + 7) / 8;
    return launch_kernel(k_causal_rows<T, D>, dim3(unsigned(blocks)), dim3(256), 0, stream, 1, p);
}

}  // namespace

size_t causal_workspace(const CausalLaunch& a) { return (size_t(a.ntok) * sizeof(int2) + 255) / 256 * 256; }

cudaError_t launch_causal(const CausalLaunch& a, cudaStream_t stream) {
    int2* rng = static_cast<int2*>(a.workspace);
    RangeParams rp{a.q_seqs, a.kv_seqs, a.nseq, a.ntok, a.nkv, a.window, rng};
    cudaError_t e = launch_kernel(k_causal_ranges, dim3(1), dim3(1024), 0, stream, 1, rp);
    if (e != cudaSuccess) return e;
    RowParams p{a.q, a.k, a.v, a.pk, a.pv, a.out, a.q_stride, a.k_stride, a.v_stride, a.pk_stride, a.pv_stride, a.out_stride,
                a.heads, a.heads / a.kv_heads, a.ntok, a.prefix, a.scale * kLog2e, rng};
    if (a.bf16) {
        if (a.hd == 64) return launch_rows<__nv_bfloat16, 64>(a, p, stream);
        if (a.hd == 128) return launch_rows<__nv_bfloat16, 128>(a, p, stream);
        return launch_rows<__nv_bfloat16, 256>(a, p, stream);
    }
    if (a.hd == 64) return launch_rows<__half, 64>(a, p, stream);
    if (a.hd == 128) return launch_rows<__half, 128>(a, p, stream);
    return launch_rows<__half, 256>(a, p, stream);
}

}  // namespace ge
