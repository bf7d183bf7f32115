// attention_rows.cuh -- one attention row of ge_attention_causal / ge_attention_prefix by one warp,
// straight from the definition: lane l holds dims [l * D / 32, (l + 1) * D / 32) of the row, and the
// running maximum m (log2 units), sum l and output of a softmax are kept in fp32 over its keys.  The output is
// a mean of the values so far throughout, weights summing to 1, so that values up to the type's largest
// do not overflow on the way.  It reads the visible keys and values only, so nothing a masked place holds can
// reach the row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace ge {

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t u);
template <>
__device__ __forceinline__ float2 pair_to_float<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 pair_to_float<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t float_to_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t float_to_pair<__half>(float a, float b) {
    return pack_half2(a, b);
}
template <>
__device__ __forceinline__ uint32_t float_to_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The same, finite values past the type's largest as that: a mean whose weights were rounded may pass it, the values'
// own mean cannot.
template <typename T>
__device__ __forceinline__ uint32_t mean_to_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t mean_to_pair<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <>
__device__ __forceinline__ uint32_t mean_to_pair<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

template <int D>
struct RowState {
    static constexpr int kPer = D / 32;  // dims of one lane
    float q[kPer], o[kPer], m, l;
};

template <typename T, int D>
__device__ __forceinline__ void row_load(const T* p, int lane, float (&x)[D / 32]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p + lane * (D / 32));
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
        const float2 f = pair_to_float<T>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// q is the row's query; the state starts empty (m = -inf).
template <typename T, int D>
__device__ __forceinline__ void row_begin(RowState<D>& s, const T* q, int lane) {
    row_load<T, D>(q, lane, s.q);
#pragma unroll
    for (int i = 0; i < D / 32; i++) s.o[i] = 0.f;
    s.m = -INFINITY;
    s.l = 0.f;
}

// Adds keys [0, n) at k, v (rows `k_stride`, `v_stride` elements apart), eight at a time: their loads and
// sums are independent, so a key costs a fraction of a trip to memory.
template <typename T, int D>
__device__ void row_keys(RowState<D>& s, const T* k, const T* v, int64_t k_stride, int64_t v_stride, int n,
                         float scale_log2e, int lane) {
    constexpr int B = 8, W = D / 64;  // keys at a time; a lane's words of a row
    for (int j = 0; j < n; j += B) {
        const int count = min(B, n - j);
        uint32_t kw[B][W], vw[B][W];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int64_t at = j + min(b, count - 1);
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(k + at * k_stride + lane * (D / 32));
            const uint32_t* vp = reinterpret_cast<const uint32_t*>(v + at * v_stride + lane * (D / 32));
#pragma unroll
            for (int i = 0; i < W; i++) kw[b][i] = kp[i], vw[b][i] = vp[i];
        }
        float d[B], m = s.m;
#pragma unroll
        for (int b = 0; b < B; b++) {
            d[b] = 0.f;
#pragma unroll
            for (int i = 0; i < W; i++) {
                const float2 x = pair_to_float<T>(kw[b][i]);
                d[b] = fmaf(s.q[2 * i + 1], x.y, fmaf(s.q[2 * i], x.x, d[b]));
            }
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            d[b] = warp_sum(d[b]) * scale_log2e;
            m = fmaxf(m, d[b]);
        }
        const float before = s.m == m ? s.l : s.l * ex2_approx(s.m - m);  // the sum so far, under the new maximum
        s.m = m;
        s.l = before;
#pragma unroll
        for (int b = 0; b < B; b++) {
            // A score of -inf under a finite maximum weighs 0; with no finite score yet it counts nothing either
            // (m stays -inf).  A NaN score, which the maximum passes over, makes the sum NaN.
            d[b] = b >= count || (m == -INFINITY && !isnan(d[b])) ? 0.f : ex2_approx(d[b] - m);
            s.l += d[b];
        }
        const float inv = s.l == 0.f ? 0.f : 1.0f / s.l, keep = before * inv;
#pragma unroll
        for (int i = 0; i < D / 32; i++) s.o[i] *= keep;
#pragma unroll
        for (int b = 0; b < B; b++) {
            if (b >= count) break;
            const float p = d[b] * inv;
#pragma unroll
            for (int i = 0; i < W; i++) {
                const float2 x = pair_to_float<T>(vw[b][i]);
                s.o[2 * i] = fmaf(p, x.x, s.o[2 * i]);
                s.o[2 * i + 1] = fmaf(p, x.y, s.o[2 * i + 1]);
            }
        }
    }
}

}  // namespace ge
