// linear_q4.cu -- ge_linear_q4: products of a few rows with 4-bit weights and group scales,
// out[r][n] = sum_k x[r][k] w[n][k].
#include "attention_rows.cuh"
#include "operators.hpp"

namespace ge {

namespace {

// One warp per (output column, row): a lane takes 8 consecutive weights (one 32-bit word) at a time.
template <typename T>
__global__ void __launch_bounds__(256) k_linear_q4(Q4Launch p) {
    pdl_wait();
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5), r = blockIdx.y, lane = threadIdx.x & 31;
    if (n >= p.n) return;
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.values + int64_t(n) * (p.k / 2));
    const int64_t g0 = int64_t(n) * (p.k / p.group);
    float acc = 0.f;
    for (int i = lane; i < p.k / 8; i += 32) {
        const int g = i * 8 / p.group;
        const float sc = __half2float(p.scales[g0 + g]), mn = p.mins ? __half2float(p.mins[g0 + g]) : -8.0f * sc;
        const uint32_t u = w[i];
        float qs = 0.f, xs = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float xv = float(x[i * 8 + e]);
            qs = fmaf(float((u >> (4 * e)) & 15u), xv, qs);
            xs += xv;
        }
        acc = fmaf(sc, qs, fmaf(mn, xs, acc));
    }
    acc = warp_sum(acc);
    if (lane == 0) static_cast<T*>(p.out)[r * p.out_stride + n] = T(acc);
}

}  // namespace

cudaError_t launch_linear_q4(const Q4Launch& a, cudaStream_t stream) {
    const dim3 grid(unsigned((a.n + 7) / 8), unsigned(a.rows));
    if (a.bf16) return launch_kernel(k_linear_q4<__nv_bfloat16>, grid, dim3(256), 0, stream, 1, a);
    return launch_kernel(k_linear_q4<__half>, grid, dim3(256), 0, stream, 1, a);
}

}  // namespace ge
