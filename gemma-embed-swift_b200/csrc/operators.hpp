// operators.hpp -- host-side launchers of the operators on caller-owned device tensors
// (ge_attention_causal, ge_attention_prefix, ge_linear_q4).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "kernels.hpp"

namespace ge {

// Raises `kern`'s dynamic shared-memory limit, once per device and kernel (legal during a capture).
template <typename K>
cudaError_t allow_smem(K* kern, int bytes, std::atomic<uint64_t>& devices) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (devices.load(std::memory_order_acquire) >> dev) & 1)) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) devices.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    return e;
}

// Launches with programmatic stream serialisation whatever the calling thread's policy: every kernel
// of the operators waits for its predecessor (pdl_wait) before it touches memory.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, int cluster,
                       Args&&... args) {
    const bool was = programmatic_launch();
    set_programmatic_launch(true);
    const cudaError_t e = launch_kernel(kern, dim3(grid), dim3(block), smem, stream, cluster, std::forward<Args>(args)...);
    set_programmatic_launch(was);
    return e;
}

// ------------------------------------------------------------------ causal and shared-prefix attention
// Query row r of head h attends to the prefix rows [0, prefix) and to its own key rows [lo, hi),
// which the ranges of its sequence give.
struct CausalLaunch {
    bool bf16 = false;
    int heads = 0, kv_heads = 0, hd = 0;
    float scale = 1.0f;
    int window = 0;  // 0: none
    const void *q = nullptr, *k = nullptr, *v = nullptr, *pk = nullptr, *pv = nullptr;
    void* out = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0, pk_stride = 0, pv_stride = 0, out_stride = 0;  // elements
    int ntok = 0, nkv = 0, prefix = 0;
    const uint32_t* q_seqs = nullptr;   // (start, length) pairs
    const uint32_t* kv_seqs = nullptr;
    int nseq = 0;
    void* workspace = nullptr;
    int num_sms = 148;
};
// Bytes of workspace a launch with these sizes needs (only the sizes and types are read).
size_t causal_workspace(const CausalLaunch& a);
cudaError_t launch_causal(const CausalLaunch& a, cudaStream_t stream);

// ------------------------------------------------------------------ 4-bit products
// out[r][n] = sum_k x[r][k] w[n][k], w = scale * (q - 8), or scale * q + min when mins is set; the
// scale and min of group k / group.  values [n][k / 2]: element 2 i in the low half of byte i.
struct Q4Launch {
    bool bf16 = false;
    const void* x = nullptr;
    int64_t x_stride = 0;
    int rows = 0, n = 0, k = 0, group = 32;
    const uint8_t* values = nullptr;
    const __half *scales = nullptr, *mins = nullptr;
    void* out = nullptr;
    int64_t out_stride = 0;
    int num_sms = 148;
};
constexpr int kQ4MaxRows = 64;
cudaError_t launch_linear_q4(const Q4Launch& a, cudaStream_t stream);

}  // namespace ge
