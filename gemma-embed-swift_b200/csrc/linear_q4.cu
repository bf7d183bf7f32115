// linear_q4.cu -- ge_linear_q4: products of a few rows with 4-bit weights and group scales,
// out[r][n] = sum_k x[r][k] w[n][k].
//
// Bound by reading the weights once, so they stream from memory to shared memory (cp.async, a ring of
// its own per warp, no barrier in the way) and are widened on the fly to 16-bit integers, which are
// exact, for the warp's 16 x 8 x 16 tensor products with fp32 sums (a warp's product costs fewer
// issue slots than one multiply-add per weight and row, and a 128-row tcgen05 tile would be empty
// but for a few rows).  Every 32 weights the integer sums are scaled in fp32: acc += scale * sum, plus
// min * (sum of x) with minima, so no weight is ever rounded.
//
// One CTA per SM, 16 warps.  A warp owns 16 output columns n (a row tile) and, where the CTA's tiles
// leave warps over, one of S slices of k; the slices' sums are joined in shared memory in order.
// Stage of a warp: 16 rows x 256 weights (16 x 128 bytes, chunk c of row r at c ^ (r & 7), so that the
// 32-bit reads of a fragment hit 32 banks).  The lane's word of a 32-weight group holds the group's
// elements 8 c .. 8 c + 7; their nibbles come out as pairs (0, 4), (1, 5), (2, 6), (3, 7), which x is
// stored to match: the products' k order is permuted the same on both sides.
// x is staged 16 bytes at a time for all warps in two buffers of kXElems elements per 8 rows.
#include <algorithm>

#include "attention_rows.cuh"
#include "operators.hpp"

namespace ge {

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kStageK = 256;                   // weights of a row per stage
constexpr int kStageBytes = 16 * kStageK / 2;  // 2 KB
constexpr int kDepth = 4;
constexpr int kXElems = 2048;                  // x elements of 8 rows per buffer

template <int NB>
struct Q4Cfg {
    static constexpr int KC = kXElems / NB;           // k elements per row and buffer
    static constexpr int kXRow = KC * 2 + 64;         // bytes; 64 over a multiple of 128: two rows, no conflict
    static constexpr int kXBytes = 8 * NB * kXRow;
    static constexpr int kSums = 8 * NB * (KC / 32);  // sums of x per row and 32 elements
    static constexpr int kOffX = kWarps * kDepth * kStageBytes;
    static constexpr int kOffSum = kOffX + 2 * kXBytes;
    static constexpr int kSmem = kOffSum + 2 * kSums * 4;
    static constexpr int kMaxSplit = KC / kStageK;
};

struct Q4Params {
    const void* x;
    int64_t x_stride;
    int rows, n, k, group;
    const uint8_t* values;
    const __half *scales, *mins;
    void* out;
    int64_t out_stride;
    int tiles, R, S, Ks;  // row tiles in all; tiles and k slices of a CTA at a time; k per slice
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Eight 4-bit values as four exact pairs (0, 4), (1, 5), (2, 6), (3, 7), less 8 each where `kSigned`.
// fp16: 1024 + q has q as its low bits (and 1024 + 16 q the bits four places up, brought back by an
// exact multiply-add); bf16 holds 128 + q alike.
template <bool kSigned>
__device__ __forceinline__ void widen_f16(uint32_t u, uint32_t (&t)[4]) {
    const __half2 off = __float2half2_rn(kSigned ? -1032.f : -1024.f);
    const __half2 sixteenth = __float2half2_rn(0.0625f), off16 = __float2half2_rn(kSigned ? -72.f : -64.f);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t v = i ? u >> 8 : u;
        const uint32_t a = (v & 0x000f000fu) | 0x64006400u, b = (v & 0x00f000f0u) | 0x64006400u;
        const __half2 ha = __hadd2(*reinterpret_cast<const __half2*>(&a), off);
        const __half2 hb = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, off16);
        t[2 * i] = *reinterpret_cast<const uint32_t*>(&ha);
        t[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hb);
    }
}
template <bool kSigned>
__device__ __forceinline__ void widen_bf16(uint32_t u, uint32_t (&t)[4]) {
    const __nv_bfloat162 off = __float2bfloat162_rn(kSigned ? -136.f : -128.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t a = ((u >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 h = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), off);
        t[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// NB: tiles of 8 rows of x.
template <typename T, int NB, bool kMins>
__global__ void __launch_bounds__(kThreads, 1) k_linear_q4(const __grid_constant__ Q4Params p) {
    using C = Q4Cfg<NB>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int rt = warp % p.R, sp = warp / p.R;
    const int t_begin = int(int64_t(blockIdx.x) * p.tiles / gridDim.x), t_end = int(int64_t(blockIdx.x + 1) * p.tiles / gridDim.x);
    const int kcs = C::KC / p.S / kStageK * kStageK;  // k of a slice per buffer
    const int chunk_stages = kcs / kStageK;
    const int stages = (p.Ks + kStageK - 1) / kStageK, chunks = (stages + chunk_stages - 1) / chunk_stages;
    const int groups = p.k / p.group, gshift = p.group == 32 ? 5 : p.group == 64 ? 6 : 7;
    uint8_t* ring = smem + warp * kDepth * kStageBytes;
    const uint32_t ring_addr = smem_u32(ring);
    pdl_wait();
    pdl_launch();

    // x of buffer `i` (elements [s Ks + i kcs, + kcs) of every slice s): up to four 16-byte units per thread.
    constexpr int kUnits = 8 * NB * C::KC / 8 / kThreads;
    const int units_row = p.S * kcs / 8;
    uint4 xr[kUnits];
    auto load_x = [&](int i) {
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int id = u * kThreads + threadIdx.x, r = id / units_row, e = (id - r * units_row) * 8;
            const int s = e / kcs, off = i * kcs + (e - s * kcs), kk = s * p.Ks + off;
            xr[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < p.rows && off < p.Ks && kk < p.k)
                xr[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + r * p.x_stride + kk);
        }
    };
    auto store_x = [&](int i) {
        uint8_t* buf = smem + C::kOffX + (i & 1) * C::kXBytes;
        float* sums = reinterpret_cast<float*>(smem + C::kOffSum) + (i & 1) * C::kSums;
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int id = u * kThreads + threadIdx.x, r = id / units_row, e = (id - r * units_row) * 8;
            const uint4 v = xr[u];
            if (kMins) {
                float s = 0.f;
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = pair_to_float<T>(w[j]);
                    s += f.x + f.y;
                }
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                if (r < p.rows && (threadIdx.x & 3) == 0) sums[r * (C::KC / 32) + e / 32] = s;
            }
            if (r < p.rows) {
                uint4 o;  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
                o.x = __byte_perm(v.x, v.z, 0x5410);
                o.y = __byte_perm(v.x, v.z, 0x7632);
                o.z = __byte_perm(v.y, v.w, 0x5410);
                o.w = __byte_perm(v.y, v.w, 0x7632);
                *reinterpret_cast<uint4*>(buf + r * C::kXRow + e * 2) = o;
            }
        }
    };

    for (int base = t_begin; base < t_end; base += p.R) {
        const bool works = sp < p.S && base + rt < t_end;
        const int n0 = (base + rt) * 16, k0 = sp * p.Ks, k1 = min(p.k, k0 + p.Ks);
        const int mine = works ? max(0, (k1 - k0 + kStageK - 1) / kStageK) : 0;  // this warp's stages
        // The four 16-byte chunks of a stage this lane copies: rows 4 i + lane / 8, chunk lane % 8.
        auto copy = [&](int st) {
            if (st < mine) {
                const int kk = k0 + st * kStageK + (lane & 7) * 32;
                const uint32_t bytes = kk < k1 ? 16u : 0u;  // zeros past the slice
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int rr = i * 4 + (lane >> 3), n = min(n0 + rr, p.n - 1);
                    cp16(ring_addr + uint32_t((st % kDepth) * kStageBytes + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4)),
                         p.values + int64_t(n) * (p.k >> 1) + (min(kk, p.k - 32) >> 1), bytes);
                }
            }
            cp_commit();
        };
        // Scales (and mins) of rows g and g + 8, 32-weight groups 2 c and 2 c + 1 of a stage.
        const int64_t ga = int64_t(min(n0 + g, p.n - 1)) * groups, gb = int64_t(min(n0 + g + 8, p.n - 1)) * groups;
        struct Scales {
            __half2 a, b, ma, mb;
        };
        auto load_scales = [&](int st) {
            Scales s;
            const __half2 zero = __half2half2(__ushort_as_half(0));
            s.a = s.b = s.ma = s.mb = zero;
            if (st >= mine) return s;
            const int kk = k0 + st * kStageK + c * 64;
            const int i0 = kk >> gshift, i1 = (kk + 32) >> gshift;
            const bool in0 = kk < k1, in1 = kk + 32 < k1;
            const __half z = __ushort_as_half(0);
            s.a = __halves2half2(in0 ? p.scales[ga + i0] : z, in1 ? p.scales[ga + i1] : z);
            s.b = __halves2half2(in0 ? p.scales[gb + i0] : z, in1 ? p.scales[gb + i1] : z);
            if (kMins) {
                s.ma = __halves2half2(in0 ? p.mins[ga + i0] : z, in1 ? p.mins[ga + i1] : z);
                s.mb = __halves2half2(in0 ? p.mins[gb + i0] : z, in1 ? p.mins[gb + i1] : z);
            }
            return s;
        };
        float acc[NB][4];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[b][i] = 0.f;

        for (int st = 0; st < kDepth - 1; st++) copy(st);
        Scales cur = load_scales(0), nxt = load_scales(1);
        load_x(0);
        store_x(0);
        __syncthreads();
        for (int ch = 0; ch < chunks; ch++) {
            if (ch + 1 < chunks) load_x(ch + 1);
            const uint8_t* xb = smem + C::kOffX + (ch & 1) * C::kXBytes + g * C::kXRow + (sp * kcs + c * 8) * 2;
            const float* sums = reinterpret_cast<const float*>(smem + C::kOffSum) + (ch & 1) * C::kSums + sp * kcs / 32;
            for (int q = 0; q < chunk_stages; q++) {
                const int st = ch * chunk_stages + q;
                if (st >= mine) break;
                const Scales later = load_scales(st + 2);
                cp_wait<kDepth - 2>();
                __syncwarp();
                copy(st + kDepth - 1);
                const uint8_t* w = ring + (st % kDepth) * kStageBytes + g * 128 + c * 4;
#pragma unroll
                for (int j = 0; j < kStageK / 32; j++) {
                    const uint32_t ua = *reinterpret_cast<const uint32_t*>(w + ((j ^ g) << 4));
                    const uint32_t ub = *reinterpret_cast<const uint32_t*>(w + 1024 + ((j ^ g) << 4));
                    uint32_t ta[4], tb[4];
                    if constexpr (std::is_same<T, __half>::value) {
                        widen_f16<!kMins>(ua, ta);
                        widen_f16<!kMins>(ub, tb);
                    } else {
                        widen_bf16<!kMins>(ua, ta);
                        widen_bf16<!kMins>(ub, tb);
                    }
                    const int src = (lane & 28) | (j >> 1);
                    auto pick = [&](const __half2& h) {
                        const __half2 v = __shfl_sync(0xffffffffu, h, src);
                        return (j & 1) ? __high2float(v) : __low2float(v);
                    };
                    const float sa = pick(cur.a), sb = pick(cur.b);
                    const float ma = kMins ? pick(cur.ma) : 0.f, mb = kMins ? pick(cur.mb) : 0.f;
                    const uint32_t a0[4] = {ta[0], tb[0], ta[1], tb[1]}, a1[4] = {ta[2], tb[2], ta[3], tb[3]};
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint4 xv = make_uint4(0u, 0u, 0u, 0u);
                        if (b * 8 + g < p.rows)
                            xv = *reinterpret_cast<const uint4*>(xb + b * 8 * C::kXRow + (q * kStageK + j * 32) * 2);
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816<T>(d, a0, xv.x, xv.y);
                        mma16816<T>(d, a1, xv.z, xv.w);
                        acc[b][0] = fmaf(sa, d[0], acc[b][0]);
                        acc[b][1] = fmaf(sa, d[1], acc[b][1]);
                        acc[b][2] = fmaf(sb, d[2], acc[b][2]);
                        acc[b][3] = fmaf(sb, d[3], acc[b][3]);
                        if (kMins) {
                            const int r0 = b * 8 + 2 * c, at = q * (kStageK / 32) + j;
                            const float x0 = r0 < p.rows ? sums[r0 * (C::KC / 32) + at] : 0.f;
                            const float x1 = r0 + 1 < p.rows ? sums[(r0 + 1) * (C::KC / 32) + at] : 0.f;
                            acc[b][0] = fmaf(ma, x0, acc[b][0]);
                            acc[b][1] = fmaf(ma, x1, acc[b][1]);
                            acc[b][2] = fmaf(mb, x0, acc[b][2]);
                            acc[b][3] = fmaf(mb, x1, acc[b][3]);
                        }
                    }
                }
                cur = nxt;
                nxt = later;
            }
            if (ch + 1 < chunks) store_x(ch + 1);
            __syncthreads();
        }
        cp_wait<0>();
        __syncwarp();
        // Sums of the k slices, in order, through the ring (every stage has been read).
        float4* red = reinterpret_cast<float4*>(smem);
        if (p.S > 1) {
            __syncthreads();
            if (works && sp > 0)
#pragma unroll
                for (int b = 0; b < NB; b++) red[(warp * NB + b) * 32 + lane] = make_float4(acc[b][0], acc[b][1], acc[b][2], acc[b][3]);
            __syncthreads();
            if (works && sp == 0)
                for (int s = 1; s < p.S; s++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float4 v = red[((s * p.R + rt) * NB + b) * 32 + lane];
                        acc[b][0] += v.x, acc[b][1] += v.y, acc[b][2] += v.z, acc[b][3] += v.w;
                    }
        }
        if (works && sp == 0) {
            T* out = static_cast<T*>(p.out);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = n0 + g + (i >> 1) * 8, r = b * 8 + 2 * c + (i & 1);
                    if (n < p.n && r < p.rows) out[r * p.out_stride + n] = T(acc[b][i]);
                }
        }
        __syncthreads();  // the next tiles' copies and x reuse the memory read above
    }
}

template <typename T, int NB, bool kMins>
cudaError_t launch_t(const Q4Launch& a, cudaStream_t stream) {
    using C = Q4Cfg<NB>;
    cudaError_t e = cudaFuncSetAttribute(k_linear_q4<T, NB, kMins>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    Q4Params p{a.x, a.x_stride, a.rows, a.n, a.k, a.group, a.values, a.scales, a.mins, a.out, a.out_stride, 0, 0, 0, 0};
    p.tiles = (a.n + 15) / 16;
    const int grid = std::min(p.tiles, a.num_sms);
    p.R = std::min(kWarps, (p.tiles + grid - 1) / grid);
    const int stages = (a.k + kStageK - 1) / kStageK;
    p.S = std::max(1, std::min(std::min(kWarps / p.R, C::kMaxSplit), stages));
    p.Ks = (stages + p.S - 1) / p.S * kStageK;
    return launch_pdl(k_linear_q4<T, NB, kMins>, unsigned(grid), kThreads, size_t(C::kSmem), stream, 1, p);
}

template <typename T, int NB>
cudaError_t launch_m(const Q4Launch& a, cudaStream_t stream) {
    return a.mins ? launch_t<T, NB, true>(a, stream) : launch_t<T, NB, false>(a, stream);
}

template <typename T>
cudaError_t launch_e(const Q4Launch& a, cudaStream_t stream) {
    if (a.rows <= 8) return launch_m<T, 1>(a, stream);
    if (a.rows <= 16) return launch_m<T, 2>(a, stream);
    if (a.rows <= 32) return launch_m<T, 4>(a, stream);
    return launch_m<T, 8>(a, stream);
}

}  // namespace

cudaError_t launch_linear_q4(const Q4Launch& a, cudaStream_t stream) {
    return a.bf16 ? launch_e<__nv_bfloat16>(a, stream) : launch_e<__half>(a, stream);
}

}  // namespace ge
