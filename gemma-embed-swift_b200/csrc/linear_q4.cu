// linear_q4.cu -- ge_linear_q4: products of a few rows with 4-bit weights and group scales,
// out[r][n] = sum_k x[r][k] w[n][k].
//
// Bound by reading the weights once, so they stream from memory to shared memory (cp.async, a ring of
// its own per warp, no barrier in the way) and are widened on the fly to 16-bit integers, which are
// exact, for the warp's 16 x 8 x 16 tensor products with fp32 sums (a warp's product costs fewer
// issue slots than one multiply-add per weight and row, and a 128-row tcgen05 tile would be empty
// but for a few rows).  Every group's integer sums are scaled in fp32: acc += scale * sum, plus
// min * (sum of x) with minima, so no weight is ever rounded; results that are not finite are summed again from the
// definition (from_definition).
//
// One CTA per SM, 16 warps.  A warp owns 16 output columns n (a row tile) or, where the CTA has fewer
// tiles than warps, a part of k of one; the parts' sums are joined in shared memory in order.
// Stage of a warp: 16 rows x 256 weights (16 x 128 bytes, chunk c of row r at c ^ (r & 7), so that the
// 32-bit reads of a fragment hit 32 banks).  The lane's word of a 32-weight group holds the group's
// elements 8 c .. 8 c + 7; their nibbles come out as pairs (0, 4), (1, 5), (2, 6), (3, 7), which x is
// stored to match: the products' k order is permuted the same on both sides.  A stage's scales and minima
// come along in its slot, by cp.async where k is a multiple of the stage and the planes start on 16 bytes; else by
// loads the warp waits for (below).
// x is staged for all warps in two buffers of kXElems elements (all of it where it fits, so that the
// warps never meet while they stream).
//
// What bounds it now: neither memory (2 to 3.5 of 6.6 TB/s) nor one pipe (12 rows: 44 % of the issue slots, 48 % of
// shared memory's, 23 % of the tensor products'), but a warp's dependent steps from a stage's arrival through widening,
// products and scaling, at four warps to a scheduler; for many rows also the chunks of x, whose ends the warps wait for
// together.  A CTA takes as many of its tiles at once as it has warps: fewer, with parts of k on more warps, were slower
// (16384 x 8192, 1 row: 7 tiles at once 21.4 us, 4 + 3 24.7, one by one 34.5; 28671 x 8192, 12 rows: 13 at once 64,
// 7 + 6 67, 5 + 5 + 3 76), and sharing a chunk's stages of all tiles out evenly, up to two tiles a warp, won nothing
// either (23.3 and 67).  Measured, weights from memory:
//   16384 x 8192, groups of 32, 1 row, fp16              22.0 us, 3.4 TB/s
//   16384 x 8224, the same, k no multiple of 256         32.0 us, 2.4 TB/s
//   28671 x 8192, groups of 128 with mins, 12 rows, bf16   63 us, 2.0 TB/s
//   28671 x 8320, the same, k no multiple of 256           71 us, 1.8 TB/s
//   41003 x 4096, groups of 32, 4 rows, fp16               33 us, 2.8 TB/s
//    2304 x 768, groups of 32, 1 row, fp16                3.1 us (a launch and one trip to memory)
//     768 x 1152, the same                                3.6 us
#include <algorithm>

#include "attention_rows.cuh"
#include "operators.hpp"

namespace ge {

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kStageK = 256;                   // weights of a row per stage
constexpr int kScaleRow = 16;                  // bytes of a row's scales (or mins) in a stage: up to 8 groups
constexpr int kWeightBytes = 16 * kStageK / 2; // 2 KB
constexpr int kStageBytes = kWeightBytes + 2 * 16 * kScaleRow;  // weights, scales, mins
constexpr int kDepth = 3;
constexpr int kXElems = 16384;                 // elements of x per buffer, all rows
constexpr int kOffX = kWarps * kDepth * kStageBytes;
constexpr int kRows = 32;                      // of a launch
constexpr int kXBytes = kXElems * 2 + kRows * 64;  // rows are 64 bytes over a multiple of 128 apart
constexpr int kOffSum = kOffX + 2 * kXBytes;            // sums of x per group and row, 8 NB rows apart
constexpr int kSumBytes = 4096;
constexpr int kSmem = kOffSum + 2 * kSumBytes;
static_assert(kSmem <= 227 * 1024, "shared memory");

struct Q4Params {
    const void* x;
    int64_t x_stride;
    int rows, n, k;
    const uint8_t* values;
    const __half *scales, *mins;
    void* out;
    int64_t out_stride;
    int tiles, R, kc;          // row tiles in all; tiles of a CTA at a time; k per x buffer
    int whole;                 // 1: k is a multiple of the stage; 2: and the scales are aligned to 16 bytes
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// (a & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
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
        const uint32_t a = and_or(v, 0x000f000fu, 0x64006400u), b = and_or(v, 0x00f000f0u, 0x64006400u);
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
        const uint32_t a = and_or(u >> (4 * i), 0x000f000fu, 0x43004300u);
        const __nv_bfloat162 h = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), off);
        t[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}

// d = a b (+ d), not volatile: the products of several groups may be interleaved.
template <typename T, bool kFirst>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float z = 0.f;
    if constexpr (std::is_same<T, __half>::value) {
        if constexpr (kFirst)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        if constexpr (kFirst)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The sum of a warp's results that are not finite, again from the definition, in 64 bits: an infinite x times a
// weight's two parts may be inf - inf, and the integer sums of bf16 values above 1e35 may pass fp32 where the scaled ones
// do not.  Bit 4 b + i of `bad` is the lane's acc[b][i].  What is finite needs none of this: it had finite terms only.
// Out of line, since next to no call takes it.  One infinity in one row of 12 of 28671 x 8192: 0.38 ms, without it 0.06;
// in each of 64 rows of 16384 x 4096 6.3 and 0.07.  Rows full of NaN (padding never written) end at their first
// elements: 64 of them 0.62 ms.
template <typename T, int NB, bool kMins, int kPer>
__device__ __noinline__ void from_definition(const Q4Params& p, int n0, uint32_t bad) {
    constexpr int gshift = kPer == 1 ? 5 : kPer == 2 ? 6 : 7;
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int bit = 0; bit < 4 * NB; bit++) {
        unsigned lanes = __ballot_sync(0xffffffffu, (bad >> bit) & 1u);
#pragma unroll 1
        while (lanes) {
            const int of = __ffs(lanes) - 1;
            lanes &= lanes - 1;
            const int n = n0 + (of >> 2) + ((bit >> 1) & 1) * 8, r = (bit >> 2) * 8 + 2 * (of & 3) + (bit & 1);
            const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
            const uint8_t* values = p.values + int64_t(n) * (p.k >> 1);
            const int64_t row = int64_t(n) * (p.k >> gshift);
            double sum = 0.0;
#pragma unroll 1
            for (int e0 = 0; e0 < p.k; e0 += 256) {
                const int e = e0 + lane * 8;
                if (e < p.k) {
                    const uint32_t q = *reinterpret_cast<const uint32_t*>(values + (e >> 1));
                    const uint4 xv = *reinterpret_cast<const uint4*>(x + e);
                    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
                    const double scale = double(__half2float(p.scales[row + (e >> gshift)]));
                    const double low = kMins ? double(__half2float(p.mins[row + (e >> gshift)])) : 0.0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float2 f = pair_to_float<T>(xw[j >> 1]);
                        const int v = int((q >> (4 * j)) & 15u);
                        // The weight is exact: 4 bits times 11, 40 places apart from the minimum at most.
                        const double w = kMins ? fma(scale, double(v), low) : scale * double(v - 8);
                        sum = fma(double(j & 1 ? f.y : f.x), w, sum);
                    }
                }
                if (__any_sync(0xffffffffu, isnan(sum))) break;  // so is the result: a row full of NaN ends here
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == of) static_cast<T*>(p.out)[r * p.out_stride + n] = T(sum);
        }
    }
}

// NB: tiles of 8 rows of x; kPer: 32-weight units of a group, summed by the products before they are scaled.
template <typename T, int NB, bool kMins, int kPer>
__global__ void __launch_bounds__(kThreads, 1) k_linear_q4(const __grid_constant__ Q4Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    // Warp w takes part w / R of tile w % R; the first tiles have a part more where 16 is no multiple of R.
    const int rt = warp % p.R, part = warp / p.R, parts = kWarps / p.R + (rt < kWarps % p.R ? 1 : 0);
    const int t_begin = int(int64_t(blockIdx.x) * p.tiles / gridDim.x), t_end = int(int64_t(blockIdx.x + 1) * p.tiles / gridDim.x);
    // k runs in chunks of an x buffer, a chunk's stages are shared out over the parts.
    const int stages = (p.k + kStageK - 1) / kStageK, chunk_stages = p.kc / kStageK, chunks = (stages + chunk_stages - 1) / chunk_stages;
    const auto part_of = [&](int ch, int& from, int& to) {
        const int lo = ch * chunk_stages, n = min(stages - lo, chunk_stages);
        from = lo + n * part / parts;
        to = lo + n * (part + 1) / parts;
    };
    constexpr int gshift = kPer == 1 ? 5 : kPer == 2 ? 6 : 7;
    const int groups = p.k >> gshift;
    const int x_row = p.kc * 2 + 64;  // bytes between x's rows in a buffer
    uint8_t* ring = smem + warp * kDepth * kStageBytes;
    const uint32_t ring_addr = smem_u32(ring);
    pdl_wait();
    pdl_launch();

    // x of chunk `i`: up to four 16-byte units per thread.
    constexpr int kUnits = kXElems / 8 / kThreads;
    const int units_row = p.kc / 8;
    uint4 xr[kUnits];
    int unit[kUnits];  // each unit's row (high half) and first element (low half)
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
        const int id = u * kThreads + threadIdx.x, r = id / units_row;
        unit[u] = r << 16 | (id - r * units_row) * 8;
    }
    auto load_x = [&](int i) {
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int r = unit[u] >> 16, kk = i * p.kc + (unit[u] & 0xffff);
            xr[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < p.rows && kk < p.k) xr[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + r * p.x_stride + kk);
        }
    };
    auto store_x = [&](int i) {
        uint8_t* buf = smem + kOffX + (i & 1) * kXBytes;
        float* sums = reinterpret_cast<float*>(smem + kOffSum + (i & 1) * kSumBytes);
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int r = unit[u] >> 16, e = unit[u] & 0xffff;
            const uint4 v = xr[u];
            if (kMins) {
                float s = 0.f;
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = pair_to_float<T>(w[j]);
                    s += f.x + f.y;
                }
#pragma unroll
                for (int o = 1; o < 4 * kPer; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (r < p.rows && (threadIdx.x & (4 * kPer - 1)) == 0) sums[(e >> gshift) * 8 * NB + r] = s;
            }
            if (r < p.rows) {
                uint4 o;  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
                o.x = __byte_perm(v.x, v.z, 0x5410);
                o.y = __byte_perm(v.x, v.z, 0x7632);
                o.z = __byte_perm(v.y, v.w, 0x5410);
                o.w = __byte_perm(v.y, v.w, 0x7632);
                *reinterpret_cast<uint4*>(buf + r * x_row + e * 2) = o;
            }
        }
    };
    // Rows past the last repeat it: their products are not stored.
    int xrow[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) xrow[b] = min(b * 8 + g, p.rows - 1) * x_row + c * 16;

    for (int base = t_begin; base < t_end; base += p.R) {
        const bool works = base + rt < t_end;
        const int n0 = (base + rt) * 16;
        // The stages copied so far: the next one, the end of its chunk's part and the chunk.
        int cs = 0, ce = 0, cch = -1;
        const auto settle = [&]() {  // past empty parts; cch == chunks: nothing is left
            while (cs >= ce && ++cch < chunks) part_of(cch, cs, ce);
        };
        if (works) settle();
        else cch = chunks;
        // The four 16-byte chunks of a stage this lane copies: rows 4 i + lane / 8, chunk lane % 8 (swizzled, it
        // differs by 4 between odd and even i); the pointers move on by a stage with every copy.
        const uint8_t* src[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            src[i] = p.values + int64_t(min(n0 + i * 4 + (lane >> 3), p.n - 1)) * (p.k >> 1) + (lane & 7) * 16;
        const uint32_t dst = ring_addr + uint32_t((lane >> 3) * 128), c0 = uint32_t(((lane & 7) ^ (lane >> 3)) << 4), c1 = c0 ^ 64u;
        // Scales by lanes 0-15, mins by lanes 16-31, a row each.
        const __half* ssrc = (lane < 16 || !kMins ? p.scales : p.mins) + int64_t(min(n0 + (lane & 15), p.n - 1)) * groups;
        const uint32_t sdst = ring_addr + uint32_t(kWeightBytes + lane * kScaleRow);
        auto copy = [&](int at) {  // the next stage in turn, into the slot at byte `at` of the ring
            if (cch < chunks) {
                const int off = cs * (kStageK / 2);
                if (p.whole) {  // k is a multiple of the stage
#pragma unroll
                    for (int i = 0; i < 4; i++) cp16(dst + uint32_t(at + i * 512) + (i & 1 ? c1 : c0), src[i] + off, 16u);
                } else {
                    const bool in = cs * kStageK + (lane & 7) * 32 < p.k;  // zeros past k
#pragma unroll
                    for (int i = 0; i < 4; i++) cp16(dst + uint32_t(at + i * 512) + (i & 1 ? c1 : c0), in ? src[i] + off : p.values, in ? 16u : 0u);
                }
                if (kMins || lane < 16) {
                    const __half* from = ssrc + ((cs * kStageK) >> gshift);
                    if (p.whole == 2) {  // and the scales' rows are aligned: a row of the stage's at once
                        cp_small<16 / kPer>(sdst + uint32_t(at), from);
                    } else {
                        __half* out = reinterpret_cast<__half*>(ring + at + kWeightBytes + lane * kScaleRow);
                        for (int i = 0; i < (kStageK >> gshift); i++)
                            out[i] = cs * kStageK + (i << gshift) < p.k ? from[i] : __ushort_as_half(0);
                    }
                }
                cs++;
                settle();
            }
            cp_commit();
        };
        float acc[NB][4];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[b][i] = 0.f;

        for (int i = 0; i < kDepth - 1; i++) copy(i * kStageBytes);
        int slot = 0;  // of the stage in turn, in bytes
        load_x(0);
        store_x(0);
        __syncthreads();
        for (int ch = 0; ch < chunks; ch++) {
            if (ch + 1 < chunks) load_x(ch + 1);
            const uint8_t* xb = smem + kOffX + (ch & 1) * kXBytes;
            const float* sums = reinterpret_cast<const float*>(smem + kOffSum + (ch & 1) * kSumBytes) + 2 * c;
            int from = 0, to = 0;
            if (works) part_of(ch, from, to);
            for (int st = from; st < to; st++) {
                const int q = st - ch * chunk_stages;
                cp_wait<kDepth - 2>();
                __syncwarp();
                copy(slot == 0 ? (kDepth - 1) * kStageBytes : slot - kStageBytes);
                // Group j's words lie at w ^ 16 j (row g, chunk j ^ g) and 1 KB on (row g + 8).
                const int w = warp * kDepth * kStageBytes + slot + g * 128 + (g << 4) + c * 4;
                const uint8_t* scr = ring + slot + kWeightBytes + g * kScaleRow;
                slot = slot == (kDepth - 1) * kStageBytes ? 0 : slot + kStageBytes;
                // A row's scales of the stage's 8 / kPer groups, two to a word.
                const auto scales = [&](int off, uint32_t (&v)[4]) {
                    const uint4 u = *reinterpret_cast<const uint4*>(scr + off);
                    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
                };
                const auto pick = [](const uint32_t (&v)[4], int j) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[j >> 1]));
                    return j & 1 ? f.y : f.x;
                };
                uint32_t sav[4], sbv[4], mav[4], mbv[4];
                scales(0, sav);
                scales(8 * kScaleRow, sbv);
                if (kMins) {
                    scales(16 * kScaleRow, mav);
                    scales(24 * kScaleRow, mbv);
                }
                const uint8_t* const xq = xb + q * kStageK * 2;
#pragma unroll
                for (int j = 0; j < kStageK / 32 / kPer; j++) {
                    float d[NB][4];
#pragma unroll
                    for (int u = 0; u < kPer; u++) {
                        const int at = (j * kPer + u) << 4;
                        const uint32_t ua = *reinterpret_cast<const uint32_t*>(smem + (w ^ at));
                        const uint32_t ub = *reinterpret_cast<const uint32_t*>(smem + (w ^ at) + 1024);
                        uint32_t ta[4], tb[4];
                        if constexpr (std::is_same<T, __half>::value) {
                            widen_f16<!kMins>(ua, ta);
                            widen_f16<!kMins>(ub, tb);
                        } else {
                            widen_bf16<!kMins>(ua, ta);
                            widen_bf16<!kMins>(ub, tb);
                        }
                        const uint32_t a0[4] = {ta[0], tb[0], ta[1], tb[1]}, a1[4] = {ta[2], tb[2], ta[3], tb[3]};
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const uint4 xv = *reinterpret_cast<const uint4*>(xq + xrow[b] + (j * kPer + u) * 64);
                            if (u == 0) mma16816<T, true>(d[b], a0, xv.x, xv.y);
                            else mma16816<T, false>(d[b], a0, xv.x, xv.y);
                            mma16816<T, false>(d[b], a1, xv.z, xv.w);
                        }
                    }
                    const float sa = pick(sav, j), sb = pick(sbv, j);
                    const float ma = kMins ? pick(mav, j) : 0.f, mb = kMins ? pick(mbv, j) : 0.f;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        acc[b][0] = fmaf(sa, d[b][0], acc[b][0]);
                        acc[b][1] = fmaf(sa, d[b][1], acc[b][1]);
                        acc[b][2] = fmaf(sb, d[b][2], acc[b][2]);
                        acc[b][3] = fmaf(sb, d[b][3], acc[b][3]);
                        if (kMins) {
                            // Sums of rows 8 b + 2 c and the next (what lies there past the last row is not stored).
                            const float2 xs = *reinterpret_cast<const float2*>(sums + (q * (kStageK / 32 / kPer) + j) * 8 * NB + b * 8);
                            acc[b][0] = fmaf(ma, xs.x, acc[b][0]);
                            acc[b][1] = fmaf(ma, xs.y, acc[b][1]);
                            acc[b][2] = fmaf(mb, xs.x, acc[b][2]);
                            acc[b][3] = fmaf(mb, xs.y, acc[b][3]);
                        }
                    }
                }
            }
            if (ch + 1 < chunks) store_x(ch + 1);
            __syncthreads();
        }
        cp_wait<0>();
        __syncwarp();
        // Sums of the parts, in order, through the ring (every stage has been read).
        float4* red = reinterpret_cast<float4*>(smem);
        if (p.R < kWarps) {
            if (works && part > 0)
#pragma unroll
                for (int b = 0; b < NB; b++) red[(warp * NB + b) * 32 + lane] = make_float4(acc[b][0], acc[b][1], acc[b][2], acc[b][3]);
            __syncthreads();
            if (works && part == 0)
                for (int i = 1; i < parts; i++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float4 v = red[((i * p.R + rt) * NB + b) * 32 + lane];
                        acc[b][0] += v.x, acc[b][1] += v.y, acc[b][2] += v.z, acc[b][3] += v.w;
                    }
        }
        if (works && part == 0) {
            T* out = static_cast<T*>(p.out);
            uint32_t bad = 0;  // results that are not finite
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = n0 + g + (i >> 1) * 8, r = b * 8 + 2 * c + (i & 1);
                    if (n < p.n && r < p.rows) {
                        out[r * p.out_stride + n] = T(acc[b][i]);
                        if (!isfinite(acc[b][i])) bad |= 1u << (4 * b + i);
                    }
                }
            if (__any_sync(0xffffffffu, bad != 0)) from_definition<T, NB, kMins, kPer>(p, n0, bad);
        }
        __syncthreads();  // the next tiles' copies and x reuse the memory read above
    }
}

template <typename T, int NB, bool kMins, int kPer>
cudaError_t launch_t(const Q4Launch& a, cudaStream_t stream) {
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = allow_smem(k_linear_q4<T, NB, kMins, kPer>, kSmem, devices);
    if (e != cudaSuccess) return e;
    Q4Params p{a.x, a.x_stride, a.rows, a.n, a.k, a.values, a.scales, a.mins, a.out, a.out_stride, 0, 0, 0, 0};
    p.tiles = (a.n + 15) / 16;
    const int grid = std::min(p.tiles, a.num_sms);
    p.R = std::min(kWarps, (p.tiles + grid - 1) / grid);
    const int stages = (a.k + kStageK - 1) / kStageK;
    int per_buffer = kXElems / a.rows / kStageK;  // stages of all rows in an x buffer
    if (kMins) per_buffer = std::min(per_buffer, kSumBytes / (4 * 8 * NB * (kStageK / 32 / kPer)));
    p.kc = std::min(per_buffer, stages) * kStageK;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.scales) | reinterpret_cast<uintptr_t>(a.mins);
    p.whole = a.k % kStageK ? 0 : at % 16 ? 1 : 2;
    return launch_pdl(k_linear_q4<T, NB, kMins, kPer>, unsigned(grid), kThreads, size_t(kSmem), stream, 1, p);
}

template <typename T, int NB, bool kMins>
cudaError_t launch_g(const Q4Launch& a, cudaStream_t stream) {
    if (a.group == 32) return launch_t<T, NB, kMins, 1>(a, stream);
    if (a.group == 64) return launch_t<T, NB, kMins, 2>(a, stream);
    return launch_t<T, NB, kMins, 4>(a, stream);
}

template <typename T, int NB>
cudaError_t launch_m(const Q4Launch& a, cudaStream_t stream) {
    return a.mins ? launch_g<T, NB, true>(a, stream) : launch_g<T, NB, false>(a, stream);
}

template <typename T>
cudaError_t launch_e(const Q4Launch& a, cudaStream_t stream) {
    if (a.rows <= 8) return launch_m<T, 1>(a, stream);
    if (a.rows <= 16) return launch_m<T, 2>(a, stream);
    if (a.rows <= kRows) return launch_m<T, 4>(a, stream);
    // More rows in two halves, each over all weights (the second from the L2 cache where they fit): sums of 64 rows
    // spill into local memory in earnest (those of 32 store 32 to 52 bytes a thread, next to nothing), and their x leaves
    // room for one stage at a time, which only one part of k works on (16384 x 4096, groups of 64 with mins, bf16, 64
    // rows: 115 us at once, 72 in halves; 33 rows of groups of 32: 78 and 45).
    Q4Launch half = a;
    half.rows = (a.rows + 1) / 2;
    cudaError_t e = launch_e<T>(half, stream);
    if (e != cudaSuccess) return e;
    half.x = static_cast<const T*>(a.x) + half.rows * a.x_stride;
    half.out = static_cast<T*>(a.out) + half.rows * a.out_stride;
    half.rows = a.rows - half.rows;
    return launch_e<T>(half, stream);
}

}  // namespace

cudaError_t launch_linear_q4(const Q4Launch& a, cudaStream_t stream) {
    return a.bf16 ? launch_e<__nv_bfloat16>(a, stream) : launch_e<__half>(a, stream);
}

}  // namespace ge
