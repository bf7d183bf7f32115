// attention_causal.cu -- ge_attention_causal and ge_attention_prefix: attention of query rows over a
// shared prefix and over their own sequences' keys up to their own place, on the tensor cores.
//
// Every query row r reduces to a pair of key ranges: the prefix rows [0, P), the same for every row,
// and its own key rows [lo(r), hi(r)):
//   query i of n in a sequence whose own keys are rows [s, s + m):  hi = s + m - n + i + 1 (cut to
//   [s, s + m]), lo = s, or max(s, hi - window) under a window.
// A causal prompt is the case P = 0, m = n.  With that, sequences need no tiles of their own: a tile is
// T = 128 / G consecutive query rows (G = heads / KV heads) with all G heads that read one KV head, row
// t * G + g of its 128, whatever sequences its rows belong to.  Short texts fill a tile together, and
// the prefix' tiles serve the rows of many sequences at once.
//
// Kernels, each waiting for the one before (programmatic dependent launch):
//   k_rows_*        only for more than kPlanSeqs sequences: (lo, hi) of every row ahead of the plan
//   k_causal_plan   (lo, hi) per row where a tile mixes sequences, per item (below) the disjoint key segments its
//                   rows see, and the list of work pieces.  A warp plans an item; one CTA up to 64 items, which
//                   hand their results on through shared memory, else a cluster of 4 or 8.  Items that fill the
//                   SMs more than once go costliest first (a counting sort); fewer are cut into pieces of their key
//                   blocks that fill the SMs once, unless there are few keys.  Bound by latency: 5 us for 8
//                   queries, 10 us for 64 documents (300 items), 17 us for 50,000 tokens of one KV head of 256
//                   (1240 items); sorting by all CTAs of the cluster won 2 us at 1100 items and lost 1 at 300.
//   k_causal_tc     persistent, one CTA per SM: walks the pieces in turn (below)
//   k_causal_merge  only where tiles may be cut: joins the pieces' partial rows by their maxima and sums, a CTA per
//                   row and head; bound by latency (5 to 7 us).
// The result of a row depends only on its own ranges and, through the pieces, on the call's sizes:
// which CTA takes a piece changes nothing.
//
// k_causal_tc.  A work item is NT = 2 neighbouring tiles (head dims 64, 128; NT = 1 for 256, whose O
// takes half of tensor memory), one KV head and a run of key blocks of 128, each K and V tile serving
// both tiles' products.  Per tile x and block j: S = Q K^T (128 x 128, fp32 in tensor memory); a warpgroup
// per tile, one thread per row, turns S into P = 2^(S scale log2e - m) in 16 bits, written over S; O += P V
// (fp32 in tensor memory).  One warp issues every product, in the order PV_0(j - 1), S_0(j), PV_1(j - 1),
// S_1(j), so that one tile's softmax runs under the other tile's products; head dim 256 has two S
// buffers instead and runs S(j) ahead of PV(j - 1).  The running maximum of a row is moved (and its O
// rescaled) only when it grows by more than 2^8; until then every term of the row shares the old one, so
// the result is exact and P stays within 2^8 (2^15 as fp16 holds it, kRaise).  P in 16 bits is the operand the product takes; sums are
// taken over the unrounded fp32 values.
//   warp 0   TMA producer of Q and K      warp 1   MMA issuer
//   warp 2   TMA producer of V            warp 3   owns tensor memory
//   warps 4-7 (and 8-11 for tile 1)       softmax, then O / l to the output (or the partial rows)
// K and V blocks come in boxes of 32 rows, so a short segment loads few rows it does not need; rows of
// the V block past its last key, up to the product's step of 16, are zeroed, so whatever lies behind a
// segment never meets the product.  Keys masked for some rows of a tile only (later tokens, other
// sequences) do meet it, with P = 0: where their values are infinite or NaN, 0 x V leaves NaN in rows that
// must not see it, and the epilogue recomputes rows with non-finite outputs from the definition
// (attention_rows.cuh), which reads a row's own keys only, as it does rows with scores past kFar.
//
// What bounds it: on long sequences the softmax beside the products (of a tile's block, about 1350 cycles for a warp
// that has the scheduler to itself, for 1090 of the tensor core); on texts of a few hundred tokens the turn from one
// item to the next (Q's load, the first softmax and the epilogue have nothing beside them).  Measured:
//   2 x 4096 tokens, 32 heads of 128 on 8      0.243 ms, 1131 TFLOP/s
//   4 x 8000 tokens, 32 heads of 128 on 8       2.04 ms, 1028 TFLOP/s (runs long enough for the power limit's clock)
//   4 x 4096 tokens, 4 heads of 256 on 2       0.122 ms, 1131 TFLOP/s
//   2 x 8192 tokens, 12 heads of 64            0.282 ms,  731 TFLOP/s (a 64 wide S costs half the product, the
//                                              same softmax)
//   64 x 300 tokens, 32 heads of 128 on 8      0.125 ms,  379 TFLOP/s; 394 MB of tensors, 3.1 TB/s
#include <stdlib.h>

#include <algorithm>

#include "attention_rows.cuh"
#include "operators.hpp"

namespace ge {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.0f;  // log2 units a row's maximum may grow before it is moved
// Row maxima (log2 units) from which on a row is recomputed: scores times scale are rounded there to steps that an
// exponent feels (1/8; from 2^23 on 1, where 2^(S scale - m) of the largest key itself would be 0 or infinite).
constexpr float kFar = 1048576.0f;
constexpr int kKeys = 128;     // keys of a block
// Probabilities are held times 2^kRaise: fp16's smallest numbers then stand for probabilities of 2^-31, not 2^-24,
// so that many small ones beside a large one keep their sum (P stays within 2^(kGrow + 7), below fp16's largest).
template <typename E>
constexpr float kRaise = 0.f;
template <>
constexpr float kRaise<__half> = 7.f;
constexpr int kMaxPieces = 128;
constexpr int kBuckets = 1024;
constexpr int kMaxSms = 256;  // room for a cut call's items (fewer than SMs)

// ------------------------------------------------------------------------------------ sizes
constexpr int tiles_per_item(int hd) { return hd == 256 ? 1 : 2; }

struct Sizes {
    int group, T, TI, tiles, lmax;  // TI = rows of an item
};
Sizes sizes_of(const CausalLaunch& a) {
    Sizes s;
    s.group = a.heads / a.kv_heads;
    s.T = 128 / s.group;
    s.TI = s.T * tiles_per_item(a.hd);
    s.tiles = (a.ntok + s.TI - 1) / s.TI;
    // Pieces an item may be cut into: enough to fill the SMs twice (the plan fills them once), one where the items
    // do so already.
    const int64_t units = std::max<int64_t>(int64_t(s.tiles) * a.kv_heads, 1);
    // Calls over few keys are not cut: a block costs about 2 us, the merge's launch and run 6.
    s.lmax = units >= a.num_sms || int64_t(a.prefix) + a.nkv <= 4 * kKeys ? 1 : int(std::min<int64_t>(kMaxPieces, (2 * a.num_sms + units - 1) / units));
    return s;
}

struct Header {
    int err;    // a wait that gave up
    int nwork;  // pieces in the work list
};
// An item: NT neighbouring tiles.
struct alignas(16) TileInfo {
    int nblk, nseg, pieces, live;  // key blocks, own-key segments, pieces; bit x: tile x has rows of a sequence
    int lo0, hi0, lo1, hi1;        // per tile the hull of its rows' own keys
    // Items inside one sequence (simple): row i sees [ks, ke) up to key see + i, as own_range has it; the
    // others' rows have theirs in rng.
    int simple, see, ks, ke;
    int pos, end, spare[2];        // the first own-key segment
};
// A piece of an item, all that the main kernel's roles need of it but further segments and mixed rows.
struct alignas(16) Work {
    int tile, b0, b1, piece;     // blocks [b0, b1) of the item; piece -1: the whole item, straight to the output
    int seg, nseg, pos, end;     // where b0's own keys start, and that segment's end
    int lo0, hi0, lo1, hi1;
    int flags, see, ks, ke;      // flags: live, and 4 for simple
};

struct Layout {
    Header* head;
    int2 *rng, *segs;
    TileInfo* info;
    Work* work;
    float* o;    // [piece][row][head][hd]
    float2* ml;  // [piece][row][head]: maximum (log2 units), sum
    size_t bytes;
};
Layout layout_of(const CausalLaunch& a, const Sizes& s) {
    Layout l;
    size_t at = 0;
    const auto take = [&](size_t n) {
        char* p = static_cast<char*>(a.workspace) + at;
        at += (n + 255) / 256 * 256;
        return p;
    };
    l.head = reinterpret_cast<Header*>(take(sizeof(Header)));
    l.rng = reinterpret_cast<int2*>(take(size_t(a.ntok) * sizeof(int2)));
    l.segs = reinterpret_cast<int2*>(take(size_t(s.tiles) * s.TI * sizeof(int2)));
    l.info = reinterpret_cast<TileInfo*>(take(size_t(s.tiles) * sizeof(TileInfo)));
    // With pieces, (pieces of all tiles) x (KV heads) stays within the SMs (k_causal_plan).
    l.work = reinterpret_cast<Work*>(take(size_t(std::max(s.tiles, s.lmax > 1 ? a.num_sms : 0)) * sizeof(Work)));
    const size_t part = s.lmax > 1 ? size_t(s.lmax) * a.ntok * a.heads : 0;
    l.ml = reinterpret_cast<float2*>(take(part * sizeof(float2)));
    l.o = reinterpret_cast<float*>(take(part * a.hd * sizeof(float)));
    l.bytes = at;
    return l;
}

// ------------------------------------------------------------------------------------ plan
struct PlanParams {
    const uint32_t* q_seqs;
    const uint32_t* kv_seqs;
    int nseq, ntok, nkv, window, T, TI, tiles, kv_heads, prefix_blocks, lmax, sms;
    bool by_rows;  // rng is there already (k_rows_range)
    Header* head;
    int2 *rng, *segs;
    TileInfo* info;
    Work* work;
};

__device__ __forceinline__ int warp_max_i(int v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_min_i(int v) { return __reduce_min_sync(0xffffffffu, v); }

// The own keys of a row that may see keys below `see` of the range [ks, ke).
__device__ __forceinline__ int2 own_range(int see, int ks, int ke, int window) {
    const int hi = max(ks, min(see, ke));
    const int lo = window > 0 ? min(hi, max(ks, see - window)) : ks;
    return make_int2(lo, hi);
}

// A sequence's rows [q0, q1) and keys [ks, ke), cut to the tensors; row q0 + i sees keys below see + i.
struct Seq {
    int q0, q1, ks, ke, see;
};
__device__ __forceinline__ Seq seq_of(const PlanParams& p, int s) {
    const int64_t q = p.q_seqs[2 * s], n = p.q_seqs[2 * s + 1], k = p.kv_seqs[2 * s], m = p.kv_seqs[2 * s + 1];
    Seq r;
    r.q0 = int(min(q, int64_t(p.ntok)));
    r.q1 = int(min(q + n, int64_t(p.ntok)));
    r.ks = int(min(k, int64_t(p.nkv)));
    r.ke = int(min(k + m, int64_t(p.nkv)));
    // Rows and keys stay below 2^30, so a clamped value decides every row the same way.
    r.see = int(max(int64_t(-(1 << 30)), min(k + m - n + 1, int64_t(1 << 30))));
    return r;
}

// Up to kPlanSeqs sequences are kept in shared memory, where every item looks through them all.  Texts of 20 tokens, 4
// heads of 64 / 32 of 128: 600 of them 23.5 / 68 us so and 27 / 72 by rows (below); 1000 29 / 112 and 31 / 104; 2000
// 68 / 232 and 44 / 187; 4000 167 / 538 and 71 / 354.
constexpr int kPlanSeqs = 1024, kMaxItemRows = 256, kPlanItems = 64;  // items planned by one CTA
struct Seqs {
    int4* range;  // q0, q1, ks, ke
    int* see;
};
constexpr size_t plan_smem(int kept) {
    return size_t((kept + 3) / 4 * 4) * (sizeof(int4) + sizeof(int)) + 32 * 2 * kMaxItemRows * sizeof(int2);
}
__device__ __forceinline__ Seq seq_at(const Seqs& seqs, int s) {
    const int4 r = seqs.range[s];
    return Seq{r.x, r.y, r.z, r.w, seqs.see[s]};
}
// Rows sequence s has among [r0, r1), as offsets from r0: [x, y), empty unless x < y.
__device__ __forceinline__ int2 rows_within(const PlanParams& p, const Seqs& seqs, int s, int r0, int r1) {
    const int2 q = s < p.nseq ? *reinterpret_cast<const int2*>(&seqs.range[s]) : make_int2(0, 0);
    return make_int2(max(q.x, r0) - r0, min(q.y, r1) - r0);
}

// The disjoint ascending segments of n ranges whose lo never falls (empty ones aside), into seg, which may be
// the ranges' own memory; false where a lo falls.
__device__ bool find_segments(const PlanParams& p, const int2* ranges, int2* seg, int n, int lane, int& nseg) {
    int end = -1, low = -1;  // running maximum of hi and lo over the ranges so far
    nseg = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const int2 rg = i < n ? ranges[i] : make_int2(0, -1);
        const bool some = rg.y > rg.x;
        // Inclusive running maxima over the lanes, then those of the ranges before each lane's.
        int e = some ? rg.y : -1, l = some ? rg.x : -1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int pe = __shfl_up_sync(0xffffffffu, e, o), pl = __shfl_up_sync(0xffffffffu, l, o);
            if (lane >= o) {
                e = max(e, pe);
                l = max(l, pl);
            }
        }
        int be = __shfl_up_sync(0xffffffffu, e, 1), bl = __shfl_up_sync(0xffffffffu, l, 1);
        be = lane ? max(be, end) : end;
        bl = lane ? max(bl, low) : low;
        if (__any_sync(0xffffffffu, some && rg.x < bl)) return false;
        const bool fresh = some && rg.x > be;  // keys between be and lo are no row's
        const unsigned fm = __ballot_sync(0xffffffffu, fresh);
        if (fresh) {
            const int at = nseg + __popc(fm & ((1u << lane) - 1));
            seg[at].x = rg.x;
            if (at > 0) seg[at - 1].y = be;
        }
        nseg += __popc(fm);
        end = max(end, __shfl_sync(0xffffffffu, e, 31));
        low = max(low, __shfl_sync(0xffffffffu, l, 31));
        __syncwarp();
    }
    if (nseg > 0 && lane == 0) seg[nseg - 1].y = end;
    __syncwarp();
    return true;
}

// The n ranges of rng in ascending order of lo, empty ones last, into the kMaxItemRows places of seg (a bitonic
// sort by the warp).
__device__ void sort_ranges(const int2* rng, int2* seg, int n, int lane) {
#pragma unroll 1
    for (int i = lane; i < kMaxItemRows; i += 32) {
        const int2 rg = i < n ? rng[i] : make_int2(0, -1);
        seg[i] = rg.y > rg.x ? rg : make_int2(INT_MAX, INT_MAX);
    }
    __syncwarp();
#pragma unroll 1
    for (int size = 2; size <= kMaxItemRows; size *= 2)
#pragma unroll 1
        for (int step = size / 2; step > 0; step /= 2) {
#pragma unroll 1
            for (int t = lane; t < kMaxItemRows / 2; t += 32) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const int2 a = seg[i], b = seg[j];
                if ((a.x > b.x) == ((i & size) == 0)) seg[i] = b, seg[j] = a;
            }
            __syncwarp();
        }
}

// More sequences: the rows' ranges are written to rng before the plan, so that the time is that of the rows and
// sequences, not of the product of items and sequences (4 heads of 64: 10,000 texts of 20 tokens 0.15 ms, 100,000 of
// them 1.4, a million of 2 tokens 1.1; looking through all of them took 1.36 ms for 10,000 and 100 times that for
// each ten times more).  Every sequence s adds (1, s + 1) where it starts and takes
// it away where it ends, in 64 bits; the sum up to a row then holds how many sequences have it and, where that is
// one, which.  Rows of several are left out like rows of none.  Sums of whole numbers: the atomics' order is free.
constexpr int kRowBlock = 1024;  // rows of a CTA
__device__ __forceinline__ uint64_t* row_marks(const PlanParams& p) { return reinterpret_cast<uint64_t*>(p.rng); }
__device__ __forceinline__ uint64_t* block_sums(const PlanParams& p) { return reinterpret_cast<uint64_t*>(p.segs); }

__global__ void __launch_bounds__(256) k_rows_clear(PlanParams p) {
    pdl_wait();
    pdl_launch();
    for (int row = int(blockIdx.x) * 256 + int(threadIdx.x); row < p.ntok; row += int(gridDim.x) * 256) row_marks(p)[row] = 0;
}

__global__ void __launch_bounds__(256) k_rows_mark(PlanParams p) {
    pdl_wait();
    pdl_launch();
    unsigned long long* marks = reinterpret_cast<unsigned long long*>(row_marks(p));
    for (int s = int(blockIdx.x) * 256 + int(threadIdx.x); s < p.nseq; s += int(gridDim.x) * 256) {
        const Seq q = seq_of(p, s);
        if (q.q0 >= q.q1) continue;
        const unsigned long long one = (1ull << 32) + uint32_t(s + 1);
        atomicAdd(&marks[q.q0], one);
        if (q.q1 < p.ntok) atomicAdd(&marks[q.q1], 0ull - one);
    }
}

// The exclusive sum of v over the CTA's 32 W threads, and in `all` the whole.
template <int W>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t& all) {
    __shared__ uint64_t warps[W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warps[warp] = inc;
    __syncthreads();
    uint64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w < warp) before += warps[w];
        all += warps[w];
    }
    __syncthreads();
    return before + inc - v;
}

__device__ __forceinline__ void load_marks(const PlanParams& p, int row, uint64_t (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = row + i < p.ntok ? row_marks(p)[row + i] : 0;
}

__global__ void __launch_bounds__(256) k_rows_sum(PlanParams p) {
    pdl_wait();
    pdl_launch();
    uint64_t v[4], all;
    load_marks(p, int(blockIdx.x) * kRowBlock + int(threadIdx.x) * 4, v);
    block_scan<8>(v[0] + v[1] + v[2] + v[3], all);
    if (threadIdx.x == 0) block_sums(p)[blockIdx.x] = all;
}

__global__ void __launch_bounds__(1024) k_rows_scan(PlanParams p) {
    pdl_wait();
    pdl_launch();
    const int blocks = (p.ntok + kRowBlock - 1) / kRowBlock;
    uint64_t carry = 0, all;
    for (int b0 = 0; b0 < blocks; b0 += 1024) {
        const int b = b0 + int(threadIdx.x);
        const uint64_t at = carry + block_scan<32>(b < blocks ? block_sums(p)[b] : 0, all);
        if (b < blocks) block_sums(p)[b] = at;
        carry += all;
    }
}

__global__ void __launch_bounds__(256) k_rows_range(PlanParams p) {
    pdl_wait();
    pdl_launch();
    const int row = int(blockIdx.x) * kRowBlock + int(threadIdx.x) * 4;
    uint64_t v[4], all;
    load_marks(p, row, v);
    uint64_t at = block_sums(p)[blockIdx.x] + block_scan<8>(v[0] + v[1] + v[2] + v[3], all);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        at += v[i];
        if (row + i >= p.ntok) break;
        int2 rg = make_int2(0, -1);
        if (at >> 32 == 1) {
            const Seq q = seq_of(p, int(uint32_t(at)) - 1);
            rg = own_range(q.see + (row + i - q.q0), q.ks, q.ke, p.window);
        }
        p.rng[row + i] = rg;
    }
}

// One item, by one warp: rng and seg are the warp's own shared memory.  Its segments and (mixed) rows go to the
// workspace.
__device__ TileInfo plan_item(const PlanParams& p, const Seqs& seqs, int2* rng, int2* seg, int t, int lane) {
    const int r0 = t * p.TI, n = min(p.TI, p.ntok - r0);
    TileInfo f{};
    bool any = false;
    const int scan = p.by_rows ? 0 : p.nseq;
    if (p.by_rows) {
#pragma unroll 1
        for (int i = lane; i < p.TI; i += 32) {
            rng[i] = i < n ? p.rng[r0 + i] : make_int2(0, -1);
            any |= rng[i].y >= 0;
        }
        __syncwarp();
    }
#pragma unroll 1
    for (int s0 = 0; s0 < scan; s0 += 32) {
        const int2 in = rows_within(p, seqs, s0 + lane, r0, r0 + n);
        any |= in.x < in.y;
        const unsigned whole = __ballot_sync(0xffffffffu, in.x == 0 && in.y == n);
        if (whole) {  // the item lies inside one sequence
            const Seq q = seq_at(seqs, s0 + __ffs(whole) - 1);
            const int see = q.see + (r0 - q.q0), n0 = min(p.T, n);
            const int2 a = own_range(see, q.ks, q.ke, p.window), b = own_range(see + n0 - 1, q.ks, q.ke, p.window);
            const int2 e = own_range(see + n - 1, q.ks, q.ke, p.window);
            f.live = n > n0 ? 3 : 1;
            f.lo0 = a.x, f.hi0 = b.y;
            f.lo1 = f.live == 3 ? own_range(see + n0, q.ks, q.ke, p.window).x : INT_MAX;
            f.hi1 = f.live == 3 ? e.y : 0;
            f.nseg = e.y > a.x ? 1 : 0;
            f.nblk = p.prefix_blocks + (e.y - a.x + kKeys - 1) / kKeys;
            f.simple = 1, f.see = see, f.ks = q.ks, f.ke = q.ke;
            f.pieces = 1;
            f.pos = a.x, f.end = e.y;
            return f;
        }
    }
    if (!__any_sync(0xffffffffu, any)) return f;  // live 0: no row of a sequence, no work
#pragma unroll 1
    for (int i = p.by_rows ? p.TI : lane; i < p.TI; i += 32) rng[i] = make_int2(0, -1);
    __syncwarp();
#pragma unroll 1
    for (int s0 = 0; s0 < scan; s0 += 32) {
        const int2 in = rows_within(p, seqs, s0 + lane, r0, r0 + n);
        unsigned m = __ballot_sync(0xffffffffu, in.x < in.y);
        if (__popc(m) > 4) {  // many short ones: a lane each
            if (in.x < in.y) {
                const Seq q = seq_at(seqs, s0 + lane);
#pragma unroll 1
                for (int i = in.x; i < in.y; i++) rng[i] = own_range(q.see + (r0 + i - q.q0), q.ks, q.ke, p.window);
            }
        } else {
#pragma unroll 1
            while (m) {
                const int src = __ffs(m) - 1;
                m &= m - 1;
                const Seq q = seq_at(seqs, s0 + src);
                const int x = __shfl_sync(0xffffffffu, in.x, src), y = __shfl_sync(0xffffffffu, in.y, src);
#pragma unroll 1
                for (int i = x + lane; i < y; i += 32) rng[i] = own_range(q.see + (r0 + i - q.q0), q.ks, q.ke, p.window);
            }
        }
        __syncwarp();
    }
    // Tiles with rows, and the hulls of their keys.
    int lo_x[2] = {INT_MAX, INT_MAX}, hi_x[2] = {0, 0};
#pragma unroll 1
    for (int i0 = 0; i0 < p.TI; i0 += 32) {
        const int i = i0 + lane;
        const int2 rg = i < n ? rng[i] : make_int2(0, -1);
        const bool in = rg.y >= 0, x = i >= p.T;
        if (__any_sync(0xffffffffu, in && !x)) f.live |= 1;
        if (__any_sync(0xffffffffu, in && x)) f.live |= 2;
        if (rg.y > rg.x) {  // per lane, reduced once behind the loop
            lo_x[0] = min(lo_x[0], x ? INT_MAX : rg.x), hi_x[0] = max(hi_x[0], x ? 0 : rg.y);
            lo_x[1] = min(lo_x[1], x ? rg.x : INT_MAX), hi_x[1] = max(hi_x[1], x ? rg.y : 0);
        }
    }
    // The rows' own keys as disjoint ascending segments, by one pass over the ranges in ascending order (lo
    // never falls): as the rows have them, or, where a row's lo falls, sorted into seg first.
    if (!find_segments(p, rng, seg, n, lane, f.nseg)) {
        sort_ranges(rng, seg, n, lane);
        find_segments(p, seg, seg, kMaxItemRows, lane, f.nseg);
    }
    f.lo0 = warp_min_i(lo_x[0]), f.hi0 = warp_max_i(hi_x[0]);
    f.lo1 = warp_min_i(lo_x[1]), f.hi1 = warp_max_i(hi_x[1]);
    int nblk = 0;
#pragma unroll 1
    for (int i = lane; i < f.nseg; i += 32) {
        nblk += (seg[i].y - seg[i].x + kKeys - 1) / kKeys;
        p.segs[int64_t(t) * p.TI + i] = seg[i];
    }
#pragma unroll 1
    for (int i = p.by_rows ? n : lane; i < n; i += 32) p.rng[r0 + i] = rng[i];
    if (f.nseg > 0) f.pos = seg[0].x, f.end = seg[0].y;
    f.nblk = __reduce_add_sync(0xffffffffu, nblk) + p.prefix_blocks;
    f.pieces = 1;
    __syncwarp();
    return f;
}

// One cluster: the items by the warps of all its CTAs, then their pieces and order by the first CTA.
__global__ void __launch_bounds__(1024) k_causal_plan(PlanParams p) {
    extern __shared__ __align__(16) uint8_t plan_shared[];
    __shared__ int hist[kBuckets], warp_sum_s[32], s_nblk[kMaxSms], s_at[kMaxSms], s_chunk;
    __shared__ TileInfo s_info[kPlanItems];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = int(gridDim.x);
    const int kept = p.by_rows ? 0 : p.nseq, room = (kept + 3) / 4 * 4;
    const Seqs seqs{reinterpret_cast<int4*>(plan_shared), reinterpret_cast<int*>(plan_shared + size_t(room) * sizeof(int4))};
    int2* rng = reinterpret_cast<int2*>(seqs.see + room) + warp * 2 * kMaxItemRows;
    hist[tid] = 0;
    if (tid == 0) s_chunk = INT_MAX;
    pdl_wait();
    pdl_launch();
#pragma unroll 1
    for (int s = tid; s < kept; s += 1024) {
        const Seq r = seq_of(p, s);
        seqs.range[s] = make_int4(r.q0, r.q1, r.ks, r.ke);
        seqs.see[s] = r.see;
    }
    if (blockIdx.x == 0 && tid == 0) p.head->err = 0;
    __syncthreads();
    // A single CTA keeps the items' infos at hand; a cluster's come back through global memory.
    const TileInfo* info = ctas == 1 ? s_info : p.info;
#pragma unroll 1
    for (int t = int(blockIdx.x) + warp * ctas; t < p.tiles; t += ctas * 32) {
        const TileInfo f = plan_item(p, seqs, rng, rng + kMaxItemRows, t, lane);
        if (lane == 0) {
            p.info[t] = f;
            if (ctas == 1) s_info[t] = f;
        }
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    if (blockIdx.x != 0) return;
    const auto whole = [&](int t, const TileInfo& f) {
        return Work{t, 0, f.nblk, -1, 0, f.nseg, f.pos, f.end, f.lo0, f.hi0, f.lo1, f.hi1, f.live | (f.simple << 2), f.see, f.ks, f.ke};
    };
    if (int64_t(p.tiles) * p.kv_heads > p.sms) {
        // Several rounds of the SMs: whole items, costliest first, by a counting sort over their blocks; the order
        // within a bucket does not matter.  The lanes of a bucket add as one.
        const auto add = [&](int bucket, bool one) {  // counts into the bucket; gives the count before
            const unsigned peers = __match_any_sync(0xffffffffu, bucket), ones = __ballot_sync(0xffffffffu, one) & peers;
            const int leader = __ffs(peers) - 1, at = lane == leader ? atomicAdd(&hist[bucket], __popc(ones)) : 0;
            return __shfl_sync(0xffffffffu, at, leader) + __popc(ones & ((1u << lane) - 1));
        };
#pragma unroll 1
        for (int t0 = warp * 32; t0 < p.tiles; t0 += 1024) {
            const int t = t0 + lane;
            const int4 f = t < p.tiles ? *reinterpret_cast<const int4*>(info + t) : make_int4(0, 0, 0, 0);  // nblk, nseg, pieces, live
            add(min(f.x, kBuckets - 1), f.w != 0);
        }
        __syncthreads();
        // Exclusive sums from the costliest bucket down: thread i holds bucket kBuckets - 1 - i.
        const int v = hist[kBuckets - 1 - tid];
        int inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_sum_s[warp] = inc;
        __syncthreads();
        const int u = lane < warp ? warp_sum_s[lane] : 0;
        const int before = __reduce_add_sync(0xffffffffu, u);
        hist[kBuckets - 1 - tid] = before + inc - v;
        if (tid == 1023) p.head->nwork = before + inc;
        __syncthreads();
#pragma unroll 1
        for (int t0 = warp * 32; t0 < p.tiles; t0 += 1024) {
            const int t = t0 + lane;
            TileInfo f{};
            if (t < p.tiles) f = info[t];
            const int at = add(min(f.nblk, kBuckets - 1), f.live != 0);
            if (f.live) p.work[at] = whole(t, f);
        }
        return;
    }
    // One round of the SMs (fewer items than SMs): items in order, cut into pieces where that is allowed.
    int chunk = INT_MAX;
    if (tid < p.tiles) s_nblk[tid] = info[tid].nblk;
    __syncthreads();
    if (p.lmax > 1) {
        // Blocks per piece: the fewest for which the pieces of all items and KV heads still fit one round (a
        // second, short round would cost as much as the first).  Every warp tries a size.
        int most = 1;
#pragma unroll 1
        for (int t = lane; t < p.tiles; t += 32) most = max(most, s_nblk[t]);
        most = warp_max_i(most);
#pragma unroll 1
        for (int c0 = max(1, (most + p.lmax - 1) / p.lmax); chunk == INT_MAX; c0 += 32) {
            const int c = min(c0 + warp, most);  // `most`, one piece per item, always fits
            int n = 0;
#pragma unroll 1
            for (int t = lane; t < p.tiles; t += 32) n += max(1, (s_nblk[t] + c - 1) / c);
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0 && (c == most || int64_t(n) * p.kv_heads <= p.sms)) atomicMin(&s_chunk, c);
            __syncthreads();
            chunk = s_chunk;
            __syncthreads();
        }
    }
    const auto pieces_of = [&](int nblk, int& sz) {
        const int want = chunk == INT_MAX ? 1 : max(1, (nblk + chunk - 1) / chunk);
        sz = (nblk + want - 1) / want;
        return sz ? (nblk + sz - 1) / sz : 1;  // the last piece may come out empty, and is dropped
    };
    if (warp == 0) {  // where each item's pieces start in the list
        int base = 0;
#pragma unroll 1
        for (int t0 = 0; t0 < p.tiles; t0 += 32) {
            const int t = t0 + lane;
            int sz, n = t < p.tiles && info[t].live ? pieces_of(s_nblk[t], sz) : 0, inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int w = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += w;
            }
            if (t < p.tiles) s_at[t] = base + inc - n;
            base += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) p.head->nwork = base;
    }
    __syncthreads();
#pragma unroll 1
    for (int t = warp; t < p.tiles; t += 32) {  // a lane per piece
        const TileInfo f = info[t];
        if (!f.live) continue;
        const int at = s_at[t];
        int sz;
        const int n = pieces_of(f.nblk, sz);
        if (n == 1) {
            if (lane == 0) p.work[at] = whole(t, f);
            continue;
        }
        if (lane == 0) p.info[t].pieces = n;
        const int2* seg = p.segs + int64_t(t) * p.TI;
#pragma unroll 1
        for (int i = lane; i < n; i += 32) {
            const int b0 = i * sz, b1 = min(f.nblk, b0 + sz);
            int s = 0, first = p.prefix_blocks;  // segment s starts at block `first`
            int2 g = make_int2(0, 0);
            if (f.nseg > 0) {
                g = make_int2(f.pos, f.end);
#pragma unroll 1
                for (; s + 1 < f.nseg; s++, g = seg[s]) {
                    const int m = (g.y - g.x + kKeys - 1) / kKeys;
                    if (b0 < first + m) break;
                    first += m;
                }
                g.x += max(0, b0 - first) * kKeys;
            }
            p.work[at + i] = Work{t, b0, b1, i, s, f.nseg, g.x, g.y, f.lo0, f.hi0, f.lo1, f.hi1, f.live | (f.simple << 2), f.see, f.ks, f.ke};
        }
    }
}

// ------------------------------------------------------------------------------------ main kernel
template <int D>
struct Cfg {
    static constexpr int NT = tiles_per_item(D);
    static constexpr int DS = D < 128 ? D : 128;         // dims of a K or V stage
    static constexpr int DH = D / DS;                    // stages of a block
    static constexpr int QC = D / 64, SC = DS / 64;      // 64-dim chunks of [128 rows][128 bytes]
    static constexpr int ST = D == 64 ? 4 : 2;           // ring depth, K and V each
    static constexpr int kChunk = 128 * 128;
    static constexpr int kStage = SC * kChunk;
    static constexpr int kQ = NT * QC * kChunk;
    static constexpr int kOffK = kQ, kOffV = kOffK + ST * kStage, kOffOut = kOffV + ST * kStage;
    static constexpr bool kBoxes = D == 128;             // outputs leave as boxes where they can
    static constexpr int kOutBuf = 32 * 64;              // 32 columns of a warp's rows on their way out, two per warp
    static constexpr int kOffBar = kOffOut + (kBoxes ? NT * 4 * 2 * kOutBuf : 0);
    static constexpr int kSmem = kOffBar + 512 + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static constexpr int kThreads = 128 + 128 * NT;
    static constexpr uint32_t kTmemS = 256;              // O in [0, 256), S and P in [256, 512)
};

struct TcParams {
    const void *q, *k, *v, *pk, *pv;
    void* out;
    int64_t q_stride, k_stride, v_stride, pk_stride, pv_stride, out_stride;
    int heads, kv_heads, group, T, TI, ntok, window, prefix, prefix_blocks;
    bool out_wide;      // rows of out start on 32-byte boundaries
    bool out_boxes;     // a warp's 32 rows of a tile are a box of out
    uint32_t kv_magic;  // ceil(2^32 / kv_heads)
    float scale_log2e;
    int64_t wait_cycles;
    Header* head;
    const int2 *rng, *segs;
    const Work* work;
    float* o;
    float2* ml;
};

__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok));
    return ok != 0;
}

// A word with its n lowest bits set (0 below 0, all above 32).
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// Waits for the phase of parity `parity`, at most `limit` cycles: then the error is recorded and every role comes
// to its end, each within its own next wait.  Little code: the roles hold dozens of waits, and at an item's turn
// code that has left the instruction cache costs more than the work.
template <bool kSleep>
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, int* err, int64_t limit) {
    if (mbar_test(bar, parity)) return true;
    const int64_t t0 = clock64();
    do {
        if (clock64() - t0 >= limit) {
            *err = kErrTimeout;
            return false;
        }
        if (kSleep) __nanosleep(32);
    } while (!mbar_test(bar, parity));
    return true;
}
// The same by a whole warp, whose lanes agree.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err, int64_t limit) {
    if (__all_sync(0xffffffffu, mbar_poll(bar, parity))) return true;
    const int64_t t0 = clock64();
    do {
        if (__any_sync(0xffffffffu, clock64() - t0 >= limit)) {
            *err = kErrTimeout;
            return false;
        }
    } while (!__all_sync(0xffffffffu, mbar_test(bar, parity)));
    return true;
}
// kWaitLimitNs at 2 GHz, and more over many keys: a warp recomputes 32 rows over all of them at most, at about 0.1 us
// for a key of a row (8 heads of 128 wide, 8192 rows that all see an infinite value: 27 ms, 0.13 ms without it); 1 us
// is allowed.
// GE_ATTENTION_WAIT_NS in the environment of the process' first call stands in its place (0: whatever is not there
// at the first look has run out).
int64_t wait_limit(int64_t keys) {
    static const int64_t given = [] {
        const char* ns = getenv("GE_ATTENTION_WAIT_NS");
        return ns ? int64_t(std::max(0LL, std::min(atoll(ns), 1LL << 60))) : int64_t(-1);
    }();
    return 2 * (given >= 0 ? given : int64_t(kWaitLimitNs) + keys * 32 * 1000);
}
// 32 bytes at once, to a 32-byte boundary: a store touches a line for every lane's row, so half as many go out.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// Two fp32 operations at a time.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A piece of work as every role walks it.
struct Piece {
    int tile, kvh, b0, b1, piece, flags;
    int lo[2], hi[2];
    int seg, nseg, pos, end;
    int see, ks, ke;
    const int2* segs;
};
// A piece's words, asked for one piece ahead so that their way from memory is under the work before.
struct RawPiece {
    int4 a, b, c, d;
    int id;
};
// The piece of work item `id` (one per KV head): id / kv_heads, by a multiplication that is at most one off.
__device__ __forceinline__ int piece_index(const TcParams& p, int id) {
    if (p.kv_heads == 1) return id;
    const int q = int(__umulhi(uint32_t(id), p.kv_magic));
    return q * p.kv_heads > id ? q - 1 : q;
}
__device__ __forceinline__ RawPiece fetch_piece(const TcParams& p, int id, int total) {
    RawPiece r;
    r.id = id;
    r.a = r.b = r.c = r.d = make_int4(0, 0, 0, 0);
    if (id < total) {
        const int4* src = reinterpret_cast<const int4*>(p.work + piece_index(p, id));
        r.a = src[0], r.b = src[1], r.c = src[2], r.d = src[3];
    }
    return r;
}
__device__ __forceinline__ Piece piece_of(const TcParams& p, const RawPiece& r) {
    Piece s;
    s.kvh = r.id - piece_index(p, r.id) * p.kv_heads;
    s.tile = r.a.x, s.b0 = r.a.y, s.b1 = r.a.z, s.piece = r.a.w;
    s.seg = r.b.x, s.nseg = r.b.y, s.pos = r.b.z, s.end = r.b.w;
    s.lo[0] = r.c.x, s.hi[0] = r.c.y, s.lo[1] = r.c.z, s.hi[1] = r.c.w;
    s.flags = r.d.x, s.see = r.d.y, s.ks = r.d.z, s.ke = r.d.w;
    s.segs = p.segs + int64_t(r.a.x) * p.TI;
    return s;
}
// For the warps short of registers: the next piece's words into the L1 cache.
__device__ __forceinline__ void prefetch_piece(const TcParams& p, int id, int total) {
    if (id < total) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.work + piece_index(p, id)));
}
// Walks a piece's key blocks: prefix blocks, then blocks of the own-key segments.
struct Cursor {
    int b, seg, pos, end;
    bool prefix;
    int row, nv;  // the block's first row and its keys
    __device__ __forceinline__ void set(const TcParams& p) {
        prefix = b < p.prefix_blocks;
        row = prefix ? b * kKeys : pos;
        nv = min(kKeys, (prefix ? p.prefix : end) - row);
    }
    __device__ __forceinline__ Cursor(const TcParams& p, const Piece& s) {
        b = s.b0;
        seg = s.seg;
        pos = s.pos;
        end = s.end;
        set(p);
    }
    __device__ __forceinline__ void next(const TcParams& p, const Piece& s) {
        if (!prefix) {
            pos += kKeys;
            if (pos >= end && b + 1 < s.b1) {
                const int2 g = s.segs[++seg];
                pos = g.x;
                end = g.y;
            }
        }
        b++;
        set(p);
    }
    // Whether tile x has a row that may see a key of the block.
    __device__ __forceinline__ bool active(const Piece& s, int x) const {
        return prefix ? (s.flags >> x) & 1 : (row < s.hi[x] && row + nv > s.lo[x]);
    }
};
// Pieces are taken in turn, every second round backwards, so that the CTA with a round's costliest
// piece gets the next round's cheapest.
__device__ __forceinline__ int piece_id(int round) {
    const int g = int(gridDim.x), c = int(blockIdx.x);
    return round * g + ((round & 1) ? g - 1 - c : c);
}

__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = globaltimer();
    while (!mbar_test(bar, parity) && globaltimer() - t0 < kWaitLimitNs) {
    }
}

template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int M, int N, int b_mn);
template <>
__host__ __device__ constexpr uint32_t idesc_of<__half>(int M, int N, int b_mn) {
    return idesc_f16(M, N, 0, b_mn);
}
template <>
__host__ __device__ constexpr uint32_t idesc_of<__nv_bfloat16>(int M, int N, int b_mn) {
    return idesc_f16(M, N, 0, b_mn) | (1u << 7) | (1u << 10);  // A and B: bf16
}

// 1 / l for a row's sum l.  A finite score leaves a sum of 2^-8 and more, so l = 0 is a row that sees no key, whose
// result is 0, or keys whose scores are all -infinity, a softmax of 0 / 0.
__device__ __forceinline__ float inverse_sum(float l, bool sees) { return l != 0.f ? 1.0f / l : sees ? NAN : 0.f; }

// One row of piece `id` from the definition, by a whole warp; stored like the epilogue does.  It reads the
// piece again: one handed over would live in memory for all of the callers' work.
template <typename E, int D>
__device__ __forceinline__ void exact_row(const TcParams& p, int id, int row, int head, int2 rg) {
    const int lane = threadIdx.x & 31;
    const Piece s = piece_of(p, fetch_piece(p, id, id + 1));
    RowState<D> st;
    row_begin<E, D>(st, static_cast<const E*>(p.q) + row * p.q_stride + int64_t(head) * D, lane);
    const int64_t col = int64_t(s.kvh) * D;
    Cursor c(p, s);
    for (; c.b < s.b1; c.next(p, s)) {
        const int j0 = c.prefix ? c.row : max(c.row, rg.x), j1 = c.prefix ? c.row + c.nv : min(c.row + c.nv, rg.y);
        if (j0 >= j1) continue;
        const E* k = static_cast<const E*>(c.prefix ? p.pk : p.k) + j0 * (c.prefix ? p.pk_stride : p.k_stride) + col;
        const E* v = static_cast<const E*>(c.prefix ? p.pv : p.v) + j0 * (c.prefix ? p.pv_stride : p.v_stride) + col;
        row_keys<E, D>(st, k, v, c.prefix ? p.pk_stride : p.k_stride, c.prefix ? p.pv_stride : p.v_stride, j1 - j0,
                       p.scale_log2e, lane);
    }
    if (s.piece < 0) {
        const float inv = st.l != 0.f ? 1.0f : inverse_sum(0.f, p.prefix > 0 || rg.y > rg.x);
        uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<E*>(p.out) + row * p.out_stride + int64_t(head) * D + lane * (D / 32));
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] = float_to_pair<E>(st.o[2 * i] * inv, st.o[2 * i + 1] * inv);
    } else {
        const int64_t at = (int64_t(s.piece) * p.ntok + row) * p.heads + head;
        if (lane == 0) p.ml[at] = make_float2(st.m, -st.l);  // a negative sum: divided by it already
        float2* o = reinterpret_cast<float2*>(p.o + at * D + lane * (D / 32));
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] = make_float2(st.o[2 * i], st.o[2 * i + 1]);
    }
}

// Where a wait of a CTA's softmax warps ran out: the rows of all its pieces become NaN, so that what `out` held before
// cannot pass for a result.  By the softmax warps (others may not have the registers), a row a thread.  Rows done
// before go too: to know how far each warp came would hold registers throughout (200 bytes of spills).
template <typename E, int D>
__device__ __noinline__ void rows_lost(const TcParams& p) {
    const int i = int(threadIdx.x) - 128, x = i >> 7, r = i & 127, token = r / p.group, total = p.head->nwork * p.kv_heads;
#pragma unroll 1
    for (int round = 0; piece_id(round) < total; round++) {
        const Piece s = piece_of(p, fetch_piece(p, piece_id(round), total));
        const int row = s.tile * p.TI + x * p.T + token, head = s.kvh * p.group + (r - token * p.group);
        if (r >= p.group * p.T || row >= p.ntok || (!(s.flags & 4) && p.rng[row].y < 0)) continue;
        if (s.piece >= 0) {  // the merge makes the row of it
            p.ml[(int64_t(s.piece) * p.ntok + row) * p.heads + head] = make_float2(0.f, NAN);
            continue;
        }
        const uint32_t nan = float_to_pair<E>(NAN, NAN);
        uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(p.out) + row * p.out_stride + int64_t(head) * D);
#pragma unroll 1
        for (int c = 0; c < D / 8; c++) dst[c] = make_uint4(nan, nan, nan, nan);
    }
}

template <typename E, int D>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1)
    k_causal_tc(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                const __grid_constant__ CUtensorMap mapV, const __grid_constant__ CUtensorMap mapPK,
                const __grid_constant__ CUtensorMap mapPV, const __grid_constant__ CUtensorMap mapO,
                const __grid_constant__ TcParams p) {
    using C = Cfg<D>;
    constexpr int NT = C::NT, ST = C::ST, DH = C::DH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
    uint64_t *q_full = bars, *q_empty = bars + 1;
    uint64_t *k_full = bars + 2, *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
    uint64_t *s_full = v_empty + ST, *p_full = s_full + 2;  // per S buffer
    uint64_t *o_full = p_full + 2, *o_empty = o_full + 2;   // per tile
    uint64_t *pv_done = o_empty + 2, *idle = pv_done + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
    volatile uint32_t* lost = tmem_slot + 1;
    int* err = &p.head->err;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int live_rows = p.group * p.T;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < ST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], 4);
        }
        mbar_init(pv_done, 1);
        mbar_init(idle, 1);
        *lost = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch(&mapQ);
        tma_prefetch(&mapK);
        tma_prefetch(&mapV);
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    // Rows [live_rows, 128) of the Q chunks are never loaded: zeroed once, their scores stay finite.
    {
        const int dead = 128 - live_rows;
        for (int i = threadIdx.x; i < NT * C::QC * dead * 8; i += C::kThreads) {
            const int c = i / (dead * 8), rr = live_rows + (i / 8) % dead;
            *reinterpret_cast<uint4*>(smem + c * C::kChunk + rr * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch();
    const int total = p.head->nwork * p.kv_heads;

    if (warp < 4) {
        if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 0 || warp == 2) {
            // ---------------------------------------------------------- TMA producers (Q and K; V)
            if (lane == 0) {
                const bool keys = warp == 0;
                uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
                uint8_t* ring = smem + (keys ? C::kOffK : C::kOffV);
                const CUtensorMap* own = keys ? &mapK : &mapV;
                const CUtensorMap* shared = keys ? &mapPK : &mapPV;
                bool ok = true;
                int issued = 0, issued_q = 0;
                for (int round = 0, id; ok && (id = piece_id(round)) < total; round++) {
                    const Piece s = piece_of(p, fetch_piece(p, id, total));
                    prefetch_piece(p, piece_id(round + 1), total);
                    if (s.b0 >= s.b1) continue;
                    if (keys) {
                        if (!wait_on<true>(q_empty, uint32_t(issued_q & 1) ^ 1u, err, p.wait_cycles)) break;
                        mbar_expect_tx(q_full, uint32_t(NT * C::QC * 128 * live_rows));
#pragma unroll 1
                        for (int x = 0; x < NT; x++)
#pragma unroll 1
                            for (int c = 0; c < C::QC; c++)
                                tma_load_3d(smem + (x * C::QC + c) * C::kChunk, &mapQ, q_full, c * 64, s.kvh * p.group,
                                            s.tile * p.TI + x * p.T);
                        issued_q++;
                    }
                    for (Cursor c(p, s); ok && c.b < s.b1; c.next(p, s)) {
                        const int boxes = (c.nv + 31) / 32;
                        const CUtensorMap* map = c.prefix ? shared : own;
                        for (int h = 0; h < DH; h++) {
                            const int st = issued % ST;
                            if (!wait_on<true>(&empty[st], uint32_t((issued / ST) & 1) ^ 1u, err, p.wait_cycles)) {
                                ok = false;
                                break;
                            }
                            mbar_expect_tx(&full[st], uint32_t(boxes * C::SC * 4096));
#pragma unroll 1
                            for (int ch = 0; ch < C::SC; ch++)
#pragma unroll 1
                                for (int b = 0; b < boxes; b++)
                                    tma_load_2d(ring + st * C::kStage + ch * C::kChunk + b * 4096, map, &full[st],
                                                s.kvh * D + h * C::DS + ch * 64, c.row + b * 32);
                            issued++;
                        }
                    }
                }
                // Every issued load lands before the CTA exits, also after an error.
                if (issued_q > 0) drain(q_full, uint32_t((issued_q - 1) & 1));
#pragma unroll 1
                for (int st = 0; st < ST; st++) {
                    const int n = issued / ST + (st < issued % ST ? 1 : 0);
                    if (n > 0) drain(&full[st], uint32_t((n - 1) & 1));
                }
            }
        } else if (warp == 1) {
            // ---------------------------------------------------------- MMA issuer (the whole warp walks along)
            const uint32_t id_s = idesc_of<E>(128, kKeys, 0);      // K-major Q and K
            const uint32_t id_o = idesc_of<E>(128, C::DS, 1);      // P from tensor memory, MN-major V
            // Descriptors of the tiles' starts; others lie (bytes / 16) further.
            const uint64_t q_desc = sw128_desc(smem_u32(smem), 16, 1024), k_desc = sw128_desc(smem_u32(smem + C::kOffK), 16, 1024);
            const uint64_t v_desc = sw128_desc(smem_u32(smem + C::kOffV), C::kChunk, 1024);
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = wait_warp(bar, parity, err, p.wait_cycles);
                return ok;
            };
            int nq = 0, nk = 0, nv = 0;            // Q tiles, K stages and V stages used so far
            int ns[2] = {0, 0}, np[2] = {0, 0};    // S and PV products per S buffer (NT 2) or in all (NT 1, [0])
            int no[2] = {0, 0};                    // items with an O, per tile
            for (int round = 0, id; ok && (id = piece_id(round)) < total; round++) {
                const Piece s = piece_of(p, fetch_piece(p, id, total));
                prefetch_piece(p, piece_id(round + 1), total);
                if (s.b0 >= s.b1) continue;
                if (!wait(q_full, uint32_t(nq & 1))) break;
                nq++;
                tc_fence_after();
                Cursor c(p, s);
                int prev = 0, prev_nv = 0;  // the block before: the tiles it is active for, its keys
                int used = 0;               // tiles with an O in this item
                for (;;) {
                    const bool more = c.b < s.b1;
                    int act = 0;
                    if (more)
                        for (int x = 0; x < NT; x++) act |= NT == 1 || c.active(s, x) ? 1 << x : 0;
                    if constexpr (NT == 2) {
                        // This block's K and the block before's V first: once a tile's P has come, its PV and then its S
                        // (over the P just read) go out together, and the other tile's softmax runs under them.
                        const int ks = nk % ST, vs = nv % ST, steps = (prev_nv + 15) / 16;
                        if (more && !wait(&k_full[ks], uint32_t((nk / ST) & 1))) break;
                        if (prev_nv) {
                            if (!wait(&v_full[vs], uint32_t((nv / ST) & 1))) break;
                            if (prev_nv & 15) {
                                // Rows behind the block's last key, up to the product's step.
#pragma unroll 1
                                for (int i = lane; i < (steps * 16 - prev_nv) * C::SC * 8; i += 32) {
                                    const int rr = prev_nv + i / (C::SC * 8), ch = (i >> 3) % C::SC;
                                    *reinterpret_cast<uint4*>(smem + C::kOffV + vs * C::kStage + ch * C::kChunk + rr * 128 + (i & 7) * 16) =
                                        make_uint4(0u, 0u, 0u, 0u);
                                }
                                fence_proxy_async_smem();
                                __syncwarp();
                            }
                        }
                        const uint64_t kd = k_desc + uint32_t(__shfl_sync(0xffffffffu, ks, 0) * (C::kStage >> 4));
                        const uint64_t vd = v_desc + uint32_t(__shfl_sync(0xffffffffu, vs, 0) * (C::kStage >> 4));
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const bool pv = (prev >> x) & 1, sc = (act >> x) & 1;
                            const uint32_t begun = uint32_t(used >> x) & 1u;
                            if (pv) {
                                if (!begun && no[x] > 0 && !wait(&o_empty[x], uint32_t((no[x] - 1) & 1))) break;
                                if (!wait(&p_full[x], uint32_t(np[x] & 1))) break;
                                np[x]++;
                                if (!begun) no[x]++;
                                used |= 1 << x;
                            }
                            tc_fence_after();
                            const uint32_t od = tmem + uint32_t(x * D), sd = tmem + C::kTmemS + uint32_t(x * kKeys);
                            if (elect_one()) {
                                if (pv) {
                                    if (steps == 8) {
#pragma unroll
                                        for (int kk = 0; kk < 8; kk++)
                                            umma_f16_ta(od, sd + kk * 8, vd + uint32_t(kk * 128), id_o, kk ? 1u : begun);
                                    } else {
#pragma unroll 1
                                        for (int kk = 0; kk < steps; kk++)
                                            umma_f16_ta(od, sd + kk * 8, vd + uint32_t(kk * 128), id_o, kk ? 1u : begun);
                                    }
                                }
                                if (sc) {
#pragma unroll
                                    for (int kk = 0; kk < C::DS / 16; kk++)
                                        umma_f16(sd, q_desc + uint32_t(((x * C::QC + (kk >> 2)) * C::kChunk + (kk & 3) * 32) >> 4),
                                                 kd + uint32_t(((kk >> 2) * C::kChunk + (kk & 3) * 32) >> 4), id_s, kk != 0);
                                    umma_commit(&s_full[x]);
                                }
                                if (!more && (pv || begun)) umma_commit(&o_full[x]);
                                if (x == 1) {
                                    if (prev_nv) umma_commit(&v_empty[vs]);
                                    if (more) umma_commit(&k_empty[ks]);
                                }
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                        if (prev_nv) nv++;
                        if (more) nk++;
                    } else {
                        if (more) {
                            // S into the other of the two buffers, ahead of the block before's PV.
                            const int b = ns[0] & 1;
                            for (int h = 0; h < DH; h++) {
                                const int st = (nk + h) % ST;
                                if (!wait(&k_full[st], uint32_t(((nk + h) / ST) & 1))) break;
                                tc_fence_after();
                                const uint64_t kd = k_desc + uint32_t(__shfl_sync(0xffffffffu, st, 0) * (C::kStage >> 4));
                                const uint32_t sd = tmem + C::kTmemS + uint32_t(__shfl_sync(0xffffffffu, b, 0) * kKeys);
                                if (elect_one()) {
#pragma unroll
                                    for (int kk = 0; kk < C::DS / 16; kk++)
                                        umma_f16(sd, q_desc + uint32_t(((h * C::SC + (kk >> 2)) * C::kChunk + (kk & 3) * 32) >> 4),
                                                 kd + uint32_t(((kk >> 2) * C::kChunk + (kk & 3) * 32) >> 4), id_s, (h | kk) != 0);
                                    umma_commit(&k_empty[st]);
                                    if (h == DH - 1) umma_commit(&s_full[b]);
                                }
                                __syncwarp();
                            }
                            if (!ok) break;
                            ns[0]++;
                            nk += DH;
                        }
                        if (prev_nv) {
                            const int b = np[0] & 1, steps = (prev_nv + 15) / 16;
                            if (!used && no[0] > 0 && !wait(&o_empty[0], uint32_t((no[0] - 1) & 1))) break;
                            for (int h = 0; h < DH; h++) {
                                const int st = (nv + h) % ST;
                                if (!wait(&v_full[st], uint32_t(((nv + h) / ST) & 1))) break;
                                if (prev_nv & 15) {
#pragma unroll 1
                                    for (int i = lane; i < (steps * 16 - prev_nv) * C::SC * 8; i += 32) {
                                        const int rr = prev_nv + i / (C::SC * 8), ch = (i >> 3) % C::SC;
                                        *reinterpret_cast<uint4*>(smem + C::kOffV + st * C::kStage + ch * C::kChunk + rr * 128 + (i & 7) * 16) =
                                            make_uint4(0u, 0u, 0u, 0u);
                                    }
                                    fence_proxy_async_smem();
                                    __syncwarp();
                                }
                                if (h == 0 && !wait(&p_full[b], uint32_t((np[0] >> 1) & 1))) break;
                                tc_fence_after();
                                const uint64_t vd = v_desc + uint32_t(__shfl_sync(0xffffffffu, st, 0) * (C::kStage >> 4));
                                const uint32_t pd = tmem + C::kTmemS + uint32_t(__shfl_sync(0xffffffffu, b, 0) * kKeys), od = tmem + uint32_t(h * C::DS);
                                const uint32_t begun = uint32_t(used);
                                if (elect_one()) {
                                    if (steps == 8) {
#pragma unroll
                                        for (int kk = 0; kk < 8; kk++)
                                            umma_f16_ta(od, pd + kk * 8, vd + uint32_t(kk * 128), id_o, kk ? 1u : begun);
                                    } else {
#pragma unroll 1
                                        for (int kk = 0; kk < steps; kk++)
                                            umma_f16_ta(od, pd + kk * 8, vd + uint32_t(kk * 128), id_o, kk ? 1u : begun);
                                    }
                                    umma_commit(&v_empty[st]);
                                    if (h == DH - 1) {
                                        umma_commit(pv_done);
                                        if (!more) umma_commit(&o_full[0]);
                                    }
                                }
                                __syncwarp();
                            }
                            if (!ok) break;
                            np[0]++;
                            if (!used) no[0]++;
                            used = 1;
                            nv += DH;
                        }
                    }
                    if (!more) break;
                    prev = act;
                    prev_nv = c.nv;
                    c.next(p, s);
                    // Every S of the item has read Q.
                    if (c.b >= s.b1 && elect_one()) umma_commit(q_empty);
                    __syncwarp();
                }
            }
            // The products in flight end before the CTA gives its memory back.
            if (elect_one()) {
                umma_commit(idle);
                drain(idle, 0);
            }
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------- softmax and output, one thread per row
        if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int x = NT == 2 ? (warp - 4) >> 2 : 0;
        const int quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lane_base = tmem + (uint32_t(quad * 32) << 16);
        const int token = r / p.group;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            ok = wait_warp(bar, parity, err, p.wait_cycles);
            return ok;
        };
        int nb = 0, no = 0;  // blocks and items with an O so far
        int round = 0;
        RawPiece next = fetch_piece(p, piece_id(0), total);
        // The row of the piece in `next`, and its range where the plan wrote it.
        const auto row_of = [&]() { return next.a.x * p.TI + x * p.T + token; };
        const auto range_of = [&]() {
            const bool stored = next.id < total && r < live_rows && row_of() < p.ntok && !(next.d.x & 4);
            return stored ? p.rng[row_of()] : make_int2(0, -1);
        };
        int2 range = range_of();
        while (ok && next.id < total) {
            const Piece s = piece_of(p, next);
            const int id = next.id, row = row_of();
            int2 rg = range;
            if ((s.flags & 4) && r < live_rows && row < p.ntok) rg = own_range(s.see + (row - s.tile * p.TI), s.ks, s.ke, p.window);
            next = fetch_piece(p, piece_id(++round), total);
            // Rows of no query take every score: never stored.
            const bool in = rg.y >= 0;
            const int row_lo = in ? rg.x : 0, row_hi = in ? rg.y : INT_MAX;
            const int warp_lo = __reduce_max_sync(0xffffffffu, row_lo), warp_hi = __reduce_min_sync(0xffffffffu, row_hi);
            const int tile_lo = x ? s.lo[1] : s.lo[0], tile_hi = x ? s.hi[1] : s.hi[0];
            const bool tile_live = (s.flags >> x) & 1;
            float m = -INFINITY, l = 0.f;
            const int nb0 = nb;
            // Runs of blocks: the prefix' and each segment's (of this piece), those the tile has rows for.
            int b = s.b0, seg = s.seg, pos = s.pos, end = s.end;
            while (ok && b < s.b1) {
                const bool prefix = b < p.prefix_blocks;
                int key = prefix ? b * kKeys : pos, lim = prefix ? p.prefix : end;
                const int blocks = min(prefix ? p.prefix_blocks - b : (end - pos + kKeys - 1) / kKeys, s.b1 - b);
                lim = min(lim, key + blocks * kKeys);
                b += blocks;
                if (!prefix && b < s.b1) {
                    const int2 g = s.segs[++seg];
                    pos = g.x, end = g.y;
                }
                // A block is active where the issuers' test says so: key < tile_hi and its end > tile_lo.
                int stop = lim;
                if (NT == 2) {
                    if (prefix ? !tile_live : tile_lo >= lim) continue;
                    if (!prefix) {
                        if (tile_lo > key) key += (tile_lo - key) / kKeys * kKeys;
                        stop = min(lim, tile_hi);
                    }
                }
                // Blocks below `free` (and from warp_lo on) need no mask in this warp.
                const int free = prefix ? lim : min(lim, warp_hi), from = prefix ? 0 : warp_lo;
                for (; key < stop; key += kKeys, nb++) {
                    const int buf = NT == 2 ? x : nb & 1;
                    if (!wait(&s_full[buf], uint32_t((NT == 2 ? nb : nb >> 1) & 1))) break;
                    tc_fence_after();
                    const uint32_t scol = lane_base + C::kTmemS + uint32_t(buf * kKeys);
                    uint32_t sr[kKeys];
#pragma unroll
                    for (int i = 0; i < kKeys / 32; i++) tmem_ld32(scol + i * 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[i * 32]));
                    tmem_wait_ld();
                    if (key + kKeys > free || key < from) {
                        // Keys of the row among the block's (a later segment's may start within a block's
                        // length of this one's end).
                        const int lo = prefix ? 0 : row_lo - key, hi = (in ? prefix ? lim : min(row_hi, lim) : INT_MAX) - key;
#pragma unroll
                        for (int w = 0; w < kKeys / 32; w++) {  // bit i: key 32 w + i is the row's
                            const uint32_t bits = low_bits(hi - 32 * w) & ~low_bits(lo - 32 * w);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(bits & (1u << i))) sr[32 * w + i] = __float_as_uint(-INFINITY);
                        }
                    }
                    float mp[4];  // four independent chains of three-way maxima
#pragma unroll
                    for (int i = 0; i < 4; i++) mp[i] = max3(__uint_as_float(sr[3 * i]), __uint_as_float(sr[3 * i + 1]), __uint_as_float(sr[3 * i + 2]));
#pragma unroll
                    for (int i = 12; i < kKeys; i += 2)
                        mp[(i >> 1) & 3] = max3(mp[(i >> 1) & 3], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
                    const float mb = fmaxf(max3(mp[0], mp[1], mp[2]), mp[3]) * p.scale_log2e;
                    const bool grow = mb > m + kGrow;
                    if (__any_sync(0xffffffffu, grow)) {
                        // Also a row's first visible key: O and l are still 0 then (or not begun, in the item's first
                        // block).
                        const float alpha = m == -INFINITY || !grow ? 1.0f : ex2_approx(m - mb);
                        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
                            // O is complete up to the block before: S came behind that PV (of head dim 256: ahead).
                            if (NT == 1 && !wait(&pv_done[0], uint32_t((nb - 1) & 1))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int i = 0; i < D / 32; i++) {
                                uint32_t o[32];
                                tmem_ld32(lane_base + uint32_t(x * D + i * 32), o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                                tmem_st32(lane_base + uint32_t(x * D + i * 32), o);
                            }
                            l *= alpha;
                        }
                        if (grow) m = mb;
                    }
                    const float mu = m == -INFINITY ? 0.f : kRaise<E> - m;
                    const uint64_t scale2 = pack2(p.scale_log2e, p.scale_log2e), mu2 = pack2(mu, mu);
                    uint64_t ps[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int h = 0; h < kKeys / 64; h++) {
                        uint32_t pk[32];
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            float p0, p1;
                            unpack2(fma2(pack2(__uint_as_float(sr[h * 64 + 2 * e]), __uint_as_float(sr[h * 64 + 2 * e + 1])), scale2, mu2), p0, p1);
                            p0 = ex2_approx(p0), p1 = ex2_approx(p1);
                            ps[e & 3] = add2(ps[e & 3], pack2(p0, p1));
                            pk[e] = float_to_pair<E>(p0, p1);
                        }
                        tmem_st32(scol + h * 32, pk);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[buf]);
                    float l0, l1;
                    unpack2(add2(add2(ps[0], ps[1]), add2(ps[2], ps[3])), l0, l1);
                    l += l0 + l1;
                }
            }
            const int count = nb - nb0;
            if (!ok) break;
            // ---- output
            range = range_of();  // of the next piece
            const int head = s.kvh * p.group + (r - token * p.group);
            const int64_t at = (int64_t(s.piece) * p.ntok + row) * p.heads + head;  // of a partial row
            const float inv = s.piece >= 0 ? 1.0f : inverse_sum(l, p.prefix > 0 || rg.y > rg.x);
            if (in && s.piece >= 0) p.ml[at] = make_float2(m - kRaise<E>, l);
            bool bad = fabsf(m) >= kFar && m != -INFINITY;
            // Whole rows of head dim 128 leave as boxes through shared memory, where all of the warp's belong to a sequence:
            // the threads do not wait for the stores (64 texts of 300 tokens, 32 heads: 129 us, by stores 140).  Head dim
            // 64 gains nothing (88 us both ways), 256 loses with its four warps (148 us for 141).
            const bool box = C::kBoxes && p.out_boxes && s.piece < 0 && __all_sync(0xffffffffu, in || row >= p.ntok);
            if (count) {
                if (!wait(&o_full[x], uint32_t(no & 1))) break;
                no++;
                tc_fence_after();
            }
#pragma unroll 1
            for (int i = 0; i < D / 32; i++) {
                uint32_t o[32];
                if (count) {
                    tmem_ld32(lane_base + uint32_t(x * D + i * 32), o);
                    tmem_wait_ld();
                    if (i == D / 32 - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&o_empty[x]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0u;
                }
                float z = 0.f;
#pragma unroll
                for (int e = 0; e < 32; e++) z = fmaf(__uint_as_float(o[e]), 0.f, z);
                bad |= z != 0.f;  // NaN: a value is infinite or NaN
                if (box) {
                    uint8_t* buf = smem + C::kOffOut + ((warp - 4) * 2 + (i & 1)) * C::kOutBuf;
                    if (lane == 0) bulk_wait_read<1>();  // the copy before the last has left the buffer
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t w[4];
#pragma unroll
                        for (int f = 0; f < 4; f++)
                            w[f] = mean_to_pair<E>(__uint_as_float(o[8 * e + 2 * f]) * inv, __uint_as_float(o[8 * e + 2 * f + 1]) * inv);
                        *reinterpret_cast<uint4*>(buf + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && row < p.ntok) {
                        tma_store_3d(&mapO, buf, i * 32, head, row);
                        bulk_commit();
                    }
                } else if (in && s.piece < 0) {
                    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<E*>(p.out) + row * p.out_stride + int64_t(head) * D + i * 32);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t w[8];
#pragma unroll
                        for (int f = 0; f < 8; f++)
                            w[f] = mean_to_pair<E>(__uint_as_float(o[16 * e + 2 * f]) * inv, __uint_as_float(o[16 * e + 2 * f + 1]) * inv);
                        if (p.out_wide) {
                            store32(dst + 8 * e, w);
                        } else {
                            *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(dst + 8 * e + 4) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                } else if (in) {
                    float* dst = p.o + at * D + i * 32;
#pragma unroll
                    for (int e = 0; e < 4; e++) store32(dst + 8 * e, *reinterpret_cast<const uint32_t(*)[8]>(&o[8 * e]));
                }
                __syncwarp();
            }
            unsigned redo = __ballot_sync(0xffffffffu, in && bad);
            __syncwarp();
            while (redo) {
                const int src = __ffs(redo) - 1;
                redo &= redo - 1;
                if (C::kBoxes) bulk_wait_all();  // lane 0's copies of the rows are behind
                __syncwarp();
                const int2 g = make_int2(__shfl_sync(0xffffffffu, rg.x, src), __shfl_sync(0xffffffffu, rg.y, src));
                exact_row<E, D>(p, id, __shfl_sync(0xffffffffu, row, src), __shfl_sync(0xffffffffu, head, src), g);
            }
        }
        if (!ok) *lost = 1;
    }

    if (C::kBoxes && warp >= 4 && lane == 0) bulk_wait_all();
    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (warp >= 4 && *lost) rows_lost<E, D>(p);
}

// ------------------------------------------------------------------------------------ merge
struct MergeParams {
    void* out;
    int64_t out_stride;
    int heads, ntok, TI, lmax, prefix, window;
    const int2* rng;
    const TileInfo* info;
    const float* o;
    const float2* ml;
};

// One CTA of W warps per (row, head): out = sum_c 2^(m_c - m) O_c / sum_c 2^(m_c - m) l_c, m the
// largest m_c (O_c l_c in O_c's place for recomputed rows, which come divided, their sums negative).
// Thread c weighs piece c; the warps add every W-th piece each, joined in order.  The
// loads that say whether and how many pieces there are go out together with the pieces' maxima.
template <typename E, int D, int W>
__global__ void __launch_bounds__(32 * W) k_causal_merge(MergeParams p) {
    static_assert(32 * W >= kMaxPieces && 32 * W >= D / 2, "a thread per piece and per pair of columns");
    __shared__ float w[kMaxPieces], red_m[W], red_l[W], part[W][D];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch();
    const int row = int(blockIdx.x) / p.heads, head = int(blockIdx.x) - row * p.heads;
    const int64_t step = int64_t(p.ntok) * p.heads, id = int64_t(row) * p.heads + head;
    const TileInfo* f = p.info + row / p.TI;
    const int4 info = *reinterpret_cast<const int4*>(f);  // nblk, nseg, pieces, live
    const int simple = f->simple;
    const int2 rng = p.rng[row];
    float2 ml = tid < p.lmax ? p.ml[tid * step + id] : make_float2(-INFINITY, 0.f);
    const int n = info.z;
    if (n <= 1 || !info.w || (!simple && rng.y < 0)) return;
    if (tid >= n) ml = make_float2(-INFINITY, 0.f);
    const bool nan = __syncthreads_or(isnan(ml.y));  // of a piece: its row is NaN whatever its weight
    float m = warp_max(ml.x);
    if (lane == 0) red_m[warp] = m;
    __syncthreads();
    m = red_m[0];
#pragma unroll
    for (int i = 1; i < W; i++) m = fmaxf(m, red_m[i]);
    const float wt = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);  // 0: no visible key, and no row was left
    const float part_l = wt * fabsf(ml.y);
    // Of a recomputed row, which is a mean, and of a sum; -1: no score of the piece is finite, and its row is 0.  Any
    // other meets its weight, also one that is 0 beside a far larger one, and so does a recomputed row without a finite
    // score: 0 times an infinite value is NaN, in pieces as in one row.
    if (tid < n) w[tid] = signbit(ml.y) ? part_l : ml.x == -INFINITY ? -1.f : wt;
    const float l = warp_sum(part_l);
    if (lane == 0) red_l[warp] = l;
    __syncthreads();
    // Weights over the whole sum before they meet the pieces: no partial sum of means passes the largest value.
    float lt = 0.f;
#pragma unroll
    for (int i = 0; i < W; i++) lt += red_l[i];
    bool sees = p.prefix > 0;
    if (lt == 0.f && !sees) {
        const int2 own = simple ? own_range(f->see + (row - row / p.TI * p.TI), f->ks, f->ke, p.window) : rng;
        sees = own.y > own.x;
    }
    const float inv = nan ? NAN : inverse_sum(lt, sees);
    constexpr int P = D / 32;
    float acc[P];
#pragma unroll
    for (int i = 0; i < P; i++) acc[i] = 0.f;
#pragma unroll 4
    for (int c = warp; c < n; c += W) {
        const bool none = w[c] < 0.f;
        const float wc = (none ? 0.f : w[c]) * inv;
        const float2* src = reinterpret_cast<const float2*>(p.o + (c * step + id) * D + lane * P);
#pragma unroll
        for (int i = 0; i < P / 2; i++) {
            const float2 v = none ? make_float2(0.f, 0.f) : src[i];
            acc[2 * i] = fmaf(wc, v.x, acc[2 * i]);
            acc[2 * i + 1] = fmaf(wc, v.y, acc[2 * i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < P; i++) part[warp][lane * P + i] = acc[i];
    __syncthreads();
    if (tid < D / 2) {
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; i++) {
            v[0] += part[i][2 * tid];
            v[1] += part[i][2 * tid + 1];
        }
        uint32_t pair = mean_to_pair<E>(v[0], v[1]);
        const uint32_t plain = float_to_pair<E>(v[0], v[1]);  // of infinite values
        if (isinf(v[0])) pair = (pair & 0xffff0000u) | (plain & 0xffffu);
        if (isinf(v[1])) pair = (pair & 0xffffu) | (plain & 0xffff0000u);
        reinterpret_cast<uint32_t*>(static_cast<E*>(p.out) + row * p.out_stride + int64_t(head) * D)[tid] = pair;
    }
}

// ------------------------------------------------------------------------------------ launch
template <typename E, int D>
cudaError_t launch_t(const CausalLaunch& a, const Sizes& s, const Layout& l, cudaStream_t stream) {
    using C = Cfg<D>;
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = allow_smem(k_causal_tc<E, D>, C::kSmem, devices);
    if (e != cudaSuccess) return e;
    const __half *q = static_cast<const __half*>(a.q), *k = static_cast<const __half*>(a.k), *v = static_cast<const __half*>(a.v);
    const __half *pk = static_cast<const __half*>(a.pk), *pv = static_cast<const __half*>(a.pv);
    CUtensorMap mq, mk, mv, mpk, mpv;
    const uint64_t kw = uint64_t(a.kv_heads) * D;
    if (!encode_fp16_map_3d(&mq, q, D, uint64_t(a.heads), uint64_t(a.ntok), 64, uint32_t(s.group), uint32_t(s.T), uint64_t(a.q_stride)))
        return cudaErrorInvalidValue;
    mk = mv = mpk = mpv = mq;  // never read where there are no rows
    if (a.nkv > 0 && (!encode_fp16_map(&mk, k, kw, uint64_t(a.nkv), 64, 32, uint64_t(a.k_stride)) ||
                      !encode_fp16_map(&mv, v, kw, uint64_t(a.nkv), 64, 32, uint64_t(a.v_stride))))
        return cudaErrorInvalidValue;
    if (a.prefix > 0 && (!encode_fp16_map(&mpk, pk, kw, uint64_t(a.prefix), 64, 32, uint64_t(a.pk_stride)) ||
                         !encode_fp16_map(&mpv, pv, kw, uint64_t(a.prefix), 64, 32, uint64_t(a.pv_stride))))
        return cudaErrorInvalidValue;
    // A warp's rows of a tile: all heads of some tokens, or some heads of one.
    const bool boxes = C::kBoxes && (s.group & (s.group - 1)) == 0;
    CUtensorMap mo = mq;
    const uint32_t box_heads = uint32_t(std::min(s.group, 32));
    if (boxes && !encode_fp16_map_3d(&mo, static_cast<const __half*>(a.out), D, uint64_t(a.heads), uint64_t(a.ntok), 32, box_heads,
                                     32 / box_heads, uint64_t(a.out_stride), CU_TENSOR_MAP_SWIZZLE_64B))
        return cudaErrorInvalidValue;
    TcParams p{a.q, a.k, a.v, a.pk, a.pv, a.out, a.q_stride, a.k_stride, a.v_stride, a.pk_stride, a.pv_stride, a.out_stride,
               a.heads, a.kv_heads, s.group, s.T, s.TI, a.ntok, std::min(a.window, 1 << 30), a.prefix, (a.prefix + kKeys - 1) / kKeys,
               reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_stride % 16 == 0, boxes,
               uint32_t(((uint64_t(1) << 32) + a.kv_heads - 1) / a.kv_heads), a.scale * kLog2e,
               wait_limit(int64_t(a.prefix) + a.nkv),
               l.head, l.rng, l.segs, l.work, l.o, l.ml};
    const int64_t most = s.lmax > 1 ? a.num_sms : int64_t(s.tiles) * a.kv_heads;
    e = launch_pdl(k_causal_tc<E, D>, unsigned(std::min<int64_t>(a.num_sms, most)), C::kThreads, size_t(C::kSmem), stream, 1, mq, mk, mv,
                   mpk, mpv, mo, p);
    if (e != cudaSuccess || s.lmax == 1) return e;
    MergeParams mp{a.out, a.out_stride, a.heads, a.ntok, s.TI, s.lmax, a.prefix, p.window, l.rng, l.info, l.o, l.ml};
    // Eight warps a row where all rows are resident at once, else four, so that twice as many are (64 rows of 32
    // heads, 18 pieces: 6.7 us with four, 8.8 with eight; 2 rows of 3 heads, 128 pieces: 7.7 and 4.9).
    const int64_t rows = int64_t(a.ntok) * a.heads;
    if (rows > 8 * a.num_sms) return launch_pdl(k_causal_merge<E, D, 4>, unsigned(rows), 128, 0, stream, 1, mp);
    return launch_pdl(k_causal_merge<E, D, 8>, unsigned(rows), 256, 0, stream, 1, mp);
}

template <typename E>
cudaError_t launch_e(const CausalLaunch& a, const Sizes& s, const Layout& l, cudaStream_t stream) {
    if (a.hd == 64) return launch_t<E, 64>(a, s, l, stream);
    if (a.hd == 128) return launch_t<E, 128>(a, s, l, stream);
    return launch_t<E, 256>(a, s, l, stream);
}

}  // namespace

size_t causal_workspace(const CausalLaunch& a) { return layout_of(a, sizes_of(a)).bytes; }

cudaError_t launch_causal(const CausalLaunch& a, cudaStream_t stream) {
    const Sizes s = sizes_of(a);
    const Layout l = layout_of(a, s);
    const int window = std::min(a.window, 1 << 30);  // no range is longer
    const bool by_rows = a.nseq > kPlanSeqs;
    PlanParams pp{a.q_seqs, a.kv_seqs, a.nseq, a.ntok, a.nkv, window, s.T, s.TI, s.tiles, a.kv_heads,
                  (a.prefix + kKeys - 1) / kKeys, s.lmax, a.num_sms, by_rows, l.head, l.rng, l.segs, l.info, l.work};
    // A warp plans an item; up to 8 CTAs share them.
    const int ctas = s.tiles <= kPlanItems ? 1 : s.tiles <= 128 ? 4 : 8;
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = allow_smem(k_causal_plan, int(plan_smem(kPlanSeqs)), devices);
    if (by_rows) {
        const unsigned blocks = unsigned((a.ntok + kRowBlock - 1) / kRowBlock);
        const auto some = [&](int n) { return unsigned(std::min((n + 255) / 256, 8 * a.num_sms)); };
        const auto next = [&](void (*kern)(PlanParams), unsigned grid, unsigned threads) {
            if (e == cudaSuccess) e = launch_pdl(kern, grid, threads, 0, stream, 1, pp);
        };
        next(k_rows_clear, some(a.ntok), 256);
        next(k_rows_mark, some(a.nseq), 256);
        next(k_rows_sum, blocks, 256);
        next(k_rows_scan, 1, 1024);
        next(k_rows_range, blocks, 256);
    }
    if (e == cudaSuccess) e = launch_pdl(k_causal_plan, unsigned(ctas), 1024, plan_smem(by_rows ? 0 : a.nseq), stream, ctas, pp);
    if (e != cudaSuccess) return e;
    return a.bf16 ? launch_e<__nv_bfloat16>(a, s, l, stream) : launch_e<__half>(a, s, l, stream);
}

}  // namespace ge
