// Attention over caches whose sequences share their beginnings: the beams or samples of a
// prompt.  Per query row the same sum as nt_kvattn.cu's,
//   o = sum_j softmax_j(scale q . k_j) v_j,
// taken in two parts that a third kernel joins by their maxima and totals: the keys that
// every row of a group sees and that are shared, once for all of the group's rows, and for
// each row the rest (attend(), with the shared keys left out).
//
// The shared part is one tile of up to 128 query rows (beams x new tokens x query heads of
// a cached head) against the group's keys, so it belongs on the tensor cores: tcgen05.mma
// with M = 128 rows, S = Q K^T into TMEM, the weights back into TMEM over the scores that
// they come from, O += P V with P as the TMEM operand.  No masks are needed: the part covers
// only whole tiles of 16 keys that all rows see.
//
// Numbers.  e4m3 codes are exact in f16, and so is a bf16 query scaled per row by a power of
// two; a float32 query is a pair of f16 (22 bits) and takes its product twice.  The block
// scales of K multiply scores, in the softmax.  V becomes bf16 with its block's scale, exactly
// (four significant bits), and the weights, which lie in any range, two bf16 (16 bits, for
// bf16 outputs) or three (24 bits, float32 outputs; with a third piece for bf16 and heads of 128 one CTA's
// TMEM would leave no room for another on its SM).  attend(), which takes short reaches and the rest of each row, has pairs of f16
// there, 22 bits: a bf16 output shows neither (64 samples over 65536 keys, error against 64 bits
// 1.6855e-3 with sharing, without it and for float32 products of torch's, of which rounding the output is all).  Weights are 1 at the row's reference, which moves to
// a block's maximum when the block's weights come to more than 2^10, and values are divided by
// 2^32, so that sums of finite ones stay finite; values below 2^-94 lose bits by it, 2^-102 at most.
//
// A CTA: four warps of softmax (a thread a row), of which one thread issues the products, and
// eight that load codes one tile ahead, convert them and write the operands (K as it lies, V
// transposed by stmatrix, its dimensions in an order of their own that the join undoes).  Two
// CTAs share an SM where they fit, so that one's products run under the other's softmax; the
// softmax warps take registers from the others.  The
// tiles of all groups and heads in a row are cut into even shares, one a CTA.
//
// 64 samples of 4 query heads on each of 8 cached heads of 128 over 65536 shared keys (69 GFLOP,
// 42 us at the measured rate; half as much again is done for the weights' second halves), caches
// flushed: this kernel 124 us, the rest of the rows until 153, the join until 166.  A tile of 128
// keys takes a CTA 8400 clocks, two CTAs an SM, of which its 24 products take 1600 (65 to 68 each,
// measured alone): the softmax and the conversions beside it are the longer side (the tensor cores
// are busy 31 % of the time, a scheduler issues in 54 % of its clocks; of 10 warps an issue 4 wait for
// memory).  float32: 178, 204 and 218 us.  On
// the way: 177 us with four loading warps whose registers spilled (shared memory leaves no L1
// to catch that), 147 with eight, 131 with the look-ups in shared memory, 123 with 32 columns a step.  D = 128 in
// bf16 still spills 152 bytes a thread and reads 308.
//
// Few rows (kFewRows) take the attention of nt_kvattn.cu instead, over both parts in one kernel;
// short reaches (kSReach, kSBytes) that without sharing.
#include "nt_kvattn.cuh"

#include <cuda_bf16.h>

namespace nt {
namespace {

using namespace kva;

constexpr int kSRows = 128;            // query rows of a tile
constexpr int kSKeys = 128;            // keys of a tile
constexpr int kSGroups = 512;          // groups of a call
constexpr int kSoftWarps = 4, kLoadWarps = 8;
constexpr int kSThreads = 32 * (kSoftWarps + kLoadWarps);
constexpr float kSUp = 4294967296.f;   // 2^32: values are held divided by it
constexpr float kSMost = 1024.f;       // a block's weights that come to more move the reference to their maximum

struct SharedArgs {
    KvAttnArgs a;                      // a.part: the rest's partial rows
    int B, groups, K;                  // sequences, groups, sequences of a group
    int rows, row_tiles, rows_cap;     // query rows of a cached head of a group, tiles of them, rows of a tile at most
    int copies;                        // of a tile's rows among the 128: each takes its part of a tile's keys
    int64_t stride;                    // floats of a partial tile
    int ctas;
    const int32_t* shared;
    int64_t* info;                     // [groups][2]: tiles per head before the group, lo | hi << 32; then the total
    int32_t* rest_info;                // in even shares: tiles per head of the rest before each sequence, and the total
    float* part;                       // partial tiles: [copies * rows_cap][D] means, as many references and totals
};

// The keys [lo, hi) that the rows of a group have in common and all see, in whole tiles of 16.
struct Common { int lo, hi; };
// One sequence's part in it; a sequence without new tokens has none.
__device__ __forceinline__ bool common_of(const SharedArgs& s, int b, int* lo, int* hi) {
    const int cnt = tokens_of(s.a, b);
    if (cnt == 0) return false;
    const int len = s.a.lengths[b];
    *lo = s.a.window >= 0 && len - 1 > s.a.window ? len - 1 - s.a.window : 0;
    *hi = len - cnt + 1;
    return true;
}
__device__ __forceinline__ Common common_whole(int lo, int hi, int shared) {
    Common c;
    c.lo = (lo + kTile - 1) & ~(kTile - 1);
    c.hi = min(hi, max(shared, 0)) & ~(kTile - 1);
    if (c.hi <= c.lo) c.lo = c.hi = 0;
    return c;
}
// by one warp
__device__ __forceinline__ Common common_warp(const SharedArgs& s, int g) {
    int lo = 0, hi = 0x7fffffff;
    bool any = false;
    for (int i = threadIdx.x & 31; i < s.K; i += 32) {
        int l, h;
        if (common_of(s, g * s.K + i, &l, &h)) {
            lo = max(lo, l);
            hi = min(hi, h);
            any = true;
        }
    }
    lo = __reduce_max_sync(0xffffffffu, lo);
    hi = __reduce_min_sync(0xffffffffu, hi);
    any = __any_sync(0xffffffffu, any);
    return common_whole(lo, any ? hi : 0, s.shared[g]);
}

// ---------------------------------------------------------------------------
// The shared part
// ---------------------------------------------------------------------------
template <int DT, int D> struct SharedCfg {
    static constexpr int NQ = DT == NT_F32 ? 2 : 1;     // f16 pieces of a query
    static constexpr int NP = DT == NT_F32 ? 3 : 2;     // bf16 pieces of a weight
    static constexpr int kQ = kSRows * D * 2;           // bytes of a piece
    static constexpr int kK = kSKeys * D * 2;
    static constexpr int kCol3 = 128;                   // TMEM columns: scores and weights 0.., third piece, sums
    static constexpr int kColO = NP == 3 ? 192 : 128;
    static constexpr uint32_t kCols = kColO + D <= 256 ? 256 : 512;
    static constexpr int kData = NQ * kQ + 2 * kK;
    // two CTAs of an SM at most: their TMEM would not go round
    static constexpr int kBytes = 1024 + (kData < 76 * 1024 ? 76 * 1024 : kData);
    static constexpr int kPerSm = kCols == 256 && kBytes <= 112 * 1024 ? 2 : 1;
};

__device__ __forceinline__ void s_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void s_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void s_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void s_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void s_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
// K-major operand, 128-byte swizzle, rows of 64 two-byte elements, groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t s_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// type: 0 f16, 1 bf16; float32 sums
__host__ __device__ constexpr uint32_t s_idesc(uint32_t type, int N) {
    return 1u << 4 | type << 7 | type << 10 | (uint32_t)(N >> 3) << 17 | (uint32_t)(kSRows >> 4) << 24;
}
// 32 lanes x 16 columns, a thread a lane: asked for, and waited for
__device__ __forceinline__ void s_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
// the registers pass through, so that nothing reads them before
__device__ __forceinline__ void s_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
// the same, 32 columns
__device__ __forceinline__ void s_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void s_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void s_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at) : "memory");
}
__device__ __forceinline__ void s_ld8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) :: "memory");
}
__device__ __forceinline__ void s_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
// four 8x8 matrices of two-byte elements, stored transposed: lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void s_stmatrix_t(uint32_t at, uint32_t m0, uint32_t m1, uint32_t m2, uint32_t m3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(m0), "r"(m1), "r"(m2), "r"(m3)
                 : "memory");
}
// Where a dimension's sum stands among the columns: the order in which stmatrix leaves V's dimensions.
__host__ __device__ constexpr int column_of(int d) { return (d & ~63) + (d % 16 / 2) * 8 + (d % 64 / 16) * 2 + (d & 1); }

constexpr int kSBlocks = kSKeys / kTile;               // blocks of 16 keys of a tile
struct SharedBars { uint64_t k_full, v_full, s_full, p_full, o_done, q_full, found[4]; };
// Where a tile's blocks lie (in elements of the codes, < 0: not to be seen) and their scales (of K < 0 then).
struct SharedBlocks { int64_t off[kSBlocks]; float ks[kSBlocks], vs[kSBlocks]; };

template <int DT, int D>
__global__ void __launch_bounds__(kSThreads, SharedCfg<DT, D>::kPerSm) kv_shared_kernel(const __grid_constant__ SharedArgs s) {
    using Cfg = SharedCfg<DT, D>;
    using El = Elem<DT>;
    using T = typename El::T;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ SharedBars bars;
    __shared__ uint32_t tmem_base;
    __shared__ SharedBlocks blocks[4];                  // of tiles t, t + 1, ...
    __shared__ float row_scale[kSRows];                 // what a row's scores are multiplied by, besides their block's scale
    __shared__ int64_t before[kSGroups + 1];            // tiles per head ahead of a group
    __shared__ int c_lo[kSGroups], c_hi[kSGroups], c_lead[kSGroups];
    const KvAttnArgs& a = s.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* q_smem = smem;
    unsigned char* k_smem = smem + Cfg::NQ * Cfg::kQ;
    unsigned char* v_smem = k_smem + Cfg::kK;

    // what each group's rows have in common, and the sequence whose table is read
    for (int g = tid; g < s.groups; g += kSThreads) {
        c_lo[g] = 0;
        c_hi[g] = 0x7fffffff;
        c_lead[g] = 0x7fffffff;
    }
    __syncthreads();
    for (int b = tid; b < s.B; b += kSThreads) {
        int lo, hi;
        if (common_of(s, b, &lo, &hi)) {
            const int g = b / s.K;
            atomicMax(&c_lo[g], lo);
            atomicMin(&c_hi[g], hi);
            atomicMin(&c_lead[g], b);
        }
    }
    __syncthreads();
    for (int g = tid; g < s.groups; g += kSThreads) {
        const Common c = common_whole(c_lo[g], c_lead[g] == 0x7fffffff ? 0 : c_hi[g], s.shared[g]);
        c_lo[g] = c.lo;
        c_hi[g] = c.hi;
    }
    __syncthreads();
    if (warp == 0) {
        int64_t sum = 0;
        for (int g0 = 0; g0 < s.groups; g0 += 32) {
            int64_t n = g0 + lane < s.groups ? (c_hi[g0 + lane] - c_lo[g0 + lane] + kSKeys - 1) / kSKeys : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += up;
            }
            if (g0 + lane < s.groups) before[g0 + lane + 1] = sum + n;
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) before[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int g = tid; g <= s.groups; g += kSThreads) {
            s.info[2 * g] = before[g];
            if (g < s.groups) s.info[2 * g + 1] = (int64_t)c_hi[g] << 32 | (uint32_t)c_lo[g];
        }
    const int64_t per_head = (int64_t)a.H * s.row_tiles, total = before[s.groups] * per_head;
    const int64_t share = (total + s.ctas - 1) / s.ctas;
    const int64_t begin = blockIdx.x * share, end = begin + share < total ? begin + share : total;
    if (begin >= end) return;

    if (tid == 0) {
        mbar_init(smem_u32(&bars.k_full), kLoadWarps);
        mbar_init(smem_u32(&bars.v_full), kLoadWarps);
        mbar_init(smem_u32(&bars.s_full), 1);
        mbar_init(smem_u32(&bars.p_full), kSoftWarps);
        mbar_init(smem_u32(&bars.o_done), 1);
        mbar_init(smem_u32(&bars.q_full), kSoftWarps);
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&bars.found[i]), 2 * kSBlocks);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kSoftWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(Cfg::kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    s_fence_before();
    __syncthreads();
    s_fence_after();
    const uint32_t tmem = tmem_base;

    // The share's segments in order: (group, head, row tile) and its tiles [first, last).
    struct Segment { int g, h, rt, first, last; };
    auto segment = [&](int64_t at, int g) {
        Segment e;
        while (before[g + 1] * per_head <= at) ++g;
        const int64_t rel = at - before[g] * per_head, n = before[g + 1] - before[g];
        const int item = (int)(rel / n);
        e.g = g;
        e.h = item / s.row_tiles;
        e.rt = item % s.row_tiles;
        e.first = (int)(rel - item * n);
        e.last = (int)(end - at < n - e.first ? e.first + (end - at) : n);
        return e;
    };

    if (warp < kSoftWarps) {
        if constexpr (Cfg::kPerSm == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        // ---------------- queries, softmax, results: a thread a row ----------------
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        const uint32_t qs = smem_u32(q_smem), ks_smem = smem_u32(k_smem), vs_smem = smem_u32(v_smem);
        int it = 0, seg = 0, g = 0;
        bool ok = true;
        for (int64_t at = begin; at < end && ok; ++seg) {
            const Segment e = segment(at, g);
            g = e.g;
            const int rows = min(kSRows, s.rows - e.rt * kSRows);
            // a tile of 32 rows or fewer stands four times among the lanes, one of 64 twice: each copy takes a part of
            // the keys' columns, and has a reference, a total and sums of its own
            const int copy = warp / (4 / s.copies), row0 = warp % (4 / s.copies) * 32;
            const bool busy = row0 < rows;               // this warp has rows
            const int first_block = copy * (8 / s.copies), last_block = first_block + 8 / s.copies;
            // Queries, a row by the lanes that hold eight of its elements each, in f16, scaled by a power of two so
            // that the largest is in [2^13, 2^14); the scores' scale is positive, its sign the query's.
            {
                constexpr int LR = D / 8, RW = 32 / LR;  // lanes of a row, rows at a time
                const int row = e.rt * kSRows + row0 + lane, beam = row / (a.T * a.G), t = row / a.G % a.T;
                const int64_t b = (int64_t)e.g * s.K + beam;
                int lo, hi;
                const bool live = row0 + lane < rows && common_of(s, (int)b, &lo, &hi) && t < (a.counts ? a.counts[b] : a.T);
                // where lane's row lies, in elements; -1: no such row
                const int64_t mine = live ? b * a.q_sb + (int64_t)t * a.q_st + (int64_t)(e.h * a.G + row % a.G) * a.q_sh : -1;
                const int d = lane % LR * 8;
#pragma unroll 1
                for (int r0 = 0; r0 < 32; r0 += 4 * RW) {
                    uint4 raw[4][sizeof(T) / 2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int64_t off = __shfl_sync(0xffffffffu, mine, r0 + j * RW + lane / LR);
                        const T* q = static_cast<const T*>(a.q) + off + d;
#pragma unroll
                        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                            raw[j][i] = make_uint4(0, 0, 0, 0);
                            if (off >= 0) {
                                if (a.q_vec) raw[j][i] = __ldg(reinterpret_cast<const uint4*>(q) + i);
                                else
#pragma unroll 1
                                    for (int x = 0; x < 16 / (int)sizeof(T); ++x) {
                                        const uint32_t bits = sizeof(T) == 4 ? reinterpret_cast<const uint32_t*>(q)[4 * i + x]
                                                                             : (uint32_t)reinterpret_cast<const uint16_t*>(q)[x];
                                        const int word = sizeof(T) == 4 ? x : x / 2, at = sizeof(T) == 4 ? 0 : x % 2 * 16;
                                        raw[j][i].x |= word == 0 ? bits << at : 0u;
                                        raw[j][i].y |= word == 1 ? bits << at : 0u;
                                        raw[j][i].z |= word == 2 ? bits << at : 0u;
                                        raw[j][i].w |= word == 3 ? bits << at : 0u;
                                    }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = warp * 32 + r0 + j * RW + lane / LR;
                        float v[8], amax = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint4 w4 = raw[j][DT == NT_F32 ? i / 4 : 0];
                            const int k = DT == NT_F32 ? i % 4 : i / 2;
                            const uint32_t u = k == 0 ? w4.x : k == 1 ? w4.y : k == 2 ? w4.z : w4.w;
                            v[i] = __uint_as_float(DT == NT_F32 ? u : i & 1 ? u & 0xffff0000u : u << 16);
                            const float m = fabsf(v[i]);
                            if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
                        }
#pragma unroll
                        for (int o = 1; o < LR; o *= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                        int x = 127 + 13 - (int)(__float_as_uint(amax) >> 23);
                        x = amax > 0.f ? (x > 126 ? 126 : x) : 0;
                        float up = __uint_as_float((uint32_t)(127 + x) << 23);
                        if (lane % LR == 0) row_scale[r] = __uint_as_float((uint32_t)(127 - x) << 23) * fabsf(a.scale_log2);
                        if (a.scale_log2 < 0.f) up = -up;
                        uint32_t hi4[4], lo4[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x0 = v[2 * i] * up, x1 = v[2 * i + 1] * up;
                            hi4[i] = pack_h2(x0, x1);
                            const float2 rest = unpack_h2(hi4[i]);
                            lo4[i] = pack_h2(x0 - rest.x, x1 - rest.y);
                        }
                        const int at8 = (d / 64) * (kSRows * 128) + r * 128 + (((d % 64 / 8) ^ (r & 7)) << 4);
                        *reinterpret_cast<uint4*>(q_smem + at8) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
                        if constexpr (Cfg::NQ == 2) *reinterpret_cast<uint4*>(q_smem + Cfg::kQ + at8) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.q_full));
            const float f_row = row_scale[tid];

            float m = -INFINITY, l = 0.f;               // reference (log2) and total
            for (int tile = e.first; tile < e.last; ++tile, ++it) {
                if (tid == 0) {
                    // scores; the weights of the tile before lie where they go
                    const bool go = (tile > e.first || mbar_wait(smem_u32(&bars.q_full), seg & 1)) &&
                                    (it == 0 || mbar_wait(smem_u32(&bars.o_done), (it - 1) & 1)) && mbar_wait(smem_u32(&bars.k_full), it & 1);
                    if (go) {
                        s_fence_after();
#pragma unroll
                        for (int p = 0; p < Cfg::NQ; ++p)
#pragma unroll
                            for (int k = 0; k < D / 16; ++k)
                                s_mma_ss(tmem, s_desc(qs + p * Cfg::kQ + k / 4 * (kSRows * 128) + k % 4 * 32),
                                         s_desc(ks_smem + k / 4 * (kSKeys * 128) + k % 4 * 32), s_idesc(0, kSKeys), p || k);
                        s_commit(smem_u32(&bars.s_full));
                    } else {
                        atomicOr(a.err, ERRF_TIMEOUT_MMA);
                    }
                }
                __syncwarp();
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.s_full), it & 1));
                if (!ok) {
                    if (lane == 0) atomicOr(a.err, ERRF_TIMEOUT_EPILOGUE);
                    break;
                }
                s_fence_after();
                if (busy) {
                    const float* ks = blocks[it & 3].ks;
                    // Two blocks of 16 keys at a time, the next ones' scores on their way: a block's weights go where its
                    // scores lie, 8 columns a piece.  The other copies' keys have none here.
                    uint32_t v[32];
                    s_ld32(lanes + first_block * 16, v);
                    if (s.copies > 1) {
                        uint32_t zero[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) zero[i] = 0u;
#pragma unroll 1
                        for (int c = 0; c < kSBlocks; ++c) {
                            if (c >= first_block && c < last_block) continue;
                            s_st16(lanes + c * 16, zero);
                            if constexpr (Cfg::NP == 3) s_st8(lanes + Cfg::kCol3 + c * 8, *reinterpret_cast<uint32_t (*)[8]>(zero));
                        }
                    }
#pragma unroll 1
                    for (int c = first_block; c < last_block; c += 2) {
                        const float k0 = ks[c], k1 = ks[c + 1];
                        // a block that is not seen has no weight
                        const float f[2] = {k0 >= 0.f ? f_row * k0 : 0.f, k1 >= 0.f ? f_row * k1 : 0.f};
                        const bool seen = k0 >= 0.f || k1 >= 0.f;
                        float p[32], sum;
                        auto weigh = [&]() {
                            const float at = m == -INFINITY ? 0.f : m, base[2] = {k0 < 0.f ? INFINITY : at, k1 < 0.f ? INFINITY : at};
                            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                p[i] = ex2(fmaf(__uint_as_float(v[i]), f[i / 16], -base[i / 16]));
                                part[i & 3] += p[i];
                            }
                            sum = (part[0] + part[1]) + (part[2] + part[3]);
                        };
                        s_ld_wait(v);
                        weigh();
                        // the reference is far below the blocks' maximum (or there is none yet, or a NaN)
                        if (__any_sync(0xffffffffu, seen && (!(sum <= kSMost) || m == -INFINITY))) {
                            float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[i / 16] = fmaxf(x[i / 16], __uint_as_float(v[i]));
                            const float mx = fmaxf(k0 >= 0.f ? x[0] * f[0] : -INFINITY, k1 >= 0.f ? x[1] * f[1] : -INFINITY);
                            // to a whole number, so that what is there already is multiplied by a power of two
                            const bool move = mx > m;
                            const float next = move ? ceilf(mx) : m;
                            const float by = !move ? 1.f : next - m < 126.f ? __uint_as_float((uint32_t)(127 - (int)(next - m)) << 23) : 0.f;
                            m = next;
                            l *= by;
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            const __nv_bfloat162 by2 = __floats2bfloat162_rn(by, by);
                            auto scale = [&](int col, bool packed) {        // 8 columns
                                uint32_t w[8];
                                s_ld8(lanes + col, w);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const __nv_bfloat162 y = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), by2);
                                    w[i] = packed ? *reinterpret_cast<const uint32_t*>(&y) : __float_as_uint(__uint_as_float(w[i]) * by);
                                }
                                s_st8(lanes + col, w);
                            };
                            if (tile > e.first)
#pragma unroll 1
                                for (int d = 0; d < D; d += 8) scale(Cfg::kColO + d, false);
#pragma unroll 1
                            for (int col = first_block * 2; col < c * 2; ++col) scale(col * 8, true);
                            if constexpr (Cfg::NP == 3)
#pragma unroll 1
                                for (int col = first_block; col < c; ++col) scale(Cfg::kCol3 + col * 8, true);
                            weigh();
                        }
                        l += sum;
                        if (c + 2 < last_block) s_ld32(lanes + (c + 2) * 16, v);
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            uint32_t w[16], w2[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float p0 = p[16 * n + 2 * i], p1 = p[16 * n + 2 * i + 1];
                                const uint32_t h = pack_b2(p0, p1);
                                const float r0 = p0 - __uint_as_float(h << 16), r1 = p1 - __uint_as_float(h & 0xffff0000u);
                                const uint32_t h2 = pack_b2(r0, r1);
                                w[i] = h;
                                w[8 + i] = h2;
                                if constexpr (Cfg::NP == 3)
                                    w2[i] = pack_b2(r0 - __uint_as_float(h2 << 16), r1 - __uint_as_float(h2 & 0xffff0000u));
                            }
                            s_st16(lanes + (c + n) * 16, w);
                            if constexpr (Cfg::NP == 3) s_st8(lanes + Cfg::kCol3 + (c + n) * 8, w2);
                        }
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                s_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.p_full));
                if (tid == 0) {
                    if (mbar_wait(smem_u32(&bars.v_full), it & 1) && mbar_wait(smem_u32(&bars.p_full), it & 1)) {
                        s_fence_after();
#pragma unroll
                        for (int p = 0; p < Cfg::NP; ++p)
#pragma unroll
                            for (int k = 0; k < kSKeys / 16; ++k)
                                s_mma_ts(tmem + Cfg::kColO, tmem + (p == 2 ? Cfg::kCol3 + k * 8 : k * 16 + p * 8),
                                         s_desc(vs_smem + k / 4 * (D * 128) + k % 4 * 32), s_idesc(1, D), tile > e.first || p || k);
                        s_commit(smem_u32(&bars.o_done));
                    } else {
                        atomicOr(a.err, ERRF_TIMEOUT_MMA);
                    }
                }
                __syncwarp();
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.o_done), (it - 1) & 1));
            if (!ok) break;
            s_fence_after();
            if (busy) {
                const int64_t slot = ((int64_t)e.g * a.H + e.h) * s.row_tiles + e.rt + blockIdx.x;
                float* part = s.part + slot * s.stride;
                const float inv = l != 0.f ? kSUp / l : 0.f;
                const int r = copy * s.rows_cap + row0 + lane, n = s.copies * s.rows_cap;
                const bool mine = row0 + lane < rows;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t w[16];
                    s_ld16(lanes + Cfg::kColO + c, w);
                    s_ld_wait(w);
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<float4*>(part + r * D + c + i) =
                                make_float4(__uint_as_float(w[i]) * inv, __uint_as_float(w[i + 1]) * inv, __uint_as_float(w[i + 2]) * inv,
                                            __uint_as_float(w[i + 3]) * inv);
                    }
                }
                if (mine) {
                    part[n * D + r] = m;
                    part[n * D + n + r] = l * (float)(1 << (int)kPShift);      // as attend() leaves it
                }
            }
            s_fence_before();
            at += e.last - e.first;
        }
    } else {
        // the launch's 384 threads have 80 registers each (30720): 128 x 112 and 256 x 64 of them
        if constexpr (Cfg::kPerSm == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ---------------- codes: global memory -> registers -> operands ----------------
        constexpr int CH = D / 16;                      // 16-code pieces of a key
        constexpr int N = kSKeys * CH / (32 * kLoadWarps);      // of a thread, K and V each
        const int w = warp - kSoftWarps, lt = w * 32 + lane;
        const int n_tiles = (int)(end - begin);
        // The first of these warps looks up where blocks lie, a lane a block, for the tile three ahead of the one in
        // work: its scales are on their way into shared memory while the next one's table entries are asked for.
        Segment e = segment(begin, 0);
        int64_t at = begin;
        int entry = -2, slot = 0, head = 0;
        bool bad_page = false;
        auto ask_entry = [&]() {                        // -1: no page, -2: not wanted
            entry = -2;
            if (at >= end) return;
            const int key = c_lo[e.g] + e.first * kSKeys + lane * kTile;
            if (lane < kSBlocks && key < c_hi[e.g]) entry = max(__ldg(a.table + (int64_t)c_lead[e.g] * a.table_sb + (key >> a.page_shift)), -1);
            slot = key & ((1 << a.page_shift) - 1);
            head = e.h;
            if (++at < end && ++e.first >= e.last) e = segment(at, e.g);
        };
        auto ask_scales = [&](int tile) {
            if (lane < kSBlocks) {
                SharedBlocks& to = blocks[tile & 3];
                const bool there = entry >= 0 && entry < a.n_pages;
                const int64_t row = (int64_t)entry * a.H + head;
                to.off[lane] = there ? ((row << a.page_shift) + slot) * D : -1;
                if (there) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&to.ks[lane])), "l"(a.ks + row) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&to.vs[lane])), "l"(a.vs + row) : "memory");
                } else {
                    to.ks[lane] = -1.f;
                    to.vs[lane] = 0.f;
                    if (entry != -2) bad_page = true;
                }
                // arrives when the lane's copies have landed, and for what it has written itself
                asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&bars.found[tile & 3])) : "memory");
                mbar_arrive(smem_u32(&bars.found[tile & 3]));
            }
            __syncwarp();
        };
        if (w == 0)
            for (int i = 0; i < 3; ++i) {
                ask_entry();
                ask_scales(i);
            }
        if (w == 0) ask_entry();
        // K piece j of a thread: key (j * threads + lt) / CH; V piece j of a warp: 8 keys x 64 dimensions, key of the lane's quarter
        uint4 kr[N], vr[N];
        auto fetch = [&](const uint8_t* codes, int tile, int key, int dim) {
            const int64_t o = blocks[tile & 3].off[key / kTile];
            uint4 r = make_uint4(0, 0, 0, 0);
            if (o >= 0)
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(codes + o + key % kTile * D + dim));
            return r;
        };
        auto load_k = [&](int tile) {
#pragma unroll
            for (int j = 0; j < N; ++j) kr[j] = fetch(a.kc, tile, (j * 32 * kLoadWarps + lt) / CH, lt % CH * 16);
        };
        auto load_v = [&](int tile) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = j * kLoadWarps + w;
                vr[j] = fetch(a.vc, tile, u / (D / 64) * 8 + lane / 4, u % (D / 64) * 64 + lane % 4 * 16);
            }
        };
        bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.found[0]), 0));
        if (ok) {
            load_k(0);
            load_v(0);
        }
        for (int it = 0; it < n_tiles && ok; ++it) {
            const bool more = it + 1 < n_tiles;
            ok = (it == 0 || __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.s_full), (it - 1) & 1))) &&
                 (!more || __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.found[(it + 1) & 3]), ((it + 1) >> 2) & 1)));
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int key = (j * 32 * kLoadWarps + lt) / CH, c = lt % CH, panel = c / 4;
                uint4 h[2];
                h[0] = make_uint4(cvt_lo(kr[j].x), cvt_hi(kr[j].x), cvt_lo(kr[j].y), cvt_hi(kr[j].y));
                h[1] = make_uint4(cvt_lo(kr[j].z), cvt_hi(kr[j].z), cvt_lo(kr[j].w), cvt_hi(kr[j].w));
                unsigned char* base = k_smem + panel * (kSKeys * 128) + key * 128;
                // panel 1 writes its odd chunk first, so that eight lanes meet eight banks
                const int o = panel & 1, ch = c % 4 * 2;
                *reinterpret_cast<uint4*>(base + (((ch + o) ^ (key & 7)) << 4)) = o ? h[1] : h[0];
                *reinterpret_cast<uint4*>(base + (((ch + 1 - o) ^ (key & 7)) << 4)) = o ? h[0] : h[1];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.k_full));
            if (more) load_k(it + 1);
            ok = it == 0 || __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.o_done), (it - 1) & 1));
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = j * kLoadWarps + w, ko = u / (D / 64), half = u % (D / 64);
                const float f = blocks[it & 3].vs[ko / 2] * (1.f / kSUp);
                const uint32_t words[4] = {vr[j].x, vr[j].y, vr[j].z, vr[j].w};
                uint32_t b[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = unpack_h2(cvt_lo(words[i])), y = unpack_h2(cvt_hi(words[i]));
                    b[2 * i] = pack_b2(x.x * f, x.y * f);
                    b[2 * i + 1] = pack_b2(y.x * f, y.y * f);
                }
                // matrix i: dimensions 16c + 2i, + 1 of the four lanes of a key, as rows 8i + 2c, + 1
                const uint32_t base = smem_u32(v_smem) + ko / 8 * (D * 128) + half * (64 * 128) + (((ko & 7) ^ (lane & 7)) << 4) + lane * 128;
                s_stmatrix_t(base, b[0], b[1], b[2], b[3]);
                s_stmatrix_t(base + 32 * 128, b[4], b[5], b[6], b[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.v_full));
            if (more) load_v(it + 1);
            if (w == 0) {                               // what stood in these places was read for tile it - 1
                ask_scales(it + 3);
                ask_entry();
            }
        }
        if (!ok && lane == 0) atomicOr(a.err, ERRF_TIMEOUT_PRODUCER);
        if (bad_page) atomicOr(a.err, ERRF_BAD_ARG);
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    s_fence_before();
    __syncthreads();
    if (warp == kSoftWarps) {
        __syncwarp();
        s_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kCols));
    }
}

// ---------------------------------------------------------------------------
// The rest of each row, always to partial rows
// ---------------------------------------------------------------------------
__device__ __forceinline__ Span rest_of(const SharedArgs& s, int64_t b, int row_tile, Common c) {
    Span e = span_of(s.a, b, row_tile);
    e.skip = 0x7fffffff;
    e.gap = 0;
    if (e.tiles && c.hi > c.lo) {                       // lo16 <= c.lo and c.hi <= hi: all of the group's rows see [c.lo, c.hi)
        e.skip = (c.lo - e.lo16) / kTile;
        e.gap = c.hi - c.lo;
        e.tiles = e.skip + (e.hi - c.hi + kTile - 1) / kTile;
    }
    return e;
}

template <int DT, int D, int W, bool HALF>
__global__ void __launch_bounds__(W * 32, 16 / W) kv_rest_kernel(const __grid_constant__ SharedArgs s) {
    extern __shared__ __align__(128) unsigned char smem[];
    const KvAttnArgs& a = s.a;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int split = blockIdx.x, h = blockIdx.y / a.row_tiles, row_tile = blockIdx.y % a.row_tiles;
    const int64_t b = blockIdx.z;
    const Span e = rest_of(s, b, row_tile, common_warp(s, (int)b / s.K));
    if (e.bad && split == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
    const int first = split * a.chunk, last = min(first + a.chunk, e.tiles);
    if (first < e.tiles) {
        float* part = a.part + ((b * gridDim.y + blockIdx.y) * a.splits + split) * (kRows * (D + 2));
        attend<DT, D, W, HALF, ROWS_WITH_GAP>(a, b, h, row_tile, e, first, last, part, smem);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the join follows this kernel alone, and needs the one before too
}

// Tiles per head (and `more` for each) of the sequences before i, for i <= B, by all threads of a CTA, with the
// groups' common keys.
__device__ __forceinline__ void rest_before(const SharedArgs& s, int* before, int* c_lo, int* c_hi, int more = 0) {
    for (int g = threadIdx.x; g < s.groups; g += blockDim.x) {
        c_lo[g] = 0;
        c_hi[g] = 0x7fffffff;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < s.B; b += blockDim.x) {
        int lo, hi;
        if (common_of(s, b, &lo, &hi)) {
            atomicMax(&c_lo[b / s.K], lo);
            atomicMin(&c_hi[b / s.K], hi);
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < s.groups; g += blockDim.x) {
        const Common c = common_whole(c_lo[g], c_hi[g] == 0x7fffffff ? 0 : c_hi[g], s.shared[g]);
        c_lo[g] = c.lo;
        c_hi[g] = c.hi;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int sum = 0;
        for (int i0 = 0; i0 < s.B; i0 += 32) {
            int n = 0;
            if (i0 + lane < s.B) {
                const int g = (i0 + lane) / s.K;
                const Span e = rest_of(s, i0 + lane, 0, Common{c_lo[g], c_hi[g]});
                n = e.tiles ? e.tiles + more : 0;
                if (e.bad && blockIdx.x == 0) atomicOr(s.a.err, ERRF_BAD_ARG);
            }
#pragma unroll
            for (int k = 1; k < 32; k *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, n, k);
                if (lane >= k) n += up;
            }
            if (i0 + lane < s.B) before[i0 + lane + 1] = sum + n;
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) before[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0)                                // for the join
        for (int i = threadIdx.x; i <= s.B; i += blockDim.x) s.rest_info[i] = before[i];
}

// In even shares, for ragged sequences (see kv_attention_even_kernel): two partial rows a CTA.
template <int DT, int D, int W, bool HALF>
__global__ void __launch_bounds__(W * 32, 16 / W) kv_rest_even_kernel(const __grid_constant__ SharedArgs s) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int before[kEvenBatch + 1], c_lo[kEvenBatch], c_hi[kEvenBatch];
    const KvAttnArgs& a = s.a;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    rest_before(s, before, c_lo, c_hi);
    const int64_t total = (int64_t)before[s.B] * a.H, share = share_of(total, gridDim.x);
    const int64_t begin = blockIdx.x * share, end = begin + share < total ? begin + share : total;
    // a share can hold many short heads, so each has a slot of its own: head and CTA counted together
    int b = 0;
    for (int64_t at = begin; at < end;) {
        while ((int64_t)before[b + 1] * a.H <= at) ++b;
        const Span e = rest_of(s, b, 0, Common{c_lo[b / s.K], c_hi[b / s.K]});
        const int64_t rel = at - (int64_t)before[b] * a.H;
        const int h = (int)(rel / e.tiles), first = (int)(rel - (int64_t)h * e.tiles);
        const int last = (int)(end - at < e.tiles - first ? first + (end - at) : e.tiles);
        attend<DT, D, W, HALF, ROWS_WITH_GAP>(a, b, h, 0, e, first, last, a.part + ((int64_t)b * a.H + h + blockIdx.x) * (kRows * (D + 2)), smem);
        at += last - first;
        __syncthreads();                                // the sums are read before the next ring is filled
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------------------
// Few rows a group: the shared part and the rest by attend(), in one kernel.  The shared
// part takes the group's rows, eight at a time, as the columns of one product; all tiles
// of both parts lie in a row (the groups' shared ones, then the sequences' rests) and are cut
// into even shares of CTAs of two warps; a head, which takes as long to begin and to end as
// kFewBegin tiles, counts as so many more.  Every head of either has a slot of its own for
// each CTA that it reaches: its number and the CTA's, added up.
// ---------------------------------------------------------------------------
constexpr int kFewBegin = 12;
template <int DT, int D, bool HALF_C, bool HALF_R>
__global__ void __launch_bounds__(64, 8) kv_few_kernel(const __grid_constant__ SharedArgs s) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int before[kEvenBatch + 1], c_lo[kEvenBatch], c_hi[kEvenBatch], c_before[kEvenBatch + 1], c_lead[kEvenBatch];
    const KvAttnArgs& a = s.a;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int g = threadIdx.x; g < s.groups; g += 64) c_lead[g] = 0x7fffffff;
    rest_before(s, before, c_lo, c_hi, kFewBegin);
    for (int b = threadIdx.x; b < s.B; b += 64)
        if (tokens_of(a, b)) atomicMin(&c_lead[b / s.K], b);
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int sum = 0;
        for (int i0 = 0; i0 < s.groups; i0 += 32) {
            int n = i0 + lane < s.groups ? (c_hi[i0 + lane] - c_lo[i0 + lane]) / kTile : 0;
            if (n) n += kFewBegin;
#pragma unroll
            for (int k = 1; k < 32; k *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, n, k);
                if (lane >= k) n += up;
            }
            if (i0 + lane < s.groups) c_before[i0 + lane + 1] = sum + n;
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) c_before[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int g = threadIdx.x; g <= s.groups; g += 64) {
            s.info[2 * g] = c_before[g];
            if (g < s.groups) s.info[2 * g + 1] = (int64_t)c_hi[g] << 32 | (uint32_t)c_lo[g];
        }
    const int64_t per_head = (int64_t)a.H * s.row_tiles, common = c_before[s.groups] * per_head, total = common + (int64_t)before[s.B] * a.H;
    const int64_t share = share_of(total, gridDim.x);
    const int64_t begin = blockIdx.x * share, end = begin + share < total ? begin + share : total;
    int g = 0, b = 0;
    for (int64_t at = begin; at < end;) {
        int64_t rel, item;
        int units;                                      // of the head: its tiles and kFewBegin
        const bool together = at < common;
        Span e;
        if (together) {
            while (c_before[g + 1] * per_head <= at) ++g;
            e.lo = e.lo16 = c_lo[g];
            e.hi = c_hi[g];
            e.lead = c_lead[g];
            e.tiles = (e.hi - e.lo) / kTile;
            units = c_before[g + 1] - c_before[g];
            rel = at - c_before[g] * per_head;
            item = g * per_head;
        } else {
            while (common + (int64_t)before[b + 1] * a.H <= at) ++b;
            e = rest_of(s, b, 0, Common{c_lo[b / s.K], c_hi[b / s.K]});
            units = before[b + 1] - before[b];
            rel = at - common - (int64_t)before[b] * a.H;
            item = s.groups * per_head + (int64_t)b * a.H;
        }
        const int n = (int)(rel / units), from = (int)(rel - (int64_t)n * units), to = (int)(end - at < units - from ? from + (end - at) : units);
        const int first = max(from - kFewBegin, 0), last = to - kFewBegin;
        if (last > 0) {
            float* part = a.part + (item + n + blockIdx.x) * (kRows * (D + 2));
            if (together) attend<DT, D, 2, HALF_C, ROWS_TOGETHER>(a, (int64_t)g * s.K, n / s.row_tiles, n % s.row_tiles, e, first, last, part, smem);
            else attend<DT, D, 2, HALF_R, ROWS_WITH_GAP>(a, b, n, 0, e, first, last, part, smem);
        }
        at += to - from;
        __syncthreads();                                // the sums are read before the next ring is filled
    }
}

// ---------------------------------------------------------------------------
// Joins a query row's parts: those of the shared tiles, then those of the rest.
// ---------------------------------------------------------------------------
constexpr int kSJoinWarps = 8;
// W warps a row: one where there are rows enough, which needs no barrier, else all of a CTA.
enum { REST_IN_CHUNKS = 0, REST_IN_SHARES = 1, ALL_IN_SHARES = 2 };
template <int DT, int D, int HOW, int W>
__global__ void __launch_bounds__(kSJoinWarps * 32) kv_shared_join_kernel(const __grid_constant__ SharedArgs s, int rest_ctas) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int E = D / 32;
    const KvAttnArgs& a = s.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.H * a.G;
    const int64_t at = (int64_t)blockIdx.x * (kSJoinWarps / W) + warp / W;      // row (b, t, head)
    if (at >= (int64_t)s.B * a.T * heads) return;       // a whole CTA when W is all its warps
    const int hq = (int)(at % heads), t = (int)(at / heads % a.T), h = hq / a.G;
    const int64_t b = at / heads / a.T;
    const int g = (int)b / s.K, beam = (int)b % s.K;
    constexpr int kPart = kRows * (D + 2);
    const bool live = t < tokens_of(a, b);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t info0 = s.info[2 * g], info1 = s.info[2 * g + 1], info2 = s.info[2 * g + 2];
    constexpr bool kFew = HOW == ALL_IN_SHARES;          // both parts in rows of eight
    // the shared tiles
    constexpr int kTileRows = kFew ? kRows : kSRows;
    const int srow = (beam * a.T + t) * a.G + hq % a.G, rt = srow / kTileRows, r1 = srow % kTileRows;
    const int64_t per_head = (int64_t)a.H * s.row_tiles, common = s.info[2 * s.groups] * per_head;
    const int64_t tiles = info2 - info0, item = (int64_t)g * per_head + (int64_t)h * s.row_tiles + rt;
    int rest_first = 0, rest_n = 0, rest_all = 0;
    if constexpr (HOW != REST_IN_CHUNKS) {
        rest_first = s.rest_info[b];
        rest_n = s.rest_info[b + 1] - rest_first;
        rest_all = s.rest_info[s.B];
    }
    const int64_t share = kFew ? share_of(common + (int64_t)rest_all * a.H, rest_ctas) : (common + s.ctas - 1) / s.ctas;
    constexpr int begin = kFew ? kFewBegin : 0;          // units of a head ahead of its tiles
    int n1 = 0, n2 = 0;
    const float* part1 = kFew ? a.part : s.part;
    if (tiles > 0) {
        const int64_t g0 = info0 * per_head + ((int64_t)h * s.row_tiles + rt) * tiles, c0 = (g0 + begin) / share;
        n1 = (int)((g0 + tiles - 1) / share - c0 + 1) * (kFew ? 1 : s.copies);
        part1 += (item + c0) * (kFew ? kPart : s.stride);
    }
    // the rest
    const int row = t * a.G + hq % a.G, row_tile = row / kRows, r2 = row % kRows;
    const float* part2 = a.part;
    if constexpr (HOW != REST_IN_CHUNKS) {
        if (rest_n > 0) {
            const int64_t sh = kFew ? share : share_of((int64_t)rest_all * a.H, rest_ctas);
            const int64_t g0 = (kFew ? common : 0) + (int64_t)rest_first * a.H + (int64_t)h * rest_n, c0 = (g0 + begin) / sh;
            n2 = (int)((g0 + rest_n - 1) / sh - c0 + 1);
            part2 += ((kFew ? s.groups * per_head : 0) + b * a.H + h + c0) * kPart;
        }
    } else {
        const Span e = rest_of(s, b, row_tile, Common{(int)(uint32_t)info1, (int)(info1 >> 32)});
        n2 = (e.tiles + a.chunk - 1) / a.chunk;
        part2 += (b * (int64_t)(a.H * a.row_tiles) + h * a.row_tiles + row_tile) * a.splits * kPart;
    }
    const int n = live ? n1 + n2 : 0;
    const int copies = kFew ? 1 : s.copies, cap = kFew ? kRows : s.rows_cap, held = copies * cap;      // rows of a partial tile
    // part i's row: its means; its reference lies `refs` floats behind the tile's begin, its total as many rows on
    auto tile_of = [&](int i) { return i < n1 ? part1 + i / copies * (kFew ? (int64_t)kPart : s.stride) : part2 + (int64_t)(i - n1) * kPart; };
    auto row_of = [&](int i) { return i < n1 ? i % copies * cap + r1 : r2; };
    auto ref_of = [&](int i, float* l) {
        const int rows = i < n1 ? held : kRows;
        const float* p = tile_of(i) + rows * D + row_of(i);
        *l = p[rows];
        return *p;
    };
    // the row's reference and total: every warp takes them from all parts, a lane a part
    float m = -INFINITY, tot = 0.f, m_own = -INFINITY, l_own = 0.f;      // of part `lane`
    for (int i = lane; i < n; i += 32) {
        float li;
        const float mi = ref_of(i, &li), up = fmaxf(m, mi), base = up == -INFINITY ? 0.f : up;
        if (i == lane) m_own = mi, l_own = li;
        tot = fmaf(ex2(mi - base), li, tot * ex2(m - base));
        m = up;
    }
#pragma unroll
    for (int k = 16; k; k /= 2) {
        const float mi = __shfl_xor_sync(0xffffffffu, m, k), li = __shfl_xor_sync(0xffffffffu, tot, k);
        const float up = fmaxf(m, mi), base = up == -INFINITY ? 0.f : up;
        tot = __fadd_rn(__fmul_rn(ex2(m - base), tot), __fmul_rn(ex2(mi - base), li));     // alike in every lane
        m = up;
    }
    const float base = m == -INFINITY ? 0.f : m, inv = tot != 0.f ? 1.f / tot : 0.f;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    // 32 parts at a time: their weights a lane each, then their rows, eight on their way
    for (int i0 = 0; i0 < n; i0 += 32) {
        if (i0 && i0 + lane < n) m_own = ref_of(i0 + lane, &l_own);
        const float f_own = i0 + lane < n ? ex2(m_own - base) * l_own * inv : 0.f;
        const int upto = min(32, n - i0);
        for (int j0 = warp % W; j0 < upto; j0 += 8 * W) {
            float2 x[8][E / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = i0 + j0 + j * W;
                const bool shared = !kFew && i < n1;
                const float* p = tile_of(i) + row_of(i) * D;
#pragma unroll
                for (int e = 0; e < E; e += 2)
                    x[j][e / 2] = j0 + j * W < upto ? *reinterpret_cast<const float2*>(p + (shared ? column_of(lane * E + e) : lane * E + e))
                                                    : make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = __shfl_sync(0xffffffffu, f_own, (j0 + j * W) & 31);
                if (j0 + j * W < upto)
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        sum[e] = fmaf(f, x[j][e / 2].x, sum[e]);
                        sum[e + 1] = fmaf(f, x[j][e / 2].y, sum[e + 1]);
                    }
            }
        }
    }
    if constexpr (W > 1) {
        __shared__ float ws[kSJoinWarps][D];
#pragma unroll
        for (int e = 0; e < E; ++e) ws[warp][lane * E + e] = sum[e];
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sum[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kSJoinWarps; ++w) sum[e] += ws[w][lane * E + e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        static_cast<T*>(a.out)[at * D + lane * E + e] = El::from_f(live && tot != 0.f ? sum[e] : 0.f);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Query rows of a cached head of a group up to which attend() takes them.  us a call, attend() : tcgen05, 16
// heads of 128: 8 rows over 65536 keys 64 : 146; 32 rows over 4096 31 : 44, over 65536 171 : 159; 64 rows over
// 4096 46 : 60, over 16384 104 : 82, over 65536 317 : 168.
constexpr int64_t kFewRows = 32;
// What a call must be able to reach for the sharing to pay: keys a sequence, and bytes of codes of all of them.
// us a call, without sharing : with it, 4 beams of 16 heads of 128: 512 keys 8.7 : 14.8, 2048 keys 17.8 : 15.4; 16 such
// groups in a window of 512 keys 27 : 31, over 2048 keys 89 : 45; 8 beams of 10 heads of 64 over 1024 keys 13.4 : 14.5,
// over 2048 15.6 : 14.8.
constexpr int64_t kSReach = 1024, kSBytes = 16 << 20;
// attend() takes kEvenBatch sequences at most; of more, groups of few rows take tcgen05 where at least so many sequences
// share. us a call, without sharing : on tcgen05, 600 to 640 sequences of 8 heads of 128, bf16: groups of 2 over 4096 keys 609 : 1236,
// of 4 603 : 647, of 8 635 : 378 (over 1024 keys 181 : 153), of 16 635 : 225; 4 heads of 64, of 4 251 : 200, of 8 250 : 126 (72 : 63);
// float32 within a few percent of that. One head of 128 in groups of 8: 114 : 82 over 4096 keys, 40 : 53 over 1024.
constexpr int64_t kSMany = 8;
constexpr int64_t kSJoinRows = 1024;    // rows from which on a warp joins one alone
struct SharedPlan { bool use, few; Plan rest; int rows, row_tiles, rows_cap, copies, ctas; int64_t stride, info, rest_info, part, rest_part, bytes; };

SharedPlan shared_plan(int dtype, int64_t B, int64_t groups, int64_t T, int64_t G, int64_t H, int64_t D, int64_t page, int64_t n_blocks,
                       int64_t window) {
    SharedPlan p{};
    const int64_t K = B / groups, rows = K * T * G;
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    p.rows = (int)std::min<int64_t>(rows, 1 << 20);
    int64_t reach = n_blocks * page;
    if (window >= 0) reach = std::min(reach, window + T);
    p.few = rows <= kFewRows && T * G <= kRows && B <= kEvenBatch;
    const bool tiles = groups <= kSGroups && rows <= (1 << 20) && (rows > kFewRows || T * G > kRows || K >= kSMany);
    p.use = K > 1 && reach >= kSReach && B * H * reach * 2 * D >= kSBytes && (p.few || tiles);
    if (!p.use) return p;
    p.info = up((2 * groups + 2) * 8);
    if (p.few) {
        p.row_tiles = (int)((rows + kRows - 1) / kRows);
        p.rest_info = up((B + 1) * 4);
        p.ctas = 8 * 148;
        p.rest_part = up((groups * H * p.row_tiles + B * H + p.ctas) * kRows * (D + 2) * 4);
        p.bytes = p.info + p.rest_info + p.rest_part;
        return p;
    }
    p.rest = plan_of(B, T, G, H, D, page, n_blocks, window);
    if (!p.rest.even && p.rest.warps == 8) p.rest.splits = 1;
    p.row_tiles = (int)((rows + kSRows - 1) / kSRows);
    p.rows_cap = (int)std::min<int64_t>(rows, kSRows);
    const bool two = dtype == NT_BF16 ? true : D == 64;
    p.ctas = 148 * (two ? 2 : 1);
    p.rest_info = p.rest.even ? up((B + 1) * 4) : 0;
    p.copies = p.rows_cap <= 32 ? 4 : p.rows_cap <= 64 ? 2 : 1;
    p.stride = (p.copies * p.rows_cap * (D + 2) + 3) / 4 * 4;      // written 16 bytes at a time
    p.part = up((groups * H * p.row_tiles + p.ctas) * p.stride * 4);
    const int64_t slots = p.rest.even ? B * H + p.rest.even : B * H * p.rest.row_tiles * p.rest.splits;
    p.rest_part = up(slots * kRows * (D + 2) * 4);
    p.bytes = p.info + p.rest_info + p.part + p.rest_part;
    return p;
}

int launch_after(const void* kernel, const char* name, dim3 grid, dim3 block, size_t smem, void** args, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NT_ERR_CUDA, "%s launch failed: %s", name, cudaGetErrorString(e));
    }
    return check_launch(name);
}

template <int DT, int D, int HOW>
int launch_shared_join(const SharedArgs& s, int ctas, cudaStream_t stream) {
    SharedArgs args = s;
    void* two[] = {&args, &ctas};
    const int64_t rows = (int64_t)s.B * s.a.T * s.a.H * s.a.G;
    const bool one_warp = rows >= kSJoinRows;
    const void* f = one_warp ? (const void*)kv_shared_join_kernel<DT, D, HOW, 1> : (const void*)kv_shared_join_kernel<DT, D, HOW, kSJoinWarps>;
    return launch_after(f, "kv_shared_join_kernel", dim3((unsigned)(one_warp ? (rows + kSJoinWarps - 1) / kSJoinWarps : rows)),
                        dim3(kSJoinWarps * 32), 0, two, stream);
}

template <int DT, int D, bool HALF_C, bool HALF_R>
int launch_few(const SharedArgs& s, cudaStream_t stream) {
    const size_t smem = std::max(kRingBytes<D, 2>, sizeof(float) * 2 * kRows * (D + 2));
    kv_few_kernel<DT, D, HALF_C, HALF_R><<<s.ctas, 64, smem, stream>>>(s);
    const int rc = check_launch("kv_few_kernel");
    return rc != NT_OK ? rc : launch_shared_join<DT, D, ALL_IN_SHARES>(s, s.ctas, stream);
}

template <int DT, int D, int W, bool HALF>
int launch_rest(const SharedArgs& s, const SharedPlan& p, cudaStream_t stream) {
    const size_t smem = std::max(kRingBytes<D, W>, sizeof(float) * W * kRows * (D + 2));
    SharedArgs args = s;
    void* one[] = {&args};
    if constexpr (W == 2) {
        if (p.rest.even) {
            const int rc = launch_after((const void*)kv_rest_even_kernel<DT, D, W, HALF>, "kv_rest_even_kernel", dim3(p.rest.even), dim3(W * 32), smem, one, stream);
            return rc != NT_OK ? rc : launch_shared_join<DT, D, REST_IN_SHARES>(s, p.rest.even, stream);
        }
    }
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_rest_kernel<DT, D, W, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_kv_attention_shared: %s", cudaGetErrorString(e));
    }
    const dim3 grid((unsigned)s.a.splits, (unsigned)(s.a.H * s.a.row_tiles), (unsigned)s.B);
    const int rc = launch_after((const void*)kv_rest_kernel<DT, D, W, HALF>, "kv_rest_kernel", grid, dim3(W * 32), smem, one, stream);
    return rc != NT_OK ? rc : launch_shared_join<DT, D, REST_IN_CHUNKS>(s, 0, stream);
}

template <int DT, int D>
int launch_shared(const SharedArgs& s, const SharedPlan& p, cudaStream_t stream) {
    if (p.few) {
        if (p.rows <= kRows / 2) return launch_few<DT, D, true, true>(s, stream);
        return 2 * s.a.T * s.a.G <= kRows ? launch_few<DT, D, false, true>(s, stream) : launch_few<DT, D, false, false>(s, stream);
    }
    using Cfg = SharedCfg<DT, D>;
    const cudaError_t e = cudaFuncSetAttribute(kv_shared_kernel<DT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kBytes);
    if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_kv_attention_shared: %s", cudaGetErrorString(e));
    kv_shared_kernel<DT, D><<<p.ctas, kSThreads, Cfg::kBytes, stream>>>(s);
    const int rc = check_launch("kv_shared_kernel");
    if (rc != NT_OK) return rc;
    const bool half = 2 * s.a.T * s.a.G <= kRows;
    if (p.rest.warps == 8) return half ? launch_rest<DT, D, 8, true>(s, p, stream) : launch_rest<DT, D, 8, false>(s, p, stream);
    return half ? launch_rest<DT, D, 2, true>(s, p, stream) : launch_rest<DT, D, 2, false>(s, p, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_kv_attention_shared_workspace_bytes(int dtype, int64_t B, int64_t groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                               int64_t page, int64_t n_blocks, int64_t window) {
    if (B < 1 || groups < 1 || B % groups || T < 1 || Hkv < 1 || Hq < Hkv || D < 1 || page < 1 || n_blocks < 0) return 0;
    const SharedPlan p = shared_plan(dtype, B, groups, T, Hq / Hkv, Hkv, D, page, n_blocks, window);
    return p.use ? p.bytes : nt_kv_attention_workspace_bytes(B, T, Hq, Hkv, D, page, n_blocks, window);
}

int nt_kv_attention_shared(int dtype, int64_t B, int64_t groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t page,
                           int64_t n_pages, int64_t n_blocks, int64_t window, float scale, const void* q, int64_t q_sb, int64_t q_st,
                           int64_t q_sh, const void* k_codes, const float* k_scale, const void* v_codes, const float* v_scale,
                           const int32_t* table, int64_t table_sb, const int32_t* lengths, const int32_t* counts,
                           const int32_t* shared, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
    if (groups < 1 || B < 0 || B % groups) return fail(NT_ERR_ARG, "nt_kv_attention_shared: %lld sequences in %lld groups", (long long)B, (long long)groups);
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_kv_attention_shared: dtype %d", dtype);
    if (D != 64 && D != 128) return fail(NT_ERR_ARG, "nt_kv_attention_shared: head_dim %lld (64 or 128 supported)", (long long)D);
    if (page != 16 && page != 32 && page != 64)
        return fail(NT_ERR_ARG, "nt_kv_attention_shared: page of %lld tokens (16, 32 or 64 supported)", (long long)page);
    if (T < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv || n_pages < 0 || n_blocks < 0 || B > 65535 || T > (1 << 20) || Hq > 65535 ||
        n_blocks * page > (int64_t)INT32_MAX - 4096)
        return fail(NT_ERR_ARG, "nt_kv_attention_shared: bad sizes");
    if (B == 0 || T == 0) return NT_OK;
    if (!q || !k_codes || !k_scale || !v_codes || !v_scale || !table || !lengths || !shared || !out)
        return fail(NT_ERR_ARG, "nt_kv_attention_shared: null pointer");
    if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15)
        return fail(NT_ERR_ARG, "nt_kv_attention_shared: codes need 16-byte alignment");
    const int64_t G = Hq / Hkv;
    const SharedPlan p = shared_plan(dtype, B, groups, T, G, Hkv, D, page, n_blocks, window);
    if (!p.use)
        return nt_kv_attention(dtype, B, T, Hq, Hkv, D, page, n_pages, n_blocks, window, scale, q, q_sb, q_st, q_sh, k_codes, k_scale,
                               v_codes, v_scale, table, table_sb, lengths, counts, out, workspace, workspace_bytes, stream);
    if ((!p.few && Hkv * p.rest.row_tiles > 65535) || B * T * Hq > INT32_MAX)
        return fail(NT_ERR_ARG, "nt_kv_attention_shared: %lld query rows in one call", (long long)(T * Hq));
    if (!workspace || workspace_bytes < p.bytes)
        return fail(NT_ERR_WORKSPACE, "nt_kv_attention_shared: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)p.bytes);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(NT_ERR_ARG, "nt_kv_attention_shared: the workspace needs 16-byte alignment");
    int dev = 0;
    cudaGetDevice(&dev);
    SharedArgs s{};
    KvAttnArgs& a = s.a;
    a.T = (int)T; a.G = (int)G; a.H = (int)Hkv;
    a.page_shift = page == 16 ? 4 : page == 32 ? 5 : 6;
    a.n_pages = n_pages; a.n_blocks = n_blocks;
    a.window = window < 0 ? -1 : (int)std::min<int64_t>(window, INT32_MAX / 2);
    a.chunk = p.rest.chunk; a.splits = p.rest.splits; a.row_tiles = p.rest.row_tiles;
    a.scale_log2 = scale * kLog2e;
    a.q = q; a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
    const int64_t es = dtype == NT_F32 ? 4 : 2;
    a.q_vec = ((reinterpret_cast<uintptr_t>(q) | (uint64_t)((q_sb | q_st | q_sh) * es)) & 15) == 0;
    a.kc = static_cast<const uint8_t*>(k_codes); a.ks = k_scale;
    a.vc = static_cast<const uint8_t*>(v_codes); a.vs = v_scale;
    a.table = table; a.table_sb = table_sb; a.lengths = lengths; a.counts = counts;
    a.out = out;
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_attention_shared: error word unavailable");
    s.B = (int)B; s.groups = (int)groups; s.K = a.beams = (int)(B / groups);
    s.rows = p.rows; s.row_tiles = p.row_tiles; s.rows_cap = p.rows_cap; s.copies = p.copies; s.stride = p.stride; s.ctas = p.ctas;
    s.shared = shared;
    char* ws = static_cast<char*>(workspace);
    s.info = reinterpret_cast<int64_t*>(ws);
    s.rest_info = reinterpret_cast<int32_t*>(ws + p.info);
    s.part = reinterpret_cast<float*>(ws + p.info + p.rest_info);
    a.part = reinterpret_cast<float*>(ws + p.info + p.rest_info + p.part);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32) return D == 64 ? launch_shared<NT_F32, 64>(s, p, st) : launch_shared<NT_F32, 128>(s, p, st);
    return D == 64 ? launch_shared<NT_BF16, 64>(s, p, st) : launch_shared<NT_BF16, 128>(s, p, st);
}

}  // extern "C"
