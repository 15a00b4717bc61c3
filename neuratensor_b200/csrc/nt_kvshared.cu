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
// bf16 outputs) or three (24 bits).  Weights are 1 at the row's reference, which follows
// its maximum when that is 2^8 larger, and values are divided by 2^32, so that sums of finite
// ones stay finite; values below 2^-94 lose bits by it, 2^-102 at most.
//
// A CTA: four warps of softmax (a thread a row), of which one thread issues the products, and
// four that load codes one tile ahead, convert them and write the operands (K as it lies, V
// transposed by stmatrix, its dimensions in an order of their own that the join undoes).  Two
// CTAs share an SM where they fit, so that one's products run under the other's softmax.  The
// tiles of all groups and heads in a row are cut into even shares, one a CTA.
#include "nt_kvattn.cuh"

#include <cuda_bf16.h>

namespace nt {
namespace {

using namespace kva;

constexpr int kSRows = 128;            // query rows of a tile
constexpr int kSKeys = 128;            // keys of a tile
constexpr int kSGroups = 512;          // groups of a call
constexpr int kSoftWarps = 4, kLoadWarps = 4;
constexpr int kSThreads = 32 * (kSoftWarps + kLoadWarps);
constexpr float kSUp = 4294967296.f;   // 2^32: values are held divided by it
constexpr float kSLag = 8.f;           // a maximum this much (log2) above the reference moves it

struct SharedArgs {
    KvAttnArgs a;                      // a.part: the rest's partial rows
    int B, groups, K;                  // sequences, groups, sequences of a group
    int rows, row_tiles, rows_cap;     // query rows of a cached head of a group, tiles of them, rows of a partial tile
    int64_t stride;                    // floats of a partial tile
    int ctas;
    const int32_t* shared;
    int64_t* info;                     // [groups][2]: tiles per head before the group, lo | hi << 32; then the total
    float* part;                       // partial tiles: [rows_cap][D] means, [rows_cap] references, [rows_cap] totals
};

// The keys [lo, hi) that the rows of a group have in common and all see, in whole tiles of 16.
struct Common { int lo, hi; };
// One sequence's part in it; a sequence without new tokens has none.
__device__ __forceinline__ bool common_of(const SharedArgs& s, int b, int* lo, int* hi) {
    const int len = s.a.lengths[b], cnt = s.a.counts ? s.a.counts[b] : s.a.T;
    if (cnt <= 0 || cnt > s.a.T || len < cnt || len > (s.a.n_blocks << s.a.page_shift)) return false;
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
// 32 lanes x 32 columns, a thread a lane
__device__ __forceinline__ void s_ld32(uint32_t at, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void s_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at) : "memory");
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

struct SharedBars { uint64_t k_full, v_full, s_full, p_full, o_done, q_full; };

template <int DT, int D>
__global__ void __launch_bounds__(kSThreads, SharedCfg<DT, D>::kPerSm) kv_shared_kernel(const __grid_constant__ SharedArgs s) {
    using Cfg = SharedCfg<DT, D>;
    using El = Elem<DT>;
    using T = typename El::T;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ SharedBars bars;
    __shared__ uint32_t tmem_base;
    __shared__ float k_scale[2][kSKeys / kTile];        // of a tile's blocks of 16 keys; < 0: not to be seen
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
        // ---------------- queries, softmax, results: a thread a row ----------------
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        const uint32_t qs = smem_u32(q_smem), ks_smem = smem_u32(k_smem), vs_smem = smem_u32(v_smem);
        int it = 0, seg = 0, g = 0;
        bool ok = true;
        for (int64_t at = begin; at < end && ok; ++seg) {
            const Segment e = segment(at, g);
            g = e.g;
            const int row = e.rt * kSRows + tid, rows = min(kSRows, s.rows - e.rt * kSRows);
            const bool busy = warp * 32 < rows;          // this warp has rows
            float f_row = 0.f;
            {
                const int beam = row / (a.T * a.G), t = row / a.G % a.T;
                const int64_t b = (int64_t)e.g * s.K + beam;
                int lo, hi;
                const bool live = row < s.rows && common_of(s, (int)b, &lo, &hi) && t < (a.counts ? a.counts[b] : a.T);
                const T* q = static_cast<const T*>(a.q) + (live ? b * a.q_sb + (int64_t)t * a.q_st + (int64_t)(e.h * a.G + row % a.G) * a.q_sh : 0);
                auto read8 = [&](int d, float (&v)[8]) {
                    if (!live) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = 0.f;
                    } else if (a.q_vec) {
                        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
                        for (int i = 0; i < 8; i += E) {
                            const uint4 w = __ldg(reinterpret_cast<const uint4*>(q + d + i));
                            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
                            for (int j = 0; j < E; ++j) v[i + j] = El::to_f(x[j]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = El::load(q + d + i);
                    }
                };
                float amax = 0.f;
#pragma unroll 4
                for (int d = 0; d < D; d += 8) {
                    float v[8];
                    read8(d, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float m = fabsf(v[i]);
                        if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
                    }
                }
                // a power of two that brings the largest to [2^13, 2^14); the scores' scale is positive, its sign the query's
                int x = 127 + 13 - (int)(__float_as_uint(amax) >> 23);
                x = amax > 0.f ? (x > 126 ? 126 : x) : 0;
                float up = __uint_as_float((uint32_t)(127 + x) << 23);
                f_row = __uint_as_float((uint32_t)(127 - x) << 23) * fabsf(a.scale_log2);
                if (a.scale_log2 < 0.f) up = -up;
#pragma unroll 2
                for (int d = 0; d < D; d += 8) {
                    float v[8];
                    read8(d, v);
                    uint32_t hi[4], lo4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x0 = v[2 * i] * up, x1 = v[2 * i + 1] * up;
                        hi[i] = pack_h2(x0, x1);
                        const float2 r = unpack_h2(hi[i]);
                        lo4[i] = pack_h2(x0 - r.x, x1 - r.y);
                    }
                    const int at8 = (d / 64) * (kSRows * 128) + tid * 128 + (((d % 64 / 8) ^ (tid & 7)) << 4);
                    *reinterpret_cast<uint4*>(q_smem + at8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (Cfg::NQ == 2) *reinterpret_cast<uint4*>(q_smem + Cfg::kQ + at8) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.q_full));

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
                    const float* ks = k_scale[it & 1];
                    float mx = -INFINITY;
#pragma unroll
                    for (int c = 0; c < kSKeys / 32; ++c) {
                        float v[32];
                        s_ld32(lanes + c * 32, v);
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const float k = ks[2 * c + n];
                            if (k >= 0.f) {
                                float x = v[16 * n];
#pragma unroll
                                for (int i = 1; i < 16; ++i) x = fmaxf(x, v[16 * n + i]);
                                mx = fmaxf(mx, x * (f_row * k));
                            }
                        }
                    }
                    const bool move = mx > m + kSLag;
                    if (__any_sync(0xffffffffu, move)) {
                        const float next = move ? mx : m, f = m == -INFINITY ? 0.f : ex2(m - next);
                        const float by = move ? f : 1.f;
                        if (tile > e.first) {
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) {
                                float v[32];
                                s_ld32(lanes + Cfg::kColO + c * 32, v);
                                uint32_t w[16];
#pragma unroll
                                for (int n = 0; n < 2; ++n) {
#pragma unroll
                                    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[16 * n + i] * by);
                                    s_st16(lanes + Cfg::kColO + c * 32 + 16 * n, w);
                                }
                            }
                        }
                        l *= by;
                        m = next;
                    }
                    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int c = 0; c < kSKeys / 32; ++c) {
                        float v[32];
                        s_ld32(lanes + c * 32, v);
                        uint32_t w0[16], w1[16], w2[16];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const float k = ks[2 * c + n], f = f_row * k;
                            const bool seen = k >= 0.f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float p0 = seen ? ex2(fmaf(v[16 * n + 2 * i], f, -base)) : 0.f;
                                const float p1 = seen ? ex2(fmaf(v[16 * n + 2 * i + 1], f, -base)) : 0.f;
                                l += p0 + p1;
                                const uint32_t h = pack_b2(p0, p1);
                                const float r0 = p0 - __uint_as_float(h << 16), r1 = p1 - __uint_as_float(h & 0xffff0000u);
                                const uint32_t h2 = pack_b2(r0, r1);
                                w0[8 * n + i] = h;
                                w1[8 * n + i] = h2;
                                if constexpr (Cfg::NP == 3)
                                    w2[8 * n + i] = pack_b2(r0 - __uint_as_float(h2 << 16), r1 - __uint_as_float(h2 & 0xffff0000u));
                            }
                        }
                        s_st16(lanes + c * 32, w0);
                        s_st16(lanes + c * 32 + 16, w1);
                        if constexpr (Cfg::NP == 3) s_st16(lanes + Cfg::kCol3 + c * 16, w2);
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
                                s_mma_ts(tmem + Cfg::kColO, tmem + (p == 2 ? Cfg::kCol3 + k * 8 : k / 2 * 32 + k % 2 * 8 + p * 16),
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
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float v[32];
                    s_ld32(lanes + Cfg::kColO + c * 32, v);
                    if (tid < rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<float4*>(part + tid * D + c * 32 + i) =
                                make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
                    }
                }
                if (tid < rows) {
                    part[s.rows_cap * D + tid] = m;
                    part[s.rows_cap * D + s.rows_cap + tid] = l * (float)(1 << (int)kPShift);      // as attend() leaves it
                }
            }
            s_fence_before();
            at += e.last - e.first;
        }
    } else {
        // ---------------- codes: global memory -> registers -> operands ----------------
        constexpr int CH = D / 16;                      // 16-code pieces of a key
        constexpr int N = kSKeys * CH / (32 * kLoadWarps);      // of a thread, K and V each
        const int w = warp - kSoftWarps, lt = w * 32 + lane;
        // the tile whose codes are in registers, and what lane j < 8 knows of its j-th block of 16 keys
        struct Pages { int page; float ks, vs; };
        uint4 kr[N], vr[N];
        int64_t at = begin;
        Segment e = segment(at, 0);
        auto advance = [&]() {                          // to the next tile; false behind the last
            ++at;
            if (at >= end) return false;
            if (++e.first >= e.last) e = segment(at, e.g);
            return true;
        };
        bool bad_page = false;
        auto look_up = [&]() {
            Pages p{-1, -1.f, 0.f};
            const int key = c_lo[e.g] + e.first * kSKeys + lane * kTile;
            if (lane < kSKeys / kTile && key < c_hi[e.g]) {
                const int pg = a.table[(int64_t)c_lead[e.g] * a.table_sb + (key >> a.page_shift)];
                if (pg < 0 || pg >= a.n_pages) {
                    bad_page = true;
                } else {
                    p.page = pg;
                    p.ks = __ldg(a.ks + (int64_t)pg * a.H + e.h);
                    p.vs = __ldg(a.vs + (int64_t)pg * a.H + e.h);
                }
            }
            return p;
        };
        // K piece j of a thread: key (j * threads + lt) / CH; V piece j of a warp: 8 keys x 64 dimensions, key of the lane's quarter
        auto k_key = [&](int j) { return (j * 32 * kLoadWarps + lt) / CH; };
        auto v_unit = [&](int j) { return j * kLoadWarps + w; };
        auto code_at = [&](const uint8_t* codes, int pg, int key, int dim) {
            const int slot = (c_lo[e.g] + e.first * kSKeys + key) & ((1 << a.page_shift) - 1);
            return __ldg(reinterpret_cast<const uint4*>(codes + ((((int64_t)pg * a.H + e.h) << a.page_shift) + slot) * D + dim));
        };
        auto load_k = [&](const Pages& p) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int key = k_key(j), pg = __shfl_sync(0xffffffffu, p.page, key / kTile);
                kr[j] = pg >= 0 ? code_at(a.kc, pg, key, lt % CH * 16) : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_v = [&](const Pages& p) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = v_unit(j), key = u / (D / 64) * 8 + lane / 4;
                const int pg = __shfl_sync(0xffffffffu, p.page, key / kTile);
                vr[j] = pg >= 0 ? code_at(a.vc, pg, key, u % (D / 64) * 64 + lane % 4 * 16) : make_uint4(0, 0, 0, 0);
            }
        };
        Pages now = look_up(), next{};
        load_k(now);
        load_v(now);
        bool more = true;
        for (int it = 0; more; ++it) {
            bool ok = it == 0 || __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.s_full), (it - 1) & 1));
            if (!ok) {
                if (lane == 0) atomicOr(a.err, ERRF_TIMEOUT_PRODUCER);
                break;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int key = k_key(j), c = lt % CH, panel = c / 4;
                const uint32_t words[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
                uint4 h[2];
                h[0] = make_uint4(cvt_lo(words[0]), cvt_hi(words[0]), cvt_lo(words[1]), cvt_hi(words[1]));
                h[1] = make_uint4(cvt_lo(words[2]), cvt_hi(words[2]), cvt_lo(words[3]), cvt_hi(words[3]));
                unsigned char* base = k_smem + panel * (kSKeys * 128) + key * 128;
                // panel 1 writes its odd chunk first, so that eight lanes meet eight banks
                const int o = panel & 1, ch = c % 4 * 2;
                *reinterpret_cast<uint4*>(base + (((ch + o) ^ (key & 7)) << 4)) = o ? h[1] : h[0];
                *reinterpret_cast<uint4*>(base + (((ch + 1 - o) ^ (key & 7)) << 4)) = o ? h[0] : h[1];
            }
            if (w == 0 && lane < kSKeys / kTile) k_scale[it & 1][lane] = now.ks;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.k_full));
            const float vs = now.vs * (1.f / kSUp);
            more = advance();
            if (more) {
                next = look_up();
                load_k(next);
            }
            ok = it == 0 || __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.o_done), (it - 1) & 1));
            if (!ok) {
                if (lane == 0) atomicOr(a.err, ERRF_TIMEOUT_PRODUCER);
                break;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = v_unit(j), ko = u / (D / 64), half = u % (D / 64);
                const float f = __shfl_sync(0xffffffffu, vs, ko / 2);
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
            if (more) {
                now = next;
                load_v(now);
            }
        }
        if (bad_page) atomicOr(a.err, ERRF_BAD_ARG);
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
        attend<DT, D, W, HALF, true>(a, b, h, row_tile, e, first, last, part, smem);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the join follows this kernel alone, and needs the one before too
}

// Tiles per head of the sequences before i, for i <= B, by all threads of a CTA, with the groups' common keys.
__device__ __forceinline__ void rest_before(const SharedArgs& s, int* before, int* c_lo, int* c_hi, bool flag) {
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
                n = e.tiles;
                if (e.bad && flag) atomicOr(s.a.err, ERRF_BAD_ARG);
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
}

// In even shares, for ragged sequences (see kv_attention_even_kernel): two partial rows a CTA.
template <int DT, int D, int W, bool HALF>
__global__ void __launch_bounds__(W * 32, 16 / W) kv_rest_even_kernel(const __grid_constant__ SharedArgs s) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int before[kEvenBatch + 1], c_lo[kEvenBatch], c_hi[kEvenBatch];
    const KvAttnArgs& a = s.a;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    rest_before(s, before, c_lo, c_hi, blockIdx.x == 0);
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
        attend<DT, D, W, HALF, true>(a, b, h, 0, e, first, last, a.part + ((int64_t)b * a.H + h + blockIdx.x) * (kRows * (D + 2)), smem);
        at += last - first;
        __syncthreads();                                // the sums are read before the next ring is filled
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------------------
// Joins a query row's parts: those of the shared tiles, then those of the rest.
// ---------------------------------------------------------------------------
constexpr int kSJoinWarps = 8;
template <int DT, int D, bool EVEN>
__global__ void __launch_bounds__(kSJoinWarps * 32) kv_shared_join_kernel(const __grid_constant__ SharedArgs s, int rest_ctas) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int E = D / 32;
    const KvAttnArgs& a = s.a;
    const int heads = a.H * a.G, t = blockIdx.x / heads, hq = blockIdx.x % heads, h = hq / a.G;
    const int64_t b = blockIdx.z;
    const int g = (int)b / s.K, beam = (int)b % s.K;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kPart = kRows * (D + 2);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t info0 = s.info[2 * g], info1 = s.info[2 * g + 1], info2 = s.info[2 * g + 2];
    const Common c{(int)(uint32_t)info1, (int)(info1 >> 32)};
    const int cnt = a.counts ? a.counts[b] : a.T;
    // the shared tiles
    const int srow = (beam * a.T + t) * a.G + hq % a.G, rt = srow / kSRows;
    const int64_t per_head = (int64_t)a.H * s.row_tiles, share = (s.info[2 * s.groups] * per_head + s.ctas - 1) / s.ctas;
    const int64_t tiles = info2 - info0, item = (int64_t)g * per_head + (int64_t)h * s.row_tiles + rt;
    int n1 = 0;
    const int64_t step1 = s.stride;
    const float* part1 = s.part;
    if (tiles > 0) {
        const int64_t g0 = info0 * per_head + ((int64_t)h * s.row_tiles + rt) * tiles, c0 = g0 / share;
        n1 = (int)((g0 + tiles - 1) / share - c0 + 1);
        part1 += (item + c0) * step1;
    }
    const int r1 = srow % kSRows;
    // the rest
    const int row = t * a.G + hq % a.G, row_tile = row / kRows, r2 = row % kRows;
    int n2 = 0;
    const float* part2 = a.part;
    if constexpr (EVEN) {
        __shared__ int before[kEvenBatch + 1], c_lo[kEvenBatch], c_hi[kEvenBatch];
        rest_before(s, before, c_lo, c_hi, false);
        const int64_t sh = share_of((int64_t)before[s.B] * a.H, rest_ctas);
        const int n = before[b + 1] - before[b];
        if (n > 0) {
            const int64_t g0 = (int64_t)before[b] * a.H + (int64_t)h * n, c0 = g0 / sh;
            n2 = (int)((g0 + n - 1) / sh - c0 + 1);
            part2 += (b * a.H + h + c0) * kPart;
        }
    } else {
        const Span e = rest_of(s, b, row_tile, c);
        n2 = (e.tiles + a.chunk - 1) / a.chunk;
        part2 += (b * (int64_t)(a.H * a.row_tiles) + h * a.row_tiles + row_tile) * a.splits * kPart;
    }
    const bool live = cnt > 0 && t < cnt && cnt <= a.T && a.lengths[b] >= cnt && a.lengths[b] <= (a.n_blocks << a.page_shift);
    const int n = live ? n1 + n2 : 0;
    auto ref_of = [&](int i, float* l) {
        const float* p = i < n1 ? part1 + i * step1 + (int64_t)s.rows_cap * D + r1 : part2 + (int64_t)(i - n1) * kPart + kRows * D + r2;
        *l = p[i < n1 ? s.rows_cap : kRows];
        return *p;
    };
    // the row's reference and total: every warp takes them from all parts
    float m = -INFINITY, tot = 0.f;
    for (int i = lane; i < n; i += 32) {
        float li;
        const float mi = ref_of(i, &li), up = fmaxf(m, mi), base = up == -INFINITY ? 0.f : up;
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
#pragma unroll 4
    for (int i = warp; i < n; i += kSJoinWarps) {
        float li;
        const float mi = ref_of(i, &li), f = ex2(mi - base) * li * inv;
        float v[E];
        if (i < n1) {
            const float* p = part1 + i * step1 + (int64_t)r1 * D;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 x = *reinterpret_cast<const float2*>(p + column_of(lane * E + e));
                v[e] = x.x;
                v[e + 1] = x.y;
            }
        } else {
            const float* p = part2 + (int64_t)(i - n1) * kPart + r2 * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 x = *reinterpret_cast<const float2*>(p + e);
                v[e] = x.x;
                v[e + 1] = x.y;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = fmaf(f, v[e], sum[e]);
    }
    __shared__ float ws[kSJoinWarps][D];
#pragma unroll
    for (int e = 0; e < E; ++e) ws[warp][lane * E + e] = sum[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kSJoinWarps * 32) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kSJoinWarps; ++w) x += ws[w][d];
        static_cast<T*>(a.out)[((b * a.T + t) * (int64_t)heads + hq) * D + d] = El::from_f(live && tot != 0.f ? x : 0.f);
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct SharedPlan { bool use; Plan rest; int rows, row_tiles, rows_cap, ctas; int64_t stride, info, part, rest_part, bytes; };

SharedPlan shared_plan(int dtype, int64_t B, int64_t groups, int64_t T, int64_t G, int64_t H, int64_t D, int64_t page, int64_t n_blocks,
                       int64_t window) {
    SharedPlan p{};
    const int64_t K = B / groups, rows = K * T * G;
    p.use = K > 1 && groups <= kSGroups && rows <= (1 << 20);
    if (!p.use) return p;
    p.rest = plan_of(B, T, G, H, D, page, n_blocks, window);
    if (!p.rest.even && p.rest.warps == 8) p.rest.splits = 1;
    p.rows = (int)rows;
    p.row_tiles = (int)((rows + kSRows - 1) / kSRows);
    p.rows_cap = (int)std::min<int64_t>(rows, kSRows);
    const bool two = dtype == NT_BF16 ? true : D == 64;
    p.ctas = 148 * (two ? 2 : 1);
    const int64_t align = 256;
    auto up = [&](int64_t x) { return (x + align - 1) / align * align; };
    p.info = up((2 * groups + 2) * 8);
    p.stride = (p.rows_cap * (D + 2) + 3) / 4 * 4;      // written 16 bytes at a time
    p.part = up((groups * H * p.row_tiles + p.ctas) * p.stride * 4);
    const int64_t slots = p.rest.even ? B * H + p.rest.even : B * H * p.rest.row_tiles * p.rest.splits;
    p.rest_part = up(slots * kRows * (D + 2) * 4);
    p.bytes = p.info + p.part + p.rest_part;
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

template <int DT, int D, int W, bool HALF>
int launch_rest(const SharedArgs& s, const SharedPlan& p, cudaStream_t stream) {
    const size_t smem = std::max(kRingBytes<D, W>, sizeof(float) * W * kRows * (D + 2));
    SharedArgs args = s;
    int ctas = p.rest.even;
    void* one[] = {&args};
    void* two[] = {&args, &ctas};
    const dim3 join((unsigned)(s.a.T * s.a.H * s.a.G), 1, (unsigned)s.B);
    if constexpr (W == 2) {
        if (p.rest.even) {
            const int rc = launch_after((const void*)kv_rest_even_kernel<DT, D, W, HALF>, "kv_rest_even_kernel", dim3(ctas), dim3(W * 32), smem, one, stream);
            return rc != NT_OK ? rc : launch_after((const void*)kv_shared_join_kernel<DT, D, true>, "kv_shared_join_kernel", join, dim3(kSJoinWarps * 32), 0, two, stream);
        }
    }
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_rest_kernel<DT, D, W, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_kv_attention_shared: %s", cudaGetErrorString(e));
    }
    const dim3 grid((unsigned)s.a.splits, (unsigned)(s.a.H * s.a.row_tiles), (unsigned)s.B);
    const int rc = launch_after((const void*)kv_rest_kernel<DT, D, W, HALF>, "kv_rest_kernel", grid, dim3(W * 32), smem, one, stream);
    return rc != NT_OK ? rc : launch_after((const void*)kv_shared_join_kernel<DT, D, false>, "kv_shared_join_kernel", join, dim3(kSJoinWarps * 32), 0, two, stream);
}

template <int DT, int D>
int launch_shared(const SharedArgs& s, const SharedPlan& p, cudaStream_t stream) {
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
    if (Hkv * p.rest.row_tiles > 65535 || T * Hq > INT32_MAX)
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
    s.B = (int)B; s.groups = (int)groups; s.K = (int)(B / groups);
    s.rows = p.rows; s.row_tiles = p.row_tiles; s.rows_cap = p.rows_cap; s.stride = p.stride; s.ctas = p.ctas;
    s.shared = shared;
    char* ws = static_cast<char*>(workspace);
    s.info = reinterpret_cast<int64_t*>(ws);
    s.part = reinterpret_cast<float*>(ws + p.info);
    a.part = reinterpret_cast<float*>(ws + p.info + p.part);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32) return D == 64 ? launch_shared<NT_F32, 64>(s, p, st) : launch_shared<NT_F32, 128>(s, p, st);
    return D == 64 ? launch_shared<NT_BF16, 64>(s, p, st) : launch_shared<NT_BF16, 128>(s, p, st);
}

}  // extern "C"
