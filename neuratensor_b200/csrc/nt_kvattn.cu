// Attention of the new tokens over the paged 8-bit cache (nt_kvcache.cu).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,  k = ks[page, head] * code, v alike,
// query row t of sequence b at position p = len - cnt + t sees j <= p and, with
// a window, j >= p - window.
//
// Bound by HBM: a step reads every visible code once (one byte per element)
// and does two flops per query row with it.  Each warp streams its own tiles of
// 16 keys through a ring in shared memory (16-byte cp.async, one tile ahead of
// the arithmetic, no barrier between warps), and the tensor cores (mma m16n8k16,
// f16 in, float32 sums) do the products that would cost the CUDA cores a
// conversion and an FMA per element.  The cached operand is the 16-row one of
// each product (keys of K, then dimensions of V^T), the query rows of one cached
// head the 8 columns: up to eight shared heads of a step, or a draft of a few
// tokens.  e4m3 codes are exact in f16, and so is a bf16 query of at least 2^-30
// of its row's largest (scaled to [2^13, 2^14), where f16 ends at 2^-24; rows whose
// largest is below 2^-113 are scaled by 2^126, which brings every bf16 number into
// f16).  float32
// queries, and the weights always, are split into two f16 (22 bits) and take
// their product twice.
//
// The k order of a product is free, so a lane takes 16 consecutive dimensions
// of a key (one 16-byte read) as its part of four k-steps, with q in the same
// order; likewise lane group g of V owns D/8 consecutive dimensions of the four
// keys whose probabilities the lane holds, which come from the first product by
// one 8x8 transpose per eight keys.
//
// Softmax is online, in float32, base 2: a warp keeps its rows' running
// maximum, sum and output over its tiles; the warps of a CTA join in shared
// memory, and the CTAs that share a head in a second kernel, in a fixed order.
// Probabilities are 2^14 p as a pair of f16, the second what the first leaves, for
// bf16 outputs too, so that these are a float32 result rounded once (one f16, off
// by 2^-12, changes one bf16 output in ten).  With four query rows of a cached head
// or fewer (HALF) the first halves take columns 0..3 of the product and the second
// ones columns 4..7, whose queries repeat the rows: the pair costs one select, and the
// kernels below take what they took with one f16 (34.9 us, 103.2 against 103.0).
// With more rows it is a second product (drafts of 5 rows 14.1 against 13.9 us; 107 to
// 116 against 124 for 8 tokens of 4 heads on 8 x 8 cached heads of up to 16384 keys).
//
// The kernel alone, caches flushed, for 64 streams of 16 bf16 heads of 128 with
// window 512 (134 MB of codes) / 8 ragged caches of up to 65536 tokens, 32 heads
// over 8: 34.9 / 101.7 us with a ring of two tiles, 36.0 / 104.7 with three,
// 43.5 / 125.5 with four (two ahead; 32 KB a CTA).
#include "nt_kernels.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace nt {
namespace {

constexpr int kRows = 8;               // query rows per CTA
constexpr int kTile = 16;              // keys per tile
constexpr float kPShift = 14.f;        // probabilities are held times 2^14
constexpr float kHuge = 3e38f;         // 448 of it is infinite; no power of two, so no block's scale

struct KvAttnArgs {
    int T, G, H, page_shift;           // tokens, query heads per cached head, cached heads, log2(page)
    int64_t n_pages, n_blocks;
    int window;                        // < 0: none
    int chunk;                         // tiles per CTA
    int splits, row_tiles;
    float scale_log2;
    const void* q; int64_t q_sb, q_st, q_sh; int q_vec;
    const uint8_t* kc; const float* ks; const uint8_t* vc; const float* vs;
    const int32_t* table; int64_t table_sb;
    const int32_t* lengths; const int32_t* counts;
    void* out;
    float* part;                       // partial rows: [kRows][D] means, [kRows] maxima, [kRows] totals
    unsigned* err;
};

// What the rows of one row tile see of their sequence: keys [lo, hi), in tiles from lo16.
struct Span { int cnt, start, lo, hi, lo16, tiles; bool bad; };

__device__ __forceinline__ Span span_of(const KvAttnArgs& a, int64_t b, int row_tile) {
    Span s;
    const int len = a.lengths[b];
    s.cnt = a.counts ? a.counts[b] : a.T;
    s.bad = s.cnt < 0 || s.cnt > a.T || len < s.cnt || len > (a.n_blocks << a.page_shift);
    if (s.bad) s.cnt = 0;
    s.start = len - s.cnt;
    const int t0 = row_tile * kRows / a.G, t1 = min((row_tile * kRows + kRows - 1) / a.G, s.cnt - 1);
    s.lo = s.hi = s.lo16 = s.tiles = 0;
    if (t0 < s.cnt) {
        const int p0 = s.start + t0;
        s.lo = a.window >= 0 && p0 > a.window ? p0 - a.window : 0;
        s.hi = s.start + t1 + 1;
        s.lo16 = s.lo & ~(kTile - 1);
        s.tiles = (s.hi - s.lo16 + kTile - 1) / kTile;
    }
    return s;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// two e4m3 codes (the low or the high half of w) to two f16 values, exactly
__device__ __forceinline__ uint32_t cvt_lo(uint32_t w) {
    uint32_t r;
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, a;}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t cvt_hi(uint32_t w) {
    uint32_t r;
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, b;}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ float rcp(float x) {            // of a power of two here, or near enough
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// an 8x8 matrix of f16, one row of two columns per lane, transposed
__device__ __forceinline__ uint32_t transpose(uint32_t w) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// A warp's ring: kStages tiles of 16 keys, K then V, rows of D bytes.  16-byte
// chunk c of a row is stored at chunk c ^ swizzle(row), so that the eight lanes
// that read together (K: two rows, four chunks; V: four even or four odd rows,
// two chunks) meet different banks.
constexpr int kStages = 2;
template <int D> constexpr int kTileBytes = kTile * D;
template <int D, int W> constexpr size_t kRingBytes = (size_t)W * kStages * 2 * kTileBytes<D>;
template <int D> __device__ __forceinline__ int k_swz(int row) { return D == 128 ? (row & 1) * 4 : 0; }
template <int D> __device__ __forceinline__ int v_swz(int row) { return D == 128 ? row & 6 : (row >> 1) & 3; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Tiles [first, last) of one row tile of head h, sequence b, by the W warps of a
// CTA: the rows themselves when these are all of its tiles, else their means over
// the tiles with their maxima and totals in `part`.  HALF: there are four rows or
// fewer; columns 4..7 repeat them and take the weights' second halves.
template <int DT, int D, int W, bool HALF>
__device__ __forceinline__ void attend(const KvAttnArgs& a, int64_t b, int h, int row_tile, const Span& s, int first,
                                       int last, float* part, unsigned char* smem) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int KS = D / 16;                 // k-steps of the first product
    constexpr int MT = D / 16;                 // 16-dimension tiles of the second
    constexpr bool kPair = DT == NT_F32;       // a second product with what f16 leaves of q
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    constexpr int kMask = HALF ? 3 : 7;
    const int row = row_tile * kRows + (g & kMask), t = row / a.G;
    const bool live = t < s.cnt;
    // in the products a lane holds rows 2c and 2c + 1: their positions
    const int t0 = (row_tile * kRows + ((2 * c) & kMask)) / a.G, t1 = (row_tile * kRows + ((2 * c + 1) & kMask)) / a.G;
    const int p0 = t0 < s.cnt ? s.start + t0 : -1, p1 = t1 < s.cnt ? s.start + t1 : -1;
    // every row of the CTA sees all of a tile when it lies in [all_lo, all_hi)
    const int all_hi = s.start + row_tile * kRows / a.G + 1, all_lo = a.window >= 0 ? s.hi - 1 - a.window : 0;

    // o[j]: dimensions g*D/8 + 2j (rows 2c, 2c+1) and g*D/8 + 2j + 1 (the same rows), in units of v_unit
    float o[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, v_unit = 0.f, inv_unit = 0.f;

    // This warp's tiles are first + warp + W * i, i < mine.  Lane j holds the
    // page and the scales of the j-th of 32 tiles: f_* for the tiles being
    // fetched, c_* for those being computed, one behind.
    const int mine = last - first > warp ? (last - first - warp + W - 1) / W : 0;
    const int32_t* table = a.table + b * a.table_sb;
    int f_page = -1, c_page = -1;
    float f_ks = 0.f, f_vs = 0.f, c_ks = 0.f, c_vs = 0.f;
    bool bad_page = false;
    unsigned char* ring = smem + warp * (kStages * 2 * kTileBytes<D>);
    const uint32_t ring_u32 = smem_u32(ring);
    auto fetch = [&](int i) {
        if ((i & 31) == 0) {
            f_page = -1;
            if (i + lane < mine) {
                const int pg = table[(s.lo16 + (first + warp + W * (i + lane)) * kTile) >> a.page_shift];
                if (pg < 0 || pg >= a.n_pages) {
                    bad_page = true;
                } else {
                    f_page = pg;
                    f_ks = __ldg(a.ks + (int64_t)pg * a.H + h);
                    f_vs = __ldg(a.vs + (int64_t)pg * a.H + h);
                }
            }
        }
        const int pg = __shfl_sync(0xffffffffu, f_page, i & 31);
        if (pg >= 0 && i < mine) {
            const int slot = ((first + warp + W * i) * kTile + s.lo16) & ((1 << a.page_shift) - 1);
            const int64_t off = ((((int64_t)pg * a.H + h) << a.page_shift) + slot) * D + lane * 16;
            const uint32_t dst = ring_u32 + (i % kStages) * (2 * kTileBytes<D>);
            constexpr int CH = D / 16;                  // chunks of a row
#pragma unroll
            for (int j = 0; j < kTileBytes<D> / 512; ++j) {
                const int row = j * (32 / CH) + lane / CH, ch = lane % CH;
                cp16(dst + row * D + ((ch ^ k_swz<D>(row)) << 4), a.kc + off + j * 512);
                cp16(dst + kTileBytes<D> + row * D + ((ch ^ v_swz<D>(row)) << 4), a.vc + off + j * 512);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0);                                           // on its way while q is read

    // q rows in f16, scaled by a power of two so that the largest value is in [2^13, 2^14)
    uint32_t qh[KS][2], ql[KS][2];
    float q_inv = 1.f;
    {
        float v[D / 64][16];
        float amax = 0.f;
        const T* q = static_cast<const T*>(a.q) + b * a.q_sb + (int64_t)t * a.q_st + (int64_t)(h * a.G + row % a.G) * a.q_sh;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            if (!live) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[i][e] = 0.f;
            } else if (a.q_vec) {
                constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
                for (int e = 0; e < 16; e += E) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q + 64 * i + 16 * c + e));
                    const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
                    for (int j = 0; j < E; ++j) v[i][e + j] = El::to_f(x[j]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[i][e] = El::load(q + 64 * i + 16 * c + e);
            }
        }
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float m = fabsf(v[i][e]);
                if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int e = 127 + 13 - (int)(__float_as_uint(amax) >> 23);
        e = amax > 0.f ? (e > 126 ? 126 : e) : 0;                       // >= -114; 2^e and 2^-e are normal
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        q_inv = __uint_as_float((uint32_t)(127 - e) << 23) * a.scale_log2;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x0 = v[k / 4][4 * (k % 4) + 2 * j] * up, x1 = v[k / 4][4 * (k % 4) + 2 * j + 1] * up;
                qh[k][j] = pack_h2(x0, x1);
                if constexpr (kPair) {
                    const float2 r = unpack_h2(qh[k][j]);
                    ql[k][j] = pack_h2(x0 - r.x, x1 - r.y);
                } else {
                    ql[k][j] = 0u;
                }
            }
    }

    const float qi0 = __shfl_sync(0xffffffffu, q_inv, 8 * c), qi1 = __shfl_sync(0xffffffffu, q_inv, 8 * c + 4);

    for (int i = 0; i < mine; ++i) {
        if ((i & 31) == 0) {
            c_page = f_page;
            c_ks = f_ks;
            c_vs = f_vs;
        }
        __syncwarp();                                   // the stage that fetch writes has been read by all lanes
        fetch(i + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();                                   // every lane's part of tile i has landed
        if (__shfl_sync(0xffffffffu, c_page, i & 31) >= 0) {
            const int key0 = s.lo16 + (first + warp + W * i) * kTile;
            const unsigned char* kt = ring + (i % kStages) * (2 * kTileBytes<D>);
            const unsigned char* vt = kt + kTileBytes<D>;
            const float ks = __shfl_sync(0xffffffffu, c_ks, i & 31), vs = __shfl_sync(0xffffffffu, c_vs, i & 31);
            // scores: d[0], d[1] key g of the tile, d[2], d[3] key g + 8, for rows 2c and 2c + 1
            float d[4] = {0.f, 0.f, 0.f, 0.f}, d2[4] = {0.f, 0.f, 0.f, 0.f};     // two chains of products
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const int at = g * D + (((4 * j + c) ^ k_swz<D>(g)) << 4);
                const uint4 u = *reinterpret_cast<const uint4*>(kt + at), w = *reinterpret_cast<const uint4*>(kt + 8 * D + at);
                const uint32_t ku[4] = {u.x, u.y, u.z, u.w}, kw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t a0 = cvt_lo(ku[k]), a1 = cvt_lo(kw[k]), a2 = cvt_hi(ku[k]), a3 = cvt_hi(kw[k]);
                    float (&e)[4] = k & 1 ? d2 : d;
                    mma_f16(e, a0, a1, a2, a3, qh[4 * j + k][0], qh[4 * j + k][1], e[0], e[1], e[2], e[3]);
                    if constexpr (kPair) mma_f16(e, a0, a1, a2, a3, ql[4 * j + k][0], ql[4 * j + k][1], e[0], e[1], e[2], e[3]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] += d2[k];
            float sc[2][2] = {{d[0] * (qi0 * ks), d[1] * (qi1 * ks)}, {d[2] * (qi0 * ks), d[3] * (qi1 * ks)}};
            const bool whole = key0 >= all_lo && key0 >= s.lo && key0 + kTile <= all_hi;
            if (!whole) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int key = key0 + 8 * n + g;
                    if (key > p0 || (a.window >= 0 && key < p0 - a.window)) sc[n][0] = -INFINITY;
                    if (key > p1 || (a.window >= 0 && key < p1 - a.window)) sc[n][1] = -INFINITY;
                }
            }
            float x0 = fmaxf(sc[0][0], sc[1][0]), x1 = fmaxf(sc[0][1], sc[1][1]);
#pragma unroll
            for (int k = 4; k < 32; k *= 2) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, k));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, k));
            }
            if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1) || vs > 2.f * v_unit) {
                x0 = fmaxf(x0, m0);
                x1 = fmaxf(x1, m1);
                float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - x0), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - x1);
                m0 = x0;
                m1 = x1;
                l0 *= f0;
                l1 *= f1;
                if (vs > 2.f * v_unit) {
                    f0 *= v_unit / vs;
                    f1 *= v_unit / vs;
                    v_unit = vs;
                    inv_unit = 1.f / vs;
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    o[j][0] *= f0; o[j][1] *= f1;
                    o[j][2] *= f0; o[j][3] *= f1;
                }
            }
            // The sums are kept in units of one block's scale, so that another block's is
            // a factor of its weights.  A larger scale becomes the unit; one far below it
            // would push the weights out of f16 and multiplies its product instead.
            const float rel = vs * inv_unit;
            const bool plain = rel >= 0.00390625f;                 // 2^-8
            const float fold = plain ? rel : 1.f, unfold = plain ? rcp(rel) : 1.f;
            const float b0f = m0 == -INFINITY ? 0.f : m0 - kPShift, b1f = m1 == -INFINITY ? 0.f : m1 - kPShift;
            const float w00 = ex2(sc[0][0] - b0f) * fold, w01 = ex2(sc[0][1] - b1f) * fold;
            const float w10 = ex2(sc[1][0] - b0f) * fold, w11 = ex2(sc[1][1] - b1f) * fold;
            uint32_t pk0 = pack_h2(w00, w01), pk1 = pack_h2(w10, w11);
            const float2 rest0 = unpack_h2(pk0), rest1 = unpack_h2(pk1);
            const uint32_t lo0 = pack_h2(w00 - rest0.x, w01 - rest0.y), lo1 = pack_h2(w10 - rest1.x, w11 - rest1.y);
            uint32_t bl0 = 0u, bl1 = 0u;
            if constexpr (HALF) {
                if (c >= 2) {
                    pk0 = lo0;
                    pk1 = lo1;
                }
            } else {
                bl0 = transpose(lo0);
                bl1 = transpose(lo1);
            }
            l0 = fmaf(w00 + w10, unfold, l0);
            l1 = fmaf(w01 + w11, unfold, l1);
            uint32_t bh0 = transpose(pk0), bh1 = transpose(pk1);  // row g, keys 2c, 2c+1 and 2c+8, 2c+9
            uint32_t vw[4][D / 32];
            auto load_v = [&]() {
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int r = (n >> 1) * 8 + 2 * c + (n & 1);
                    const unsigned char* row = vt + r * D;
                    if constexpr (D == 128) {
                        const uint4 w = *reinterpret_cast<const uint4*>(row + ((g ^ v_swz<D>(2 * c)) << 4));
                        vw[n][0] = w.x; vw[n][1] = w.y; vw[n][2] = w.z; vw[n][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(row + (((g >> 1) ^ v_swz<D>(2 * c)) << 4) + (g & 1) * 8);
                        vw[n][0] = w.x; vw[n][1] = w.y;
                    }
                }
            };
            auto clear_v = [&]() {                      // slots that no row sees may hold anything, NaN too
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int key = key0 + (n >> 1) * 8 + 2 * c + (n & 1);
                    if (key < s.lo || key >= s.hi) {
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) vw[n][k] = 0u;
                    }
                }
            };
            auto nan_bytes = [](uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u; };
            load_v();
            // A NaN value among keys that some row does not see: 0 * NaN would reach
            // that row.  Rare, so it takes a second product: the values without their
            // NaNs, then infinity where a row sees one, turned to NaN (inf * 0).
            bool extra = false;
            if (!whole) {
                clear_v();
                uint32_t any = 0u;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) any |= nan_bytes(vw[n][k]);
                extra = a.T > 1 && __any_sync(0xffffffffu, any != 0u);
            }
            // 16 dimensions by 16 keys of V^T: rows g and g + 8 are dimensions g*D/8 + 2j and + 1
            auto v_tile = [&](int j, uint32_t (&f)[4]) {
                const int k = j / 2;
                const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
                const uint32_t lo = __byte_perm(vw[0][k], vw[1][k], sel), hi = __byte_perm(vw[2][k], vw[3][k], sel);
                f[0] = cvt_lo(lo); f[1] = cvt_hi(lo); f[2] = cvt_lo(hi); f[3] = cvt_hi(hi);
            };
            if (plain && !extra) {
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    uint32_t f[4];
                    v_tile(j, f);
                    mma_f16(o[j], f[0], f[1], f[2], f[3], bh0, bh1, o[j][0], o[j][1], o[j][2], o[j][3]);
                    if constexpr (!HALF) mma_f16(o[j], f[0], f[1], f[2], f[3], bl0, bl1, o[j][0], o[j][1], o[j][2], o[j][3]);
                }
            } else {
                float f_out = plain ? 1.f : rel;
                if (extra) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) vw[n][k] &= ~(nan_bytes(vw[n][k]) * 0xffu);
                }
                for (;;) {
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        uint32_t f[4];
                        float e[4];
                        v_tile(j, f);
                        mma_f16(e, f[0], f[1], f[2], f[3], bh0, bh1, 0.f, 0.f, 0.f, 0.f);
                        if constexpr (!HALF) mma_f16(e, f[0], f[1], f[2], f[3], bl0, bl1, e[0], e[1], e[2], e[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            o[j][k] = fmaf(f_out, e[k], o[j][k]);
                            if (f_out == kHuge) o[j][k] = fmaf(o[j][k], 0.f, o[j][k]);
                        }
                    }
                    if (!extra) break;
                    extra = false;
                    f_out = kHuge;
                    // which keys the rows see, as f16 ones, and the NaNs as 448
                    const int ka = key0 + g, kb = key0 + 8 + g;
                    auto sees = [&](int key, int p) { return key <= p && (a.window < 0 || key >= p - a.window); };
                    pk0 = (sees(ka, p0) ? 0x3c00u : 0u) | (sees(ka, p1) ? 0x3c000000u : 0u);
                    pk1 = (sees(kb, p0) ? 0x3c00u : 0u) | (sees(kb, p1) ? 0x3c000000u : 0u);
                    bh0 = transpose(pk0);
                    bh1 = transpose(pk1);
                    bl0 = bl1 = 0u;
                    load_v();
                    clear_v();
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) vw[n][k] = nan_bytes(vw[n][k]) * 0x7eu;
                }
            }
        }
    }
    if (bad_page) atomicOr(a.err, ERRF_BAD_ARG);
#pragma unroll
    for (int k = 4; k < 32; k *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, k);
        l1 += __shfl_xor_sync(0xffffffffu, l1, k);
    }

    if constexpr (HALF) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[j][k] += __shfl_xor_sync(0xffffffffu, o[j][k], 2);
    }
    // Join the warps.  A warp leaves the mean of the values that it saw, beside its
    // maximum and total: a mean is no larger than the largest value, where a sum of
    // cached values of 1e36 and more would pass float32's range.
    const float r0 = l0 != 0.f ? 1.f / l0 : 0.f, r1 = l1 != 0.f ? 1.f / l1 : 0.f;
    __syncthreads();                                    // all rings are read: their memory takes the means
    float (*so)[kRows][D] = reinterpret_cast<float (*)[kRows][D]>(smem);
    float (*sm)[kRows] = reinterpret_cast<float (*)[kRows]>(smem + sizeof(float) * W * kRows * D);
    float (*sl)[kRows] = sm + W;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        if (HALF && c >= 2) break;
        const int d = g * (D / 8) + 2 * j;
        *reinterpret_cast<float2*>(&so[warp][2 * c][d]) = make_float2(o[j][0] * r0 * v_unit, o[j][2] * r0 * v_unit);
        *reinterpret_cast<float2*>(&so[warp][2 * c + 1][d]) = make_float2(o[j][1] * r1 * v_unit, o[j][3] * r1 * v_unit);
    }
    if (g == 0) {
        sm[warp][2 * c] = m0;
        sm[warp][2 * c + 1] = m1;
        sl[warp][2 * c] = l0;
        sl[warp][2 * c + 1] = l1;
    }
    __syncthreads();
    const int rows = min(kRows, a.T * a.G - row_tile * kRows);
    const bool alone = last - first == s.tiles;         // this CTA has seen all keys
    for (int i = threadIdx.x; i < rows * D; i += (W * 32)) {
        const int r = i / D, d = i % D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) mm = fmaxf(mm, sm[w][r]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float f[W], sum = 0.f, tot = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {                   // a warp without keys holds zeros; a NaN row keeps its NaN
            f[w] = ex2(sm[w][r] - base) * sl[w][r];
            tot += f[w];
        }
        const float inv = tot != 0.f ? 1.f / tot : 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum = fmaf(f[w] * inv, so[w][r][d], sum);
        if (alone) {
            const int rr = row_tile * kRows + r, tt = rr / a.G;
            T* out = static_cast<T*>(a.out) + ((b * a.T + tt) * (int64_t)(a.H * a.G) + h * a.G + rr % a.G) * D + d;
            *out = El::from_f(tt < s.cnt && tot != 0.f ? sum : 0.f);
        } else {
            part[i] = sum;
            if (d == 0) {
                part[kRows * D + r] = mm;
                part[kRows * D + kRows + r] = tot;
            }
        }
    }
}

// W warps per CTA, 16 to an SM (128 registers a thread).  A CTA takes `chunk`
// tiles of one row tile.
template <int DT, int D, int W, bool HALF>
__global__ void __launch_bounds__(W * 32, 16 / W) kv_attention_kernel(const __grid_constant__ KvAttnArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    const int split = blockIdx.x, h = blockIdx.y / a.row_tiles, row_tile = blockIdx.y % a.row_tiles;
    const int64_t b = blockIdx.z;
    const Span s = span_of(a, b, row_tile);
    if (s.bad && split == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
    const int first = split * a.chunk, last = min(first + a.chunk, s.tiles);
    if (split > 0 && first >= s.tiles) return;
    float* part = a.part + ((b * gridDim.y + blockIdx.y) * a.splits + split) * (kRows * (D + 2));
    attend<DT, D, W, HALF>(a, b, h, row_tile, s, first, last, part, smem);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Ragged sequences, in even shares: all tiles of all heads and sequences in a row
// (sequence by sequence, head by head) are cut into gridDim.x shares of `share`
// tiles, so every CTA works equally long whatever the lengths.  A CTA leaves at
// most two partial rows: of the head its share begins in (slot 0) and of the one it
// ends in (slot 1).  One row tile per head; up to kEvenBatch sequences.
constexpr int kEvenBatch = 512;
constexpr int kEvenLeast = 8;          // tiles of a share at least

// before[i] = tiles per head of the sequences before i, for i <= B; all threads of the CTA take part.
__device__ __forceinline__ void tiles_before(const KvAttnArgs& a, int B, int* before, bool flag) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int sum = 0;
        for (int i0 = 0; i0 < B; i0 += 32) {
            int n = 0;
            if (i0 + lane < B) {
                const Span s = span_of(a, i0 + lane, 0);
                n = s.tiles;
                if (s.bad && flag) atomicOr(a.err, ERRF_BAD_ARG);
            }
#pragma unroll
            for (int k = 1; k < 32; k *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, n, k);
                if (lane >= k) n += up;
            }
            if (i0 + lane < B) before[i0 + lane + 1] = sum + n;
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) before[0] = 0;
    }
    __syncthreads();
}
__device__ __forceinline__ int64_t share_of(int64_t total, int ctas) {
    const int64_t n = (total + ctas - 1) / ctas;
    return n > kEvenLeast ? n : kEvenLeast;
}

template <int DT, int D, int W, bool HALF>
__global__ void __launch_bounds__(W * 32, 16 / W) kv_attention_even_kernel(const __grid_constant__ KvAttnArgs a, int B) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int before[kEvenBatch + 1];
    tiles_before(a, B, before, blockIdx.x == 0);
    const int64_t total = (int64_t)before[B] * a.H, share = share_of(total, gridDim.x);
    const int64_t begin = blockIdx.x * share, end = begin + share < total ? begin + share : total;
    int b = 0;
    for (int64_t at = begin; at < end;) {
        while ((int64_t)before[b + 1] * a.H <= at) ++b;
        const Span s = span_of(a, b, 0);
        const int64_t rel = at - (int64_t)before[b] * a.H;
        const int h = (int)(rel / s.tiles), first = (int)(rel - (int64_t)h * s.tiles);
        const int last = (int)(end - at < s.tiles - first ? first + (end - at) : s.tiles);
        attend<DT, D, W, HALF>(a, b, h, 0, s, first, last, a.part + (2 * (int64_t)blockIdx.x + (at != begin)) * (kRows * (D + 2)), smem);
        at += last - first;
        __syncthreads();                                // the sums are read before the next ring is filled
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Joins the chunks of one query row: warp w takes chunks w, w + 8, ..., a lane D/32
// dimensions, so the order of the sums is fixed.  Launched as a programmatic
// dependent of the main kernel: its own launch is over when the last chunk is written.
constexpr int kJoinWarps = 8;
template <int DT, int D, bool EVEN>
__global__ void __launch_bounds__(kJoinWarps * 32) kv_attention_join_kernel(const __grid_constant__ KvAttnArgs a, int B, int ctas) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int E = D / 32;
    const int heads = a.H * a.G, t = blockIdx.x / heads, hq = blockIdx.x % heads, h = hq / a.G;
    const int64_t b = blockIdx.z;
    const int row = t * a.G + hq % a.G, row_tile = row / kRows, r = row % kRows, y = h * a.row_tiles + row_tile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kPart = kRows * (D + 2);
    const Span s = span_of(a, b, row_tile);
    int n;                                              // partial rows, kPart apart
    const float* part;
    if constexpr (EVEN) {
        __shared__ int before[kEvenBatch + 1];
        tiles_before(a, B, before, false);
        const int64_t share = share_of((int64_t)before[B] * a.H, ctas);
        const int64_t g0 = (int64_t)before[b] * a.H + (int64_t)h * s.tiles, c0 = g0 / share;
        n = s.tiles ? (int)((g0 + s.tiles - 1) / share - c0 + 1) : 0;
        // the head begins in CTA c0, in its slot 1 unless the share begins with it, and goes on in slots 0
        part = a.part + 2 * c0 * kPart;
        if (g0 != c0 * share) part += kPart;
    } else {
        n = (s.tiles + a.chunk - 1) / a.chunk;
        part = a.part + (b * (int64_t)(a.H * a.row_tiles) + y) * a.splits * kPart;
    }
    // where partial row i is: two slots a CTA when EVEN, the first possibly the second slot
    const int64_t step = EVEN ? 2 * kPart : kPart;
    const int64_t back = EVEN && n > 1 && ((part - a.part) / kPart & 1) ? kPart : 0;
    auto at = [&](int i) { return part + i * step - (i ? back : 0); };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n == 1) return;                                 // its CTA wrote the row
    if (n == 0) {                                       // a CTA wrote it, or in even shares none
        if (EVEN)
            for (int d = threadIdx.x; d < D; d += kJoinWarps * 32)
                static_cast<T*>(a.out)[((b * a.T + t) * (int64_t)heads + hq) * D + d] = El::from_f(0.f);
        return;
    }
    const int mr = kRows * D + r;                       // a partial row's maximum; its total kRows behind
    // the row's maximum and total: every warp takes them from all partial rows
    float m = -INFINITY, tot = 0.f;
    for (int i = lane; i < n; i += 32) {
        const float mi = at(i)[mr], li = at(i)[mr + kRows], up = fmaxf(m, mi), base = up == -INFINITY ? 0.f : up;
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
    const float base = m == -INFINITY ? 0.f : m;
    const float inv = tot != 0.f ? 1.f / tot : 0.f;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
#pragma unroll 8
    for (int i = warp; i < n; i += kJoinWarps) {
        const float* pi = at(i);
        const float f = ex2(pi[mr] - base) * pi[mr + kRows] * inv;
        float v[E];
        if constexpr (E == 4) {
            const float4 q = *reinterpret_cast<const float4*>(pi + r * D + lane * E);
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
            const float2 q = *reinterpret_cast<const float2*>(pi + r * D + lane * E);
            v[0] = q.x; v[1] = q.y;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = fmaf(f, v[e], sum[e]);
    }
    __shared__ float ws[kJoinWarps][D];
#pragma unroll
    for (int e = 0; e < E; ++e) ws[warp][lane * E + e] = sum[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) x += ws[w][d];
        static_cast<T*>(a.out)[((b * a.T + t) * (int64_t)heads + hq) * D + d] = El::from_f(t < s.cnt && tot != 0.f ? x : 0.f);
    }
}

// Warps per CTA, tiles per CTA and CTAs per row tile, from sizes the host knows (not the lengths).
struct Plan { int row_tiles, warps, chunk, splits, even; int64_t part_bytes; };
Plan plan_of(int64_t B, int64_t T, int64_t G, int64_t H, int64_t D, int64_t page, int64_t n_blocks, int64_t window) {
    Plan pl{};
    window = std::min<int64_t>(window, INT32_MAX / 2);
    pl.row_tiles = (int)((T * G + kRows - 1) / kRows);
    int64_t span = n_blocks * page;
    if (window >= 0) span = std::min(span, window + std::min<int64_t>(T, kRows) + kTile);
    const int64_t tiles = span / kTile + 1, base = B * H * pl.row_tiles;
    if (base <= 2 * 148 && tiles <= 72) {
        // few short sequences: all warps of an SM on two of them, and no second launch (kernels of
        // one sequence, 10 heads of 64, 257 keys: 6.1 us against 8.8 in chunks).  The limit of 72
        // tiles lies between few heads and many (us between events, eight warps : chunks, windows of
        // 512, 1024, 1500 and 2048): 10 heads of 64 10.3 : 12.3, 14.3 : 12.3, 16.4 : 13.2, 18.4 : 14.4;
        // 256 of 128 18.4 : 21.4, 24.6 : 28.7, 30.7 : 32.9, 36.9 : 41.0.
        pl.warps = 8;
        pl.chunk = (int)tiles;
        pl.splits = 1;
    } else if (window < 0 && pl.row_tiles == 1 && B <= kEvenBatch && base <= 8 * 148 &&
               B * tiles < INT32_MAX) {
        // lengths that the host does not know: even shares for one wave of eight CTAs per SM, unless
        // there are more heads than that (us, even shares against chunks or whole heads: 8 ragged
        // caches of up to 65536 tokens x 8 heads 100 : 105, one of 131072 x 8 63 : 81, 64 of up to
        // 8192 x 16 214 : 235; but 200 of up to 2000 x 8 124 : 98)
        pl.warps = 2;
        pl.even = (int)std::min<int64_t>(8 * 148, (base * tiles + kEvenLeast - 1) / kEvenLeast);
        pl.part_bytes = 2 * (int64_t)pl.even * kRows * (D + 2) * (int64_t)sizeof(float);
        return pl;
    } else {
        // CTAs of two warps: one wave of eight per SM where a window makes the sequences
        // alike, half as many again, for a table's capacity, where they may be ragged.  Between
        // events, us, 8 : 12.  Windows: 300 heads, 1000 30.8 : 34.8; 512 ragged, 1000 38.8 : 43.0;
        // 64 ragged, 2048 20.5 : 23.5; drafts of 4 float32 tokens, 400 heads, 1000 28.7 : 32.9.
        // None: 600 ragged of up to 4000 115.9 : 96.3; drafts of 8 tokens of 2 heads, 64 cached heads,
        // ragged of up to 8192 47.1 : 44.9, all of 8192 59.4 : 67.7; 16 heads on each of 16, ragged of
        // up to 16384 36.9 : 45.0.
        pl.warps = 2;
        const int64_t want = std::max<int64_t>(1, (window >= 0 ? 8 : 12) * 148 / std::max<int64_t>(1, base));
        pl.chunk = (int)std::max<int64_t>(2 * pl.warps, (tiles + want - 1) / want);
        pl.splits = (int)((tiles + pl.chunk - 1) / pl.chunk);
    }
    pl.part_bytes = pl.splits > 1 ? base * pl.splits * kRows * (D + 2) * (int64_t)sizeof(float) : 0;
    return pl;
}

template <int DT, int D, bool EVEN>
int launch_join(const KvAttnArgs& a, int64_t B, int ctas, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.T * a.H * a.G), 1, (unsigned)B);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<DT, D, EVEN>, a, (int)B, ctas);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NT_ERR_CUDA, "kv_attention_join_kernel launch failed: %s", cudaGetErrorString(e));
    }
    return check_launch("kv_attention_join_kernel");
}

template <int DT, int D, int W, bool HALF>
int launch_kv_attention(const KvAttnArgs& a, int64_t B, int even, cudaStream_t stream) {
    const size_t smem = std::max(kRingBytes<D, W>, sizeof(float) * W * kRows * (D + 2));
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_attention_kernel<DT, D, W, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_kv_attention: %s", cudaGetErrorString(e));
    }
    if constexpr (W == 2) {
        if (even) {
            kv_attention_even_kernel<DT, D, W, HALF><<<even, W * 32, smem, stream>>>(a, (int)B);
            const int rc = check_launch("kv_attention_even_kernel");
            return rc != NT_OK ? rc : launch_join<DT, D, true>(a, B, even, stream);
        }
    }
    const dim3 grid((unsigned)a.splits, (unsigned)(a.H * a.row_tiles), (unsigned)B);
    kv_attention_kernel<DT, D, W, HALF><<<grid, W * 32, smem, stream>>>(a);
    const int rc = check_launch("kv_attention_kernel");
    return rc != NT_OK || a.splits == 1 ? rc : launch_join<DT, D, false>(a, B, 0, stream);
}

template <int DT, int D, bool HALF>
int launch_warps(const KvAttnArgs& a, int64_t B, const Plan& pl, cudaStream_t stream) {
    return pl.warps == 8 ? launch_kv_attention<DT, D, 8, HALF>(a, B, 0, stream)
                         : launch_kv_attention<DT, D, 2, HALF>(a, B, pl.even, stream);
}
// HALF wherever it can be: us a call of the 8 ragged caches above 109 against 113, of the 64 streams
// 30.7 against 31.4.
template <int DT, int D>
int launch_planned(const KvAttnArgs& a, int64_t B, const Plan& pl, cudaStream_t stream) {
    return 2 * a.T * a.G <= kRows ? launch_warps<DT, D, true>(a, B, pl, stream) : launch_warps<DT, D, false>(a, B, pl, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_kv_attention_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t page,
                                        int64_t n_blocks, int64_t window) {
    if (B < 1 || T < 1 || Hkv < 1 || Hq < Hkv || D < 1 || page < 1 || n_blocks < 0) return 0;
    return plan_of(B, T, Hq / Hkv, Hkv, D, page, n_blocks, window).part_bytes;
}

int nt_kv_attention(int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t page, int64_t n_pages,
                    int64_t n_blocks, int64_t window, float scale, const void* q, int64_t q_sb, int64_t q_st,
                    int64_t q_sh, const void* k_codes, const float* k_scale, const void* v_codes, const float* v_scale,
                    const int32_t* table, int64_t table_sb, const int32_t* lengths, const int32_t* counts, void* out,
                    void* workspace, int64_t workspace_bytes, void* stream) {
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_kv_attention: dtype %d", dtype);
    if (D != 64 && D != 128) return fail(NT_ERR_ARG, "nt_kv_attention: head_dim %lld (64 or 128 supported)", (long long)D);
    if (page != 16 && page != 32 && page != 64)
        return fail(NT_ERR_ARG, "nt_kv_attention: page of %lld tokens (16, 32 or 64 supported)", (long long)page);
    if (B < 0 || T < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv || n_pages < 0 || n_blocks < 0 || B > 65535 ||
        T > (1 << 20) || Hq > 65535 || n_blocks * page > (int64_t)INT32_MAX - 4096)
        return fail(NT_ERR_ARG, "nt_kv_attention: bad sizes");
    if (B == 0 || T == 0) return NT_OK;
    if (!q || !k_codes || !k_scale || !v_codes || !v_scale || !table || !lengths || !out)
        return fail(NT_ERR_ARG, "nt_kv_attention: null pointer");
    if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15)
        return fail(NT_ERR_ARG, "nt_kv_attention: codes need 16-byte alignment");
    const int64_t G = Hq / Hkv;
    const Plan pl = plan_of(B, T, G, Hkv, D, page, n_blocks, window);
    if (Hkv * pl.row_tiles > 65535) return fail(NT_ERR_ARG, "nt_kv_attention: %lld query rows in one call", (long long)(T * Hq));
    if (pl.part_bytes > 0 && (!workspace || workspace_bytes < pl.part_bytes))
        return fail(NT_ERR_WORKSPACE, "nt_kv_attention: workspace %lld < %lld bytes", (long long)workspace_bytes,
                    (long long)pl.part_bytes);
    int dev = 0;
    cudaGetDevice(&dev);
    KvAttnArgs a{};
    a.T = (int)T; a.G = (int)G; a.H = (int)Hkv;
    a.page_shift = page == 16 ? 4 : page == 32 ? 5 : 6;
    a.n_pages = n_pages; a.n_blocks = n_blocks;
    a.window = window < 0 ? -1 : (int)std::min<int64_t>(window, INT32_MAX / 2);
    a.chunk = pl.chunk; a.splits = pl.splits; a.row_tiles = pl.row_tiles;
    a.scale_log2 = scale * kLog2e;
    a.q = q; a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
    const int64_t es = dtype == NT_F32 ? 4 : 2;
    a.q_vec = ((reinterpret_cast<uintptr_t>(q) | (uint64_t)((q_sb | q_st | q_sh) * es)) & 15) == 0;
    a.kc = static_cast<const uint8_t*>(k_codes); a.ks = k_scale;
    a.vc = static_cast<const uint8_t*>(v_codes); a.vs = v_scale;
    a.table = table; a.table_sb = table_sb; a.lengths = lengths; a.counts = counts;
    a.out = out; a.part = static_cast<float*>(workspace);
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_attention: error word unavailable");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32) return D == 64 ? launch_planned<NT_F32, 64>(a, B, pl, st) : launch_planned<NT_F32, 128>(a, B, pl, st);
    return D == 64 ? launch_planned<NT_BF16, 64>(a, B, pl, st) : launch_planned<NT_BF16, 128>(a, B, pl, st);
}

}  // extern "C"
