// Attention of the new tokens over the paged 8-bit cache (nt_kvcache.cu).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,  k = ks[page, head] * code, v alike,
// query row t of sequence b at position p = len - cnt + t sees j <= p and, with
// a window, j >= p - window.
//
// Bound by HBM: a step reads every visible code once (one byte per element)
// and does two flops per query row with it.  So nothing is staged: the codes
// go from global memory to registers in the shape the matrix instruction
// takes, one tile of 16 keys ahead of the arithmetic, and the tensor cores
// (mma m16n8k16, f16 in, float32 sums) do the products that would cost the
// CUDA cores a conversion and an FMA per element.  The 16-row operand is the
// query rows of one cached head: eight of them (a step of eight shared heads,
// or a draft of a few tokens), and in the other eight rows what f16 leaves of
// them, which makes the product exact to float32 for float32 queries and costs
// nothing; e4m3 codes and bf16 queries are exact in f16 as they are.
//
// The k order of a product is free, so a lane takes 16 consecutive dimensions
// of a key (one 16-byte load) as its part of four k-steps, with q in the same
// order; likewise lane group g of V owns D/8 consecutive dimensions, one per
// n-tile, of the four keys whose probabilities the lane holds after the first
// product, so the probabilities never leave their registers either.
//
// Softmax is online, in float32, base 2: a warp keeps its rows' running
// maximum, sum and output over its tiles; four warps of a CTA join in shared
// memory, and the CTAs of a long sequence (`chunk` tiles each) in a second
// kernel, in chunk order.  Probabilities are held as 2^14 p in f16 (11 bits;
// small ones reach down to 2^-38 of the largest) for bf16 outputs, whose own
// rounding is 2^-9, and as an f16 pair for float32.
#include "nt_kernels.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace nt {
namespace {

constexpr int kAttnThreads = 128;
constexpr int kWarps = kAttnThreads / 32;
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
    const void* q; int64_t q_sb, q_st, q_sh;
    const uint8_t* kc; const float* ks; const uint8_t* vc; const float* vs;
    const int32_t* table; int64_t table_sb;
    const int32_t* lengths; const int32_t* counts;
    void* out;
    float* part;                       // [B, H * row_tiles, splits] x ([kRows][D] sums, [kRows] maxima, [kRows] totals)
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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
                 "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// two e4m3 codes (low 16 bits) to two f16 values, exactly
__device__ __forceinline__ uint32_t cvt2(uint32_t w) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// One tile of codes in registers: for K, rows g and g+8 of the tile, 16 bytes
// per 64 dimensions; for V, rows 2c, 2c+1, 2c+8, 2c+9, the lane group's D/8 bytes.
template <int D> struct TileRegs {
    uint32_t k[2][D / 64][4];
    uint32_t v[4][D / 32];
    float ks, vs;
    bool live;
};

template <int D>
__device__ __forceinline__ void load_tile(TileRegs<D>& r, const KvAttnArgs& a, int key0, int page, int h, int g, int c) {
    r.live = page >= 0 && page < a.n_pages;
    if (!r.live) {
        r.ks = r.vs = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) r.k[n][i][0] = r.k[n][i][1] = r.k[n][i][2] = r.k[n][i][3] = 0u;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) r.v[n][i] = 0u;
        return;
    }
    const int64_t head = (int64_t)page * a.H + h;
    const int slot = key0 & ((1 << a.page_shift) - 1);
    const int64_t off = ((head << a.page_shift) + slot) * D;
    const uint8_t* kp = a.kc + off;
    const uint8_t* vp = a.vc + off;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(kp + (n * 8 + g) * D + 64 * i + 16 * c));
            r.k[n][i][0] = w.x; r.k[n][i][1] = w.y; r.k[n][i][2] = w.z; r.k[n][i][3] = w.w;
        }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const uint8_t* p = vp + ((n >> 1) * 8 + 2 * c + (n & 1)) * D + g * (D / 8);
        if constexpr (D == 128) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
            r.v[n][0] = w.x; r.v[n][1] = w.y; r.v[n][2] = w.z; r.v[n][3] = w.w;
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
            r.v[n][0] = w.x; r.v[n][1] = w.y;
        }
    }
    r.ks = __ldg(a.ks + head);
    r.vs = __ldg(a.vs + head);
}

template <int DT, int D>
__global__ void __launch_bounds__(kAttnThreads, 3) kv_attention_kernel(const __grid_constant__ KvAttnArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int KS = D / 16;                 // k-steps of the first product
    constexpr int NT = D / 8;                  // n-tiles of the second
    constexpr bool kPair = DT == NT_F32;       // rows 8..15 hold what f16 leaves of rows 0..7
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int split = blockIdx.x, h = blockIdx.y / a.row_tiles, row_tile = blockIdx.y % a.row_tiles;
    const int64_t b = blockIdx.z;
    const Span s = span_of(a, b, row_tile);
    if (s.bad && split == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
    const int first = split * a.chunk, last = min(first + a.chunk, s.tiles);
    if (split > 0 && first >= s.tiles) return;

    const int row = row_tile * kRows + g, t = row / a.G;
    const bool live = t < s.cnt;
    const int p = live ? s.start + t : -1;
    // every row of the CTA sees all of a tile when it lies in [all_lo, all_hi)
    const int all_hi = s.start + row_tile * kRows / a.G + 1, all_lo = a.window >= 0 ? s.hi - 1 - a.window : 0;

    // q rows in f16, scaled by a power of two so that the largest value is in [2^13, 2^14)
    uint32_t qh[KS][2], ql[KS][2];
    float q_inv = 1.f;
    {
        float v[D / 64][16];
        float amax = 0.f;
        const T* q = static_cast<const T*>(a.q) + b * a.q_sb + (int64_t)t * a.q_st + (int64_t)(h * a.G + row % a.G) * a.q_sh;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                v[i][e] = live ? El::load(q + 64 * i + 16 * c + e) : 0.f;
                const float m = fabsf(v[i][e]);
                if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int e = 127 + 13 - (int)(__float_as_uint(amax) >> 23);
        e = amax > 0.f ? (e > 100 ? 100 : e) : 0;                       // >= -114
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

    float o[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = 0.f;
    float m = -INFINITY, l = 0.f;

    const int32_t* table = a.table + b * a.table_sb;
    auto page_of = [&](int tile) { return tile < last ? table[(s.lo16 + tile * kTile) >> a.page_shift] : -1; };
    int tile = first + warp;
    TileRegs<D> cur, nxt;
    bool bad_page = false;
    int page = page_of(tile), page2 = page_of(tile + kWarps);
    if (tile < last) {
        load_tile<D>(cur, a, s.lo16 + tile * kTile, page, h, g, c);
        bad_page |= !cur.live;
    }
    for (; tile < last; tile += kWarps) {
        page = page2;
        page2 = page_of(tile + 2 * kWarps);
        if (tile + kWarps < last) {
            load_tile<D>(nxt, a, s.lo16 + (tile + kWarps) * kTile, page, h, g, c);
            bad_page |= !nxt.live;
        }
        if (cur.live) {
            const int key0 = s.lo16 + tile * kTile;
            // scores of 16 keys: n-tile n, keys 8n + 2c and + 1 of row g
            float sc[2][2];
            const float f = q_inv * cur.ks;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const uint32_t w = cur.k[n][k / 4][k % 4];
                    mma_f16(d, qh[k][0], ql[k][0], qh[k][1], ql[k][1], cvt2(w), cvt2(w >> 16), d[0], d[1], d[2], d[3]);
                }
                sc[n][0] = (kPair ? d[0] + d[2] : d[0]) * f;
                sc[n][1] = (kPair ? d[1] + d[3] : d[1]) * f;
            }
            const bool whole = key0 >= all_lo && key0 >= s.lo && key0 + kTile <= all_hi;
            uint32_t ind0 = 0u, ind1 = 0u;              // which keys the row sees, as f16 ones
            if (!whole) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = key0 + 8 * n + 2 * c + e;
                        const bool see = key <= p && (a.window < 0 || key >= p - a.window);
                        if (!see) sc[n][e] = -INFINITY;
                        const uint32_t one = see ? 0x3c00u << (16 * e) : 0u;
                        if (n == 0) ind0 |= one; else ind1 |= one;
                    }
                // slots that no row sees may hold anything, NaN too
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int key = key0 + (n >> 1) * 8 + 2 * c + (n & 1);
                    if (key < s.lo || key >= s.hi) {
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) cur.v[n][i] = 0u;
                    }
                }
            }
            float mx = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx);
                const float corr = m == -INFINITY ? 0.f : ex2(m - mn);
                m = mn;
                l *= corr;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    o[j][0] *= corr;
                    o[j][1] *= corr;
                }
            }
            const float base = m == -INFINITY ? 0.f : m - kPShift;
            const float p00 = ex2(sc[0][0] - base), p01 = ex2(sc[0][1] - base);
            const float p10 = ex2(sc[1][0] - base), p11 = ex2(sc[1][1] - base);
            uint32_t a0 = pack_h2(p00, p01), a2 = pack_h2(p10, p11), a1 = 0u, a3 = 0u;
            {
                const float2 r0 = unpack_h2(a0), r1 = unpack_h2(a2);
                if constexpr (kPair) {
                    a1 = pack_h2(p00 - r0.x, p01 - r0.y);
                    a3 = pack_h2(p10 - r1.x, p11 - r1.y);
                    l += (p00 + p01) + (p10 + p11);
                } else {
                    l += (r0.x + r0.y) + (r1.x + r1.y);       // the weights that are used sum to one
                }
            }
            // A NaN value among keys that some row does not see: 0 * NaN would reach
            // that row.  Rare, so it takes a second product: the values without their
            // NaNs, then infinity where a row sees one, turned to NaN (inf * 0).
            bool extra = false;
            float vscale = cur.vs;
            uint32_t nan_at[4][D / 32];
            if (!whole && a.T > 1) {
                uint32_t any = 0u;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) any |= (cur.v[n][i] & 0x7f7f7f7fu) + 0x01010101u;
                if (__any_sync(0xffffffffu, (any & 0x80808080u) != 0u)) {
                    extra = true;
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) {
                            const uint32_t hit = (((cur.v[n][i] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
                            nan_at[n][i] = hit * 0x7eu;        // 448
                            cur.v[n][i] &= ~(hit * 0xffu);
                        }
                }
            }
            for (;;) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint32_t lo01 = __byte_perm(cur.v[0][i], cur.v[1][i], 0x5140), lo23 = __byte_perm(cur.v[0][i], cur.v[1][i], 0x7362);
                    const uint32_t hi01 = __byte_perm(cur.v[2][i], cur.v[3][i], 0x5140), hi23 = __byte_perm(cur.v[2][i], cur.v[3][i], 0x7362);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w0 = (e < 2 ? lo01 : lo23) >> (16 * (e & 1)), w1 = (e < 2 ? hi01 : hi23) >> (16 * (e & 1));
                        float d[4];
                        mma_f16(d, a0, a1, a2, a3, cvt2(w0), cvt2(w1), 0.f, 0.f, 0.f, 0.f);
                        o[4 * i + e][0] = fmaf(vscale, kPair ? d[0] + d[2] : d[0], o[4 * i + e][0]);
                        o[4 * i + e][1] = fmaf(vscale, kPair ? d[1] + d[3] : d[1], o[4 * i + e][1]);
                    }
                }
                if (!extra) {
                    if (vscale == kHuge)
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            o[j][0] = fmaf(o[j][0], 0.f, o[j][0]);
                            o[j][1] = fmaf(o[j][1], 0.f, o[j][1]);
                        }
                    break;
                }
                extra = false;
                vscale = kHuge;
                a0 = ind0; a2 = ind1; a1 = a3 = 0u;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) cur.v[n][i] = nan_at[n][i];
            }
        }
        cur = nxt;
    }
    if (bad_page && lane == 0) atomicOr(a.err, ERRF_BAD_ARG);
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // join the four warps: lane (g, c) of a warp holds row g, dimensions [c*D/4, (c+1)*D/4)
    __shared__ float so[kWarps][kRows][D];
    __shared__ float sm[kWarps][kRows], sl[kWarps][kRows];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int j = 0; j < NT; ++j) so[warp][g][(2 * c + half) * NT + j] = o[j][half];
    if (c == 0) {
        sm[warp][g] = m;
        sl[warp][g] = l;
    }
    __syncthreads();
    const int rows = min(kRows, a.T * a.G - row_tile * kRows);
    const int64_t slot = (b * gridDim.y + blockIdx.y) * a.splits + split;
    const bool alone = s.tiles <= a.chunk;              // this CTA has seen all keys
    for (int i = threadIdx.x; i < rows * D; i += kAttnThreads) {
        const int r = i / D, d = i % D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w][r]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, tot = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(sm[w][r] - base);
            // a warp without keys holds zeros; a NaN row keeps its NaN
            sum = fmaf(f, so[w][r][d], sum);
            tot = fmaf(f, sl[w][r], tot);
        }
        if (alone) {
            const int rr = row_tile * kRows + r, tt = rr / a.G;
            T* out = static_cast<T*>(a.out) + ((b * a.T + tt) * (int64_t)(a.H * a.G) + h * a.G + rr % a.G) * D + d;
            *out = El::from_f(tt < s.cnt && tot != 0.f ? sum / tot : 0.f);
        } else {
            float* part = a.part + slot * (kRows * (D + 2));
            part[i] = sum;
            if (d == 0) {
                part[kRows * D + r] = mm;
                part[kRows * D + kRows + r] = tot;
            }
        }
    }
}

// Joins the chunks of a row tile, in chunk order: one thread per (row, dimension).
template <int DT, int D>
__global__ void __launch_bounds__(D) kv_attention_join_kernel(const __grid_constant__ KvAttnArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    const int r = blockIdx.x % kRows, y = blockIdx.x / kRows, h = y / a.row_tiles, row_tile = y % a.row_tiles;
    const int64_t b = blockIdx.z;
    const int rr = row_tile * kRows + r, tt = rr / a.G, d = threadIdx.x;
    if (rr >= a.T * a.G) return;
    const Span s = span_of(a, b, row_tile);
    if (s.tiles <= a.chunk) return;                     // its CTA wrote the rows
    const int n = (s.tiles + a.chunk - 1) / a.chunk;
    const float* part = a.part + (b * (int64_t)(a.H * a.row_tiles) + y) * a.splits * (kRows * (D + 2));
    float mm = -INFINITY;
    for (int i = 0; i < n; ++i) mm = fmaxf(mm, part[(int64_t)i * (kRows * (D + 2)) + kRows * D + r]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float sum = 0.f, tot = 0.f;
    for (int i = 0; i < n; ++i) {
        const float* pi = part + (int64_t)i * (kRows * (D + 2));
        const float f = ex2(pi[kRows * D + r] - base);
        sum = fmaf(f, pi[r * D + d], sum);
        tot = fmaf(f, pi[kRows * D + kRows + r], tot);
    }
    T* out = static_cast<T*>(a.out) + ((b * a.T + tt) * (int64_t)(a.H * a.G) + h * a.G + rr % a.G) * D + d;
    *out = El::from_f(tt < s.cnt && tot != 0.f ? sum / tot : 0.f);
}

// Tiles per CTA and CTAs per row tile, from sizes the host knows (not the lengths).
struct Plan { int row_tiles, chunk, splits; int64_t part_bytes; };
Plan plan_of(int64_t B, int64_t T, int64_t G, int64_t H, int64_t D, int64_t page, int64_t n_blocks, int64_t window) {
    Plan pl;
    pl.row_tiles = (int)((T * G + kRows - 1) / kRows);
    int64_t span = n_blocks * page;
    if (window >= 0) span = std::min(span, window + std::min<int64_t>(T, kRows) + kTile);
    const int64_t tiles = span / kTile + 1, base = B * H * pl.row_tiles;
    // four waves of three CTAs per SM, at least two tiles for each warp
    const int64_t want = std::max<int64_t>(1, 4 * 3 * 148 / std::max<int64_t>(1, base));
    pl.chunk = (int)std::max<int64_t>(2 * kWarps, (tiles + want - 1) / want);
    pl.splits = (int)((tiles + pl.chunk - 1) / pl.chunk);
    pl.part_bytes = pl.splits > 1 ? base * pl.splits * kRows * (D + 2) * (int64_t)sizeof(float) : 0;
    return pl;
}

template <int DT, int D>
int launch_kv_attention(const KvAttnArgs& a, int64_t B, cudaStream_t stream) {
    const dim3 grid((unsigned)a.splits, (unsigned)(a.H * a.row_tiles), (unsigned)B);
    kv_attention_kernel<DT, D><<<grid, kAttnThreads, 0, stream>>>(a);
    const int rc = check_launch("kv_attention_kernel");
    if (rc != NT_OK || a.splits == 1) return rc;
    const dim3 jgrid((unsigned)(a.H * a.row_tiles * kRows), 1, (unsigned)B);
    kv_attention_join_kernel<DT, D><<<jgrid, D, 0, stream>>>(a);
    return check_launch("kv_attention_join_kernel");
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
    a.kc = static_cast<const uint8_t*>(k_codes); a.ks = k_scale;
    a.vc = static_cast<const uint8_t*>(v_codes); a.vs = v_scale;
    a.table = table; a.table_sb = table_sb; a.lengths = lengths; a.counts = counts;
    a.out = out; a.part = static_cast<float*>(workspace);
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_attention: error word unavailable");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32) return D == 64 ? launch_kv_attention<NT_F32, 64>(a, B, st) : launch_kv_attention<NT_F32, 128>(a, B, st);
    return D == 64 ? launch_kv_attention<NT_BF16, 64>(a, B, st) : launch_kv_attention<NT_BF16, 128>(a, B, st);
}

}  // extern "C"
