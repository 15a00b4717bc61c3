// Rotary positions at given positions (the rotation of apply_rotary,
// neuratensor/core/model.py:119-126, which the reference applies at
// positions 0..T-1 only): half and interleaved pairs, a part of the head,
// any frequencies, forward and backwards in angle (the gradient).
//
// y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a), a = p F_i.
// The angle is taken in turns: t = p (F_i / 2 pi) in float64, reduced to
// t - rint(t), then sincospi in float32, so a position in the millions loses
// nothing (float32 would be off by p 2^-24 radians).
//
// Bound by HBM: every element is read and written once, and the angles cost
// two float64 products and one sincospi per token and pair, shared by the heads.
// A CTA takes a few tokens: it puts their sines into shared memory once and then
// walks their heads' vectors in the order they lie in memory, four units of a
// thread in flight.  (A thread that kept one pair's sines in registers and walked
// the heads left too few threads and half-used lines: 29 against 19 us for 8 x
// 2048 tokens of 20 bf16 heads of 64, 178 against 124 us for 32767 tokens of 24
// float32 heads of 128, half of each rotated.)
#include "nt_kernels.cuh"

#include <algorithm>

namespace nt {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxHead = 2048;         // dimensions of a head: its sines are held in shared memory
constexpr int kMaxTokens = 256;        // of a CTA
constexpr double kInvTwoPi = 0.15915494309189533577;

// Exact n / d for n < 2^16 and 0 < d < 2^16.
struct Div16 {
    uint32_t d, m;
    Div16() = default;
    explicit Div16(uint32_t v) : d(v), m(v == 1 ? 0u : (uint32_t)((1ull << 32) / v + 1)) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return d == 1 ? n : __umulhi(n, m); }
};

struct RotArgs {
    int64_t N, T;                      // tokens B*T, tokens per sequence
    int H, D, R;
    float mscale, sgn;                 // sgn: mscale with the sine's sign
    const void* x; int64_t x_sb, x_st, x_sh;
    const int64_t* pos; int64_t p_sb;
    const float* freq;
    void* y; int64_t y_sb, y_st, y_sh;
    int units, rot_units;              // units of work per token and head: those that turn come first
    int tokens, heads;                 // per CTA
    Div16 by_units, by_heads, by_pairs;
};

template <typename T, int E> struct Vec { T v[E]; };
template <typename T, int E>
__device__ __forceinline__ Vec<T, E> ld(const T* p) {
    Vec<T, E> r;
    if constexpr (E * sizeof(T) == 16) *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
    else {
#pragma unroll
        for (int e = 0; e < E; ++e) r.v[e] = p[e];
    }
    return r;
}
template <typename T, int E>
__device__ __forceinline__ void st(T* p, const Vec<T, E>& r) {
    if constexpr (E * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
    else {
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = r.v[e];
    }
}

// Written out so that every layout rounds alike: the results do not depend on the vector width.
__device__ __forceinline__ float turn1(float x1, float x2, float c, float s) { return fmaf(-x2, s, __fmul_rn(x1, c)); }
__device__ __forceinline__ float turn2(float x1, float x2, float c, float s) { return fmaf(x1, s, __fmul_rn(x2, c)); }

// A unit is two vectors of E elements, E pairs: dimensions d and d + R/2 in the
// half layout (E >= 1), 2E neighbouring ones in the interleaved layout; or, past
// R, 2E dimensions to copy (the last unit of a head may have E only).
template <int DT, int E, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    extern __shared__ __align__(16) float2 turns_cs[];                // [tokens][R/2] (m cos, m sin)
    __shared__ int64_t x_at[kMaxTokens], y_at[kMaxTokens];
    __shared__ double pos_of[kMaxTokens];
    const int pairs = a.R / 2;
    const int64_t n0 = (int64_t)blockIdx.x * a.tokens;
    const int tokens = (int)(a.N - n0 < a.tokens ? a.N - n0 : a.tokens);
    const int h0 = blockIdx.y * a.heads, heads = a.H - h0 < a.heads ? a.H - h0 : a.heads;
    if (threadIdx.x < tokens) {
        const int64_t n = n0 + threadIdx.x, b = n / a.T, t = n - b * a.T;
        pos_of[threadIdx.x] = (double)a.pos[b * a.p_sb + t];
        x_at[threadIdx.x] = b * a.x_sb + t * a.x_st;
        y_at[threadIdx.x] = b * a.y_sb + t * a.y_st;
    }
    __syncthreads();
    constexpr int U = E * sizeof(T) == 16 ? 2 : 4;      // units of a thread in flight
    const int work = tokens * heads * a.units;
    Vec<T, E> x1[U], x2[U];
    T* dst[U];
    int d1[U], d2[U], at[U];                            // at: of the unit's first pair, -1 to copy
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = i0 + u * kRotThreads;
            if (i >= work) continue;
            const uint32_t th = a.by_units(i), unit = i - th * a.units, t = heads == a.heads ? a.by_heads(th) : th / heads,
                           h = th - t * heads;
            const T* src = static_cast<const T*>(a.x) + x_at[t] + (int64_t)(h0 + h) * a.x_sh;
            dst[u] = static_cast<T*>(a.y) + y_at[t] + (int64_t)(h0 + h) * a.y_sh;
            const bool rot = unit < a.rot_units;
            at[u] = rot ? (int)(t * pairs + unit * E) : -1;
            d1[u] = rot ? (INTER ? 2 : 1) * (int)unit * E : a.R + 2 * (int)(unit - a.rot_units) * E;
            d2[u] = rot && !INTER ? d1[u] + pairs : d1[u] + E;
            x1[u] = ld<T, E>(src + d1[u]);
            if (d2[u] < a.D) x2[u] = ld<T, E>(src + d2[u]);
        }
    };
    load(threadIdx.x);                                  // on their way while the sines are taken
    for (int i = threadIdx.x; i < tokens * pairs; i += kRotThreads) {
        const uint32_t t = a.by_pairs(i), k = i - t * pairs;
        const double turns = __dmul_rn(pos_of[t], __dmul_rn((double)a.freq[k], kInvTwoPi));
        float sn, cs;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
        turns_cs[i] = make_float2(cs * a.mscale, sn * a.sgn);
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < work; i0 += U * kRotThreads) {
        if (i0 != threadIdx.x) load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * kRotThreads >= work) continue;
            if (at[u] >= 0) {
                Vec<float, 2 * E> cs;                   // cos and sine of E pairs
                if constexpr (E == 1) {
                    *reinterpret_cast<float2*>(&cs) = turns_cs[at[u]];
                } else {
#pragma unroll
                    for (int k = 0; k < E / 2; ++k)
                        reinterpret_cast<float4*>(&cs)[k] = reinterpret_cast<const float4*>(turns_cs + at[u])[k];
                }
                // element e of the two vectors in a row: e < E from x1, else from x2
                Vec<T, E> o1, o2;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float co = cs.v[2 * k], si = cs.v[2 * k + 1];
                    if constexpr (!INTER) {
                        const float p = El::to_f(x1[u].v[k]), q = El::to_f(x2[u].v[k]);
                        o1.v[k] = El::from_f(turn1(p, q, co, si));
                        o2.v[k] = El::from_f(turn2(p, q, co, si));
                    } else {
                        auto in = [&](int e) { return El::to_f(e < E ? x1[u].v[e < E ? e : 0] : x2[u].v[e < E ? 0 : e - E]); };
                        auto out = [&](int e, float v) { (e < E ? o1.v[e < E ? e : 0] : o2.v[e < E ? 0 : e - E]) = El::from_f(v); };
                        const float p = in(2 * k), q = in(2 * k + 1);
                        out(2 * k, turn1(p, q, co, si));
                        out(2 * k + 1, turn2(p, q, co, si));
                    }
                }
                x1[u] = o1;
                x2[u] = o2;
            }
            st(dst[u] + d1[u], x1[u]);
            if (d2[u] < a.D) st(dst[u] + d2[u], x2[u]);
        }
    }
}

template <int DT, int E>
int launch(RotArgs a, bool inter, bool in_place, cudaStream_t stream) {
    a.rot_units = a.R / 2 / E;
    a.units = a.rot_units + (in_place ? 0 : (a.D - a.R + 2 * E - 1) / (2 * E));
    // about 1024 units a CTA, so that four or more CTAs an SM run while the work lasts
    const int64_t all = a.N * a.H * a.units;
    const int64_t most = std::max<int64_t>(kRotThreads, std::min<int64_t>(1024, all / (4 * 148)));
    a.heads = (int)std::min<int64_t>(a.H, std::max<int64_t>(1, most / a.units));
    a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(most / ((int64_t)a.heads * a.units), std::min(2 * kMaxHead / a.R, kMaxTokens)));
    a.by_units = Div16((uint32_t)a.units);
    a.by_heads = Div16((uint32_t)a.heads);
    a.by_pairs = Div16((uint32_t)(a.R / 2));
    const int64_t blocks = (a.N + a.tokens - 1) / a.tokens, rows = (a.H + a.heads - 1) / a.heads;
    if (blocks > 2147483647LL || rows > 65535) return fail(NT_ERR_ARG, "nt_rotary: too many tokens or heads");
    const dim3 grid((unsigned)blocks, (unsigned)rows);
    const size_t smem = (size_t)a.tokens * (a.R / 2) * sizeof(float2);       // 16 KB at most
    if (inter) rotary_kernel<DT, E, true><<<grid, kRotThreads, smem, stream>>>(a);
    else rotary_kernel<DT, E, false><<<grid, kRotThreads, smem, stream>>>(a);
    return check_launch("rotary_kernel");
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_rotary(int dtype, int64_t B, int64_t T, int64_t H, int64_t D, int64_t R, int interleaved, int inverse,
                         float mscale, const void* x, int64_t x_sb, int64_t x_st, int64_t x_sh, const int64_t* positions,
                         int64_t p_sb, const float* inv_freq, void* y, int64_t y_sb, int64_t y_st, int64_t y_sh,
                         void* stream) {
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_rotary: dtype %d", dtype);
    if (B < 0 || T < 0 || H < 0 || D < 1 || D > kMaxHead || H > 65535 || (T > 0 && B > INT64_MAX / 65536 / kMaxHead / T))
        return fail(NT_ERR_ARG, "nt_rotary: bad sizes (B %lld, T %lld, H %lld, D %lld; heads of at most %d)", (long long)B,
                    (long long)T, (long long)H, (long long)D, kMaxHead);
    if (R < 2 || R > D || R % 2) return fail(NT_ERR_ARG, "nt_rotary: rotated part %lld of %lld must be even, 2..D",
                                             (long long)R, (long long)D);
    if (B == 0 || T == 0 || H == 0) return NT_OK;
    if (!x || !positions || !inv_freq || !y) return fail(NT_ERR_ARG, "nt_rotary: null pointer");
    const bool in_place = x == y;
    if (in_place && (x_sb != y_sb || x_st != y_st || x_sh != y_sh))
        return fail(NT_ERR_ARG, "nt_rotary: in place needs equal strides");
    const int64_t es = dtype == NT_F32 ? 4 : 2, E = 16 / es;
    const uint64_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) |
                          (uint64_t)((x_sb | x_st | x_sh | y_sb | y_st | y_sh) * es);
    const bool vec = (bits & 15) == 0 && D % E == 0 && (R / 2) % E == 0;
    RotArgs a{};
    a.N = B * T; a.T = T; a.H = (int)H; a.D = (int)D; a.R = (int)R;
    a.mscale = mscale; a.sgn = inverse ? -mscale : mscale;
    a.x = x; a.x_sb = x_sb; a.x_st = x_st; a.x_sh = x_sh;
    a.pos = positions; a.p_sb = p_sb; a.freq = inv_freq;
    a.y = y; a.y_sb = y_sb; a.y_st = y_st; a.y_sh = y_sh;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32) return vec ? launch<NT_F32, 4>(a, interleaved, in_place, st) : launch<NT_F32, 1>(a, interleaved, in_place, st);
    return vec ? launch<NT_BF16, 8>(a, interleaved, in_place, st) : launch<NT_BF16, 1>(a, interleaved, in_place, st);
}
