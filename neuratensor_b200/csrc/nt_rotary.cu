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
// one float64 product and one sincospi per token and pair.  So a thread keeps
// one token's vector of pairs, takes its sines once and walks the heads with
// it; few tokens are spread over several threads per pair instead, each with
// its share of the heads.
#include "nt_kernels.cuh"

#include <algorithm>

namespace nt {
namespace {

constexpr int kRotThreads = 256;
constexpr double kInvTwoPi = 0.15915494309189533577;

struct RotArgs {
    int64_t N, T;                      // tokens B*T, tokens per sequence
    int H, D, R;
    float mscale;                      // sign of the sine included in `sgn`
    float sgn;
    const void* x; int64_t x_sb, x_st, x_sh;
    const int64_t* pos; int64_t p_sb;
    const float* freq;
    void* y; int64_t y_sb, y_st, y_sh;
    int units;                         // vectors of work per token and head: rotated, then copied
    int rot_units;
    int per_block;                     // tokens per block
    int head_step;                     // heads of a token are spread over gridDim.y blocks
};

// `n` elements at once: 16 bytes, 4 bytes (a bf16 pair) or one element
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

// E elements per vector.  Half layout: a unit is E pairs, one vector from each
// half.  Interleaved: a unit is E/2 pairs in one vector (one pair as two
// elements when E == 1).
template <int DT, int E, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    constexpr int PAIRS = INTER ? (E == 1 ? 1 : E / 2) : E;
    const int unit0 = threadIdx.x % a.units, local = threadIdx.x / a.units;
    const int64_t n = (int64_t)blockIdx.x * a.per_block + local;
    if (local >= a.per_block || n >= a.N) return;
    const int64_t b = n / a.T, t = n - b * a.T;
    const T* x = static_cast<const T*>(a.x) + b * a.x_sb + t * a.x_st;
    T* y = static_cast<T*>(a.y) + b * a.y_sb + t * a.y_st;
    const double p = (double)a.pos[b * a.p_sb + t];
    const int h0 = blockIdx.y;
    for (int unit = unit0; unit < a.units; unit += kRotThreads) {      // one turn unless a token has more units than threads
        if (unit < a.rot_units) {
            float c[PAIRS], s[PAIRS];
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const double turns = __dmul_rn(p, __dmul_rn((double)a.freq[unit * PAIRS + k], kInvTwoPi));
                const float r = (float)(turns - rint(turns));
                float sn, cs;
                sincospif(2.f * r, &sn, &cs);
                c[k] = cs * a.mscale;
                s[k] = sn * a.sgn;
            }
            if constexpr (!INTER) {
                const int d1 = unit * E, d2 = d1 + a.R / 2;
#pragma unroll 4
                for (int h = h0; h < a.H; h += a.head_step) {
                    const Vec<T, E> u = ld<T, E>(x + h * a.x_sh + d1), v = ld<T, E>(x + h * a.x_sh + d2);
                    Vec<T, E> o1, o2;
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        const float x1 = El::to_f(u.v[k]), x2 = El::to_f(v.v[k]);
                        o1.v[k] = El::from_f(turn1(x1, x2, c[k], s[k]));
                        o2.v[k] = El::from_f(turn2(x1, x2, c[k], s[k]));
                    }
                    st(y + h * a.y_sh + d1, o1);
                    st(y + h * a.y_sh + d2, o2);
                }
            } else {
                constexpr int W = E == 1 ? 2 : E;
                const int d = unit * W;
#pragma unroll 4
                for (int h = h0; h < a.H; h += a.head_step) {
                    const Vec<T, W> u = ld<T, W>(x + h * a.x_sh + d);
                    Vec<T, W> o;
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        const float x1 = El::to_f(u.v[2 * k]), x2 = El::to_f(u.v[2 * k + 1]);
                        o.v[2 * k] = El::from_f(turn1(x1, x2, c[k], s[k]));
                        o.v[2 * k + 1] = El::from_f(turn2(x1, x2, c[k], s[k]));
                    }
                    st(y + h * a.y_sh + d, o);
                }
            }
        } else {
            const int d = a.R + (unit - a.rot_units) * E;
            for (int h = h0; h < a.H; h += a.head_step) st(y + h * a.y_sh + d, ld<T, E>(x + h * a.x_sh + d));
        }
    }
}

template <int DT, int E>
int launch(RotArgs a, bool inter, bool in_place, cudaStream_t stream) {
    a.rot_units = inter ? a.R / (E == 1 ? 2 : E) : a.R / 2 / E;
    a.units = a.rot_units + (in_place ? 0 : (a.D - a.R) / E);
    a.per_block = std::max(1, kRotThreads / a.units);
    const int64_t blocks = (a.N + a.per_block - 1) / a.per_block;
    if (blocks > 2147483647LL) return fail(NT_ERR_ARG, "nt_rotary: too many tokens");
    // heads over blocks until the device has two blocks per SM to run
    a.head_step = (int)std::min<int64_t>(a.H, std::max<int64_t>(1, 2 * 148 / blocks));
    const dim3 grid((unsigned)blocks, (unsigned)a.head_step);
    if (inter) rotary_kernel<DT, E, true><<<grid, kRotThreads, 0, stream>>>(a);
    else rotary_kernel<DT, E, false><<<grid, kRotThreads, 0, stream>>>(a);
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
    if (B < 0 || T < 0 || H < 0 || D < 1 || D > 65536 || H > 65535 || B > INT64_MAX / 2 / (T > 0 ? T : 1))
        return fail(NT_ERR_ARG, "nt_rotary: bad sizes (B %lld, T %lld, H %lld, D %lld)", (long long)B, (long long)T,
                    (long long)H, (long long)D);
    if (R < 2 || R > D || R % 2) return fail(NT_ERR_ARG, "nt_rotary: rotated part %lld of %lld must be even, 2..D",
                                             (long long)R, (long long)D);
    if (B == 0 || T == 0 || H == 0) return NT_OK;
    if (!x || !positions || !inv_freq || !y) return fail(NT_ERR_ARG, "nt_rotary: null pointer");
    const bool in_place = x == y;
    if (in_place && (x_sb != y_sb || x_st != y_st || x_sh != y_sh))
        return fail(NT_ERR_ARG, "nt_rotary: in place needs equal strides");
    const int64_t es = dtype == NT_F32 ? 4 : 2, E = 16 / es;
    const int64_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | (uint64_t)(x_sb * es) |
                         (uint64_t)(x_st * es) | (uint64_t)(x_sh * es) | (uint64_t)(y_sb * es) |
                         (uint64_t)(y_st * es) | (uint64_t)(y_sh * es);
    const bool vec = (bits & 15) == 0 && D % E == 0 && (interleaved ? R % E == 0 : (R / 2) % E == 0);
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
