// New keys and values into the paged 8-bit attention cache.
//
// The reference's attention keeps nothing between calls
// (neuratensor/core/model.py:148-181); this cache is what a generation step
// needs to see the tokens before it.  Codes are e4m3, and every block (the
// page's tokens of one head) has one scale, a power of two:
//   s' = min { 2^e >= 2^-126 : max|x| <= 448 * 2^e },  s = max(s', old s),
//   code = e4m3(x / s), old codes of the block become e4m3(code * old s / s).
// A power of two costs a floating code no precision (it moves the exponent
// only) and makes x / s exact, so a code is one rounding of x; and re-encoding
// a block whose scale grows is exact down to e4m3's subnormals, so filling a
// block token by token loses nothing against filling it at once.
//
// One CTA of 64 or 128 threads per (sequence, touched page, head) and side (k or
// v): the new values are read once into registers, their largest magnitude is
// reduced, and the codes are written; 8 values per thread and step (16 bytes of
// bf16 in, 8 bytes of codes out).  Bound by HBM for prompts (8 of up to 8192
// tokens, 16 heads of 128: 112 us with 128 threads that looked the page up before
// they read, 72 us so; several units to a CTA of 256 threads 92 us), by launch
// latency for single tokens.
#include "nt_kernels.cuh"

#include <cuda_fp8.h>

namespace nt {
namespace {

// Threads of a block of P x D values, eight vectors of eight values each or fewer.
template <int D, int P> constexpr int kAppThreadsOf = P * D / 64 > 64 ? P * D / 64 : 64;

struct AppendArgs {
    int64_t T; int H; int64_t n_pages, n_blocks;
    const void* x[2]; int64_t sb[2], st[2], sh[2];
    uint8_t* codes[2]; float* scale[2];
    const int32_t* table; int64_t table_sb;
    const int32_t* lengths; const int32_t* counts;
    unsigned* err;
};

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ void from_e4m3x4(uint32_t w, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Exponent of the smallest power of two with amax <= 448 * 2^e (448 = 1.75 * 2^8), at least -126.
__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
    return e < -126 ? -126 : e;           // zero and float32 subnormals too
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight values as they are read.
template <int DT> struct Raw {
    using T = typename Elem<DT>::T;
    static constexpr int W = 8 * (int)sizeof(T) / 16;
    uint4 w[W];
    template <bool VEC> __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w)[i] = p[i];
        }
    }
    __device__ __forceinline__ float at(int i) const {
        const uint32_t u = reinterpret_cast<const uint32_t*>(w)[DT == NT_BF16 ? i / 2 : i];
        return __uint_as_float(DT != NT_BF16 ? u : i & 1 ? u & 0xffff0000u : u << 16);
    }
    // Largest magnitude, NaN ignored; infinity where there is one.
    __device__ __forceinline__ float amax() const {
        float m = 0.f;
        if constexpr (DT == NT_BF16) {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
            uint32_t p = u[0] & 0x7fff7fffu;
#pragma unroll
            for (int i = 1; i < 4; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(p) : "r"(u[i] & 0x7fff7fffu));
            m = fmaxf(fmaxf(m, __uint_as_float(p << 16)), __uint_as_float(p & 0xffff0000u));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(at(i)));
        }
        return m;
    }
    __device__ __forceinline__ float amax_finite() const {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = fabsf(at(i));
            if (v <= 3.402823466e38f) m = fmaxf(m, v);
        }
        return m;
    }
};

// VEC: rows allow 16-byte loads.
template <int DT, int D, int P, bool VEC>
__global__ void __launch_bounds__(kAppThreadsOf<D, P>) kv_append_kernel(const __grid_constant__ AppendArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int kAppThreads = kAppThreadsOf<D, P>;
    constexpr int CH = D / 8;                           // vectors of a row
    constexpr int NV = P * CH / kAppThreads;            // vectors of a thread
    static_assert(NV >= 1 && NV * kAppThreads == P * CH, "a block's vectors divide among the threads");
    const int h = blockIdx.x % a.H, side = blockIdx.x / a.H;
    const int64_t b = blockIdx.z;
    const int64_t len = a.lengths[b], cnt = a.counts ? a.counts[b] : a.T, start = len - cnt;
    if (cnt < 0 || cnt > a.T || start < 0 || len > a.n_blocks * P) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
        return;
    }
    const int64_t blk = start / P + blockIdx.y, base = blk * P;
    if (cnt == 0 || base >= len) return;
    const int lo = (int)(start > base ? start - base : 0);                // first new slot; older ones before it
    const int hi = (int)(len - base < P ? len - base : P);
    const bool full = lo == 0 && hi == P;               // all pages of a prompt but its first and last
    const int64_t st = side ? a.st[1] : a.st[0];
    const T* x = static_cast<const T*>(side ? a.x[1] : a.x[0]) + b * (side ? a.sb[1] : a.sb[0]) +
                 (int64_t)h * (side ? a.sh[1] : a.sh[0]) + (base - start + threadIdx.x / CH) * st + threadIdx.x % CH * 8;
    const int64_t step = kAppThreads / CH * st;
    // the values are on their way before the page is known
    Raw<DT> raw[NV];
    if (full) {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i].template load<VEC>(x + i * step);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int slot = (threadIdx.x + i * kAppThreads) / CH;
            if (slot >= lo && slot < hi) raw[i].template load<VEC>(x + i * step);
        }
    }
    const int64_t page = a.table[b * a.table_sb + blk];
    if (page < 0 || page >= a.n_pages) {
        if (threadIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
        return;
    }
    uint8_t* codes = (side ? a.codes[1] : a.codes[0]) + (page * a.H + h) * (int64_t)(P * D);
    float* sp = (side ? a.scale[1] : a.scale[0]) + page * a.H + h;
    const float s_old = lo > 0 ? *sp : 0.f;

    float amax = 0.f;
    if (full) {
#pragma unroll
        for (int i = 0; i < NV; ++i) amax = fmaxf(amax, raw[i].amax());
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int slot = (threadIdx.x + i * kAppThreads) / CH;
            if (slot >= lo && slot < hi) amax = fmaxf(amax, raw[i].amax());
        }
    }
    if (amax > 3.402823466e38f) {                       // an infinity: the finite values' maximum is wanted
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int slot = (threadIdx.x + i * kAppThreads) / CH;
            if (slot >= lo && slot < hi) amax = fmaxf(amax, raw[i].amax_finite());
        }
    }
    __shared__ float red[kAppThreads / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();                                                       // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kAppThreads / 32; ++w) amax = fmaxf(amax, red[w]);
    const float s_blk = exp2i(block_exponent(amax));
    const float s = fmaxf(s_blk, s_old);
    const float inv = 1.f / s;                          // exact: scales are powers of two
    uint2* dst = reinterpret_cast<uint2*>(codes) + threadIdx.x;
    auto encode = [&](int i) {
        uint2 w;
        w.x = e4m3x4(raw[i].at(0) * inv, raw[i].at(1) * inv, raw[i].at(2) * inv, raw[i].at(3) * inv);
        w.y = e4m3x4(raw[i].at(4) * inv, raw[i].at(5) * inv, raw[i].at(6) * inv, raw[i].at(7) * inv);
        dst[i * kAppThreads] = w;
    };
    if (full) {
#pragma unroll
        for (int i = 0; i < NV; ++i) encode(i);
    } else {
        const float ratio = s_old * inv;
        const bool grown = lo > 0 && s > s_old;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int slot = (threadIdx.x + i * kAppThreads) / CH;
            if (slot >= lo && slot < hi) {
                encode(i);
            } else if (grown && slot < lo) {
                uint2 w = dst[i * kAppThreads];
                float f[4];
                from_e4m3x4(w.x, f);
                w.x = e4m3x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
                from_e4m3x4(w.y, f);
                w.y = e4m3x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
                dst[i * kAppThreads] = w;
            }
        }
    }
    if (threadIdx.x == 0) *sp = s;
}

template <int DT, int D, int P>
int launch_append(const AppendArgs& a, int64_t B, int vec, cudaStream_t stream) {
    const int64_t blocks = (a.T + P - 2) / P + 1;      // pages that T tokens can touch
    if (blocks > 65535) return fail(NT_ERR_ARG, "nt_kv_append: %lld tokens in one call", (long long)a.T);
    const dim3 grid((unsigned)(2 * a.H), (unsigned)blocks, (unsigned)B);
    if (vec) kv_append_kernel<DT, D, P, true><<<grid, kAppThreadsOf<D, P>, 0, stream>>>(a);
    else kv_append_kernel<DT, D, P, false><<<grid, kAppThreadsOf<D, P>, 0, stream>>>(a);
    return check_launch("kv_append_kernel");
}

template <int DT, int D>
int launch_append_page(const AppendArgs& a, int64_t B, int64_t page, int vec, cudaStream_t stream) {
    if (page == 16) return launch_append<DT, D, 16>(a, B, vec, stream);
    if (page == 32) return launch_append<DT, D, 32>(a, B, vec, stream);
    return launch_append<DT, D, 64>(a, B, vec, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_kv_append(int dtype, int64_t B, int64_t T, int64_t Hkv, int64_t D, int64_t page, int64_t n_pages,
                            int64_t n_blocks, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v,
                            int64_t v_sb, int64_t v_st, int64_t v_sh, void* k_codes, float* k_scale, void* v_codes,
                            float* v_scale, const int32_t* table, int64_t table_sb, const int32_t* lengths,
                            const int32_t* counts, void* stream) {
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_kv_append: dtype %d", dtype);
    if (D != 64 && D != 128) return fail(NT_ERR_ARG, "nt_kv_append: head_dim %lld (64 or 128 supported)", (long long)D);
    if (page != 16 && page != 32 && page != 64)
        return fail(NT_ERR_ARG, "nt_kv_append: page of %lld tokens (16, 32 or 64 supported)", (long long)page);
    if (B < 0 || T < 0 || Hkv < 1 || n_pages < 0 || n_blocks < 0 || B > 65535 || Hkv > 65535 || T > INT32_MAX)
        return fail(NT_ERR_ARG, "nt_kv_append: bad sizes");
    if (B == 0 || T == 0) return NT_OK;
    if (!k || !v || !k_codes || !k_scale || !v_codes || !v_scale || !table || !lengths)
        return fail(NT_ERR_ARG, "nt_kv_append: null pointer");
    if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15)
        return fail(NT_ERR_ARG, "nt_kv_append: codes need 16-byte alignment");
    int dev = 0;
    cudaGetDevice(&dev);
    AppendArgs a{};
    a.T = T; a.H = (int)Hkv; a.n_pages = n_pages; a.n_blocks = n_blocks;
    a.x[0] = k; a.sb[0] = k_sb; a.st[0] = k_st; a.sh[0] = k_sh;
    a.x[1] = v; a.sb[1] = v_sb; a.st[1] = v_st; a.sh[1] = v_sh;
    a.codes[0] = static_cast<uint8_t*>(k_codes); a.codes[1] = static_cast<uint8_t*>(v_codes);
    a.scale[0] = k_scale; a.scale[1] = v_scale;
    a.table = table; a.table_sb = table_sb; a.lengths = lengths; a.counts = counts;
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_append: error word unavailable");
    const int64_t es = dtype == NT_F32 ? 4 : 2;
    const uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                          (uint64_t)((k_sb | k_st | k_sh | v_sb | v_st | v_sh) * es);
    const int vec = (bits & 15) == 0;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NT_F32)
        return D == 64 ? launch_append_page<NT_F32, 64>(a, B, page, vec, st) : launch_append_page<NT_F32, 128>(a, B, page, vec, st);
    return D == 64 ? launch_append_page<NT_BF16, 64>(a, B, page, vec, st) : launch_append_page<NT_BF16, 128>(a, B, page, vec, st);
}
