// Penalties for repeated tokens, per-request biases and grammar masks on
// logits, in one pass (NeuraTensorModel.generate's repetition penalty,
// neuratensor/core/model.py:336-342, is a host loop over every token of the
// history; frequency and presence penalties, biases and masks are what callers
// add around it).
//
// Bound by HBM: logits in and out once, one mask bit per entry, the history
// once.  The history has to be counted per vocabulary entry before a logit is
// final, so a CTA owns a slice of one row's vocabulary, with a counter per entry
// in shared memory: it reads the row's whole history (from L2 for all slices
// but the first), counts what falls into its slice, and then streams the slice.
// Five CTAs share an SM, so some stream while others count.  Integer counters:
// the order of arrival changes nothing.
//
// 250 x 131072 float32 with 4000 tokens of history, 300 biases and a mask: 67 us,
// where the stream alone takes 44, the history 13, lookups at its touched entries,
// biases and mask the rest; 64 x 32000 bf16 with 8704 tokens 14 us.  Measured
// against this at the first size: the history counted once per cluster into
// distributed shared memory 96 to 131 us; a list of touched entries put right
// after an unchanged stream 89; a second kernel with a hash table per row 86.
// The registers of a CTA decide: four vectors and eight tokens of a thread in
// flight cost a CTA per SM or spills (69 to 78 us).
//
// A counter holds the index (plus one) of the last bias entry of the token, the
// number of occurrences after the prompt, and one bit for an occurrence at all:
// 16 + 15 + 1 bits of one word while the history is below 2^15 tokens and the
// biases below 2^16, else two words.
//
// In place and without a mask nothing else changes, so only the entries with a
// counter are read and written.
#include "nt_kernels.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nt {
namespace {

constexpr int kLogThreads = 256;

struct LogArgs {
    int64_t V;
    const void* x; int64_t ld;
    const int64_t* tokens; int64_t tok_ld; int L;
    const int32_t* lengths; const int32_t* prompts;
    const float* rep; const float* freq; const float* pres;
    float rep_all, rep_inv, freq_all, pres_all;   // rep_inv: 1 / rep_all, rounded from float64 as generate's loop has it
    const int64_t* ids; int64_t ids_ld; const float* bias; int64_t bias_ld; int NB;
    const uint32_t* allowed; int64_t allowed_ld;
    void* out; int64_t ldo;
    int slice;                         // vocabulary entries per CTA, a multiple of 128
    int slices;
};

// Where a counter's parts lie.  Narrow: bit 31 seen, bits 16..30 the
// occurrences, bits 0..15 the bias index.  Wide: bit 31 and bits 0..30 of one
// word, the bias index in another `slice` words further.
template <bool WIDE> struct Count {
    static constexpr uint32_t kSeen = 1u << 31, kOne = WIDE ? 1u : 1u << 16;
    static constexpr int kWords = WIDE ? 2 : 1;
};

// One logit: the penalties of its counter w, bias entry j - 1 (0: none).  Without
// branches for the penalties: an entry that was not met is multiplied by one and
// loses zero, which leaves it as it is, and the lanes of a warp stay together.
template <int DT, bool WIDE, bool EACH>
__device__ __forceinline__ float process(float x, uint32_t w, uint32_t j, float r, float r_inv, float fq, float ps,
                                         const float* bias) {
    const uint32_t made = WIDE ? w & 0x7fffffffu : (w >> 16) & 0x7fffu;
    if (!WIDE) j = w & 0xffffu;
    if constexpr (EACH) {
        for (uint32_t i = 0; i < made; ++i) x = Elem<DT>::rnd(x > 0.f ? x * r_inv : x * r);
    } else {
        const float f = x > 0.f ? r_inv : r;
        x *= (WIDE ? w : w >> 16) ? f : 1.f;
    }
    x -= made ? fmaf(fq, (float)made, ps) : 0.f;
    if (j) x += __ldg(bias + (j - 1));
    return x;
}

// COUNTED: there is a history or there are biases.  MASK: there is a mask.
template <int DT, bool COUNTED, bool MASK, bool WIDE, bool EACH>
__global__ void __launch_bounds__(kLogThreads, 5) logits_kernel(const __grid_constant__ LogArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    using K = Count<WIDE>;
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint32_t smem[];
    const int64_t b = blockIdx.x / a.slices;
    const int lo = (int)(blockIdx.x % a.slices) * a.slice;
    const int n = (int)(a.V - lo < a.slice ? a.V - lo : a.slice);
    const T* x = static_cast<const T*>(a.x) + b * a.ld + lo;
    T* y = static_cast<T*>(a.out) + b * a.ldo + lo;
    // Entries before the first 16-byte boundary of x.  Entry i's counter is
    // words[i], shifted so that those of a vector are 16-byte aligned too.
    const int head_x = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    const int head_y = (int)((16 - (reinterpret_cast<uintptr_t>(y) & 15)) & 15) / (int)sizeof(T);
    uint32_t* words = smem + ((E - head_x) & (E - 1));
    const int stride = a.slice + E;                     // from the counters to the bias indices when wide
    const uint32_t* mask = MASK ? a.allowed + b * a.allowed_ld : nullptr;
    float r = 1.f, r_inv = 1.f, fq = 0.f, ps = 0.f;
    const float* bias = nullptr;
    if constexpr (COUNTED) {
        r = a.rep ? a.rep[b] : a.rep_all;
        r_inv = a.rep ? 1.f / r : a.rep_inv;
        fq = a.freq ? a.freq[b] : a.freq_all;
        ps = a.pres ? a.pres[b] : a.pres_all;
        if (a.NB) bias = a.bias + b * a.bias_ld;
        int len = a.L > 0 ? (a.lengths ? a.lengths[b] : a.L) : 0;
        len = len < 0 ? 0 : (len > a.L ? a.L : len);
        for (int i = threadIdx.x; i < stride * K::kWords / 4; i += kLogThreads)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int prompt = a.prompts ? a.prompts[b] : 0;
        const int64_t* tok = a.tokens + b * a.tok_ld;
        constexpr int R = 4;                            // tokens of a thread in flight
        auto count = [&](int i0, auto all) {
            constexpr bool whole = decltype(all)::value;
            uint32_t v[R];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const int i = i0 + k * kLogThreads;
                v[k] = ~0u;
                if (whole || i < len) {
                    const int2 t = __ldg(reinterpret_cast<const int2*>(tok) + i);
                    if (t.y == 0) v[k] = (uint32_t)t.x - (uint32_t)lo;
                }
            }
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (v[k] < (uint32_t)n) {
                    if (i0 + k * kLogThreads >= prompt) atomicAdd(words + v[k], K::kOne);
                    else atomicOr(words + v[k], K::kSeen);
                }
        };
        int i0 = threadIdx.x;
        for (; i0 + (R - 1) * kLogThreads < len; i0 += R * kLogThreads) count(i0, std::true_type{});
        if (i0 < len) count(i0, std::false_type{});
        __syncthreads();
        if (a.NB) {
            const int64_t* ids = a.ids + b * a.ids_ld;
            for (int j = threadIdx.x; j < a.NB; j += kLogThreads) {
                const uint64_t v = (uint64_t)(__ldg(ids + j) - lo);
                if (v < (uint64_t)n) {
                    uint32_t* w = words + v + (WIDE ? stride : 0);
                    // the upper bits no longer change, so the maximum is that of the index
                    atomicMax(w, WIDE ? (uint32_t)(j + 1) : (*w & 0xffff0000u) | (uint32_t)(j + 1));
                }
            }
            __syncthreads();
        }
    }
    auto one = [&](int i) {                             // a single entry
        float v = El::to_f(x[i]);
        if (COUNTED) v = process<DT, WIDE, EACH>(v, words[i], WIDE ? words[stride + i] : 0u, r, r_inv, fq, ps, bias);
        if (MASK && !((mask[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u)) v = -INFINITY;
        y[i] = El::from_f(v);
    };
    if (!MASK && static_cast<const void*>(x) == static_cast<const void*>(y)) {
        if (COUNTED)
            for (int i = threadIdx.x; i < n; i += kLogThreads)
                if (words[i] || (WIDE && words[stride + i])) one(i);
        return;
    }
    const int head = head_x == head_y ? (head_x < n ? head_x : n) : n;      // all singly when no boundary is shared
    const int nv = (n - head) / E;
    constexpr int U = 3;                                // vectors of a thread in flight, with their mask bits
    auto vectors = [&](int i0, auto all) {
        constexpr bool whole = decltype(all)::value;
        const uint4* src = reinterpret_cast<const uint4*>(x + head) + i0;
        uint4* dst = reinterpret_cast<uint4*>(y + head) + i0;
        uint4 q[U];
        uint32_t off[U];                                // which entries the mask takes out
#pragma unroll
        for (int u = 0; u < U; ++u) {
            off[u] = 0u;
            if (whole || i0 + u * kLogThreads < nv) {
                q[u] = __ldcs(src + u * kLogThreads);
                if constexpr (MASK) {
                    const uint32_t at = (uint32_t)(lo + head + (i0 + u * kLogThreads) * E), sh = at & 31;
                    uint32_t bits = __ldg(mask + (at >> 5)) >> sh;
                    if (head && sh + E > 32) bits |= __ldg(mask + (at >> 5) + 1) << (32 - sh);
                    off[u] = ~bits & ((1u << E) - 1u);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!(whole || i0 + u * kLogThreads < nv)) continue;
            T v[E];
            if constexpr (COUNTED) {
                const uint32_t* c = words + head + (i0 + u * kLogThreads) * E;
                uint32_t w[E], any = 0u;
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const uint4 t = *reinterpret_cast<const uint4*>(c + e);
                    w[e] = t.x; w[e + 1] = t.y; w[e + 2] = t.z; w[e + 3] = t.w;
                    any |= t.x | t.y | t.z | t.w;
                    if (WIDE) {
                        const uint4 d = *reinterpret_cast<const uint4*>(c + stride + e);
                        any |= d.x | d.y | d.z | d.w;
                    }
                }
                if (any) {
                    *reinterpret_cast<uint4*>(v) = q[u];
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        v[e] = El::from_f(process<DT, WIDE, EACH>(El::to_f(v[e]), w[e], WIDE ? c[stride + e] : 0u, r, r_inv,
                                                                  fq, ps, bias));
                    q[u] = *reinterpret_cast<const uint4*>(v);
                }
            }
            if (MASK && off[u]) {
                *reinterpret_cast<uint4*>(v) = q[u];
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if ((off[u] >> e) & 1u) v[e] = El::from_f(-INFINITY);
                q[u] = *reinterpret_cast<const uint4*>(v);
            }
            __stcs(dst + u * kLogThreads, q[u]);
        }
    };
    int i0 = threadIdx.x;
    for (; i0 + (U - 1) * kLogThreads < nv; i0 += U * kLogThreads) vectors(i0, std::true_type{});
    if (i0 < nv) vectors(i0, std::false_type{});
    for (int i = threadIdx.x; i < head; i += kLogThreads) one(i);
    for (int i = head + nv * E + threadIdx.x; i < n; i += kLogThreads) one(i);
}

template <int DT, bool COUNTED, bool WIDE, bool EACH>
int launch(LogArgs a, int64_t B, cudaStream_t stream) {
    // Slices of 1024 to 8192 entries: four CTAs per SM if the rows allow it, and
    // no more slices than that, since each reads the whole history of its row.
    const int64_t want = std::max<int64_t>(1, 4 * 148 / B);
    int64_t slice = std::min<int64_t>(8192, std::max<int64_t>(1024, (a.V + want - 1) / want));
    slice = (slice + 127) / 128 * 128;
    a.slice = (int)slice;
    a.slices = (int)((a.V + slice - 1) / slice);
    if (B * a.slices > INT32_MAX) return fail(NT_ERR_ARG, "nt_logits_process: too many rows");
    const size_t smem = COUNTED ? (size_t)(slice + 16 / (DT == NT_F32 ? 4 : 2)) * 4 * Count<WIDE>::kWords : 0;
    auto kern = a.allowed ? logits_kernel<DT, COUNTED, true, WIDE, EACH> : logits_kernel<DT, COUNTED, false, WIDE, EACH>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_logits_process: %s", cudaGetErrorString(e));
    }
    kern<<<(unsigned)(B * a.slices), kLogThreads, smem, stream>>>(a);
    return check_launch("logits_kernel");
}

template <int DT>
int launch_dt(const LogArgs& a, int64_t B, bool each, cudaStream_t stream) {
    if (a.L == 0 && a.NB == 0) return launch<DT, false, false, false>(a, B, stream);
    const bool wide = a.L >= (1 << 15) || a.NB >= (1 << 16) - 1;
    if (wide) return each ? launch<DT, true, true, true>(a, B, stream) : launch<DT, true, true, false>(a, B, stream);
    return each ? launch<DT, true, false, true>(a, B, stream) : launch<DT, true, false, false>(a, B, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_logits_process(int dtype, int64_t B, int64_t V, const void* logits, int64_t ld, const int64_t* tokens,
                                 int64_t tok_ld, int64_t L, const int32_t* lengths, const int32_t* prompt_lengths, int each,
                                 const float* repetition, double repetition_all, const float* frequency, float frequency_all,
                                 const float* presence, float presence_all, const int64_t* bias_ids, int64_t ids_ld,
                                 const float* bias, int64_t bias_ld, int64_t NB, const uint32_t* allowed, int64_t allowed_ld,
                                 void* out, int64_t ldo, void* stream) {
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_logits_process: dtype %d", dtype);
    if (B < 0 || V < 1 || V > INT32_MAX / 2 || B > (1 << 24) || L < 0 || L > INT32_MAX / 2 || NB < 0 || NB > INT32_MAX / 2)
        return fail(NT_ERR_ARG, "nt_logits_process: bad sizes");
    if (B == 0) return NT_OK;
    if (!logits || !out || (L > 0 && !tokens) || (NB > 0 && (!bias_ids || !bias)))
        return fail(NT_ERR_ARG, "nt_logits_process: null pointer");
    if (out == logits && ld != ldo) return fail(NT_ERR_ARG, "nt_logits_process: in place needs equal row strides");
    if (!repetition && !each && !(repetition_all > 0.0))
        return fail(NT_ERR_ARG, "nt_logits_process: repetition penalty must be above 0");
    if (!repetition && each && (!std::isfinite(repetition_all) || repetition_all == 0.0))
        return fail(NT_ERR_ARG, "nt_logits_process: a repetition penalty per occurrence must be finite and not 0");
    if (each && prompt_lengths) return fail(NT_ERR_ARG, "nt_logits_process: a penalty per occurrence takes no prompt lengths");
    LogArgs a{};
    a.V = V; a.x = logits; a.ld = ld;
    a.tokens = L > 0 ? tokens : nullptr; a.tok_ld = tok_ld; a.L = (int)L; a.lengths = lengths; a.prompts = prompt_lengths;
    a.rep = repetition; a.freq = frequency; a.pres = presence;
    a.rep_all = (float)repetition_all; a.rep_inv = (float)(1.0 / repetition_all); a.freq_all = frequency_all; a.pres_all = presence_all;
    a.ids = bias_ids; a.ids_ld = ids_ld; a.bias = bias; a.bias_ld = bias_ld; a.NB = (int)NB;
    a.allowed = allowed; a.allowed_ld = allowed_ld;
    a.out = out; a.ldo = ldo;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == NT_F32 ? launch_dt<NT_F32>(a, B, each != 0, st) : launch_dt<NT_BF16>(a, B, each != 0, st);
}
