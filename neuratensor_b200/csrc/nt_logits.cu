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
// Several CTAs share an SM, so one streams while another counts.  (A cluster of
// CTAs per row that read the history once and counted into each other's shared
// memory was slower: 131 us against 70 us for 250 x 131072 float32 with 4000 tokens of
// history, 21.5 against 13.3 us for 64 x 32000 bf16 with 8704.)  Integer counters: the
// order of arrival changes nothing.
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

namespace nt {
namespace {

constexpr int kLogThreads = 256;

struct LogArgs {
    int64_t V;
    const void* x; int64_t ld;
    const int64_t* tokens; int64_t tok_ld; int L;
    const int32_t* lengths; const int32_t* prompts;
    const float* rep; const float* freq; const float* pres;
    float rep_all, freq_all, pres_all;
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

// One logit: the penalties of its counter w, bias entry j - 1 (0: none).
template <int DT, bool WIDE, bool EACH>
__device__ __forceinline__ float process(float x, uint32_t w, uint32_t j, float r, float r_inv, float fq, float ps,
                                         const float* bias) {
    if ((w | j) != 0) {
        const uint32_t made = WIDE ? w & 0x7fffffffu : (w >> 16) & 0x7fffu;
        if constexpr (EACH) {
            for (uint32_t i = 0; i < made; ++i) x = Elem<DT>::rnd(x > 0.f ? x * r_inv : x * r);
        } else {
            if (made || (w >> 31)) x = x > 0.f ? x * r_inv : x * r;
        }
        if (made) x -= fmaf(fq, (float)made, ps);
        if (!WIDE) j = w & 0xffffu;
        if (j) x += __ldg(bias + (j - 1));
    }
    return x;
}

template <int DT, bool WIDE, bool EACH>
__global__ void __launch_bounds__(kLogThreads, 6) logits_kernel(const __grid_constant__ LogArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    using K = Count<WIDE>;
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint32_t smem[];
    const int64_t b = blockIdx.x / a.slices;
    const int64_t lo = (int64_t)(blockIdx.x % a.slices) * a.slice;
    const int n = (int)(a.V - lo < a.slice ? a.V - lo : a.slice);
    const T* x = static_cast<const T*>(a.x) + b * a.ld + lo;
    T* y = static_cast<T*>(a.out) + b * a.ldo + lo;
    // Entries before the first 16-byte boundary of x.  Entry i's counter is
    // words[i], shifted so that those of a vector are 16-byte aligned too.
    const int head_x = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    const int head_y = (int)((16 - (reinterpret_cast<uintptr_t>(y) & 15)) & 15) / (int)sizeof(T);
    const int pad = (E - head_x) & (E - 1);
    uint32_t* words = smem + pad;
    const int stride = a.slice + E;                     // from the counters to the bias indices when wide
    const float r = a.rep ? a.rep[b] : a.rep_all, fq = a.freq ? a.freq[b] : a.freq_all, ps = a.pres ? a.pres[b] : a.pres_all;
    const float r_inv = 1.f / r;
    const uint32_t* mask = a.allowed ? a.allowed + b * a.allowed_ld : nullptr;
    const float* bias = a.NB ? a.bias + b * a.bias_ld : nullptr;
    int len = a.tokens ? (a.lengths ? a.lengths[b] : a.L) : 0;
    len = len < 0 ? 0 : (len > a.L ? a.L : len);
    const bool counted = len > 0 || a.NB > 0;

    const bool touched_only = static_cast<const void*>(x) == static_cast<const void*>(y) && !mask;
    const int head = head_x == head_y ? (head_x < n ? head_x : n) : n;      // all singly when no boundary is shared
    const int nv = touched_only ? 0 : (n - head) / E;
    // vectors of a thread in flight, with their mask bits (loading the first ones before
    // the history is counted cost registers, and so CTAs per SM: 84 us against 70)
    constexpr int U = 4;
    uint4 q[U];
    uint32_t bits[U];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kLogThreads;
            bits[u] = ~0u;
            if (i >= nv) continue;
            q[u] = __ldcs(reinterpret_cast<const uint4*>(x + head) + i);
            if (mask) {
                const uint32_t at = (uint32_t)lo + head + i * E, sh = at & 31;
                bits[u] = __ldg(mask + (at >> 5)) >> sh;
                if (sh + E > 32) bits[u] |= __ldg(mask + (at >> 5) + 1) << (32 - sh);
            }
        }
    };
    if (counted) {
        for (int i = threadIdx.x; i < stride * K::kWords / 4; i += kLogThreads)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int prompt = a.prompts ? a.prompts[b] : 0;
        const int64_t* tok = a.tokens + b * a.tok_ld;
        constexpr int R = 8;                            // tokens of a thread in flight
        for (int i0 = threadIdx.x; i0 < len; i0 += R * kLogThreads) {
            uint32_t v[R];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const int i = i0 + k * kLogThreads;
                const int64_t t = i < len ? __ldg(tok + i) : -1;
                v[k] = (uint64_t)t >> 32 ? ~0u : (uint32_t)t - (uint32_t)lo;
            }
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (v[k] < (uint32_t)n) {
                    if (i0 + k * kLogThreads >= prompt) atomicAdd(words + v[k], K::kOne);
                    else atomicOr(words + v[k], K::kSeen);
                }
        }
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
        const uint32_t w = counted ? words[i] : 0u, j = WIDE && counted ? words[stride + i] : 0u;
        const float v = process<DT, WIDE, EACH>(El::to_f(x[i]), w, j, r, r_inv, fq, ps, bias);
        const bool ok = !mask || ((mask[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u);
        y[i] = El::from_f(ok ? v : -INFINITY);
    };
    if (touched_only) {
        if (counted)
            for (int i = threadIdx.x; i < n; i += kLogThreads)
                if (words[i] || (WIDE && words[stride + i])) one(i);
        return;
    }
    for (int i0 = threadIdx.x; i0 < nv; i0 += U * kLogThreads) {
        load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kLogThreads, first = head + i * E;
            if (i >= nv) break;
            T xv[E];
            *reinterpret_cast<uint4*>(xv) = q[u];
            uint32_t w[E], any = 0u;
            if (counted) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const uint4 c = *reinterpret_cast<const uint4*>(words + first + e);
                    w[e] = c.x; w[e + 1] = c.y; w[e + 2] = c.z; w[e + 3] = c.w;
                    any |= c.x | c.y | c.z | c.w;
                    if (WIDE) {
                        const uint4 d = *reinterpret_cast<const uint4*>(words + stride + first + e);
                        any |= d.x | d.y | d.z | d.w;
                    }
                }
            }
            if (any) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    xv[e] = El::from_f(process<DT, WIDE, EACH>(El::to_f(xv[e]), w[e], WIDE ? words[stride + first + e] : 0u,
                                                               r, r_inv, fq, ps, bias));
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!((bits[u] >> e) & 1u)) xv[e] = El::from_f(-INFINITY);
            __stcs(reinterpret_cast<uint4*>(y + head) + i, *reinterpret_cast<const uint4*>(xv));
        }
    }
    for (int i = threadIdx.x; i < head; i += kLogThreads) one(i);
    for (int i = head + nv * E + threadIdx.x; i < n; i += kLogThreads) one(i);
}

template <int DT, bool WIDE, bool EACH>
int launch(LogArgs a, int64_t B, cudaStream_t stream) {
    // Slices of 1024 to 8192 entries: four CTAs per SM if the rows allow it, and
    // no more slices than that, since each reads the whole history of its row.
    const int64_t want = std::max<int64_t>(1, 4 * 148 / B);
    int64_t slice = std::min<int64_t>(8192, std::max<int64_t>(1024, (a.V + want - 1) / want));
    slice = (slice + 127) / 128 * 128;
    a.slice = (int)slice;
    a.slices = (int)((a.V + slice - 1) / slice);
    if (B * a.slices > INT32_MAX) return fail(NT_ERR_ARG, "nt_logits_process: too many rows");
    const bool counted = (a.tokens && a.L > 0) || a.NB > 0;
    const size_t smem = counted ? (size_t)(slice + 16 / (DT == NT_F32 ? 4 : 2)) * 4 * Count<WIDE>::kWords : 0;
    auto kern = logits_kernel<DT, WIDE, EACH>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_logits_process: %s", cudaGetErrorString(e));
    }
    kern<<<(unsigned)(B * a.slices), kLogThreads, smem, stream>>>(a);
    return check_launch("logits_kernel");
}

template <int DT>
int launch_dt(const LogArgs& a, int64_t B, bool each, cudaStream_t stream) {
    const bool small = a.L < (1 << 15) && a.NB < (1 << 16) - 1;
    if (small) return each ? launch<DT, false, true>(a, B, stream) : launch<DT, false, false>(a, B, stream);
    return each ? launch<DT, true, true>(a, B, stream) : launch<DT, true, false>(a, B, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_logits_process(int dtype, int64_t B, int64_t V, const void* logits, int64_t ld, const int64_t* tokens,
                                 int64_t tok_ld, int64_t L, const int32_t* lengths, const int32_t* prompt_lengths, int each,
                                 const float* repetition, float repetition_all, const float* frequency, float frequency_all,
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
    if (each && prompt_lengths) return fail(NT_ERR_ARG, "nt_logits_process: a penalty per occurrence takes no prompt lengths");
    if (!repetition && !(repetition_all > 0.f)) return fail(NT_ERR_ARG, "nt_logits_process: repetition penalty must be above 0");
    LogArgs a{};
    a.V = V; a.x = logits; a.ld = ld;
    a.tokens = L > 0 ? tokens : nullptr; a.tok_ld = tok_ld; a.L = (int)L; a.lengths = lengths; a.prompts = prompt_lengths;
    a.rep = repetition; a.freq = frequency; a.pres = presence;
    a.rep_all = repetition_all; a.freq_all = frequency_all; a.pres_all = presence_all;
    a.ids = bias_ids; a.ids_ld = ids_ld; a.bias = bias; a.bias_ld = bias_ld; a.NB = (int)NB;
    a.allowed = allowed; a.allowed_ld = allowed_ld;
    a.out = out; a.ldo = ldo;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == NT_F32 ? launch_dt<NT_F32>(a, B, each != 0, st) : launch_dt<NT_BF16>(a, B, each != 0, st);
}
