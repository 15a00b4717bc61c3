// Penalties for repeated tokens, per-request biases and grammar masks on
// logits, in one pass (NeuraTensorModel.generate's repetition penalty,
// neuratensor/core/model.py:336-342, is a host loop over every token of the
// history; frequency and presence penalties, biases and masks are what callers
// add around it).
//
// Bound by HBM: logits in and out once, one mask bit per entry, and the
// history once.  The history has to be counted per vocabulary entry before a
// logit is final, so a cluster of CTAs owns a row: each CTA holds the counters
// of its slice of the vocabulary in shared memory, reads its share of the
// history and adds to whichever CTA of the cluster owns the token (distributed
// shared memory), and after one cluster barrier streams its slice.  Integer
// counters: their order of arrival changes nothing.
//
// A counter holds the index (plus one) of the last bias entry of the token, the
// number of occurrences after the prompt, and one bit for an occurrence at all:
// 16 + 15 + 1 bits of one word while the history is below 2^15 tokens and the
// biases below 2^16, else two words (the index in the second; not one of 64
// bits, whose atomics in another CTA's shared memory lost updates when tried).
#include "nt_kernels.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

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
    int slice;                         // vocabulary entries per CTA and turn, a multiple of 128
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
__global__ void __launch_bounds__(kLogThreads) logits_kernel(const __grid_constant__ LogArgs a) {
    using El = Elem<DT>;
    using T = typename El::T;
    using K = Count<WIDE>;
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint32_t words[];       // [slice] counters, [slice] bias indices when wide
    cg::cluster_group cluster = cg::this_cluster();
    const int CS = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t b = blockIdx.x / CS;
    const T* x = static_cast<const T*>(a.x) + b * a.ld;
    T* y = static_cast<T*>(a.out) + b * a.ldo;
    const float r = a.rep ? a.rep[b] : a.rep_all, fq = a.freq ? a.freq[b] : a.freq_all, ps = a.pres ? a.pres[b] : a.pres_all;
    const float r_inv = 1.f / r;
    const uint32_t* mask = a.allowed ? a.allowed + b * a.allowed_ld : nullptr;
    const int64_t* ids = a.ids + b * a.ids_ld;
    const float* bias = a.bias + b * a.bias_ld;
    int len = a.tokens ? (a.lengths ? a.lengths[b] : a.L) : 0;
    len = len < 0 ? 0 : (len > a.L ? a.L : len);
    const int prompt = a.prompts ? a.prompts[b] : 0;
    const int64_t* tok = a.tokens + b * a.tok_ld;
    const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;

    for (int64_t base = 0; base < a.V; base += (int64_t)CS * a.slice) {
        const int64_t lo = base + (int64_t)rank * a.slice;
        const int n = lo < a.V ? (int)(a.V - lo < a.slice ? a.V - lo : a.slice) : 0;
        for (int i = threadIdx.x; i < a.slice * K::kWords; i += kLogThreads) words[i] = 0;
        cluster.sync();
        for (int i = rank * kLogThreads + threadIdx.x; i < len; i += CS * kLogThreads) {
            const int64_t v = tok[i];
            if (v < base || v >= a.V) continue;
            const int64_t rel = v - base;
            if (rel >= (int64_t)CS * a.slice) continue;
            const int owner = (int)((uint32_t)rel / (uint32_t)a.slice);
            uint32_t* w = cluster.map_shared_rank(words, owner) + ((uint32_t)rel - (uint32_t)owner * a.slice);
            if (i >= prompt) atomicAdd(w, K::kOne);
            else atomicOr(w, K::kSeen);
        }
        cluster.sync();
        for (int j = threadIdx.x; j < a.NB; j += kLogThreads) {
            const int64_t v = ids[j];
            if (v < lo || v >= lo + n) continue;
            uint32_t* w = words + (v - lo) + (WIDE ? a.slice : 0);
            // the upper bits no longer change, so the maximum is that of the index
            atomicMax(w, WIDE ? (uint32_t)(j + 1) : (*w & 0xffff0000u) | (uint32_t)(j + 1));
        }
        __syncthreads();
        auto idx = [&](int i) { return WIDE ? words[a.slice + i] : 0u; };
        auto allowed = [&](int i) { return !mask || ((mask[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u); };
        const int nv = vec ? n / E : 0;
        for (int i = threadIdx.x; i < nv; i += kLogThreads) {
            const uint4 q = *reinterpret_cast<const uint4*>(x + lo + (int64_t)i * E);
            const T* xv = reinterpret_cast<const T*>(&q);
            uint4 o;
            T* ov = reinterpret_cast<T*>(&o);
            const int64_t at = lo + (int64_t)i * E;
            const uint32_t bits = mask ? mask[at >> 5] >> (at & 31) : ~0u;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float v = El::to_f(xv[e]);
                v = process<DT, WIDE, EACH>(v, words[i * E + e], idx(i * E + e), r, r_inv, fq, ps, bias);
                ov[e] = El::from_f((bits >> e) & 1u ? v : -INFINITY);
            }
            *reinterpret_cast<uint4*>(y + at) = o;
        }
        for (int i = nv * E + threadIdx.x; i < n; i += kLogThreads) {
            const float v = process<DT, WIDE, EACH>(El::to_f(x[lo + i]), words[i], idx(i), r, r_inv, fq, ps, bias);
            y[lo + i] = El::from_f(allowed(i) ? v : -INFINITY);
        }
        cluster.sync();                 // the next turn, or the end: nobody writes to a CTA that has left
    }
}

template <int DT, bool WIDE, bool EACH>
int launch(LogArgs a, int64_t B, cudaStream_t stream) {
    constexpr int kCluster = 8;
    int64_t slice = ((a.V + kCluster - 1) / kCluster + 127) / 128 * 128;
    slice = std::min<int64_t>(slice, 196608 / (4 * Count<WIDE>::kWords) / 128 * 128);
    a.slice = (int)slice;
    const size_t smem = (size_t)slice * 4 * Count<WIDE>::kWords;
    auto kern = logits_kernel<DT, WIDE, EACH>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(NT_ERR_CUDA, "nt_logits_process: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(B * kCluster));
    cfg.blockDim = dim3(kLogThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NT_ERR_CUDA, "logits_kernel launch failed: %s", cudaGetErrorString(e));
    }
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
