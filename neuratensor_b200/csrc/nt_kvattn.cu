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
#include "nt_kvattn.cuh"

namespace nt {
namespace {

using namespace kva;

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
