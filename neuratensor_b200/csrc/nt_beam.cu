// The best continuations of a beam search over beams and vocabulary.
//
// A live beam k of an item offers every token v with
//   s = score_k + x_kv - log sum_u exp x_ku,
// a finished one itself alone with s = score_k; candidates rank by s / length^alpha
// and the n best of the item's K beams are wanted, in order, ties to the lower (k, v).
//
// Bound by HBM: every logit is read once and takes a subtraction, two products, one
// exponential and a comparison.  A CTA streams a slice of one row: each thread keeps its
// vectors in registers, its running maximum and sum of exponentials, and candidates are
// the values that reach a bound that n values of the slice are known to reach: first the r-th
// largest of each warp's lane maxima, the smallest of that over the warps, with
// r * warps >= n, which a few dozen of thousands reach, then the n-th best so far.  They are
// ranked by counting in shared memory.  A slice in which too many reach the bound (constant logits) takes its n best
// one after the other instead.  A second kernel, launched as a programmatic dependent,
// joins an item's slices: logarithms and sums in float64 (candidates of two beams may lie
// closer together than float32 can tell), then n rounds of one warp over the heads of the
// sorted lists.
//
// Both kernels, caches flushed: 256 rows of 131072 float32 logits, 32 wanted, 48.5 + 15 us (the
// 134 MB take 20.5; the candidates, their ranking and the waves' ends the rest: without candidates 36);
// 64 rows of 32000 bf16 7.3 + 6; four rows 7.8 + 7.4, which is launch, one trip to memory each and the
// ranking.  On the way, at the first size: every tile's own bound 182 us; four vectors a thread
// and two CTAs an SM 57; a ranking in which each entry took one thread 122.
#include "nt_kernels.cuh"

#include <algorithm>

namespace nt {
namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamVecs = 2;           // 16-byte vectors of a thread in work, and as many on their way
constexpr int kBeamList = 1024;        // candidates a slice can hold
constexpr int kBeamMost = 64;          // n, and beams of an item
constexpr int kBeamLists = 1024;       // slices of an item's beams
constexpr int kJoinThreads = 256;
constexpr int kJoinHeld = 2048;        // list entries whose ranks the joining kernel keeps in shared memory

struct BeamArgs {
    int64_t V;
    int K, n, slices, per;             // beams, wanted, slices of a row, vectors of a slice
    const void* x; int64_t ld;
    const float* scores; const uint8_t* finished; const int32_t* lengths;
    double alpha;
    int64_t pad; int stay;
    unsigned long long* keys;          // [rows][slices][n], largest first, 0 where there are fewer
    float2* sums;                      // [rows][slices]: maximum, sum of exp(x - maximum)
    float* out_scores; int32_t* out_rows; int64_t* out_tokens;
};

// Whether a beam's logits matter: it is not finished and can still win.
__device__ __forceinline__ bool beam_open(const BeamArgs& a, int64_t row) {
    return !(a.finished && a.finished[row]) && a.scores[row] > -INFINITY && a.scores[row] < INFINITY;
}

// Order of floats as that of unsigned words; both zeros alike.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// The larger value first, of equal ones the lower token.
__device__ __forceinline__ unsigned long long beam_key(float f, uint32_t token) {
    return (unsigned long long)ordered(f) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
        if (other > k) k = other;
    }
    return k;
}

// The 16 bytes that lie `off` bytes into lo and hi.
__device__ __forceinline__ uint4 beam_pick(const uint4& lo, const uint4& hi, int off) {
    const uint32_t w[9] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, 0u};
    const int odd = (off & 2) * 8;                      // bits
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)                         // one of the four, the same for the row
        if (off >> 2 == k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(w[i + k], w[i + k + 1], odd);
    return make_uint4(o[0], o[1], o[2], o[3]);
}
// Elements at .. at + 15 / sizeof(T) of a row of V, -inf behind its end.  What a thread takes does
// not depend on the row's alignment, so that equal rows have equal sums: a row off 16-byte
// alignment takes two aligned vectors and picks.
template <typename T>
__device__ __forceinline__ uint4 beam_load(const T* x, int off, int64_t at, int64_t V) {
    constexpr int E = 16 / (int)sizeof(T);
    const int before = off / (int)sizeof(T);            // elements of the first aligned vector that come before `at`
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
    if (off == 0 && at + E <= V) {
        out = __ldcs(reinterpret_cast<const uint4*>(x + at));
    } else if (off != 0 && at >= before && at - before + 2 * E <= V) {
        const uint4* p = reinterpret_cast<const uint4*>(x + at - before);
        out = beam_pick(__ldg(p), __ldg(p + 1), off);
    } else {
        // element by element, across the row's end too
        auto bits = [&](int e) -> uint32_t {
            if constexpr (sizeof(T) == 4) return at + e < V ? reinterpret_cast<const uint32_t*>(x)[at + e] : 0xff800000u;
            else return at + e < V ? (uint32_t)reinterpret_cast<const uint16_t*>(x)[at + e] : 0xff80u;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) o[i] = bits(i);
            else o[i] = bits(2 * i) | bits(2 * i + 1) << 16;
        }
    }
    return out;
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ unsigned long long list[kBeamList];
    __shared__ uint32_t warp_bound[kBeamWarps];
    __shared__ unsigned long long warp_key[kBeamWarps];
    __shared__ float warp_m[kBeamWarps], warp_s[kBeamWarps];
    __shared__ int found[3];                            // candidates of the tiles t, t + 1 and t + 2 (mod 3)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.y;
    if (!beam_open(a, row)) return;
    if (tid < 3) found[tid] = 0;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15);       // bytes by which the row is off 16-byte alignment
    const int64_t n_vec = (a.V + E - 1) / E;
    const int64_t begin = (int64_t)blockIdx.x * a.per, end = begin + a.per < n_vec ? begin + a.per : n_vec;

    const uint4 none = DT == NT_F32 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)
                                    : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    auto value = [](const uint4& w, int e) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w);
        return DT == NT_F32 ? __uint_as_float(u[e]) : __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
    };
    // keeps the n best of the first m entries of the list, in order
    auto shrink = [&](int m) {
        if (m <= kBeamThreads) {
            // several lanes an entry, each against its part of the others
            const int q = m <= 32 ? 8 : m <= 64 ? 4 : m <= 128 ? 2 : 1, c = tid / q;
            const unsigned long long mine = c < m ? list[c] : 0ull;
            int rank = 0;
            for (int j = tid % q; j < m; j += q) rank += list[j] > mine;
            for (int o = 1; o < q; o *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, o);
            __syncthreads();
            if (tid % q == 0 && c < m && rank < a.n) list[rank] = mine;
        } else {
            unsigned long long mine[kBeamList / kBeamThreads];
            int rank[kBeamList / kBeamThreads];
#pragma unroll
            for (int i = 0; i < kBeamList / kBeamThreads; ++i) {
                mine[i] = tid + i * kBeamThreads < m ? list[tid + i * kBeamThreads] : 0ull;
                rank[i] = 0;
            }
            for (int j = 0; j < m; ++j) {
                const unsigned long long k = list[j];
#pragma unroll
                for (int i = 0; i < kBeamList / kBeamThreads; ++i) rank[i] += k > mine[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kBeamList / kBeamThreads; ++i)
                if (tid + i * kBeamThreads < m && rank[i] < a.n) list[rank[i]] = mine[i];
        }
        __syncthreads();
        return m < a.n ? m : a.n;
    };

    float top = -INFINITY, sum = 0.f, bound = -INFINITY;
    int held = 0, bound_of = 0;                         // entries when the bound was taken
    const int rounds = (a.n + kBeamWarps - 1) / kBeamWarps;
    uint4 raw[kBeamVecs], next[kBeamVecs];
    // tiles of whole vectors need no checks: of an aligned row up to `plain`, of another from vector 1 to `picked`
    constexpr int kTileVecs = kBeamVecs * kBeamThreads;
    const int64_t plain = off == 0 ? min(end, a.V / E) - kTileVecs : -1;
    const int64_t picked = off != 0 ? min(end, (a.V + off / (int)sizeof(T)) / E - 1) - kTileVecs : -1;
    const uint4* mine = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x) - off) + tid;
    auto load = [&](int64_t v0, uint4 (&to)[kBeamVecs]) {
        if (v0 <= plain) {
#pragma unroll
            for (int j = 0; j < kBeamVecs; ++j) to[j] = __ldcs(mine + v0 + j * kBeamThreads);
        } else if (v0 > 0 && v0 <= picked) {
#pragma unroll
            for (int j = 0; j < kBeamVecs; ++j) {
                const uint4 lo = __ldg(mine + v0 + j * kBeamThreads), hi = __ldg(mine + v0 + j * kBeamThreads + 1);
                to[j] = beam_pick(lo, hi, off);
            }
        } else {
#pragma unroll 1
            for (int j = 0; j < kBeamVecs; ++j) {
                const int64_t v = v0 + j * kBeamThreads + tid;
                const uint4 w = v < end ? beam_load<T>(x, off, v * E, a.V) : none;
#pragma unroll
                for (int i = 0; i < kBeamVecs; ++i)
                    if (i == j) to[i] = w;
            }
        }
    };
    load(begin, next);
    __syncthreads();
    int slot = 0;
    for (int64_t v0 = begin; v0 < end; v0 += kBeamThreads * kBeamVecs) {
#pragma unroll
        for (int j = 0; j < kBeamVecs; ++j) raw[j] = next[j];
        if (v0 + kBeamThreads * kBeamVecs < end) load(v0 + kBeamThreads * kBeamVecs, next);
        float tops[kBeamVecs], best = -INFINITY;        // of each vector, and of all
#pragma unroll
        for (int j = 0; j < kBeamVecs; ++j) {
            if constexpr (DT == NT_F32) {
                tops[j] = fmaxf(fmaxf(value(raw[j], 0), value(raw[j], 1)), fmaxf(value(raw[j], 2), value(raw[j], 3)));
            } else {
                const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&raw[j]);
                const __nv_bfloat162 two = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
                tops[j] = fmaxf(__low2float(two), __high2float(two));
            }
            best = fmaxf(best, tops[j]);
        }
        if (held < a.n) {
            // no bound yet: the r-th largest of each warp's lane maxima, the smallest of that over the warps
            uint32_t o = ordered(best), bw = 0u;
            for (int r = 0; r < rounds; ++r) {
                bw = __reduce_max_sync(0xffffffffu, o);
                const unsigned who = __ballot_sync(0xffffffffu, o == bw);
                if (lane == __ffs(who) - 1) o = 0u;
            }
            if (lane == 0) warp_bound[warp] = bw;
        }
        if (best > top) {
            sum = top == -INFINITY ? sum : sum * ex2((top - best) * kLog2e);
            top = best;
        }
        const float base = top == -INFINITY ? 0.f : top;
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kBeamVecs; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) part[e & 1] += ex2((value(raw[j], e) - base) * kLog2e);
        sum += part[0] + part[1];
        if (held < a.n) {
            __syncthreads();
            uint32_t least = warp_bound[0];
#pragma unroll
            for (int w = 1; w < kBeamWarps; ++w) least = min(least, warp_bound[w]);
            bound = least ? from_ordered(least) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < kBeamVecs; ++j)
            if (tops[j] >= bound && tops[j] > -INFINITY) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float f = value(raw[j], e);
                    if (f >= bound && f > -INFINITY) {
                        const int at = held + atomicAdd(&found[slot], 1);
                        if (at < kBeamList) list[at] = beam_key(f, (uint32_t)((v0 + j * kBeamThreads + tid) * E + e));
                    }
                }
            }
        __syncthreads();
        // A warp may count the next tile's candidates before another has read this tile's: each tile has a
        // count of its own.  The one that the tile before has used, which all have read ahead of the barrier
        // above, is cleared for the tile after the next, whose warps have passed that one's barrier.
        const int now = held + found[slot], last = slot == 0 ? 2 : slot - 1;
        if (tid == 0) found[last] = 0;
        slot = slot == 2 ? 0 : slot + 1;
        if (now > kBeamList) {
            // too many: the list as it was, and the n best of this tile one after the other
            held = shrink(held);
            unsigned long long prev = ~0ull;
            for (int r = 0; r < a.n; ++r) {
                unsigned long long k = 0ull;
#pragma unroll
                for (int j = 0; j < kBeamVecs; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float f = value(raw[j], e);
                        if (f > -INFINITY) {
                            const unsigned long long c = beam_key(f, (uint32_t)((v0 + j * kBeamThreads + tid) * E + e));
                            if (c < prev && c > k) k = c;
                        }
                    }
                k = warp_max(k);
                if (lane == 0) warp_key[warp] = k;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kBeamWarps; ++w)
                    if (warp_key[w] > k) k = warp_key[w];
                __syncthreads();
                if (k == 0ull) break;
                if (tid == 0) list[held] = k;
                ++held;
                prev = k;
            }
            __syncthreads();
        } else {
            held = now;
        }
        // the n-th best so far is the bound of what follows
        if (held >= a.n && (bound_of == 0 || held >= bound_of + 64) && v0 + kBeamThreads * kBeamVecs < end) {
            held = shrink(held);
            bound_of = held;
            bound = from_ordered((uint32_t)(list[a.n - 1] >> 32));
        }
    }
    // the slice's maximum and sum, and its n best
    float m = top;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_m[warp] = m;
    held = shrink(held);
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) m = fmaxf(m, warp_m[w]);
    sum = top == -INFINITY ? sum : sum * ex2((top - m) * kLog2e);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_s[warp] = sum;
    __syncthreads();
    const int64_t at = row * a.slices + blockIdx.x;
    if (tid == 0) {
        float s = 0.f;
        for (int w = 0; w < kBeamWarps; ++w) s += warp_s[w];
        a.sums[at] = make_float2(m, s);
    }
    if (tid < a.n) a.keys[at * a.n + tid] = tid < held ? list[tid] : 0ull;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Order of float64 as that of unsigned words, 0 for what cannot be chosen.
__device__ __forceinline__ unsigned long long ordered64(double r) {
    if (!(r > -INFINITY && r < INFINITY)) return 0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(r + 0.0);
    return u ^ ((unsigned long long)((long long)u >> 63) | 0x8000000000000000ull);
}

__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
    __shared__ double lse[kBeamMost], norm[kBeamMost];
    __shared__ unsigned long long ranks[kJoinHeld];
    __shared__ uint32_t tokens[kJoinHeld];
    __shared__ uint16_t head_at[kBeamLists];
    __shared__ uint8_t kind[kBeamMost];                 // 0 nothing to offer, 1 live, 2 finished
    __shared__ int chosen[kBeamMost], chosen_from[kBeamMost];
    __shared__ uint32_t chosen_token[kBeamMost];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row0 = (int64_t)blockIdx.x * a.K;
    const int S = a.slices, lists = a.K * S, n = a.n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int k = warp; k < a.K; k += kJoinThreads / 32) {
        const int64_t row = row0 + k;
        const bool done = a.finished && a.finished[row];
        const float score = a.scores[row];
        int what = !(score > -INFINITY && score < INFINITY) ? 0 : done ? 2 : 1;
        double l = 0.0;
        if (what == 1) {
            float m = -INFINITY;
            for (int s = lane; s < S; s += 32) m = fmaxf(m, a.sums[row * S + s].x);
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            double sum = 0.0;
            for (int s = lane; s < S; s += 32) {
                const float2 p = a.sums[row * S + s];
                sum += p.x == m || p.x == -INFINITY ? (double)p.y : (double)p.y * exp((double)p.x - (double)m);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = (double)m + log(sum);
            if (!(l > -INFINITY && l < INFINITY)) what = 0;         // NaN or infinity among the logits, or nothing left
        }
        if (lane == 0) {
            lse[k] = l;
            kind[k] = (uint8_t)what;
            const double len = a.lengths ? (double)a.lengths[row] + (what == 1 ? 1.0 : 0.0) : 1.0;
            norm[k] = a.alpha != 0.0 ? pow(len > 1.0 ? len : 1.0, a.alpha) : 1.0;
        }
    }
    const bool near = lists * n <= kJoinHeld;
    const unsigned long long* keys = a.keys + row0 * S * n;
    __syncthreads();
    // the sum of the candidate at place i of list l, which is there
    auto sum_of = [&](int l, int i) {
        const int k = l / S;
        const double s = a.scores[row0 + k];
        return kind[k] == 2 ? s : s + ((double)from_ordered((uint32_t)(keys[l * n + i] >> 32)) - lse[k]);
    };
    // its rank (0: it is not) and token
    auto look = [&](int l, int i, uint32_t* token) -> unsigned long long {
        const int k = l / S;
        *token = (uint32_t)a.pad;
        if (kind[k] == 2 ? l != k * S || i > 0 : kind[k] != 1 || i >= n) return 0ull;
        if (kind[k] == 1) {
            const unsigned long long c = keys[l * n + i];
            if (!c) return 0ull;
            *token = ~(uint32_t)c;
        }
        return ordered64(a.alpha != 0.0 ? sum_of(l, i) / norm[k] : sum_of(l, i));
    };
    if (near)
        for (int i = tid; i < lists * n; i += kJoinThreads) {
            uint32_t token;
            ranks[i] = look(i / n, i % n, &token);
            tokens[i] = token;
        }
    __syncthreads();
    if (warp == 0) {
        // a lane has lists lane, lane + 32, ...; its best head
        unsigned long long best = 0ull;
        uint32_t beam = ~0u, token = ~0u;
        int from = -1;
        auto pick = [&]() {
            best = 0ull, beam = token = ~0u, from = -1;
            for (int l = lane; l < lists; l += 32) {
                const int i = head_at[l];
                uint32_t t = 0u;
                unsigned long long r = 0ull;
                if (i < n) {
                    if (near) r = ranks[l * n + i], t = tokens[l * n + i];
                    else r = look(l, i, &t);
                }
                const uint32_t k = l / S;
                if (r > best || (r && r == best && (k < beam || (k == beam && keys[l * n + i] > keys[from * n + head_at[from]]))))
                    best = r, beam = k, token = t, from = l;
            }
        };
        // with a list a lane or none, its next two candidates are in registers
        const bool each = near && lists <= 32;
        int at = 0;
        unsigned long long then = 0ull;
        uint32_t then_token = 0u;
        if (each) {
            if (lane < lists) {
                best = ranks[lane * n], token = tokens[lane * n], beam = lane / S, from = lane;
                if (n > 1) then = ranks[lane * n + 1], then_token = tokens[lane * n + 1];
            }
        } else {
            for (int l = lane; l < lists; l += 32) head_at[l] = 0;
            pick();
        }
        for (int i = 0; i < n; ++i) {
            // the largest rank, of equal ones the lowest beam, of its own the largest logit, then the lowest token
            const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
            bool mine = (uint32_t)(best >> 32) == hi;
            const uint32_t lo = __reduce_max_sync(0xffffffffu, mine ? (uint32_t)best : 0u);
            mine = mine && (uint32_t)best == lo;
            if (!(hi | lo)) {                           // nothing left
                if (lane == 0) chosen[i] = -1;
                continue;
            }
            if (__popc(__ballot_sync(0xffffffffu, mine)) > 1) {
                const uint32_t k = __reduce_min_sync(0xffffffffu, mine ? beam : ~0u);
                mine = mine && beam == k;
                if (__popc(__ballot_sync(0xffffffffu, mine)) > 1) {
                    // a beam's own, from several slices: sums alike, but the logits need not be (float64 drops what tells them apart
                    // beside scores of 1e10 and more), so by these, then by token, as the slices' lists are
                    const unsigned long long key = mine ? keys[from * n + (each ? at : head_at[from])] : 0ull;
                    const uint32_t x = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
                    mine = mine && (uint32_t)(key >> 32) == x;
                    const uint32_t t = __reduce_max_sync(0xffffffffu, mine ? (uint32_t)key : 0u);
                    mine = mine && (uint32_t)key == t;
                }
            }
            if (mine) {
                chosen[i] = (int)beam;
                chosen_token[i] = token;
                if (each) {
                    chosen_from[i] = lane * n + at++;
                    best = then, token = then_token;
                    then = 0ull;
                    if (at + 1 < n) then = ranks[lane * n + at + 1], then_token = tokens[lane * n + at + 1];
                } else {
                    chosen_from[i] = from * n + head_at[from];
                    ++head_at[from];
                    pick();
                }
            }
            __syncwarp();
        }
        __syncwarp();
        // places: in order, or the first child of a beam in the beam's own
        __shared__ int8_t place[kBeamMost];
        if (lane == 0) {
            unsigned long long taken = 0ull;
            for (int i = 0; i < n; ++i) {
                place[i] = (int8_t)(a.stay ? -1 : i);
                if (a.stay && chosen[i] >= 0 && !(taken >> chosen[i] & 1)) {
                    place[i] = (int8_t)chosen[i];
                    taken |= 1ull << chosen[i];
                }
            }
            for (int i = 0; i < n; ++i)
                if (place[i] < 0) {
                    place[i] = (int8_t)(__ffsll((long long)~taken) - 1);
                    taken |= 1ull << place[i];
                }
        }
        __syncwarp();
        for (int i = lane; i < n; i += 32) {
            const int64_t at = (int64_t)blockIdx.x * n + place[i];
            const bool some = chosen[i] >= 0;
            a.out_scores[at] = some ? (float)sum_of(chosen_from[i] / n, chosen_from[i] % n) : -INFINITY;
            a.out_rows[at] = (int32_t)(row0 + (some ? chosen[i] : place[i] % a.K));
            a.out_tokens[at] = some ? (int64_t)chosen_token[i] : a.pad;
        }
    }
}

// Slices of a row: enough CTAs for the device, a vector a thread at least, and no more lists
// of an item than the joining kernel holds.
struct BeamPlan { int slices, per; int64_t bytes; };
BeamPlan beam_plan(int64_t B, int64_t K, int64_t V, int64_t n, int es) {
    const int64_t n_vec = (V + 16 / es - 1) / (16 / es), rows = B * K;
    int64_t s = std::max<int64_t>(1, 148 * 4 / std::max<int64_t>(1, rows));
    s = std::min({s, (n_vec + kBeamThreads - 1) / kBeamThreads, (int64_t)kBeamLists / K, (int64_t)64});
    s = std::max<int64_t>(1, s);
    BeamPlan p;
    const int64_t step = kBeamThreads;
    p.per = (int)(((n_vec + s - 1) / s + step - 1) / step * step);
    p.slices = (int)((n_vec + p.per - 1) / p.per);
    p.bytes = rows * p.slices * (n * 8 + 8);
    return p;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_beam_select_workspace_bytes(int dtype, int64_t B, int64_t K, int64_t V, int64_t n) {
    if (B < 1 || K < 1 || K > kBeamMost || V < 1 || n < 1 || n > kBeamMost) return 0;
    return beam_plan(B, K, V, n, dtype == NT_F32 ? 4 : 2).bytes;
}

int nt_beam_select(int dtype, int64_t B, int64_t K, int64_t V, int64_t n, const void* logits, int64_t ld, const float* scores,
                   const uint8_t* finished, const int32_t* lengths, double length_penalty, int64_t pad, int stay,
                   float* out_scores, int32_t* out_rows, int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                   void* stream) {
    if (dtype != NT_F32 && dtype != NT_BF16) return fail(NT_ERR_DTYPE, "nt_beam_select: dtype %d", dtype);
    if (B < 0 || V < 1 || V > (int64_t)INT32_MAX || B * K > 65535)
        return fail(NT_ERR_ARG, "nt_beam_select: bad sizes (at most 65535 rows)");
    if (K < 1 || K > kBeamMost || n < 1 || n > kBeamMost)
        return fail(NT_ERR_ARG, "nt_beam_select: %lld beams, %lld wanted (1 to %d of each)", (long long)K, (long long)n, kBeamMost);
    if (stay && n != K) return fail(NT_ERR_ARG, "nt_beam_select: children in their parents' places need n == K");
    if (!(length_penalty > -1e300 && length_penalty < 1e300)) return fail(NT_ERR_ARG, "nt_beam_select: length penalty must be finite");
    if (length_penalty != 0.0 && !lengths) return fail(NT_ERR_ARG, "nt_beam_select: a length penalty needs lengths");
    if (pad < 0 || pad > (int64_t)INT32_MAX) return fail(NT_ERR_ARG, "nt_beam_select: pad %lld", (long long)pad);
    if (B == 0) return NT_OK;
    if (!logits || !scores || !out_scores || !out_rows || !out_tokens) return fail(NT_ERR_ARG, "nt_beam_select: null pointer");
    const int es = dtype == NT_F32 ? 4 : 2;
    const BeamPlan p = beam_plan(B, K, V, n, es);
    if (!workspace || workspace_bytes < p.bytes)
        return fail(NT_ERR_WORKSPACE, "nt_beam_select: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)p.bytes);
    if ((reinterpret_cast<uintptr_t>(logits) & (es - 1)) || (reinterpret_cast<uintptr_t>(workspace) & 7))
        return fail(NT_ERR_ARG, "nt_beam_select: alignment");
    BeamArgs a{};
    a.V = V; a.K = (int)K; a.n = (int)n; a.slices = p.slices; a.per = p.per;
    a.x = logits; a.ld = ld; a.scores = scores; a.finished = finished; a.lengths = lengths;
    a.alpha = length_penalty; a.pad = pad; a.stay = stay;
    a.keys = static_cast<unsigned long long*>(workspace);
    a.sums = reinterpret_cast<float2*>(a.keys + B * K * p.slices * n);
    a.out_scores = out_scores; a.out_rows = out_rows; a.out_tokens = out_tokens;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)p.slices, (unsigned)(B * K));
    if (dtype == NT_F32) beam_scan_kernel<NT_F32><<<grid, kBeamThreads, 0, st>>>(a);
    else beam_scan_kernel<NT_BF16><<<grid, kBeamThreads, 0, st>>>(a);
    const int rc = check_launch("beam_scan_kernel");
    if (rc != NT_OK) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)B);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, beam_join_kernel, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NT_ERR_CUDA, "beam_join_kernel launch failed: %s", cudaGetErrorString(e));
    }
    return check_launch("beam_join_kernel");
}

}  // extern "C"
