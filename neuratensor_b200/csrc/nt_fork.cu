// Sequences that go on from others without copying their cache: pages are shared, counted,
// made own where they will be written, and free when no sequence has them.
//
// kv_fork rewrites a page table [R, blocks] for the rows that go on: row r takes the live
// entries of row parents[r] (those its window can still see).  refs[p] counts the entries
// of page p, with whatever else holds it.  The page of the next token is made own: of the
// rows in which it is begun and not full, one keeps it when nothing else has it (one that
// had it before, else the first), the others get a new page each and a place in the list of
// copies.  New pages, these and those of the new tokens, are the free ones of lowest index,
// row by row and block by block, so the result does not depend on any order of arrival.
//
// Two kernels, both short: the table column by column (every row of a few blocks in shared
// memory, so it is rewritten in place; counts change only where entries do), then one CTA
// that hands out pages.  They are bound by the trips to memory that depend on each other
// (parents, lengths, table, counts).  The copies themselves (kv_copy_pages, all layers in one
// launch) are bound by HBM, or by launch where they are few.  Kernels, caches flushed: 64 rows of 272
// blocks, 4 layers 4.4 + 11.8 + 5.4 us; 256 rows of 626 blocks 6.2 + 17 + 6 (24 + 101 with
// 16 CTAs for the table and the shared blocks found by the one CTA behind it).
#include "nt_kernels.cuh"

#include <algorithm>

namespace nt {
namespace {

constexpr int kForkRows = 1024;
constexpr int kForkThreads = 1024;
constexpr int kTableThreads = 512;
constexpr int kTableWords = 7680;      // table entries of a CTA in shared memory

struct ForkArgs {
    int R, group; int64_t n_pages, n_blocks; int page, tokens; int64_t window;   // window < 0: none
    int32_t* table; int64_t table_sb;
    int32_t* refs; int32_t* lengths; const int32_t* parents;
    int32_t* copies; int32_t* shared;
    int32_t* alike;                    // [groups][column CTAs]: first block of the columns that the group's rows do not share
    int columns, column_ctas;
    unsigned* err;
};

// Length of the sequence that row r goes on from, 0 for none (or a bad one).
__device__ __forceinline__ int fork_length(const ForkArgs& a, int r, bool* bad) {
    const int p = a.parents[r];
    if (p < 0 || p >= a.R) {
        if (p != -1) *bad = true;
        return 0;
    }
    const int n = a.lengths[p];
    if (n < 0 || n > a.n_blocks * a.page) {
        *bad = true;
        return 0;
    }
    return n;
}

__global__ void __launch_bounds__(kTableThreads) fork_table_kernel(const __grid_constant__ ForkArgs a) {
    __shared__ int32_t old[kTableWords];
    __shared__ int32_t from[kForkRows];                 // the row that a row goes on from; its live blocks [low, high)
    __shared__ int32_t low[kForkRows], high[kForkRows];
    __shared__ int32_t differ[kForkRows];               // first block of these columns that a group's rows do not share
    const int j0 = blockIdx.x * a.columns, m = (int)(a.n_blocks - j0 < a.columns ? a.n_blocks - j0 : a.columns);
    bool bad = false;
    for (int i = threadIdx.x; i < a.R * m; i += kTableThreads) old[i] = a.table[i / m * a.table_sb + j0 + i % m];
    for (int r = threadIdx.x; r < a.R; r += kTableThreads) {
        const int len = fork_length(a, r, &bad);
        from[r] = len ? a.parents[r] : 0;
        low[r] = a.window >= 0 && len > a.window ? (int)((len - a.window) / a.page) : 0;
        high[r] = (len + a.page - 1) / a.page;
        differ[r] = 0x7fffffff;
    }
    __syncthreads();
    auto entry = [&](int r, int c, bool* wrong) {
        const int j = j0 + c, now = j >= low[r] && j < high[r] ? old[from[r] * m + c] : -1;
        if (now >= -1 && now < a.n_pages) return now;
        *wrong = true;
        return -1;
    };
    for (int i = threadIdx.x; i < a.R * m; i += kTableThreads) {
        const int r = i / m, c = i % m, before = old[i], now = entry(r, c, &bad);
        if (now != before) {
            a.table[r * a.table_sb + j0 + c] = now;
            if (now >= 0) atomicAdd(a.refs + now, 1);
            if (before >= 0 && before < a.n_pages) atomicAdd(a.refs + before, -1);
        }
        if (a.group > 0 && r % a.group && now != entry(r - r % a.group, c, &bad)) atomicMin(&differ[r / a.group], j0 + c);
    }
    if (bad) atomicOr(a.err, ERRF_BAD_ARG);
    __syncthreads();
    if (a.group > 0)
        for (int g = threadIdx.x; g < a.R / a.group; g += kTableThreads) a.alike[g * a.column_ctas + blockIdx.x] = differ[g];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Exclusive prefix sum over the CTA's threads; `total` gets the sum.
__device__ __forceinline__ int prefix(int v, int* warps, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int w = warps[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += up;
        }
        warps[lane] = w;
    }
    __syncthreads();
    *total = warps[31];
    return sum - v + (warp ? warps[warp - 1] : 0);
}

__global__ void __launch_bounds__(kForkThreads) fork_pages_kernel(const __grid_constant__ ForkArgs a) {
    static_assert(kForkThreads == kForkRows, "a thread per row");
    __shared__ int tail[kForkRows];                     // the begun page of a row, -1: none
    __shared__ int warps[32];
    __shared__ int lens[kForkRows];
    const int r = threadIdx.x;
    bool bad = false;
    int len = 0, before = -1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (r < a.R) {
        len = fork_length(a, r, &bad);
        bad = bad && a.n_blocks == 0;                   // flagged by the kernel before, which a table of no blocks does not have
        if (len % a.page) before = a.table[r * a.table_sb + len / a.page];
    }
    tail[r] = before;
    lens[r] = len;
    __syncthreads();
    bool copy = false;
    if (before >= 0) {
        int same = 0, keeper = -1;
        bool stays = false;
        for (int i = 0; i < a.R; ++i)
            if (tail[i] == before) {
                ++same;
                const bool own = a.parents[i] == i;
                if (keeper < 0 || (own && !stays)) {
                    keeper = i;
                    stays = own;
                }
            }
        copy = keeper != r || a.refs[before] != same;
    }
    // blocks of the new tokens that their window will see, behind the row's last one
    const int64_t have = (len + a.page - 1) / a.page;
    int64_t from = have, to = ((int64_t)len + a.tokens + a.page - 1) / a.page;
    if (r >= a.R || a.parents[r] < 0 || a.parents[r] >= a.R) to = from;
    if (to > a.n_blocks) {
        to = a.n_blocks;
        bad = true;
    }
    if (a.window >= 0 && (int64_t)len + a.tokens > a.window) {
        const int64_t seen = ((int64_t)len + a.tokens - a.window) / a.page;
        from = seen > from ? seen : from;
    }
    const int fresh = (int)(to > from ? to - from : 0);
    int want;
    const int first = prefix(fresh + copy, warps, &want);
    // every thread has read the counts that decide; now they change
    if (copy) atomicAdd(a.refs + before, -1);
    if (r < a.R) {
        a.copies[2 * r] = copy ? before : -1;
        a.copies[2 * r + 1] = -1;
    }
    // the `want` free pages of lowest index; a page that a copy has just let go stays taken by another
    __shared__ int starts[kForkRows + 1];
    __shared__ int froms[kForkRows];
    starts[r] = first;
    froms[r] = (int)from;
    if (r == 0) starts[kForkRows] = want;
    __shared__ uint8_t copied[kForkRows];
    copied[r] = copy;
    __syncthreads();
    int found = 0;
    for (int64_t p0 = 0; p0 < a.n_pages && found < want; p0 += 4 * kForkThreads) {
        const int64_t p = p0 + 4 * r;
        int32_t held[4];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) held[i] = p + i < a.n_pages ? a.refs[p + i] : 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += held[i] == 0;
        int here;
        int nth = found + prefix(mine, warps, &here);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (held[i] != 0) continue;
            if (nth < want) {
                int lo = 0, hi = kForkRows;             // the last row that starts at or before nth
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (starts[mid] <= nth) lo = mid; else hi = mid;
                }
                const int k = nth - starts[lo];
                int64_t j;
                if (copied[lo] && k == 0) {
                    j = lens[lo] / a.page;
                    a.copies[2 * lo + 1] = (int)(p + i);
                } else {
                    j = froms[lo] + k - copied[lo];
                }
                a.table[lo * a.table_sb + j] = (int)(p + i);
                a.refs[p + i] = 1;
            }
            ++nth;
        }
        found += here;
        __syncthreads();
    }
    if (found < want) {
        // no page left: those rows' entries are empty, and nothing is copied
        if (first + fresh + copy > found) {
            bad = true;
            int k = found > first ? found - first : 0;
            for (; k < fresh + copy; ++k) {
                if (copy && k == 0) {
                    a.table[r * a.table_sb + len / a.page] = -1;
                    a.copies[2 * r] = -1;
                } else {
                    a.table[r * a.table_sb + from + k - copy] = -1;
                }
            }
        }
    }
    if (bad) atomicOr(a.err, ERRF_BAD_ARG);
    __syncthreads();                                    // the lengths are read, the table is written
    if (r < a.R) a.lengths[r] = len;
    if (!a.shared) return;
    // leading full blocks that a group's rows have in common, a warp a group
    const int lane = r & 31;
    for (int g = r >> 5; g < a.R / a.group; g += kForkThreads / 32) {
        int least = INT32_MAX;
        for (int i = lane; i < a.group; i += 32) least = min(least, lens[g * a.group + i] / a.page);
        for (int i = lane; i < a.column_ctas; i += 32) least = min(least, a.alike[g * a.column_ctas + i]);
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) a.shared[g] = least * a.page;
    }
}

// ---------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyLayers = 64;
constexpr int kCopyChunk = 16384;

struct CopyArgs {
    const int32_t* pages; int64_t n_pages; int64_t side_bytes, heads;
    int chunks;                        // CTAs of a page and side
    struct { const char* codes[2]; const float* scale[2]; } layer[kCopyLayers];
    unsigned* err;
};

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    const int64_t src = a.pages[2 * (int64_t)blockIdx.x], dst = a.pages[2 * (int64_t)blockIdx.x + 1];
    if (src == -1 && dst == -1) return;
    const int layer = blockIdx.z, side = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks;
    if (src < 0 || dst < 0 || src >= a.n_pages || dst >= a.n_pages) {
        if (threadIdx.x == 0 && blockIdx.y == 0 && layer == 0) atomicOr(a.err, ERRF_BAD_ARG);
        return;
    }
    char* codes = const_cast<char*>(a.layer[layer].codes[side]);
    const int64_t at = (int64_t)chunk * kCopyChunk;
    const int n = (int)((a.side_bytes - at < kCopyChunk ? a.side_bytes - at : kCopyChunk) / 16);
    const uint4* s = reinterpret_cast<const uint4*>(codes + src * a.side_bytes + at);
    uint4* d = reinterpret_cast<uint4*>(codes + dst * a.side_bytes + at);
    uint4 v[kCopyChunk / 16 / kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyChunk / 16 / kCopyThreads; ++i)
        if ((int)threadIdx.x + i * kCopyThreads < n) v[i] = s[threadIdx.x + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyChunk / 16 / kCopyThreads; ++i)
        if ((int)threadIdx.x + i * kCopyThreads < n) d[threadIdx.x + i * kCopyThreads] = v[i];
    if (chunk == 0) {
        float* scale = const_cast<float*>(a.layer[layer].scale[side]);
        for (int64_t h = threadIdx.x; h < a.heads; h += kCopyThreads) scale[dst * a.heads + h] = scale[src * a.heads + h];
    }
}

// Columns of a CTA: all of the device's SMs, but a few columns each, which lie next to each other in memory.
void fork_columns(int64_t R, int64_t n_blocks, int* columns, int* ctas) {
    const int64_t most = std::min<int64_t>(std::max<int64_t>(n_blocks, 1), kTableWords / std::max<int64_t>(R, 1));
    *columns = (int)std::min<int64_t>(most, std::max<int64_t>(8, (n_blocks + 147) / 148));
    *ctas = (int)((n_blocks + *columns - 1) / *columns);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_kv_fork_workspace_bytes(int64_t R, int64_t n_blocks, int64_t group) {
    if (R < 1 || R > kForkRows || n_blocks < 0 || group < 1) return 0;
    int columns, ctas;
    fork_columns(R, n_blocks, &columns, &ctas);
    return (R / group) * (int64_t)ctas * 4;
}

int nt_kv_fork(int64_t R, int64_t n_pages, int64_t n_blocks, int64_t page, int64_t tokens, int64_t window, int64_t group,
               int32_t* table, int64_t table_sb, int32_t* refs, int32_t* lengths, const int32_t* parents, int32_t* copies,
               int32_t* shared, void* workspace, int64_t workspace_bytes, void* stream) {
    if (R < 0 || R > kForkRows) return fail(NT_ERR_ARG, "nt_kv_fork: %lld rows (at most %d)", (long long)R, kForkRows);
    if (page < 1 || page > 65536 || tokens < 0 || tokens > INT32_MAX / 2 || n_pages < 0 || n_pages > INT32_MAX || n_blocks < 0 ||
        n_blocks * page > (int64_t)INT32_MAX - 4096 || group < 0 || (group > 0 && R % group) || (n_blocks > 0 && table_sb < n_blocks))
        return fail(NT_ERR_ARG, "nt_kv_fork: bad sizes");
    if (R == 0) return NT_OK;
    if ((!table && n_blocks > 0) || (!refs && n_pages > 0) || !lengths || !parents || !copies || (group > 0 && !shared)) return fail(NT_ERR_ARG, "nt_kv_fork: null pointer");
    const int64_t need = nt_kv_fork_workspace_bytes(R, n_blocks, group);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(NT_ERR_WORKSPACE, "nt_kv_fork: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
    int dev = 0;
    cudaGetDevice(&dev);
    ForkArgs a{};
    a.R = (int)R; a.group = (int)group; a.n_pages = n_pages; a.n_blocks = n_blocks; a.page = (int)page; a.tokens = (int)tokens;
    a.window = window < 0 ? -1 : window;
    a.table = table; a.table_sb = table_sb; a.refs = refs; a.lengths = lengths; a.parents = parents; a.copies = copies;
    a.shared = group > 0 ? shared : nullptr;
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_fork: error word unavailable");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (n_blocks > 0) {
        fork_columns(R, n_blocks, &a.columns, &a.column_ctas);
        a.alike = static_cast<int32_t*>(workspace);
        fork_table_kernel<<<a.column_ctas, kTableThreads, 0, st>>>(a);
        const int rc = check_launch("fork_table_kernel");
        if (rc != NT_OK) return rc;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kForkThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n_blocks > 0 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fork_pages_kernel, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NT_ERR_CUDA, "fork_pages_kernel launch failed: %s", cudaGetErrorString(e));
    }
    return check_launch("fork_pages_kernel");
}

int nt_kv_copy_pages(int64_t n_layers, const int64_t* layers, int64_t n_pages, int64_t Hkv, int64_t page, int64_t D, int64_t n,
                     const int32_t* pages, void* stream) {
    const int64_t side = Hkv * page * D;
    if (n_layers < 0 || n < 0 || n_pages < 0 || Hkv < 1 || page < 1 || D < 1 || side % 16 || side / kCopyChunk > 30000)
        return fail(NT_ERR_ARG, "nt_kv_copy_pages: bad sizes");
    if (n_layers == 0 || n == 0) return NT_OK;
    if (!layers || !pages) return fail(NT_ERR_ARG, "nt_kv_copy_pages: null pointer");
    for (int64_t i = 0; i < 4 * n_layers; ++i) {
        if (!layers[i]) return fail(NT_ERR_ARG, "nt_kv_copy_pages: null pointer");
        if (i % 2 == 0 && (layers[i] & 15)) return fail(NT_ERR_ARG, "nt_kv_copy_pages: codes need 16-byte alignment");
    }
    if (n > INT32_MAX) return fail(NT_ERR_ARG, "nt_kv_copy_pages: %lld pages", (long long)n);
    int dev = 0;
    cudaGetDevice(&dev);
    CopyArgs a{};
    a.pages = pages; a.n_pages = n_pages; a.side_bytes = side; a.heads = Hkv;
    a.chunks = (int)((side + kCopyChunk - 1) / kCopyChunk);
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_kv_copy_pages: error word unavailable");
    for (int64_t i = 0; i < n_layers; i += kCopyLayers) {
        const int64_t m = std::min<int64_t>(kCopyLayers, n_layers - i);
        for (int64_t j = 0; j < m; ++j)
            for (int s = 0; s < 2; ++s) {
                a.layer[j].codes[s] = reinterpret_cast<const char*>(static_cast<uintptr_t>(layers[4 * (i + j) + 2 * s]));
                a.layer[j].scale[s] = reinterpret_cast<const float*>(static_cast<uintptr_t>(layers[4 * (i + j) + 2 * s + 1]));
            }
        copy_pages_kernel<<<dim3((unsigned)n, (unsigned)(2 * a.chunks), (unsigned)m), kCopyThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
        const int rc = check_launch("copy_pages_kernel");
        if (rc != NT_OK) return rc;
    }
    return NT_OK;
}

}  // extern "C"
