// Rows of many tensors moved to the beams that go on from them, in place, in one launch.
//
// Row r of a group takes what row rows[r] of its group held.  A group's rows are staged
// through shared memory a piece at a time, so any map is right (a swap, a cycle, one row
// for all); where no row that is read is written, as when surviving beams keep their
// places, they are copied straight.  Rows that stay are neither read nor written.  Bound
// by HBM: each row that is followed is read once, each that changes written once.  One row in
// four of the large preset's 28 blocks and 64 rows (947 MB): 147 us, 99 % of the copy rate;
// half of 40 float32 rows of an odd length (56 MB), by 4-byte words, 17 us (with four of a thread on their way
// 18).
#include "nt_kernels.cuh"

#include <algorithm>

namespace nt {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveMost = 96;          // tensors of a launch
constexpr int kMoveGroup = 1024;       // rows of a group
constexpr int kMoveStage = 32768;      // bytes of the staged piece of a group
constexpr int kMoveChunk = 16384;      // bytes of a row that a CTA moves

struct MoveArgs {
    const int32_t* rows;
    int group, n;
    unsigned* err;
    struct { char* p; int64_t bytes, stride; int first, width; } t[kMoveMost];   // first: its first chunk in the grid
};

// `width`-byte words of one chunk: 16 where addresses allow, else what they have in common.
template <typename W>
__device__ __forceinline__ void move_straight(const MoveArgs& a, char* base, int64_t stride, int64_t n_words, const int16_t* from) {
    for (int r = 0; r < a.group; ++r) {
        const int src = from[r];
        if (src == r) continue;
        const W* s = reinterpret_cast<const W*>(base + src * stride);
        W* d = reinterpret_cast<W*>(base + r * stride);
        // a chunk's words on their way, up to 8 a thread (more registers cost a CTA an SM: 157 and 174 us for 148)
        constexpr int N = kMoveChunk / (int)sizeof(W) / kMoveThreads < 8 ? kMoveChunk / (int)sizeof(W) / kMoveThreads : 8;
        int64_t i = threadIdx.x;
        for (; i - threadIdx.x + N * kMoveThreads <= n_words; i += N * kMoveThreads) {
            W v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = s[i + j * kMoveThreads];
#pragma unroll
            for (int j = 0; j < N; ++j) d[i + j * kMoveThreads] = v[j];
        }
        for (; i - threadIdx.x < n_words; i += N / 2 * kMoveThreads) {      // the row's last chunk
            W v[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; ++j)
                if (i + j * kMoveThreads < n_words) v[j] = s[i + j * kMoveThreads];
#pragma unroll
            for (int j = 0; j < N / 2; ++j)
                if (i + j * kMoveThreads < n_words) d[i + j * kMoveThreads] = v[j];
        }
    }
}
template <typename W>
__device__ __forceinline__ void move_staged(const MoveArgs& a, char* base, int64_t stride, int64_t n_words, const int16_t* from,
                                            const uint8_t* read, unsigned char* smem) {
    W* stage = reinterpret_cast<W*>(smem);
    const int piece = kMoveStage / (int)sizeof(W) / a.group;              // words of a row at a time, 2 at least
    for (int64_t w0 = 0; w0 < n_words; w0 += piece) {
        const int m = (int)(n_words - w0 < piece ? n_words - w0 : piece);
        for (int i = threadIdx.x; i < a.group * m; i += kMoveThreads) {
            const int r = i / m;
            if (read[r]) stage[i] = reinterpret_cast<const W*>(base + r * stride)[w0 + i % m];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.group * m; i += kMoveThreads) {
            const int r = i / m, src = from[r];
            if (src != r) reinterpret_cast<W*>(base + r * stride)[w0 + i % m] = stage[src * m + i % m];
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kMoveThreads, 5) reorder_rows_kernel(const __grid_constant__ MoveArgs a) {
    __shared__ __align__(16) unsigned char smem[kMoveStage];
    __shared__ int16_t from[kMoveGroup];
    __shared__ uint8_t read[kMoveGroup];
    const int64_t row0 = (int64_t)blockIdx.y * a.group;
    int t = 0;
    for (int step = 64; step; step >>= 1)
        if (t + step < a.n && a.t[t + step].first <= (int)blockIdx.x) t += step;
    for (int r = threadIdx.x; r < a.group; r += kMoveThreads) read[r] = 0;
    __syncthreads();
    bool moved = false;
    for (int r = threadIdx.x; r < a.group; r += kMoveThreads) {
        const int64_t src = a.rows[row0 + r] - row0;
        const bool bad = src < 0 || src >= a.group;
        from[r] = (int16_t)(bad ? r : src);
        if (bad && a.rows[row0 + r] != -1 && blockIdx.x == 0) atomicOr(a.err, ERRF_BAD_ARG);
        if (!bad && src != r) {
            read[src] = 1;
            moved = true;
        }
    }
    if (!__syncthreads_or(moved)) return;
    bool clash = false;                                 // a row that is read changes
    for (int r = threadIdx.x; r < a.group; r += kMoveThreads) clash |= read[r] && from[r] != r;
    clash = __syncthreads_or(clash);
    const int64_t at = (int64_t)(blockIdx.x - a.t[t].first) * kMoveChunk, left = a.t[t].bytes - at;
    const int64_t bytes = left < kMoveChunk ? left : kMoveChunk, stride = a.t[t].stride;
    char* base = a.t[t].p + row0 * stride + at;
    auto go = [&](auto word) {
        using W = decltype(word);
        if (clash) move_staged<W>(a, base, stride, bytes / (int)sizeof(W), from, read, smem);
        else move_straight<W>(a, base, stride, bytes / (int)sizeof(W), from);
    };
    if (a.t[t].width == 16) go(uint4{});
    else if (a.t[t].width == 8) go(uint2{});
    else if (a.t[t].width == 4) go(uint32_t{});
    else if (a.t[t].width == 2) go(uint16_t{});
    else go(uint8_t{});
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_reorder_rows(int64_t n_tensors, const int64_t* tensors, int64_t R, int64_t group, const int32_t* rows, void* stream) {
    if (n_tensors < 0 || R < 0 || group < 1 || group > kMoveGroup || R % group || R / group > 65535)
        return fail(NT_ERR_ARG, "nt_reorder_rows: bad sizes (groups of 1 to %d rows, at most 65535 of them)", kMoveGroup);
    if (n_tensors == 0 || R == 0) return NT_OK;
    if (!tensors || !rows) return fail(NT_ERR_ARG, "nt_reorder_rows: null pointer");
    for (int64_t i = 0; i < n_tensors; ++i) {
        const int64_t p = tensors[3 * i], bytes = tensors[3 * i + 1], stride = tensors[3 * i + 2];
        if (bytes < 0 || (R > 1 && stride < bytes) || bytes > ((int64_t)1 << 40))
            return fail(NT_ERR_ARG, "nt_reorder_rows: tensor %lld has rows of %lld bytes, %lld apart", (long long)i, (long long)bytes,
                        (long long)stride);
        if (bytes > 0 && !p) return fail(NT_ERR_ARG, "nt_reorder_rows: null pointer");
    }
    int dev = 0;
    cudaGetDevice(&dev);
    MoveArgs a{};
    a.rows = rows;
    a.group = (int)group;
    a.err = device_error_word(dev);
    if (!a.err) return fail(NT_ERR_CUDA, "nt_reorder_rows: error word unavailable");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    for (int64_t i = 0; i < n_tensors;) {
        int64_t chunks = 0;
        a.n = 0;
        for (; i < n_tensors && a.n < kMoveMost; ++i) {
            const int64_t p = tensors[3 * i], bytes = tensors[3 * i + 1], stride = tensors[3 * i + 2];
            if (bytes == 0) continue;
            const int64_t c = (bytes + kMoveChunk - 1) / kMoveChunk;
            if (chunks + c > INT32_MAX) break;
            const uint64_t bits = (uint64_t)p | (uint64_t)bytes | (uint64_t)stride;
            auto& t = a.t[a.n++];
            t.p = reinterpret_cast<char*>(static_cast<uintptr_t>(p));
            t.bytes = bytes;
            t.stride = stride;
            t.first = (int)chunks;
            t.width = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
            chunks += c;
        }
        if (a.n == 0) break;
        reorder_rows_kernel<<<dim3((unsigned)chunks, (unsigned)(R / group)), kMoveThreads, 0, st>>>(a);
        const int rc = check_launch("reorder_rows_kernel");
        if (rc != NT_OK) return rc;
    }
    return NT_OK;
}
