// Copies of pages inside the store of keys and values, all layers and moves in one launch:
//     k[layer, dst, head, :rows] = k[layer, src, head, :rows], v the same,
// what a forked sequence needs before it writes into the page that it shares (its first rows), and what pages that
// move to other places need (all rows).  Rows of a head are one run of memory, whole pages one run over all heads.
// The moves are kernel parameters, so nothing is copied up from the host first.  Bound by bytes, read and written once: 63 last
// pages of 30 layers (48 MB read and written) 12 us; 24 whole pages of 24 layers of 32 heads (1.2 GB) 193 us, 0.97 of the
// measured copy rate; one page of 30 layers 2.8 us.
#include <stdlib.h>
#include <string.h>

#include "async_copy.cuh"
#include "common.cuh"

namespace nnis {

constexpr int kMoves = 1024, kSomeMoves = 128, kFewMoves = 32;  // of a launch: 12 KB of parameters, 1.5 KB, 384 bytes (2 us of the host less)

template <int N>
struct PageMoves {
    int src[N], dst[N], rows[N];
};

// A CTA: some words of one run.  blockIdx: x = move and which of k and v, y = layer, z = a share of the run(s).
template <typename W, int N>
__global__ void __launch_bounds__(256)
copy_pages_kernel(const __grid_constant__ PageMoves<N> moves, void* k, void* v, int pages, int kv_heads, int page_size, int k_row,
                  int v_row) {
    const int move = v ? blockIdx.x >> 1 : blockIdx.x;
    const bool values = v && (blockIdx.x & 1);
    const int row = values ? v_row : k_row;  // words of a row
    const int src = moves.src[move], dst = moves.dst[move], rows = moves.rows[move];
    const unsigned head_words = (unsigned)page_size * row;
    const bool whole = rows == page_size;
    const int runs = whole ? 1 : kv_heads;
    const unsigned words = whole ? kv_heads * head_words : (unsigned)(rows * row);  // of a run
    W* base = reinterpret_cast<W*>(values ? v : k) + (long long)blockIdx.y * pages * kv_heads * head_words;
    const W* from = base + (long long)src * kv_heads * head_words;
    W* to = base + (long long)dst * kv_heads * head_words;
    const unsigned total = words * runs, step = gridDim.z * 256u;
    if (total == 0) return;
    constexpr int kAhead = 4;  // words a thread has on their way
    unsigned at = blockIdx.z * 256u + threadIdx.x;
    W word[kAhead];
    if (runs == 1) {
        for (; at < total; at += kAhead * step) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (at + i * step < total) word[i] = from[at + i * step];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (at + i * step < total) to[at + i * step] = word[i];
        }
        return;
    }
    // Where in a run a thread's next word lies follows from the last one's place: a division a word made the launch wait for its
    // instructions (63 forks' pages 12.9 us, without 12.0).
    unsigned run = at / words, in_run = at - run * words;
    const unsigned more_runs = step / words, more = step - more_runs * words;
    for (; at < total; at += kAhead * step) {
        unsigned place[kAhead];  // (a page has less than 2^31 words)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            place[i] = run * head_words + in_run;
            if (at + i * step < total) word[i] = from[place[i]];
            run += more_runs;
            in_run += more;
            if (in_run >= words) {
                in_run -= words;
                ++run;
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (at + i * step < total) to[place[i]] = word[i];
    }
}

// One launch of at most N moves.
template <int N>
static cudaError_t launch_moves(void* k, void* v, int layers, int pages, int kv_heads, int page_size, int k_row, int v_row,
                                const int* src, const int* dst, const int* rows, int n, int sms, cudaStream_t stream) {
    PageMoves<N> p;
    int most = 1;
    for (int i = 0; i < n; ++i) {
        p.src[i] = src[i];
        p.dst[i] = dst[i];
        p.rows[i] = rows[i];
        most = rows[i] > most ? rows[i] : most;
    }
    const uintptr_t all = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_row | (uintptr_t)(v ? v_row : 0);
    const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2, tensors = v ? 2 : 1;
    const long long words = (long long)kv_heads * most * (k_row > v_row ? k_row : v_row) / unit;
    const long long ctas = (long long)n * tensors * layers;
    long long share = (words + 1023) / 1024;                // four words a thread
    const long long fill = (16LL * sms + ctas - 1) / ctas;  // ... unless there are CTAs enough
    if (share > fill) share = fill;
    if (share < 1) share = 1;
    if (share > 65535) share = 65535;
    const dim3 grid((unsigned)(n * tensors), (unsigned)layers, (unsigned)share);
    auto kernel = unit == 16 ? copy_pages_kernel<uint4, N> : unit == 4 ? copy_pages_kernel<uint32_t, N> : copy_pages_kernel<uint16_t, N>;
    kernel<<<grid, 256, 0, stream>>>(p, k, v, pages, kv_heads, page_size, k_row / unit, v_row / unit);
    return cudaGetLastError();
}

}  // namespace nnis

// k and v (or null): [layers, pages, kv_heads, page_size, row] with rows of `k_row` and `v_row` bytes, multiples of 2.
// moves, on the host: `count` sources, then targets, then numbers of rows (0 to page_size).  NNIS_ERR_ARGUMENT, with nothing
// copied, where a page is outside the store, the target of two moves, or a target and a source.
struct CopyCall {
    void *k, *v;
    int layers, pages, kv_heads, page_size, k_row, v_row;
    const int* moves;
    int count, sms;
    cudaStream_t stream;
};
NNIS_API int nnis_copy_pages(const void* call) {
    using namespace nnis;
    CopyCall c;
    memcpy(&c, call, sizeof c);
    const auto [k, v, layers, pages, kv_heads, page_size, k_row, v_row, moves, count, sms, stream] = c;
    if (!k || !moves || count < 0 || layers <= 0 || pages <= 0 || kv_heads <= 0 || page_size <= 0 || k_row <= 0 || k_row % 2 ||
        (v && (v_row <= 0 || v_row % 2)))
        return NNIS_ERR_ARGUMENT;
    const long long page_bytes = (long long)kv_heads * page_size * (k_row > v_row ? k_row : v_row);
    if (layers > 65535 || page_bytes / 2 >= (1LL << 31)) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)k | (uintptr_t)v) % 2) return NNIS_ERR_ALIGNMENT;
    const int *src = moves, *dst = moves + count, *rows = moves + 2 * count;
    unsigned char* seen = static_cast<unsigned char*>(calloc((size_t)pages, 1));  // 1: a source, 2: a target
    if (!seen) return (int)cudaErrorMemoryAllocation;
    bool good = true;
    for (int i = 0; i < count && good; ++i) {
        good = src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages && rows[i] >= 0 && rows[i] <= page_size;
        if (good) seen[src[i]] |= 1;
    }
    for (int i = 0; i < count && good; ++i) {
        good = !seen[dst[i]];
        seen[dst[i]] |= 2;
    }
    free(seen);
    if (!good) return NNIS_ERR_ARGUMENT;
    for (int first = 0; first < count; first += kMoves) {
        const int n = count - first < kMoves ? count - first : kMoves;
        auto launch = n <= kFewMoves ? launch_moves<kFewMoves> : n <= kSomeMoves ? launch_moves<kSomeMoves> : launch_moves<kMoves>;
        const cudaError_t e = launch(k, v, layers, pages, kv_heads, page_size, k_row, v_row, src + first, dst + first, rows + first, n,
                                     sms, stream);
        if (e != cudaSuccess) return (int)e;
    }
    return NNIS_OK;
}
