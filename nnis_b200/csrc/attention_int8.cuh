// What the kernels of attention over the 8-bit cache are given.
#pragma once

#include <limits.h>

#include <type_traits>

#include "common.cuh"

namespace nnis {

struct Attend8 {
    const void* q;
    long long q_stride;
    const int8_t *k, *v;
    const float *k_scales, *v_scales;
    const int *token_pos, *token_seq, *page_table;
    int table_rows, table_cols, pages;
    void* out;
    float* partial;  // records of slices
    int n, nq, nkv, d, page_size, window;
    float scale;
    int splits;      // most slices of a row
    // the tensor cores' kernel
    int slice_pieces, rows_at_once, tiles, aligned, cluster;  // cluster: CTAs that share a slice, at most 8; 0: a warp a unit
    int tile_eights, units;  // a tile's queries / 8
    unsigned* tickets;  // n * nkv * tiles, zero between launches
    int* status;
};

// Positions that a warp takes at a time (what each time costs beside its positions is a third of 32 positions of 64 values), and how
// many such pieces it has on their way or in use: three CTAs an SM, four with heads of 32.
__host__ __device__ constexpr int piece8(int d) { return d <= 64 ? 64 : 32; }
__host__ __device__ constexpr int stages8(int d) { return d <= 96 ? 2 : 3; }

__device__ __forceinline__ void fence_async_shared8() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

cudaError_t attend_int8_mma(Attend8 p, bool f32, cudaStream_t stream);

}  // namespace nnis
