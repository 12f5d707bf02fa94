// What the kernels of attention over shared pages have in common: the units that the host lists, and the records that
// the units leave.
//
// Token rows whose sequences begin with the same pages see those pages alike, so their queries are stacked: an *entry* is a
// (token row, query head of a kv head's group), and a *unit* is up to a tile of entries of one list of token rows over a
// range of pages that all of them see.  Per (token row, head, unit) a record, d unnormalised outputs, their maximum (log2
// units) and sum, goes to scratch; the merge kernel adds a row's records up.  Units of a single token row end at the
// row's position, all others cover only positions that every one of their rows sees.
#pragma once

#include <float.h>

#include "async_copy.cuh"
#include "common.cuh"

namespace nnis {

struct SharedUnit {   // eight ints of the plan
    int members;      // where the unit's list of token rows begins in the plan's members
    int entry;        // its first entry: members[entry / G], head entry % G of the group
    int entries;      // number of entries
    int page_begin, page_end;  // columns of the page table
    int slot;         // which of each row's records it writes
    int seq;          // row of the page table that names the pages
    int ends;         // 1: keys beyond the row's own position are hidden (all entries are of one token row)
};

constexpr int kSharedPage = 64;  // keys of a page

struct SharedArgs {
    const void* q;
    const void* k_cache;
    const void* v_cache;
    const int* token_pos;
    const int* page_table;
    const SharedUnit* units;
    const int* members;
    const int* record;   // [tokens + 1]: the first record of every token row
    float* partial;      // [records, nq, d]: outputs
    float* sums;         // [records, nq, 2]: maximum and sum
    unsigned* tickets;   // [tokens, nq], zero between calls: who writes a row's last record merges it; null: the merge kernel does
    void* out;           // [tokens, nq, d]
    int q_stride, table_cols, pages, nq, nkv, d;
    float scale;
    int beside;          // 1: the launch before this one is of the same call and runs beside it
};

// Programmatic dependent launch among the units' kernels of a call: the first waits for the kernel before the call (queries, and
// this step's keys and values) before it lets the second start, so the second need not wait to begin, only to end: whoever
// waits for it then waits for both.
__device__ __forceinline__ void units_begin(const SharedArgs& a) {
    if (!a.beside) pdl_wait();
    pdl_launch_dependents();
}
__device__ __forceinline__ void units_end(const SharedArgs& a) {
    if (a.beside) pdl_wait();
}

// Adds up one (token row, head)'s records: a warp; lane s holds the weights of records s, s + 32, ..., every lane sums its pairs of
// values over the records in their order, AHEAD records asked for at a time.  Where no record holds a key the result is zero.
template <typename T, int AHEAD>
__device__ __forceinline__ void merge_row(const float* partial, const float2* sums, int first, int count, int row, int head, int nq,
                                          int d, T* out) {
    const int lane = threadIdx.x & 31;
    const size_t rec = (size_t)first * nq + head;
    float m = -INFINITY;
    for (int s = lane; s < count; s += 32) {
        const float2 x = __ldcg(sums + rec + (size_t)s * nq);
        if (x.y != 0.f) m = fmaxf(m, x.x);
    }
    m = warp_max(m);
    float2 acc[4] = {};
    float l = 0.f;
    for (int s0 = 0; s0 < count; s0 += 32) {
        float w = 0.f;
        if (s0 + lane < count) {
            const float2 x = __ldcg(sums + rec + (size_t)(s0 + lane) * nq);
            w = x.y != 0.f ? exp2f(x.x - m) : 0.f;
            l += x.y * w;
        }
        const int here = min(32, count - s0);
        for (int s = 0; s < here; s += AHEAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j * 64 >= d) break;
                const int i = 2 * (lane + 32 * j);
                float2 v[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    v[k] = s + k < here && i < d ? __ldcg(reinterpret_cast<const float2*>(partial + (rec + (size_t)(s0 + s + k) * nq) * d + i))
                                                 : make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const float f = __shfl_sync(0xffffffffu, w, (s + k) & 31);
                    if (s + k < here && f != 0.f) {  // (a record that holds nothing is never added)
                        acc[j].x = fmaf(f, v[k].x, acc[j].x);
                        acc[j].y = fmaf(f, v[k].y, acc[j].y);
                    }
                }
            }
        }
    }
    l = warp_sum(l);
    const float inv = l != 0.f ? 1.0f / l : 0.f;  // (a sum that is no number stays one)
    T* to = out + ((size_t)row * nq + head) * d;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = 2 * (lane + 32 * j);
        if (i < d) store2(to + i, acc[j].x * inv, acc[j].y * inv);
    }
}

// After all threads of a CTA have written their unit's records: the rows that these complete are merged here.  `done`: an
// int per entry of shared memory.  Every thread of the CTA calls it.
template <typename T, int THREADS>
__device__ __forceinline__ void merge_finished(const SharedArgs& a, const SharedUnit& u, int hk, int G, int* done) {
    __syncthreads();  // (the fence below covers what the others wrote before this)
    const int* members = a.members + u.members;
    for (int e = threadIdx.x; e < u.entries; e += THREADS) {
        const int at = u.entry + e, row = members[at / G];
        unsigned* ticket = a.tickets + (size_t)row * a.nq + hk * G + at % G;
        __threadfence();
        const bool last = atomicAdd(ticket, 1u) == (unsigned)(a.record[row + 1] - a.record[row]) - 1u;
        if (last) *ticket = 0u;
        done[e] = last;
    }
    __syncthreads();
    __threadfence();
    for (int e = threadIdx.x >> 5; e < u.entries; e += THREADS / 32) {
        if (!done[e]) continue;
        const int at = u.entry + e, row = members[at / G], first = a.record[row];
        merge_row<T, 16>(a.partial, reinterpret_cast<const float2*>(a.sums), first, a.record[row + 1] - first, row, hk * G + at % G,
                         a.nq, a.d, static_cast<T*>(a.out));
    }
}

// One launch of the named form over `n_units` units; each is defined in its own file.
cudaError_t shared_units_any(const SharedArgs& a, int n_units, int tile, bool f32, cudaStream_t stream);
cudaError_t shared_units_mma(const SharedArgs& a, int n_units, cudaStream_t stream);
cudaError_t shared_units_tc(const SharedArgs& a, int n_units, int* status, cudaStream_t stream);

}  // namespace nnis
