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
    int ends;         // 1 + token row: all entries are of that row, and keys beyond its position are hidden; 0: all see all
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
    int* status;         // see units_end_check; null: nobody is told
    int beside;          // 1: the launch before this one is of the same call and runs beside it
};

// Programmatic dependent launch among the units' kernels of a call: the first waits for the kernel before the call (queries, this
// step's keys and values, and as a caller may write them there, too, positions and page tables; ahead of it only the plan is read, which
// is copied from the host) before it lets the second start, so the second need not wait to begin, only to end: whoever
// waits for it then waits for both.
__device__ __forceinline__ void units_begin(const SharedArgs& a) {
    if (!a.beside) pdl_wait();
    pdl_launch_dependents();
}
__device__ __forceinline__ void units_end(const SharedArgs& a) {
    if (a.beside) pdl_wait();
}

// A unit that ends a row's pages and does not reach the row's position (the row has gone on beyond what its plan was made for) tells the
// status word: the keys behind it are not seen.  One thread's work.
__device__ __forceinline__ void units_end_check(const SharedArgs& a, const SharedUnit& u, int pos) {
    if (u.ends && pos >= 0 && pos / kSharedPage >= u.page_end && a.status && a.record[u.ends - 1] + u.slot + 1 == a.record[u.ends])
        atomicExch(a.status, 2);
}

// 2^x for a weight: one that would be denormal is zero (exp2f keeps it, by four instructions instead of one).
__device__ __forceinline__ float sh_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Adds up one (token row, head)'s records: a warp; lane s holds the weights of records s, s + 32, ..., every lane sums its pairs of
// values over the records in their order, AHEAD records asked for at a time, the first ones before any weight is known.  Where no
// record holds a key the result is zero.
template <typename T, int AHEAD>
__device__ __forceinline__ void merge_row(const float* partial, const float2* sums, int first, int count, int row, int head, int nq,
                                          int d, T* out) {
    const int lane = threadIdx.x & 31;
    const size_t rec = (size_t)first * nq + head;
    auto ask_sum = [&](int s) { return s < count ? __ldcg(sums + rec + (size_t)s * nq) : make_float2(-INFINITY, 0.f); };
    auto ask = [&](int s0, int j, float2 (&v)[AHEAD]) {
        const int i = 2 * (lane + 32 * j);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            v[k] = s0 + k < count && i < d ? __ldcg(reinterpret_cast<const float2*>(partial + (rec + (size_t)(s0 + k) * nq) * d + i))
                                           : make_float2(0.f, 0.f);
    };
    float2 own = ask_sum(lane), v[AHEAD];
    ask(0, 0, v);
    float m = own.y != 0.f ? own.x : -INFINITY;
    for (int s = lane + 32; s < count; s += 32) {
        const float2 x = ask_sum(s);
        if (x.y != 0.f) m = fmaxf(m, x.x);
    }
    m = warp_max(m);
    float2 acc[4] = {};
    float l = 0.f;
    for (int s0 = 0; s0 < count; s0 += 32) {
        if (s0) own = ask_sum(s0 + lane);
        const float w = own.y != 0.f ? exp2f(own.x - m) : 0.f;
        l += own.y * w;
        const int end = min(32, count - s0);
        for (int s = 0; s < end; s += AHEAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j * 64 >= d) break;
                if (s0 + s + j) ask(s0 + s, j, v);
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const float f = __shfl_sync(0xffffffffu, w, (s + k) & 31);
                    if (s + k < end && f != 0.f) {  // (a record that holds nothing is never added)
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

// After all threads of a CTA have written their unit's records: the rows that these complete are merged here, a thread four (or
// two) values of an entry at a time, its records asked for eight at once.  For units whose entries have few records.  `done`: an
// int4 per entry of shared memory that nothing else uses.  Every thread of the CTA calls it.
template <typename T, int THREADS>
__device__ __forceinline__ void merge_finished(const SharedArgs& a, const SharedUnit& u, int hk, int G, int4* done) {
    __syncthreads();  // (the fence below covers what the others wrote before this)
    const int* members = a.members + u.members;
    const float2* sums = reinterpret_cast<const float2*>(a.sums);
    for (int e = threadIdx.x; e < u.entries; e += THREADS) {
        const int at = u.entry + e, row = members[at / G];
        unsigned* ticket = a.tickets + (size_t)row * a.nq + hk * G + at % G;
        __threadfence();
        const int first = a.record[row], count = a.record[row + 1] - first;
        const bool last = atomicAdd(ticket, 1u) == (unsigned)count - 1u;
        if (last) *ticket = 0u;
        done[e] = make_int4(last ? count : 0, first, row, hk * G + at % G);
    }
    __syncthreads();
    __threadfence();
    const int d = a.d, pairs = d / 2;
    for (int item = threadIdx.x; item < u.entries * pairs; item += THREADS) {
        const int e = item / pairs, i = 2 * (item % pairs);
        const int count = done[e].x, first = done[e].y, row = done[e].z, head = done[e].w;
        if (!count) continue;
        float m = -INFINITY, l = 0.f;
        float2 acc = make_float2(0.f, 0.f);
        constexpr int kAhead = 8;
        for (int s0 = 0; s0 < count; s0 += kAhead) {
            float2 ml[kAhead], v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const size_t rec = (size_t)(first + s0 + k) * a.nq + head;
                const bool there = s0 + k < count;
                ml[k] = there ? __ldcg(sums + rec) : make_float2(-INFINITY, 0.f);
                v[k] = there ? __ldcg(reinterpret_cast<const float2*>(a.partial + rec * d + i)) : make_float2(0.f, 0.f);
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
            const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
            l *= keep;
            acc.x *= keep;
            acc.y *= keep;
            m = top;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (ml[k].y == 0.f) continue;  // (a record that holds nothing is never added)
                const float f = exp2f(ml[k].x - m);
                l = fmaf(ml[k].y, f, l);
                acc.x = fmaf(f, v[k].x, acc.x);
                acc.y = fmaf(f, v[k].y, acc.y);
            }
        }
        const float inv = l != 0.f ? 1.0f / l : 0.f;
        store2(static_cast<T*>(a.out) + ((size_t)row * a.nq + head) * d + i, acc.x * inv, acc.y * inv);
    }
}

// One launch of the named form over `n_units` units; each is defined in its own file.
cudaError_t shared_units_any(const SharedArgs& a, int n_units, int tile, bool f32, cudaStream_t stream);
cudaError_t shared_units_f32(const SharedArgs& a, int n_units, int tile, cudaStream_t stream);
cudaError_t shared_units_warp(const SharedArgs& a, int n_units, cudaStream_t stream);
cudaError_t shared_units_mma(const SharedArgs& a, int n_units, cudaStream_t stream);
cudaError_t shared_units_tc(const SharedArgs& a, int n_units, cudaStream_t stream);

}  // namespace nnis
