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
    int entries;      // number of entries (0: nothing to do, a place kept free)
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
    int q_stride, table_cols, pages, nq, nkv, d;
    float scale;
};

// One launch of the named form over `n_units` units; each is defined in its own file.
cudaError_t shared_units_any(const SharedArgs& a, int n_units, int tile, bool f32, cudaStream_t stream);
cudaError_t shared_units_mma(const SharedArgs& a, int n_units, cudaStream_t stream);
cudaError_t shared_units_tc(const SharedArgs& a, int n_units, int* status, cudaStream_t stream);

}  // namespace nnis
