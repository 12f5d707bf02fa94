// Verification of drafted tokens: which of a sequence's drafts the target model keeps, and the token after them.
//
// Sequence b has k drafts and k + 1 rows of target logits z_i (row i follows i drafts); the drafting model's logits y_i
// give its draft's distribution, or there are none (drafts that nobody drew: q is one at the draft).  With
// p_i = softmax(z_i / T) and q_i = softmax(y_i / T) draft d_i is kept iff  u_i q_i(d_i) < p_i(d_i);  the first that is not
// kept, at i = a, ends the sequence's drafts, and its place takes a token from max(p_a - q_a, 0) over its sum, picked by
// inverse CDF in id order with the draw r: the first id whose running sum exceeds r times the total.  With all kept the
// token comes from p_k.  So every token is distributed as p, whatever drafted it.  T = 0 (or less): a draft is kept iff it is
// the row's argmax (the lower id among equals), and the pick is the argmax.
//
// Two launches.  The first sums every row once, in 32 bits (CTA: a share of a row; running maximum and sum, argmax).  In the
// second a cluster of CTAs takes a sequence: the drafts are decided in order from the rows' sums and the two logits of the
// draft itself, in 64 bits; a decision within 1e-4 of its border is taken again with the row's sums in 64 bits
// (the sums' 32-bit error is below 1e-5: terms 17 bits of exponent at most where they count, 2e-6; 32 and
// fewer additions a thread, 2e-6).  Then the one row that is drawn from is summed in 64 bits, each
// CTA a range of ids and each warp a range of that, because a draw may fall next to a border between two of 50,000
// tokens, and p - q cancels: 32 bits would pick another token every few hundred draws.
#include <cooperative_groups.h>
#include <float.h>

#include "async_copy.cuh"
#include "common.cuh"

namespace nnis {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 256;
constexpr int kVerifyShare = 8192;   // logits of a row that a CTA of the first launch sums at least
constexpr int kVerifyParts = 32;     // most CTAs a row
constexpr int kPickThreads = 512;
constexpr int kPickCtas = 8;         // of a cluster
constexpr float kBad = 1.f;

struct RowSum {
    float max, sum;  // maximum logit, sum of exp((x - max) / T)
    int best;        // id of the maximum, the lower among equals
    float bad;       // kBad: a logit is no number or +infinity
};

// log2(e) / T, within bounds that keep 0 and -infinity times it what they are (where that is another number the sums in 64
// bits decide, or all weights are one to 32 bits)
__device__ __forceinline__ float scale_of(float temperature) {
    return temperature > 0.f ? fmaxf(fminf(1.4426950408889634f / temperature, 1e30f), 1e-30f) : 1.f;
}

// (m, s, best) of two sets of ids
__device__ __forceinline__ RowSum joined(const RowSum& a, const RowSum& b, float c) {
    RowSum r;
    r.max = fmaxf(a.max, b.max);
    r.bad = fmaxf(a.bad, b.bad);
    r.best = a.max > b.max || (a.max == b.max && a.best < b.best) ? a.best : b.best;
    const float base = r.max == -INFINITY ? 0.f : r.max;
    r.sum = a.sum * exp2f((a.max - base) * c) + b.sum * exp2f((b.max - base) * c);
    return r;
}

__global__ void __launch_bounds__(kVerifyThreads)
verify_rows_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ first_row,
                   const float* __restrict__ temperature, int n_seqs, int rows, int draft_rows, int vocab, int per,
                   RowSum* __restrict__ parts) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ RowSum warp_sum_s[kVerifyThreads / 32];
    const int r = blockIdx.y;
    const bool of_draft = r >= rows;
    // the row's sequence: the last one that begins at or before it
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_row[mid] - (of_draft ? mid : 0) <= (of_draft ? r - rows : r)) lo = mid;
        else hi = mid - 1;
    }
    const float t = temperature[lo];
    const float c = scale_of(t);
    const float* row = of_draft ? draft_logits + (size_t)(r - rows) * vocab : logits + (size_t)r * vocab;
    const int begin = min(vocab, (int)blockIdx.x * per), end = min(vocab, begin + per);
    RowSum mine = {-INFINITY, 0.f, 0x7fffffff, 0.f};
    constexpr int kAhead = 8;
    for (int at = begin + threadIdx.x; at < end; at += kAhead * kVerifyThreads) {
        float x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = at + i * kVerifyThreads < end ? row[at + i * kVerifyThreads] : -INFINITY;
        float m = mine.max;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (!(x[i] < INFINITY)) mine.bad = kBad;
            if (x[i] > m) {
                m = x[i];
                mine.best = at + i * kVerifyThreads;
            }
        }
        const float base = m == -INFINITY ? 0.f : m;
        float s = mine.sum * exp2f((mine.max - base) * c);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) s += x[i] == -INFINITY ? 0.f : exp2f((x[i] - base) * c);
        mine.max = m;
        mine.sum = s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSum other;
        other.max = __shfl_xor_sync(0xffffffffu, mine.max, o);
        other.sum = __shfl_xor_sync(0xffffffffu, mine.sum, o);
        other.best = __shfl_xor_sync(0xffffffffu, mine.best, o);
        other.bad = __shfl_xor_sync(0xffffffffu, mine.bad, o);
        mine = joined(mine, other, c);
    }
    if ((threadIdx.x & 31) == 0) warp_sum_s[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kVerifyThreads / 32; ++w) mine = joined(mine, warp_sum_s[w], c);
        parts[(size_t)r * gridDim.x + blockIdx.x] = mine;
    }
}

// A row's parts joined by a warp (at most 32 of them); every lane gets the result.
__device__ __forceinline__ RowSum row_sum(const RowSum* __restrict__ parts, size_t row, int n_parts, float c) {
    const int lane = threadIdx.x & 31;
    RowSum mine = {-INFINITY, 0.f, 0x7fffffff, 0.f};
    if (lane < n_parts) mine = parts[row * n_parts + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSum other;
        other.max = __shfl_xor_sync(0xffffffffu, mine.max, o);
        other.sum = __shfl_xor_sync(0xffffffffu, mine.sum, o);
        other.best = __shfl_xor_sync(0xffffffffu, mine.best, o);
        other.bad = __shfl_xor_sync(0xffffffffu, mine.bad, o);
        mine = joined(mine, other, c);
    }
    return mine;
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ double weight64(float x, float max, double inv_t) {
    return x == -INFINITY ? 0.0 : exp(((double)x - (double)max) * inv_t);
}

struct PickShared {
    double warp[2][kPickThreads / 32];
    double cta[2];       // this CTA's sums, read by the others of its cluster
    double mass;         // ... of what is drawn from
    int picked;
};

// Sum over the whole cluster of up to two values a thread, every thread gets both.
__device__ __forceinline__ void cluster_sum(cg::cluster_group cluster, PickShared& s, double& a, double& b) {
    a = warp_sum64(a);
    b = warp_sum64(b);
    if ((threadIdx.x & 31) == 0) {
        s.warp[0][threadIdx.x >> 5] = a;
        s.warp[1][threadIdx.x >> 5] = b;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double x = 0.0, y = 0.0;
        for (int w = 0; w < kPickThreads / 32; ++w) {
            x += s.warp[0][w];
            y += s.warp[1][w];
        }
        s.cta[0] = x;
        s.cta[1] = y;
    }
    cluster.sync();
    a = b = 0.0;
    for (unsigned i = 0; i < cluster.num_blocks(); ++i) {
        const PickShared* other = cluster.map_shared_rank(&s, i);
        a += other->cta[0];
        b += other->cta[1];
    }
    cluster.sync();
}

__global__ void __launch_bounds__(kPickThreads) __cluster_dims__(kPickCtas, 1, 1)
verify_pick_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ drafts,
                   const int* __restrict__ first_row, const float* __restrict__ temperature, const double* __restrict__ accept_draws,
                   const double* __restrict__ pick_draws, const RowSum* __restrict__ parts, int n_parts, int rows, int vocab,
                   int* __restrict__ accepted, int* __restrict__ picked) {
    __shared__ PickShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int b = blockIdx.y, rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int row0 = first_row[b], draft0 = row0 - b, count = first_row[b + 1] - row0 - 1;
    if (row0 < b || count < 0 || row0 + count >= rows) {  // (offsets that no packed rows have: the whole cluster leaves)
        if (rank == 0 && tid == 0) {
            accepted[b] = 0;
            picked[b] = -1;
        }
        return;
    }
    const float t = temperature[b];
    const bool greedy = !(t > 0.f);
    const float c = scale_of(t);
    const double inv_t = greedy ? 1.0 : 1.0 / (double)t;
    // this thread's ids: a range of the row per CTA, a range of that per warp
    constexpr int kWarps = kPickThreads / 32;
    const int per_warp = (((vocab + kPickCtas * kWarps - 1) / (kPickCtas * kWarps)) + 31) & ~31;
    const int begin = min(vocab, (rank * kWarps + warp) * per_warp), end = min(vocab, begin + per_warp);

    // the sums of a row of z and of its row of y, in 64 bits
    auto exact_sums = [&](const float* z, float z_max, const float* y, float y_max, double& sp, double& sq) {
        sp = sq = 0.0;
        for (int i = begin + lane; i < end; i += 32) {
            sp += weight64(z[i], z_max, inv_t);
            if (y) sq += weight64(y[i], y_max, inv_t);
        }
        cluster_sum(cluster, s, sp, sq);
    };

    int a = 0;
    bool none = false;
    RowSum zs = {}, ys = {};
    const float *z = nullptr, *y = nullptr;
    int d = -1;
    bool all = false;
    for (;; ++a) {  // (every warp of the cluster decides for itself, all alike)
        zs = row_sum(parts, (size_t)(row0 + a), n_parts, c);
        z = logits + (size_t)(row0 + a) * vocab;
        all = a >= count;
        none = zs.bad != 0.f || zs.max == -INFINITY;
        if (all || none) break;
        d = drafts[draft0 + a];
        if (greedy) {
            if (d != zs.best) break;
            continue;
        }
        if (draft_logits) {
            ys = row_sum(parts, (size_t)(rows + draft0 + a), n_parts, c);
            y = draft_logits + (size_t)(draft0 + a) * vocab;
            none = ys.bad != 0.f || ys.max == -INFINITY;
            if (none) break;
        }
        if (d < 0 || d >= vocab) break;
        const double u = accept_draws[draft0 + a];
        const double ep = weight64(z[d], zs.max, inv_t), eq = y ? weight64(y[d], ys.max, inv_t) : 1.0;
        double left = u * eq * (double)zs.sum, right = ep * (y ? (double)ys.sum : 1.0);
        if (fabs(left - right) <= 1e-4 * right || t < 1e-29f) {
            double sp, sq;
            exact_sums(z, zs.max, y, ys.max, sp, sq);
            left = u * eq * sp;
            right = ep * (y ? sq : 1.0);
        }
        if (!(left < right)) break;
    }
    int pick = -1;
    if (!none && greedy) {
        pick = zs.best;
    } else if (!none) {
        // the distribution to draw from: p, or what of it the draft's distribution leaves
        double sp, sq;
        if (all) y = nullptr;
        exact_sums(z, zs.max, y, ys.max, sp, sq);
        const double ip = 1.0 / sp, iq = y ? 1.0 / sq : 0.0;
        auto mass_of = [&](int i, bool plain) -> double {
            const double p = __dmul_rn(weight64(z[i], zs.max, inv_t), ip);  // (rounded like q: equal ones leave nothing)
            if (plain) return p;
            if (y) return fmax(p - __dmul_rn(weight64(y[i], ys.max, inv_t), iq), 0.0);
            return i == d ? 0.0 : p;
        };
        bool plain = all;
        double mine, total, unused;
        for (;;) {
            mine = 0.0;
            for (int i = begin + lane; i < end; i += 32) mine += mass_of(i, plain);
            total = mine;
            unused = 0.0;
            cluster_sum(cluster, s, total, unused);
            if (plain || total > 0.0) break;
            plain = true;  // nothing is left: p and q are one
        }
        // (s.warp[0]: this CTA's warps' sums; s.cta[0] of every CTA: theirs)
        const double target = pick_draws[b] * total;
        double before = 0.0, held = 0.0;
        int last = 0;  // the last CTA with any weight
        for (int i = 0; i < kPickCtas; ++i) {
            const double other = cluster.map_shared_rank(&s, i)->cta[0];
            if (i < rank) before += other;
            if (i == rank) held = other;
            if (other > 0.0) last = i;
        }
        if (tid == 0) s.picked = -1;
        __syncthreads();
        // a draw at the very end of the sums belongs to the last id with any weight
        const bool here = (target >= before && target < before + held) || (rank == last && target >= before + held);
        if (here) {
            double ahead = before;
            int last_warp = 0;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) ahead += s.warp[0][w];
                if (s.warp[0][w] > 0.0) last_warp = w;
            }
            const double own = s.warp[0][warp];
            if (own > 0.0 && ((target >= ahead && target < ahead + own) || (warp == last_warp && target >= ahead + own))) {
                int found = -1, last_id = -1;
                for (int i0 = begin; i0 < end && found < 0; i0 += 32) {
                    const double m = i0 + lane < end ? mass_of(i0 + lane, plain) : 0.0;
                    double run = m;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, run, o);
                        if (lane >= o) run += up;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, m > 0.0 && ahead + run > target);
                    const unsigned some = __ballot_sync(0xffffffffu, m > 0.0);
                    if (over) found = i0 + __ffs(over) - 1;
                    if (some) last_id = i0 + 31 - __clz(some);
                    ahead += __shfl_sync(0xffffffffu, run, 31);
                }
                if (lane == 0) atomicMax(&s.picked, found >= 0 ? found : last_id);
            }
        }
        __syncthreads();
        if (here && tid == 0) picked[b] = s.picked;
        cluster.sync();  // nobody leaves while its sums may be read
        if (rank == 0 && tid == 0) accepted[b] = a;
        return;
    }
    if (rank == 0 && tid == 0) {
        accepted[b] = a;
        picked[b] = pick;
    }
}

static int verify_parts(int vocab) {
    const int n = (vocab + kVerifyShare - 1) / kVerifyShare;
    return n < 1 ? 1 : n > kVerifyParts ? kVerifyParts : n;
}

}  // namespace nnis

// Bytes of scratch that a call with `rows` rows of target and `draft_rows` rows of draft logits needs.
NNIS_API long long nnis_verify_scratch(int rows, int draft_rows, int vocab) {
    if (rows <= 0 || draft_rows < 0 || vocab <= 0) return -1;
    return (long long)(rows + draft_rows) * nnis::verify_parts(vocab) * (long long)sizeof(nnis::RowSum);
}

// first_row: n_seqs + 1 offsets into the packed rows of `logits` [rows, vocab], the last one `rows`; draft rows (drafts,
// accept_draws, draft_logits or null) lie without the sequences' last rows.
NNIS_API int nnis_verify_drafts(const float* logits, const float* draft_logits, const int* drafts, const int* first_row,
                                const float* temperature, const double* accept_draws, const double* pick_draws, void* scratch,
                                int n_seqs, int rows, int vocab, int* accepted, int* picked, cudaStream_t stream) {
    using namespace nnis;
    if (n_seqs <= 0 || rows < n_seqs || vocab <= 0 || !logits || !first_row || !temperature || !pick_draws || !scratch || !accepted ||
        !picked)
        return NNIS_ERR_ARGUMENT;
    const int draft_rows = rows - n_seqs, all_rows = rows + (draft_logits ? draft_rows : 0);
    if (draft_rows > 0 && (!drafts || !accept_draws)) return NNIS_ERR_ARGUMENT;
    if (all_rows > 65535 || n_seqs > 65535 || vocab > (1 << 30)) return NNIS_ERR_UNSUPPORTED;
    if ((uintptr_t)scratch % 16) return NNIS_ERR_ALIGNMENT;
    const int n_parts = verify_parts(vocab), per = (vocab + n_parts - 1) / n_parts;
    cudaError_t e = launch_dependent(verify_rows_kernel, dim3(n_parts, all_rows), kVerifyThreads, 0, stream, logits, draft_logits,
                                     first_row, temperature, n_seqs, rows, draft_rows, vocab, per, static_cast<RowSum*>(scratch));
    if (e != cudaSuccess) return (int)e;
    e = launch_dependent(verify_pick_kernel, dim3(kPickCtas, n_seqs), kPickThreads, 0, stream, logits, draft_logits, drafts, first_row,
                         temperature, accept_draws, pick_draws, static_cast<const RowSum*>(scratch), n_parts, rows, vocab, accepted,
                         picked);
    return e == cudaSuccess ? NNIS_OK : (int)e;
}
