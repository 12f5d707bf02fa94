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
// (the sums' 32-bit error is below 4e-5: exponents of 17 bits at most where they count, 2e-6, and 2^-24 for each of a
// thread's additions one after another, 5 with 300,000 logits, 520 with the most that are taken, 2^26).  Then the one row that is
// drawn from is summed in 64 bits, each CTA a range of ids and each warp a range of that, because a draw may fall next to a
// border between two of 50,000 tokens, and p - q cancels: 32 bits would pick another token every few hundred draws.  That walk
// sums p, q and both over the ids where p is the larger, so what q leaves of p needs no second one; only where it leaves next to
// nothing are the masses summed id by id.
//
// The first launch is bound by bytes: 960 rows of 49,152 (189 MB) 33 us, 5.7 TB/s; nine rows 3.7.  The second by the instructions of
// its 64-bit weights (45 a pair of logits, a third of them of 64 bits) and, with few sequences, by its chain of steps: draft,
// row, cluster, pick.  Both in turns, the next sequences' rows beside the last ones' picks, were slower (62 us for 58).
#include <cooperative_groups.h>
#include <float.h>
#include <string.h>

#include "async_copy.cuh"
#include "common.cuh"
#include "fma_pairs.cuh"

namespace nnis {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 256;
constexpr int kVerifyShare = 8192;   // logits of a row that a CTA of the first launch sums
constexpr int kVerifyParts = 32;     // most CTAs a row
constexpr int kPickThreads = 512;
constexpr int kPickCtas = 16;        // most of a cluster

struct __align__(16) RowSum {
    float max, sum;  // maximum logit, sum of exp((x - max) / T): no number where a logit is none, or +infinity
    int best;        // id of the maximum, the lower among equals
};

// log2(e) / T, within bounds that keep 0 and -infinity times it what they are (where that is another number the sums in 64
// bits decide, or all weights are one to 32 bits)
__device__ __forceinline__ float scale_of(float temperature) {
    return temperature > 0.f ? fmaxf(fminf(1.4426950408889634f / temperature, 1e30f), 1e-30f) : 1.f;
}

// 2^x; denormal results are zero
__device__ __forceinline__ float weight32(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Of the lanes of groups of LANES: the sums together, in every lane, and with BEST the id of the maximum, the lower among equals.
template <int LANES, bool BEST>
__device__ __forceinline__ RowSum joined(RowSum x, float c) {
    float max = x.max;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) max = fmaxf(max, __shfl_xor_sync(0xffffffffu, max, o));
    x.sum *= weight32((x.max - (max == -INFINITY ? 0.f : max)) * c);
    if (x.max != max) x.best = 0x7fffffff;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        x.sum += __shfl_xor_sync(0xffffffffu, x.sum, o);
        if (BEST) x.best = min(x.best, __shfl_xor_sync(0xffffffffu, x.best, o));
    }
    x.max = max;
    return x;
}

__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A thread's share of a row's ids from `begin` on, below `end`.  BEST: with the id of the maximum (greedy rows; else it is any).
template <bool BEST>
__device__ __forceinline__ RowSum thread_sum(const float* __restrict__ row, int begin, int end, float c) {
    // (32 bits: the maximum is taken off first, exactly, so that a large one costs no digits)
    RowSum mine = {-INFINITY, 0.f, 0x7fffffff};
    constexpr int kAhead = 4;  // quads a thread has on their way
    // quads from the row's first 16-byte boundary on; the first threads take what lies before it and what is left behind them
    const int head = min(end - begin, (int)((4 - (((uintptr_t)(row + begin) >> 2) & 3)) & 3)), quads = (end - begin - head) / 4;
    const float4* row4 = reinterpret_cast<const float4*>(row + begin + head);
    for (int at = threadIdx.x; at < quads; at += kAhead * kVerifyThreads) {
        float4 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = at + i * kVerifyThreads;
            x[i] = w < quads ? __ldcs(row4 + w) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) m = max3(max3(m, x[i].x, x[i].y), x[i].z, x[i].w);
        if (m > mine.max) {
            mine.sum *= weight32((mine.max - m) * c);
            mine.max = m;
            if (BEST) {
#pragma unroll
                for (int i = kAhead - 1; i >= 0; --i) {
                    const int id = begin + head + 4 * (at + i * kVerifyThreads);
                    mine.best = x[i].x == m ? id : x[i].y == m ? id + 1 : x[i].z == m ? id + 2 : x[i].w == m ? id + 3 : mine.best;
                }
            }
        }
        const unsigned long long off = both(mine.max == -INFINITY ? 0.f : -mine.max), cc = both(c);
        unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 u = halves(mul2(add2(h ? pair_of(x[i].z, x[i].w) : pair_of(x[i].x, x[i].y), off), cc));
                sum[h] = add2(sum[h], pair_of(weight32(u.x), weight32(u.y)));  // (a NaN or +infinity makes the sum one)
            }
        const float2 s = halves(add2(sum[0], sum[1]));
        mine.sum += s.x + s.y;
    }
    const int tail = begin + head + 4 * quads;
    if (head > 0 || tail < end) {  // at most six, a thread each
        const int t = threadIdx.x, id = t < head ? begin + t : tail + t - head;
        if (id < end && (t < head || t < head + 3)) {
            const float x = row[id];
            if (x > mine.max) {
                mine.sum *= weight32((mine.max - x) * c);
                mine.max = x;
                mine.best = id;
            } else if (BEST && x == mine.max) {
                mine.best = min(mine.best, id);
            }
            mine.sum += weight32((x - (mine.max == -INFINITY ? 0.f : mine.max)) * c);
        }
    }
    return mine;
}

__global__ void __launch_bounds__(kVerifyThreads)
verify_rows_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ first_row,
                   const float* __restrict__ temperature, int n_seqs, int rows, int vocab, int per, RowSum* __restrict__ parts) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ RowSum warp_sum_s[kVerifyThreads / 32];
    const int r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool of_draft = r >= rows;
    // the row's sequence: the last one that begins at or before it
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int)((unsigned)first_row[mid] - (of_draft ? (unsigned)mid : 0u)) <= (of_draft ? r - rows : r)) lo = mid;
        else hi = mid - 1;
    }
    const float t = temperature[lo];
    const float c = scale_of(t);
    const float* row = of_draft ? draft_logits + (size_t)(r - rows) * vocab : logits + (size_t)r * vocab;
    const int begin = min(vocab, (int)blockIdx.x * per), end = min(vocab, begin + per);
    const bool greedy = !(t > 0.f);
    RowSum mine = greedy ? joined<32, true>(thread_sum<true>(row, begin, end, c), c)
                         : joined<32, false>(thread_sum<false>(row, begin, end, c), c);
    if (lane == 0) warp_sum_s[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        mine = joined<kVerifyThreads / 32, true>(warp_sum_s[lane % (kVerifyThreads / 32)], c);
        if (lane == 0) parts[(size_t)r * gridDim.x + blockIdx.x] = mine;
    }
}

// A row's parts, a lane each (at most 32; up to eight are asked for by each quarter of the warp), and the row of them, in every lane.
__device__ __forceinline__ RowSum part_of(const RowSum* __restrict__ parts, size_t row, int n_parts) {
    const int part = n_parts <= 8 ? threadIdx.x & 7 : threadIdx.x & 31;
    return part < n_parts ? parts[row * n_parts + part] : RowSum{-INFINITY, 0.f, 0x7fffffff};
}
__device__ __forceinline__ RowSum row_of(const RowSum& part, int n_parts, float c) {
    return n_parts <= 8 ? joined<8, true>(part, c) : joined<32, true>(part, c);
}

__device__ __forceinline__ double sum64(double v, int from, int to) {  // over lanes that differ in these bits
    for (int o = from; o >= to; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum of the lanes up to this one, of sixteen.
__device__ __forceinline__ double half_scan64(double v) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, v, o, 16);
        if ((threadIdx.x & 15) >= o) v += up;
    }
    return v;
}

// exp((x - max) / T) in 64 bits for x <= max: with u = 64 (x - max) / (T ln 2) and k a whole number next to it, 2^(k / 64) from a
// table times the series of 2^((u - k) / 64) to the fourth power (what is left out is 5e-14), after P. T. P. Tang's
// table-driven method (ACM TOMS 15, 1989).  k is found in 32 bits (off by 0.01 at most from rounding u), so that seven
// instructions are of 64 bits, which the device has half as many units for; the sums of a row are bound by them.
struct Scale {
    double per;          // 64 / (T ln 2)
    double max;          // the row's maximum
    float per32, max32;  // the same
    float lowest;        // below it (700 T under the maximum, and at -infinity) a weight is zero
};
__device__ __forceinline__ Scale scale64(float max, double inv_t, float t) {
    const double per = inv_t * 92.33248261689366;
    // (a temperature below 1e-35 leaves the maximum alone: 64 / T is beyond 32 bits)
    return {per, (double)max, fminf((float)per, FLT_MAX), max, t < 1e-35f ? max : fmaxf(-FLT_MAX, max - 700.f * t)};
}
// (In constant memory, from where an instruction takes them: as numbers in the code each costs two moves whenever it is used.)
__constant__ double kSeries[4] = {5.732851688640402e-10, 2.1173137155464776e-07, 5.86490495505617e-05, 0.010830424696249145};

// The table holds 2^(j / 64) less j 2^14 in its high word, so that adding k 2^14 there leaves 2^(k / 64).
__device__ __forceinline__ double table_entry(int j) {
    const double e = exp2((double)j * (1.0 / 64.0));
    return __hiloint2double(__double2hiint(e) - (j << 14), __double2loint(e));
}
// (Where x lies below the lowest, and where it is -infinity, it may be anything.)
__device__ __forceinline__ double weight64_above(const double* table, float x, const Scale& c) {
    constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to a whole number, in the low bits
    const float k = fmaf(x - c.max32, c.per32, kRound);
    const int n = __float_as_int(k);
    const double f = fma((double)x - c.max, c.per, (double)(kRound - k));
    const double p = fma(fma(fma(kSeries[0], f, kSeries[1]), f, kSeries[2]), f, kSeries[3]);
    const double j = *reinterpret_cast<const double*>(reinterpret_cast<const char*>(table) + ((n << 3) & 504));
    const double e = __hiloint2double(__double2hiint(j) + (n << 14), __double2loint(j));
    return fma(e * f, p, e);
}
__device__ __forceinline__ double weight64(const double* table, float x, const Scale& c) {
    const double w = weight64_above(table, x, c);
    return x >= c.lowest ? w : 0.0;
}

constexpr int kPickWarps = kPickThreads / 32;

struct PickShared {
    double table[64];                // see table_entry
    double warp[4][kPickWarps];
    double cta[2][4][kPickCtas];     // every CTA's sums, written by them: [turn][which][rank]
    double chunk[kPickWarps];        // the warps' shares of the ids among which the pick lies
    float row_max[2][kPickWarps], row_sum[2][kPickWarps];  // of the row at which a warp stopped
    int stop, found, last;
};

// Sums over the whole cluster of four values a thread; every thread gets all.  Each CTA tells all others its sums, in
// one of two places by turns: a place is written again only when everybody has met once more.  A quarter of a warp has one of
// the four values from the start (shuffles are what sums of a warp's doubles cost).
__device__ __forceinline__ void cluster_sums(cg::cluster_group cluster, PickShared& s, int turn, double (&v)[4]) {
    const int lane = threadIdx.x & 31, n = lane >> 3, at = lane & 7;
    const bool high = lane & 16, odd = lane & 8;
    const double a = high ? v[2] : v[0], b = high ? v[3] : v[1];
    const double x = a + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], 16), y = b + __shfl_xor_sync(0xffffffffu, high ? v[1] : v[3], 16);
    double one = (odd ? y : x) + __shfl_xor_sync(0xffffffffu, odd ? x : y, 8);
    one = sum64(one, 4, 1);
    if (at == 0) s.warp[n][threadIdx.x >> 5] = one;
    __syncthreads();
    const int ctas = (int)cluster.num_blocks();
    if (threadIdx.x < 32) {
        one = sum64(s.warp[n][at] + s.warp[n][at + 8], 4, 1);
        for (int r = at; r < ctas; r += 8) cluster.map_shared_rank(&s, r)->cta[turn][n][cluster.block_rank()] = one;
    }
    cluster.sync();
    one = sum64((at < ctas ? s.cta[turn][n][at] : 0.0) + (at + 8 < ctas ? s.cta[turn][n][at + 8] : 0.0), 4, 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __shfl_sync(0xffffffffu, one, 8 * k);
}
static_assert(kPickWarps == 16 && kPickCtas == 16, "sums of sixteen");

__global__ void __launch_bounds__(kPickThreads, 2)
verify_pick_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ drafts,
                   const int* __restrict__ first_row, const float* __restrict__ temperature, const double* __restrict__ accept_draws,
                   const double* __restrict__ pick_draws, const RowSum* __restrict__ parts, int n_parts, int rows, int vocab,
                   int* __restrict__ accepted, int* __restrict__ picked) {
    __shared__ PickShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int b = blockIdx.y, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < 64) s.table[tid] = table_entry(tid);
    if (tid == 0) {
        s.stop = s.found = 0x7fffffff;
        s.last = -1;
    }
    // (What the call was given is older than the first launch, which has waited for it: it is read under that launch's end.)
    // (Offsets may be any numbers: differences wrap, and count for nothing where a comparison says that no packed rows have them.)
    const int row0 = first_row[b], row_end = first_row[b + 1];
    const int draft0 = (int)((unsigned)row0 - (unsigned)b), count = (int)((unsigned)row_end - (unsigned)row0 - 1u);
    const float t = temperature[b];
    const bool greedy = !(t > 0.f);
    const float c = scale_of(t);
    const double inv_t = greedy ? 1.0 : 1.0 / (double)t;
    // (good ones leave as many draft rows as there are drafts)
    const bool good = row0 >= b && row_end > row0 && row_end <= rows && row_end - b <= rows - (int)gridDim.y + 1;
    // A warp's draft: its logits in the two rows.
    struct Draft {
        int id;
        float z, y;
        double draw;
    };
    auto draft_of = [&](int i) {
        Draft x = {-1, 0.f, 0.f, 0.0};
        if (i < count) {
            x.id = drafts[draft0 + i];
            x.draw = accept_draws[draft0 + i];
            if (x.id >= 0 && x.id < vocab && !greedy) {
                x.z = logits[(size_t)(row0 + i) * vocab + x.id];
                if (draft_logits) x.y = draft_logits[(size_t)(draft0 + i) * vocab + x.id];
            }
        }
        return x;
    };
    Draft mine = draft_of(good ? warp : count);
    cluster.sync();  // (all of the cluster run: their shared memory may be written)
    pdl_wait();
    pdl_launch_dependents();
    if (!good) {  // (offsets that no packed rows have: the whole cluster leaves)
        if (rank == 0 && tid == 0) {
            accepted[b] = 0;
            picked[b] = -1;
        }
        return;
    }

    // The drafts, a warp each: where the first one lies that is not kept for sure, and why (every CTA of the cluster for
    // itself, all alike).
    enum { kKept, kRefused, kNothing, kNear };
    auto decide = [&](int i, const Draft& x) -> int {
        const bool drafted = i < count, other = drafted && draft_logits && !greedy;
        const bool known = x.id >= 0 && x.id < vocab;
        RowSum zs = part_of(parts, (size_t)(row0 + i), n_parts), ys = {0.f, 1.f, 0};
        if (other) ys = part_of(parts, (size_t)(rows + draft0 + i), n_parts);
        zs = row_of(zs, n_parts, c);
        if (other) ys = row_of(ys, n_parts, c);
        if (lane == 0) {
            s.row_max[0][warp] = zs.max;
            s.row_max[1][warp] = ys.max;
            s.row_sum[0][warp] = zs.sum;
            s.row_sum[1][warp] = ys.sum;
        }
        if (!(zs.sum >= 0.f) || zs.max == -INFINITY || zs.max == INFINITY) return kNothing;
        if (!drafted) return kRefused;
        if (greedy) return x.id == zs.best ? kKept : kRefused;
        if (!(ys.sum >= 0.f) || ys.max == -INFINITY || ys.max == INFINITY) return kNothing;
        if (!known) return kRefused;
        const double eq = other ? weight64(s.table, x.y, scale64(ys.max, inv_t, t)) : 1.0;
        const double left = x.draw * eq * (double)zs.sum, right = weight64(s.table, x.z, scale64(zs.max, inv_t, t)) * (double)ys.sum;
        if (fabs(left - right) <= 1e-4 * right || t < 1e-29f) return kNear;
        return left < right ? kKept : kRefused;
    };
    // A warp's ids lie together, 32 at a time.
    const int per_warp = (((vocab + ctas * kPickWarps - 1) / (ctas * kPickWarps)) + 31) & ~31;
    const int begin = min(vocab, (rank * kPickWarps + warp) * per_warp), end = min(vocab, begin + per_warp);
    constexpr int kAhead = 4;
    const float *z = nullptr, *y = nullptr;
    Scale zc = {}, yc = {};
    float line = 0.f;  // p is larger than q where z - y lies above it (by the sums in 32 bits)
    auto ask = [&](const float* row, int first, float (&x)[kAhead]) {  // logits of ids first, first + 32, ...
        if (first - lane + 32 * kAhead <= end) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = row[first + 32 * k];
        } else {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = first + 32 * k < end ? row[first + 32 * k] : -INFINITY;
        }
    };
    // The sums of row i, at which warp `stopped` stopped, in 64 bits: of p's weights, of q's, and of both over the ids where p is
    // the larger, by the sums in 32 bits.  The last two give what q leaves of p, sum p[more] / sum p - sum q[more] / sum q,
    // without a second walk: an id on the wrong side of that line has p and q within some 2e-5 of one another, and counts for as much.
    int turn = 0;
    double sums[4];
    auto walk = [&](int i, int stopped, int without) {
        z = logits + (size_t)(row0 + i) * vocab;
        y = draft_logits && i < count ? draft_logits + (size_t)(draft0 + i) * vocab : nullptr;
        zc = scale64(s.row_max[0][stopped], inv_t, t);
        yc = scale64(s.row_max[1][stopped], inv_t, t);
        line = y ? s.row_max[0][stopped] - s.row_max[1][stopped] + t * logf(s.row_sum[0][stopped] / s.row_sum[1][stopped]) : -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n) sums[n] = 0.0;
        float xz[kAhead], xy[kAhead];
        if (y) {
            ask(z, begin + lane, xz);
            ask(y, begin + lane, xy);
            for (int i0 = begin + lane; i0 < end; i0 += 32 * kAhead) {
                float next_z[kAhead], next_y[kAhead];  // (on their way while these are worked)
                ask(z, i0 + 32 * kAhead, next_z);
                ask(y, i0 + 32 * kAhead, next_y);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const double ez = weight64_above(s.table, xz[k], zc), ey = weight64_above(s.table, xy[k], yc);
                    const bool any = xy[k] >= yc.lowest, more = xz[k] - xy[k] > line;
                    if (xz[k] >= zc.lowest) {
                        sums[0] += ez;
                        if (more) sums[2] += ez;
                    }
                    if (any) sums[1] += ey;
                    if (any && more) sums[3] += ey;
                    xz[k] = next_z[k];
                    xy[k] = next_y[k];
                }
            }
        } else {
            ask(z, begin + lane, xz);
            for (int i0 = begin + lane; i0 < end; i0 += 32 * kAhead) {
                float next_z[kAhead];
                ask(z, i0 + 32 * kAhead, next_z);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const double ez = weight64_above(s.table, xz[k], zc);
                    const bool any = xz[k] >= zc.lowest;
                    if (any) sums[0] += ez;
                    if (any && i0 + 32 * k != without) sums[2] += ez;
                    xz[k] = next_z[k];
                }
            }
        }
        cluster_sums(cluster, s, turn, sums);
        turn ^= 1;
        if (!y) sums[1] = 1.0;
    };

    int a = 0, why = kNear;
    for (int from = 0;;) {
        for (int i = from + warp; i <= count; i += kPickWarps) {
            const int how = decide(i, mine);
            if (how != kKept) {
                if (lane == 0) atomicMin(&s.stop, i * 4 + how);
                break;
            }
            mine = draft_of(i + kPickWarps);
        }
        __syncthreads();
        a = s.stop >> 2;
        why = s.stop & 3;
        if (why == kNothing || greedy) break;
        const int d = a < count ? drafts[draft0 + a] : -1;
        walk(a, (a - from) % kPickWarps, draft_logits ? -1 : d);  // (all CTAs of the cluster come here together)
        if (why != kNear) break;
        const double eq = y ? weight64(s.table, y[d], yc) : 1.0;
        if (!(accept_draws[draft0 + a] * eq * sums[0] < weight64(s.table, z[d], zc) * sums[1])) break;
        if (tid == 0) s.stop = 0x7fffffff;  // (everybody has read it: they have met)
        __syncthreads();
        from = a + 1;
        mine = draft_of(from + warp);
    }
    if (why == kNothing || greedy) {
        if (rank == 0 && warp == 0) {
            const int best = row_of(part_of(parts, (size_t)(row0 + a), n_parts), n_parts, c).best;
            if (lane == 0) {
                accepted[b] = a;
                picked[b] = why == kNothing ? -1 : best;
            }
        }
        return;
    }
    // The distribution to draw from: p, or what of it the draft's distribution leaves.
    const int d = a < count ? drafts[draft0 + a] : -1;
    const double ip = 1.0 / sums[0], iq = y ? 1.0 / sums[1] : 0.0;
    bool plain = a >= count;
    auto mass = [&](int i, float xz, float xy) {  // of id i
        const double p = __dmul_rn(weight64(s.table, xz, zc), ip);  // (rounded like q: equal ones leave nothing)
        return plain ? p : y ? fmax(p - __dmul_rn(weight64(s.table, xy, yc), iq), 0.0) : i == d ? 0.0 : p;
    };
    // Masses of warps and CTAs, from their sums over the ids where p is the larger.  Where q leaves little (or, by
    // rounding, nothing) of p the line between those ids is too coarse: the masses are summed id by id.
    double mp = ip, mq = iq, total = mp * sums[2] - mq * sums[3];
    if (!plain && (!(total >= 0.01) || t < 1e-29f)) {
        mp = 1.0;
        mq = 0.0;
        for (;;) {
            sums[0] = sums[1] = sums[2] = sums[3] = 0.0;
            for (int i = begin + lane; i < end; i += 32) sums[2] += mass(i, z[i], y ? y[i] : 0.f);
            cluster_sums(cluster, s, turn, sums);
            turn ^= 1;
            total = sums[2];
            if (plain || total > 0.0) break;
            plain = true;  // nothing is left: p and q are one
        }
    }
    const double target = fmin(fmax(pick_draws[b], 0.0), 1.0) * total;  // (a draw of another range, or no number, is its next end)
    // Where in the row the target lies: the CTAs' masses, lane by lane, then the warps'.  A draw at the very end of the
    // sums belongs to the last id with any weight.
    auto place = [&](double mass, double& ahead) {  // of sixteen; `ahead`: what lies before the first, then before the one
        const double upto = half_scan64(mass);
        const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0) & 0xffffu;
        const unsigned over = __ballot_sync(0xffffffffu, mass > 0.0 && target < ahead + upto) & 0xffffu;
        const int one = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : 0;
        const double before = __shfl_sync(0xffffffffu, upto, max(one - 1, 0));
        if (one) ahead += before;
        return one;
    };
    if (rank == 0 && tid == 0) accepted[b] = a;
    const int at = lane & 15;
    double ahead = 0.0;
    if (place(at < ctas ? fmax(mp * s.cta[turn ^ 1][2][at] - mq * s.cta[turn ^ 1][3][at], 0.0) : 0.0, ahead) != rank) return;
    // The CTA goes through that warp's ids together.
    const int of = place(fmax(mp * s.warp[2][at] - mq * s.warp[3][at], 0.0), ahead);
    const int first = min(vocab, (rank * kPickWarps + of) * per_warp), behind = min(vocab, first + per_warp);
    for (int i0 = first;; i0 += kPickThreads) {
        if (i0 >= behind) {
            if (s.last >= 0 || plain) break;
            plain = true;  // (only ids of equal p and q are here, on the line by a rounding: one of them by p)
            i0 = first;
        }
        const int i = i0 + tid;
        const double m = i < behind ? mass(i, z[i], y ? y[i] : 0.f) : 0.0;
        double run = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += up;
        }
        if (lane == 31) s.chunk[warp] = run;
        __syncthreads();
        const double upto = half_scan64(s.chunk[at]), before = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0));
        if (m > 0.0) {  // (written between the two meetings, read between the second and the next turn's first)
            atomicMax(&s.last, i);
            if (ahead + ((warp ? before : 0.0) + run) > target) atomicMin(&s.found, i);
        }
        ahead += __shfl_sync(0xffffffffu, upto, 15);
        __syncthreads();
        if (s.found < vocab) break;
    }
    if (tid == 0) picked[b] = s.found < vocab ? s.found : s.last;
}
// CTAs a row: shares of 8,192 logits, of 4,096 where all rows together are no more than four CTAs an SM then (nine rows of 49,152:
// 4.4 -> 3.7 us; 144 rows 9.2 us with 8,192, 9.7 with 4,096, 960 rows 33 and 41).
static int verify_parts(long long rows, int vocab) {
    const int fine = (vocab + kVerifyShare / 2 - 1) / (kVerifyShare / 2);
    const int n = rows * fine <= 600 ? fine : (vocab + kVerifyShare - 1) / kVerifyShare;
    return n < 1 ? 1 : n > kVerifyParts ? kVerifyParts : n;
}

}  // namespace nnis

// Bytes of scratch that a call with `rows` rows of target and `draft_rows` rows of draft logits needs.
NNIS_API long long nnis_verify_scratch(int rows, int draft_rows, int vocab) {
    if (rows <= 0 || draft_rows < 0 || vocab <= 0) return -1;
    return (long long)(rows + draft_rows) * nnis::verify_parts(rows + draft_rows, vocab) * (long long)sizeof(nnis::RowSum);
}

// first_row: n_seqs + 1 offsets into the packed rows of `logits` [rows, vocab], the last one `rows`; draft rows (drafts,
// accept_draws, draft_logits or null) lie without the sequences' last rows.
struct VerifyCall {
    const float *logits, *draft_logits;
    const int *drafts, *first_row;
    const float* temperature;
    const double *accept_draws, *pick_draws;
    void* scratch;
    int n_seqs, rows, vocab;
    int *accepted, *picked;
    cudaStream_t stream;
};
NNIS_API int nnis_verify_drafts(const void* call) {
    using namespace nnis;
    VerifyCall v;
    memcpy(&v, call, sizeof v);
    const auto [logits, draft_logits, drafts, first_row, temperature, accept_draws, pick_draws, scratch, n_seqs, rows, vocab, accepted,
                picked, stream] = v;
    if (n_seqs <= 0 || rows < n_seqs || vocab <= 0 || !logits || !first_row || !temperature || !pick_draws || !scratch || !accepted ||
        !picked)
        return NNIS_ERR_ARGUMENT;
    const int draft_rows = rows - n_seqs, all_rows = rows + (draft_logits ? draft_rows : 0);
    if (draft_rows > 0 && (!drafts || !accept_draws)) return NNIS_ERR_ARGUMENT;
    if (all_rows > 65535 || n_seqs > 65535 || vocab > (1 << 26)) return NNIS_ERR_UNSUPPORTED;
    if ((uintptr_t)scratch % 16) return NNIS_ERR_ALIGNMENT;
    const int n_parts = verify_parts(rows + draft_rows, vocab), per = (vocab + n_parts - 1) / n_parts;
    cudaError_t e = launch_dependent(verify_rows_kernel, dim3(n_parts, all_rows), kVerifyThreads, 0, stream, logits, draft_logits,
                                     first_row, temperature, n_seqs, rows, vocab, per, static_cast<RowSum*>(scratch));
    if (e != cudaSuccess) return (int)e;
    // As many CTAs a sequence as the device holds at once (two an SM) for all of them, sixteen at most, four at least: the launch takes
    // 9.8 us with sixteen (one sequence, rows of 49,152), 10.7 with eight (24 sequences), 21.5 with four (64 sequences, which eight
    // would take in two turns).
    cudaLaunchConfig_t cfg = {};
    static const int slots = 2 * device_sms();
    int ctas = kPickCtas;
    while (ctas > 4 && n_seqs * ctas > slots) ctas /= 2;
    static std::atomic<int> large[16];
    int device = 0;
    if ((e = cudaGetDevice(&device)) != cudaSuccess) return (int)e;
    if (device >= 16 || !large[device].load(std::memory_order_relaxed)) {  // (sixteen CTAs a cluster are asked for once)
        if ((e = cudaFuncSetAttribute(verify_pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return (int)e;
        if (device < 16) large[device].store(1, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3(ctas, n_seqs);
    cfg.blockDim = dim3(kPickThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent_launches() ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, verify_pick_kernel, logits, draft_logits, drafts, first_row, temperature, accept_draws, pick_draws,
                           static_cast<const RowSum*>(scratch), n_parts, rows, vocab, accepted, picked);
    return e == cudaSuccess ? NNIS_OK : (int)e;
}
