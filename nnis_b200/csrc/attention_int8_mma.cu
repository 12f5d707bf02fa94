// Attention of single rows, or of a few rows of a sequence, over the paged cache held in 8 bits, on the tensor cores: heads of 32, 64, 96 and
// 128, pages of 64 positions, float32 and bfloat16.
//
// The key's codes are multiplied as they are.  A query's head is put into whole numbers once, N = rint(q * (top' / top)), of two signed
// bytes (bfloat16: N = 256 hi + lo, off by at most top / 65,024 a value) or three (float32: 65,536 hi + 256 mid + lo, off by 2^-24 of
// top); a product of 16 x 8 x 32 whole numbers (mma.sync) holds eight queries' first bytes in its rows 0 to 7 and their second bytes in
// rows 8 to 15, so that a thread gets both sums of a score, exact, and score = (256 hi + lo) * (top / top') * key scale * scale.
// The value's codes become float16 (a byte b of 0 to 255 behind the byte 0x64 is 1,024 + b) for products of 16 x 8 x 16 with the weights
// w_j = 2^15 p_j t_j / T, where t_j is the value's scale and T a power of two above all scales that the warp has met: w_j is below
// 2^15, and float16 holds what is 2^-29 of T to its full 11 bits.  A row whose weighted values all lie far below T, because the large values
// that its warp has met have next to no weight for it, is looked at again in float32 (attend_alone8).  bfloat16: eight more queries in rows
// 8 to 15.
// float32: what float16 has left of the weights there, so that a weight has 22 bits.  Maxima, sums and outputs are float32.
//
// Any order of a head's values serves the first product and any order of positions the second, so a thread's part of every fragment lies
// side by side in shared memory as the copies bring it: a thread of the key product holds bytes [t D / 4, (t + 1) D / 4) of a
// position's row, of the value product bytes [g D / 8, (g + 1) D / 8) of positions 4 t to 4 t + 3 (g = lane / 4, t = lane % 4).
//
// A CTA: four warps, (run of rows with one sequence, key/value head, tile of queries, slice of positions); a warp takes every fourth piece
// of 64 or 32 positions of the slice through a ring of its own, filled by bulk copies, so that nothing meets before the slice's end.  Slices are of a
// fixed number of pieces, so sequences of all lengths are cut into equal pieces (where a run's rows lie further apart than its window is
// long, the last slice has what the others leave); the slice that ends last joins them.
#include <float.h>
#include <string.h>

#include <cuda_fp16.h>

#include "async_copy.cuh"
#include "int8_rows.cuh"
#include "attention_int8.cuh"

namespace nnis {

constexpr int kPage8 = 64, kWarps8 = 4;

__host__ __device__ constexpr int stage_bytes8(int d) { return 2 * piece8(d) * (d + 4); }

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same without sums before it
__device__ __forceinline__ void mma_s8_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2_8(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Two codes (bytes of `pair`, biased by 128) as float16
__device__ __forceinline__ uint32_t code_halves(uint32_t pair, uint32_t select) {
    const uint32_t biased = __byte_perm(pair, 0x64646464u, select), bias = 0x64806480u;  // 1,024 + 128
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int kMostCluster8 = 8;
// Every thread of every CTA of the cluster
__device__ __forceinline__ void cluster_sync8() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What lies at the same place of the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 peer_load2(const float* p, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_load4(const float* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void add_part(float4& sum, float& total, const float4& v, float l, float share) {
    total = fmaf(share, l, total);
    sum.x = fmaf(share, v.x, sum.x);
    sum.y = fmaf(share, v.y, sum.y);
    sum.z = fmaf(share, v.z, sum.z);
    sum.w = fmaf(share, v.w, sum.w);
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}

// A query's D / 4 values of this thread -> bytes of the whole numbers, words of four values; the factor that turns a sum of their
// products into the query's.
template <int D, bool F32>
__device__ __forceinline__ float query_codes(const float (&x)[D / 4], uint32_t (&hi)[D / 16], uint32_t (&mid)[D / 16], uint32_t (&lo)[D / 16]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = max(top, magnitude_bits(x[i]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    constexpr float kMost = F32 ? 127.f * 65536.f : 127.f * 256.f;
    const bool none = top >= 0x7f800000u, zero = __uint_as_float(top) < 0x1p-100f;
    const float inverse = none || zero ? 0.f : __fdiv_rn(kMost, __uint_as_float(top));
#pragma unroll
    for (int w = 0; w < D / 16; ++w) {
        int h[4], m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int n = __float2int_rn(x[4 * w + i] * inverse);
            l[i] = (int)(int8_t)n;
            n = (n - l[i]) >> 8;
            m[i] = F32 ? (int)(int8_t)n : 0;
            h[i] = F32 ? (n - m[i]) >> 8 : n;
        }
        hi[w] = pack_codes(h[0], h[1], h[2], h[3]);
        mid[w] = F32 ? pack_codes(m[0], m[1], m[2], m[3]) : 0u;
        lo[w] = pack_codes(l[0], l[1], l[2], l[3]);
    }
    return none ? __uint_as_float(0x7fc00000u) : zero ? 0.f : __fdiv_rn(__uint_as_float(top), kMost);
}

// One row over a warp's pieces, by all lanes of the warp, in float32 throughout: sums of weights times values, [D] to `sums`; its maximum
// (of scores in units of log 2) and sum of weights.  For rows that float16 has lost: a weight is off by up to 2^-25, half of float16's least
// step, so a sum over n positions by up to n 127 2^-25, and where a row's sums are all below lost8 that is told from nothing no more
// (4,096 positions: 2^-6 / lost8; a row of weight one on values as large as any has 2^20).
__host__ __device__ constexpr float lost8(bool f32) { return f32 ? 4096.f : 256.f; }
template <int D, typename T>
__device__ __forceinline__ float2 attend_alone8(const Attend8& p, const int* table, int hk, const T* q, int low, int pos, int first, int last, int step,
                                             float* query, float* sums) {
    constexpr int kPiece = piece8(D), kPieces = kPage8 / kPiece, kOwn = D / 32;
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < D; i += 32) query[i] = to_float(q[i]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, acc[kOwn] = {};
    for (int piece = first; piece < last; piece += step) {
        const int page = table[(unsigned)piece / kPieces];
        if ((unsigned)page >= (unsigned)p.pages) continue;
        for (int at = 0; at < kPiece; at += 32) {
            const int key = piece * kPiece + at + lane;
            const bool seen = key >= low && key <= pos;
            if (!__any_sync(0xffffffffu, seen)) continue;
            const size_t row = ((size_t)page * p.nkv + hk) * kPage8 + piece % kPieces * kPiece + at;
            float score = -INFINITY, t = 0.f;
            if (seen) {
                const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.k + (row + lane) * D);
                float dot = 0.f;
                for (int i = 0; i < D / 4; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) dot = fmaf(query[4 * i + c], code_value(codes[i], c), dot);
                score = dot * p.k_scales[row + lane] * (p.scale * 1.4426950408889634f);
                t = p.v_scales[row + lane];
            }
            const float now = fmaxf(m, warp_max(score)), base = now == -INFINITY ? 0.f : now, shrink = ex2_8(m - base);
            float w = seen ? ex2_8(score - base) : 0.f;
            l = fmaf(l, shrink, warp_sum(w));
            m = now;
            w = w == 0.f ? 0.f : w * t;
#pragma unroll
            for (int r = 0; r < kOwn; ++r) acc[r] *= shrink;
            for (int j = 0; j < 32; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j);
                if (wj == 0.f) continue;
                const int8_t* value = p.v + (row + j) * D + lane;
#pragma unroll
                for (int r = 0; r < kOwn; ++r) acc[r] = fmaf(wj, (float)value[32 * r], acc[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kOwn; ++r) sums[lane + 32 * r] = acc[r];
    __syncwarp();
    return make_float2(m, l);
}

// The same as a call, where the row's registers beside a tile's of sixteen queries would spill the tile's
template <int D, typename T>
__device__ __noinline__ float2 attend_alone_call8(const Attend8& p, const int* table, int hk, const T* q, int low, int pos, int first, int last, int step,
                                                  float* query, float* sums) {
    return attend_alone8<D, T>(p, table, hk, q, low, pos, first, last, step, query, sums);
}

// SOLO: a warp a unit, its whole range of keys, for many rows with few keys.
template <int D, bool F32, int MT, bool SOLO>
__global__ void __launch_bounds__(kWarps8 * 32, D <= 32 ? 4 : D <= 96 ? 3 : 2) attn_int8_mma_kernel(const __grid_constant__ Attend8 p) {
    using T = std::conditional_t<F32, float, bf16>;
    constexpr int kStage = stage_bytes8(D), kTile = 8 * MT, kSteps = D / 32, kWords = D / 16, kValueWords = D / 32, kCols = D / 8;
    constexpr int kOuts = F32 ? MT : (MT + 1) / 2;  // products of the weights per step of 16 positions
    constexpr int kPiece8 = piece8(D), kStages = stages8(D), kScores = kPiece8 / 4;  // (a lane's positions of a piece: 16 s + 4 t + 0 to 3)
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[kWarps8][kStages];
    __shared__ int joins;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {  // (a warp's barriers are its own)
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();

    const int per = p.nq / p.nkv, slice = SOLO ? 0 : blockIdx.y / p.cluster, rank = SOLO ? 0 : blockIdx.y % p.cluster;
    int unit = SOLO ? blockIdx.x * kWarps8 + warp : blockIdx.x;
    if (SOLO && unit >= p.units) return;  // (whole warps: nothing below meets in this form)
    const int tile = unit % p.tiles;
    unit /= p.tiles;
    const int hk = unit % p.nkv, row_first = unit / p.nkv * p.rows_at_once, row_end = min(p.n, row_first + p.rows_at_once);
    unsigned char* ring = smem + (size_t)warp * kStages * kStage;
    int stage = 0;  // the ring's next, over all runs, and the phase of its barrier
    uint32_t phase = 0;
    // what lane 0 to 3 copies of a piece: codes of keys, of values, scales of keys, of values
    const bool codes = lane < 2;
    const unsigned char* mine = codes ? reinterpret_cast<const unsigned char*>(lane == 0 ? p.k : p.v)
                                      : reinterpret_cast<const unsigned char*>(lane == 2 ? p.k_scales : p.v_scales);
    const uint32_t row_bytes = codes ? D : 4, piece_bytes = kPiece8 * row_bytes, page_bytes = (uint32_t)p.nkv * kPage8 * row_bytes;
    const uint32_t to_lane = codes ? lane * kPiece8 * D : 2 * kPiece8 * D + (lane & 1) * kPiece8 * 4;
    mine += (size_t)hk * kPage8 * row_bytes;

    for (int r0 = row_first, r1; r0 < row_end; r0 = r1) {
        // ---- the queries of as many rows as the run may have are asked for beside its sequence and positions, before anything waits
        const int e0 = tile * kTile;
        float x[MT][D / 4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int e = min(e0 + 8 * i + g, (row_end - r0) * per - 1);
            const T* q = reinterpret_cast<const T*>(p.q) + (size_t)(r0 + e / per) * p.q_stride + (size_t)(hk * per + e % per) * D + t * (D / 4);
            if (p.aligned) {
#pragma unroll
                for (int c = 0; c < D / 4; c += 4) {
                    const float4 v = load4(q + c);
                    x[i][c] = v.x; x[i][c + 1] = v.y; x[i][c + 2] = v.z; x[i][c + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 4; ++c) x[i][c] = to_float(q[c]);
            }
        }
        // ---- the run, its keys and this slice's part of them (the same for every thread of the CTA): a lane a row, for a loop over rows
        // waits for each
        int seq = -1, top_pos = -1, low_pos = INT_MAX;
        for (int first_row = r0;; first_row += 32) {
            const bool there = first_row + lane < row_end;
            const int mine_seq = there ? p.token_seq[first_row + lane] : -1, pos = there ? p.token_pos[first_row + lane] : -1;
            if (first_row == r0) seq = __shfl_sync(0xffffffffu, mine_seq, 0);
            const uint32_t others = ~__ballot_sync(0xffffffffu, there && mine_seq == seq);
            const int count = others ? __ffs(others) - 1 : 32;
            const bool counts = lane < count && pos >= 0;
            top_pos = max(top_pos, __reduce_max_sync(0xffffffffu, counts ? pos : -1));
            low_pos = min(low_pos, __reduce_min_sync(0xffffffffu, counts ? pos : INT_MAX));
            r1 = first_row + count;
            if (count < 32 || r1 >= row_end) break;
        }
        const int low = p.window > 0 && low_pos != INT_MAX ? max(0, low_pos - p.window + 1) : 0, top_low = p.window > 0 ? max(0, top_pos - p.window + 1) : 0;
        const int entries = (r1 - r0) * per;
        if (e0 >= entries) continue;
        const bool known = seq >= 0 && seq < p.table_rows && top_pos >= 0;
        const int* table = p.page_table + (size_t)(known ? seq : 0) * p.table_cols;
        constexpr int kHalves = kPage8 / kPiece8;
        const int piece_low = known ? low / kPiece8 : 0, piece_top = known ? (int)min((long long)top_pos / kPiece8 + 1, (long long)kHalves * p.table_cols) : 0;
        // a slice's pieces are dealt out to all warps of its cluster
        const int slices = max(1, min(p.splits, (piece_top - piece_low + p.slice_pieces - 1) / p.slice_pieces));
        if (!SOLO && slice >= slices) continue;
        const int first = SOLO ? piece_low : piece_low + slice * p.slice_pieces, last = SOLO || slice == slices - 1 ? piece_top : first + p.slice_pieces;
        const int step = SOLO ? 1 : kWarps8 * p.cluster;

        // ---- copies: this warp's pieces are every step-th; those of pages outside the store are passed over.  The next
        // piece's page is asked for as a piece is copied, and looked at when its turn comes.
        int next = SOLO ? first : first + rank * kWarps8 + warp, page = next < last ? table[(unsigned)next / kHalves] : -1;
        auto copy = [&](int to) {  // the piece that is copied to this stage, -1 where none is left
            while (next < last && (unsigned)page >= (unsigned)p.pages) {
                next += step;
                page = next < last ? table[(unsigned)next / kHalves] : -1;
            }
            if (next >= last) return -1;
            if (lane < 4) {
                if (lane == 0) mbar_expect_tx(&full[warp][to], kStage);
                bulk_load(ring + to * kStage + to_lane, mine + (size_t)(unsigned)page * page_bytes + (unsigned)next % kHalves * piece_bytes, piece_bytes,
                          &full[warp][to]);
            }
            const int piece = next;
            next += step;
            page = next < last ? table[(unsigned)next / kHalves] : -1;
            return piece;
        };
        int queue[kStages];
#pragma unroll
        for (int s = 0; s < kStages; ++s) queue[s] = copy(stage + s < kStages ? stage + s : stage + s - kStages);

        // ---- the tile's queries as whole numbers
        uint32_t qa[MT][kSteps][4], ql[F32 ? MT : 1][F32 ? kSteps : 1][2];
        float factor[MT], m[MT], l[MT];
        int pos_of[MT], low_of[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int e = e0 + 8 * i + g;
            pos_of[i] = e < entries && known ? p.token_pos[r0 + e / per] : -1;
            low_of[i] = p.window > 0 ? max(0, pos_of[i] - p.window + 1) : 0;
            uint32_t hi[kWords], mid[kWords], lo[kWords];
            factor[i] = query_codes<D, F32>(x[i], hi, mid, lo) * p.scale * 1.4426950408889634f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                qa[i][s][0] = hi[2 * s];
                qa[i][s][2] = hi[2 * s + 1];
                qa[i][s][1] = F32 ? mid[2 * s] : lo[2 * s];
                qa[i][s][3] = F32 ? mid[2 * s + 1] : lo[2 * s + 1];
                if constexpr (F32) {
                    ql[i][s][0] = lo[2 * s];
                    ql[i][s][1] = lo[2 * s + 1];
                }
            }
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
        float o[kOuts][kCols][4] = {};
        float unit_t = 0.f, inverse_t = 0.f;  // T and 2^15 / T

#pragma unroll 1
        while (queue[0] >= 0) {
            const int piece = queue[0];
            const unsigned char* at = ring + stage * kStage;
            if (!mbar_wait(&full[warp][stage], phase)) {
                if (lane == 0) atomicExch(p.status, 1);
                // (copies that are on their way do not outlive the CTA)
#pragma unroll
                for (int s = 1; s < kStages; ++s) {
                    const int to = stage + s < kStages ? stage + s : stage + s - kStages;
                    if (queue[s] >= 0) mbar_wait(&full[warp][to], to < stage ? phase ^ 1u : phase);
                }
                break;
            }
            const float* ks = reinterpret_cast<const float*>(at + 2 * kPiece8 * D);
            const float* vs = ks + kPiece8;
            const int key0 = piece * kPiece8 + 4 * t;
            const bool whole = piece * kPiece8 >= top_low && piece * kPiece8 + kPiece8 - 1 <= low_pos;
            // ---- scores, in units of log 2: position 16 s + 4 t + i is value i of step s
            float sc[MT][kScores];
#pragma unroll
            for (int s = 0; s < kScores / 4; ++s) {
                int acc[MT][2][4], acl[F32 ? MT : 1][2][4];
                uint32_t w[2][kWords];
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    load_words<kWords>(w[j], at + (16 * s + 4 * (g >> 1) + 2 * j + (g & 1)) * D + t * (D / 4));
                // (products that follow one another belong to different sums: a warp waits some 30 cycles for one that its next adds to)
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if (k == 0) mma_s8_first(acc[i][j], qa[i][k], w[j][2 * k], w[j][2 * k + 1]);
                            else mma_s8(acc[i][j], qa[i][k], w[j][2 * k], w[j][2 * k + 1]);
                            if constexpr (F32) {
                                const uint32_t a[4] = {ql[i][k][0], 0u, ql[i][k][1], 0u};
                                if (k == 0) mma_s8_first(acl[i][j], a, w[j][2 * k], w[j][2 * k + 1]);
                                else mma_s8(acl[i][j], a, w[j][2 * k], w[j][2 * k + 1]);
                            }
                        }
                const float4 scales = *reinterpret_cast<const float4*>(ks + 16 * s + 4 * t);
                const float key_scale[4] = {scales.x, scales.y, scales.z, scales.w};
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int first_part = acc[i][c >> 1][c & 1], second_part = acc[i][c >> 1][(c & 1) + 2];
                        float sum;
                        if constexpr (F32)
                            sum = fmaf((float)first_part, 65536.f, fmaf((float)second_part, 256.f, (float)acl[i][c >> 1][c & 1]));
                        else
                            sum = (float)(first_part * 256 + second_part);
                        sc[i][4 * s + c] = sum * factor[i] * key_scale[c];
                    }
            }
            float ts[kScores];
#pragma unroll
            for (int s = 0; s < kScores / 4; ++s) {
                const float4 scales = *reinterpret_cast<const float4*>(vs + 16 * s + 4 * t);
                ts[4 * s] = scales.x; ts[4 * s + 1] = scales.y; ts[4 * s + 2] = scales.z; ts[4 * s + 3] = scales.w;
            }
            // (a value's scale that is no number must not meet a weight of zero: nobody's positions have none, and where one row of
            // several sees such a value and another does not, the weights are looked at one by one)
            bool looks = false;
            if (!whole) {
#pragma unroll
                for (int c = 0; c < kScores; ++c) {
                    const int key = key0 + 16 * (c >> 2) + (c & 3);
                    if (key < low || key > top_pos) ts[c] = 0.f;
                    looks = looks || ts[c] != ts[c];
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        if (key > pos_of[i] || key < low_of[i]) sc[i][c] = -INFINITY;
                }
                looks = __any_sync(0xffffffffu, looks);
            }
            float t_most = ts[0];
#pragma unroll
            for (int c = 1; c < kScores; ++c) t_most = fmaxf(t_most, ts[c]);
            float most[MT];
            bool rises = t_most >= unit_t;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                most[i] = sc[i][0];
#pragma unroll
                for (int c = 1; c < kScores; ++c) most[i] = fmaxf(most[i], sc[i][c]);
                rises = rises || most[i] > m[i];
            }
            // ---- only where some maximum or T has risen are they joined and what has been added up brought in line
            if (__any_sync(0xffffffffu, rises)) {
                t_most = fmaxf(t_most, __shfl_xor_sync(0xffffffffu, t_most, 1));
                t_most = fmaxf(t_most, __shfl_xor_sync(0xffffffffu, t_most, 2));
                float grown = 1.f;
                // (a row that is not put into zeros has a scale of 2^-107 at least; 2^15 / T is a number down to T = 2^-112)
                if (t_most >= unit_t && t_most >= 0x1p-112f) {
                    const uint32_t bits = min((__float_as_uint(t_most) & 0x7f800000u) + 0x00800000u, 0x7e800000u);  // (at most 2^126)
                    grown = unit_t * __uint_as_float(0x7f000000u - bits);  // T before / T now
                    unit_t = __uint_as_float(bits);
                    inverse_t = __uint_as_float(0x7f000000u - bits) * 32768.f;
                }
                float shrink[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 1));
                    most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 2));
                    const float now = fmaxf(m[i], most[i]);
                    shrink[i] = now == -INFINITY ? 1.f : ex2_8(m[i] - now);
                    m[i] = now;
                    l[i] *= shrink[i];
                    shrink[i] *= grown;
                }
#pragma unroll
                for (int u = 0; u < kOuts; ++u) {
                    const float a = shrink[F32 ? u : 2 * u], b = F32 ? a : 2 * u + 1 < MT ? shrink[2 * u + 1 < MT ? 2 * u + 1 : 0] : 1.f;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        o[u][c][0] *= a;
                        o[u][c][1] *= a;
                        o[u][c][2] *= b;
                        o[u][c][3] *= b;
                    }
                }
            }
            // ---- weights, then times the values' scales
#pragma unroll
            for (int c = 0; c < kScores; ++c) ts[c] *= inverse_t;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
                for (int c = 0; c < kScores; ++c) {
                    sc[i][c] = ex2_8(sc[i][c] - base);
                    l[i] += sc[i][c];
                }
                if (looks) {
#pragma unroll
                    for (int c = 0; c < kScores; ++c) sc[i][c] = sc[i][c] == 0.f ? 0.f : sc[i][c] * ts[c];
                } else {
#pragma unroll
                    for (int c = 0; c < kScores; ++c) sc[i][c] *= ts[c];
                }
            }
            // ---- outputs
#pragma unroll
            for (int s = 0; s < kScores / 4; ++s) {
                uint32_t a[kOuts][4];
#pragma unroll
                for (int u = 0; u < kOuts; ++u)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // positions 4 t + 2 half, + 1
                        const int c = 4 * s + 2 * half;
                        if constexpr (F32) {
                            const uint32_t h = half2_bits(sc[u][c], sc[u][c + 1]);
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                            a[u][2 * half] = h;
                            a[u][2 * half + 1] = half2_bits(sc[u][c] - f.x, sc[u][c + 1] - f.y);
                        } else {
                            a[u][2 * half] = half2_bits(sc[2 * u][c], sc[2 * u][c + 1]);
                            a[u][2 * half + 1] = 2 * u + 1 < MT ? half2_bits(sc[2 * u + 1 < MT ? 2 * u + 1 : 0][c], sc[2 * u + 1 < MT ? 2 * u + 1 : 0][c + 1]) : 0u;
                        }
                    }
                uint32_t vw[4][kValueWords];
#pragma unroll
                for (int r = 0; r < 4; ++r) load_words<kValueWords>(vw[r], at + kPiece8 * D + (16 * s + 4 * t + r) * D + g * (D / 8));
#pragma unroll
                for (int w = 0; w < kValueWords; ++w) {
                    uint32_t c0 = vw[0][w] ^ 0x80808080u, c1 = vw[1][w] ^ 0x80808080u, c2 = vw[2][w] ^ 0x80808080u, c3 = vw[3][w] ^ 0x80808080u;
                    const uint32_t ab0 = __byte_perm(c0, c1, 0x5140), ab1 = __byte_perm(c0, c1, 0x7362);
                    const uint32_t cd0 = __byte_perm(c2, c3, 0x5140), cd1 = __byte_perm(c2, c3, 0x7362);
                    const uint32_t b0[4] = {code_halves(ab0, 0x4140), code_halves(ab0, 0x4342), code_halves(ab1, 0x4140), code_halves(ab1, 0x4342)};
                    const uint32_t b1[4] = {code_halves(cd0, 0x4140), code_halves(cd0, 0x4342), code_halves(cd1, 0x4140), code_halves(cd1, 0x4342)};
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int u = 0; u < kOuts; ++u) mma_f16(o[u][4 * w + c], a[u], b0[c], b1[c]);
                }
            }
            __syncwarp();  // every lane is done with the stage
#pragma unroll
            for (int s = 0; s + 1 < kStages; ++s) queue[s] = queue[s + 1];
            queue[kStages - 1] = copy(stage);
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }

        // ---- rows that float16 has lost (below), a bit for each of a row's four lanes
        uint32_t lost[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float largest = 0.f;
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) largest = fmaxf(largest, fabsf(F32 ? o[i][c][half] : o[i / 2][c][2 * (i & 1) + half]));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            lost[i] = __ballot_sync(0xffffffffu, pos_of[i] >= 0 && l[i] > 0.f && unit_t > 0.f && largest < lost8(F32));
        }
        // `with`: what becomes of a lost row, given its place in the tile, maximum, sum of weights and sums
        auto again = [&](float* query, float* sums, auto with) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < MT; ++i)
                while (lost[i]) {
                    const int row = (__ffs(lost[i]) - 1) / 4, e = e0 + 8 * i + row;
                    lost[i] &= ~(15u << (4 * row));
                    const T* q = reinterpret_cast<const T*>(p.q) + (size_t)(r0 + e / per) * p.q_stride + (size_t)(hk * per + e % per) * D;
                    const int pos = __shfl_sync(0xffffffffu, pos_of[i], 4 * row), from = __shfl_sync(0xffffffffu, low_of[i], 4 * row);
                    const int mine_first = SOLO ? first : first + rank * kWarps8 + warp;
                    float* to = sums + (SOLO ? 0 : (8 * i + row) * D);
                    float2 ml;
                    if constexpr (MT == 1) ml = attend_alone8<D, T>(p, table, hk, q, from, pos, mine_first, last, step, query, to);
                    else ml = attend_alone_call8<D, T>(p, table, hk, q, from, pos, mine_first, last, step, query, to);
                    with(8 * i + row, ml);
                }
            __syncwarp();
        };
        if constexpr (SOLO) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const bool sees = pos_of[i] >= 0;
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
                const float inv = sees && l[i] != 0.f ? 1.f / l[i] : 0.f, back = unit_t * (1.f / 32768.f);
                const int e = e0 + 8 * i + g;
                if (e >= entries) continue;
                T* row = reinterpret_cast<T*>(p.out) + ((size_t)(r0 + e / per) * p.nq + hk * per + e % per) * D + t * (D / 4);
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int c = 0; c < kCols; c += 4) {
                        float y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (F32) y[j] = o[i][c + j][half] + o[i][c + j][2 + half];
                            else y[j] = o[i / 2][c + j][2 * (i & 1) + half];
                            y[j] = sees ? y[j] * inv * back : 0.f;
                        }
                        store4(row + half * (D / 8) + c, make_float4(y[0], y[1], y[2], y[3]));
                    }
            }
            float* kept = reinterpret_cast<float*>(ring);
            again(kept, kept + D, [&](int row, float2 ml) {
                const int e = e0 + row;
                T* out = reinterpret_cast<T*>(p.out) + ((size_t)(r0 + e / per) * p.nq + hk * per + e % per) * D;
                for (int d = lane; d < D; d += 32) out[d] = from_float<T>(ml.y == 0.f ? 0.f : kept[D + d] / ml.y);
                fence_async_shared8();
                __syncwarp();
            });
            continue;
        }
        // ---- the four warps' parts are joined: [queries][D] sums, then maxima and sums of weights, in the warp's own ring
        float* sums = reinterpret_cast<float*>(ring);
        float* stats = sums + kTile * D;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const bool sees = pos_of[i] >= 0;  // (a padding row among others sees nothing, whatever its lanes have added up)
            const float back = unit_t * (1.f / 32768.f);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) {
                stats[2 * (8 * i + g)] = sees ? m[i] : -INFINITY;
                stats[2 * (8 * i + g) + 1] = sees ? l[i] : 0.f;
            }
            float* row = sums + (8 * i + g) * D + t * (D / 4);  // columns 2 t and 2 t + 1 of every product: D / 4 values in a run
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                if constexpr (F32) {
                    row[c] = sees ? (o[i][c][0] + o[i][c][2]) * back : 0.f;
                    row[D / 8 + c] = sees ? (o[i][c][1] + o[i][c][3]) * back : 0.f;
                } else {
                    row[c] = sees ? o[i / 2][c][2 * (i & 1)] * back : 0.f;
                    row[D / 8 + c] = sees ? o[i / 2][c][2 * (i & 1) + 1] * back : 0.f;
                }
            }
        }
        again(stats + 2 * kTile, sums, [&](int row, float2 ml) {
            if (lane == 0) {
                stats[2 * row] = ml.x;
                stats[2 * row + 1] = ml.y;
            }
        });
        __syncthreads();
        const int count = min(kTile, entries - e0);
        auto warp_part = [&](int w) { return reinterpret_cast<const float*>(smem + (size_t)w * kStages * kStage); };
        float* together = reinterpret_cast<float*>(smem) + kTile * (D + 2);  // (behind the first warp's part)
        auto place_of = [&](int e) { return (size_t)(r0 + (e0 + e) / per) * p.nq + hk * per + (e0 + e) % per; };
        auto write = [&](int e, int d, const float4& sum, float total) {
            const float inv = total == 0.f ? 0.f : 1.f / total;
            store4(reinterpret_cast<T*>(p.out) + place_of(e) * D + d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
        };
        auto put = [&](int e, int d, const float4& sum, float most, float total) {  // the slice's sums: the output, or a record of them
            if (slices == 1) {
                write(e, d, sum, total);
                return;
            }
            float* rec = p.partial + (place_of(e) * p.splits + slice) * (D + 4);
            __stcg(reinterpret_cast<float4*>(rec + 4 + d), sum);
            if (d == 0) __stcg(reinterpret_cast<float2*>(rec), make_float2(most, total));
        };
        for (int at = threadIdx.x; at < count * (D / 4); at += kWarps8 * 32) {
            const int e = at / (D / 4), d = at % (D / 4) * 4;
            float most = -INFINITY, total = 0.f;
            float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps8; ++w) most = fmaxf(most, warp_part(w)[kTile * D + 2 * e]);
            const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
            for (int w = 0; w < kWarps8; ++w) {
                const float* part = warp_part(w);
                add_part(sum, total, *reinterpret_cast<const float4*>(part + e * D + d), part[kTile * D + 2 * e + 1],
                         ex2_8(part[kTile * D + 2 * e] - base));
            }
            if (p.cluster > 1) {
                *reinterpret_cast<float4*>(together + e * D + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(together + kTile * D + 2 * e) = make_float2(most, total);
            } else {
                put(e, d, sum, most, total);
            }
        }
        if (p.cluster > 1) {
            // ---- the cluster's CTAs share out the outputs and read each other's sums
            cluster_sync8();
            for (int at = rank * kWarps8 * 32 + threadIdx.x; at < count * (D / 4); at += p.cluster * kWarps8 * 32) {
                const int e = at / (D / 4), d = at % (D / 4) * 4;
                float2 ml[kMostCluster8];
                float4 v[kMostCluster8];
                float most = -INFINITY, total = 0.f;
                float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < kMostCluster8; ++c)
                    if (c < p.cluster) {
                        ml[c] = peer_load2(together + kTile * D + 2 * e, c);
                        v[c] = peer_load4(together + e * D + d, c);
                        most = fmaxf(most, ml[c].x);
                    }
                const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
                for (int c = 0; c < kMostCluster8; ++c)
                    if (c < p.cluster) add_part(sum, total, v[c], ml[c].y, ex2_8(ml[c].x - base));
                put(e, d, sum, most, total);
            }
        }
        if (slices > 1) {
            // ---- the slice that ends last joins the others' records, in their order (a fence of every thread: one thread's release for
            // all of them took 3 us longer)
            __threadfence();
            __syncthreads();
        }
        if (p.cluster > 1) cluster_sync8();  // every record of the slice is out, and nobody reads this CTA's sums any more
        if (slices > 1 && rank == 0) {
            if (threadIdx.x == 0) {
                unsigned* ticket = p.tickets + ((size_t)r0 * p.nkv + hk) * p.tiles + tile;
                unsigned old;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(ticket) : "memory");
                joins = old == (unsigned)slices - 1u;
                if (joins) *ticket = 0u;
            }
            __syncthreads();
            if (joins) {
                for (int at = threadIdx.x; at < count * (D / 4); at += kWarps8 * 32) {
                    const int e = at / (D / 4), d = at % (D / 4) * 4;
                    const float* rec = p.partial + place_of(e) * p.splits * (D + 4);
                    float most = -INFINITY, total = 0.f;
                    float4 sum = {0.f, 0.f, 0.f, 0.f};
                    constexpr int kAhead = 8;  // records asked for at once
                    for (int s0 = 0; s0 < slices; s0 += kAhead) {
                        float2 ml[kAhead];
                        float4 v[kAhead];
                        float now = most;
#pragma unroll
                        for (int s = 0; s < kAhead; ++s) {
                            ml[s] = make_float2(-INFINITY, 0.f);
                            v[s] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (s0 + s < slices) {
                                ml[s] = __ldcg(reinterpret_cast<const float2*>(rec + (size_t)(s0 + s) * (D + 4)));
                                v[s] = __ldcg(reinterpret_cast<const float4*>(rec + (size_t)(s0 + s) * (D + 4) + 4 + d));
                            }
                        }
#pragma unroll
                        for (int s = 0; s < kAhead; ++s) now = fmaxf(now, ml[s].x);
                        const float base = now == -INFINITY ? 0.f : now, before = ex2_8(most - base);
                        total *= before;
                        sum = make_float4(sum.x * before, sum.y * before, sum.z * before, sum.w * before);
                        most = now;
#pragma unroll
                        for (int s = 0; s < kAhead; ++s) add_part(sum, total, v[s], ml[s].y, ex2_8(ml[s].x - base));
                    }
                    write(e, d, sum, total);
                }
            }
        }
        fence_async_shared8();
        __syncthreads();  // the rings are read no more
    }
}

template <int D, bool F32, int MT, bool SOLO>
static cudaError_t launch_mma8(const Attend8& p, unsigned units, cudaStream_t stream) {
    constexpr size_t smem = (size_t)kWarps8 * stages8(D) * stage_bytes8(D);
    static_assert(stages8(D) * stage_bytes8(D) >= 2 * 8 * MT * (D + 2) * 4, "a warp's part of the outputs fits its ring, twice in the first");
    static_assert(stages8(D) * stage_bytes8(D) >= 8 * MT * (D + 2) * 4 + D * 4, "and a query behind it");
    auto kernel = attn_int8_mma_kernel<D, F32, MT, SOLO>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    const dim3 grid(SOLO ? (units + kWarps8 - 1) / kWarps8 : units, SOLO ? 1u : (unsigned)(p.splits * p.cluster));
    if (SOLO || p.cluster == 1) return launch_dependent(kernel, grid, kWarps8 * 32, smem, stream, p);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kWarps8 * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)p.cluster;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent_launches() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D>
static cudaError_t launch_mma8_of(const Attend8& p, bool f32, int mt, unsigned units, cudaStream_t stream) {
    if (p.cluster == 0)
        return f32 ? launch_mma8<D, true, 1, true>(p, units, stream) : mt == 1 ? launch_mma8<D, false, 1, true>(p, units, stream)
                                                                            : launch_mma8<D, false, 2, true>(p, units, stream);
    return f32 ? launch_mma8<D, true, 1, false>(p, units, stream) : mt == 1 ? launch_mma8<D, false, 1, false>(p, units, stream)
                                                                         : launch_mma8<D, false, 2, false>(p, units, stream);
}

cudaError_t attend_int8_mma(Attend8 p, bool f32, cudaStream_t stream) {
    const int per = p.nq / p.nkv, entries = p.rows_at_once * per, mt = f32 ? 1 : p.tile_eights;
    p.tiles = (entries + 8 * mt - 1) / (8 * mt);
    const long long units = (long long)((p.n + p.rows_at_once - 1) / p.rows_at_once) * p.nkv * p.tiles;
    if (units > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    p.units = (int)units;
    switch (p.d) {
        case 32: return launch_mma8_of<32>(p, f32, mt, (unsigned)units, stream);
        case 64: return launch_mma8_of<64>(p, f32, mt, (unsigned)units, stream);
        case 96: return launch_mma8_of<96>(p, f32, mt, (unsigned)units, stream);
        default: return launch_mma8_of<128>(p, f32, mt, (unsigned)units, stream);
    }
}

}  // namespace nnis
