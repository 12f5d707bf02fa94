// Attention of single rows, or of a few rows of a sequence, over the paged cache held in 8 bits, on the tensor cores: heads of 32, 64, 96 and
// 128, pages of 64 positions, float32 and bfloat16.
//
// The key's codes are multiplied as they are.  A query's head is put into whole numbers once, N = rint(q * (top' / top)), of two signed
// bytes (bfloat16: N = 256 hi + lo, off by at most top / 65,024 a value) or three (float32: 65,536 hi + 256 mid + lo, off by 2^-24 of
// top); a product of 16 x 8 x 32 whole numbers (mma.sync) holds eight queries' first bytes in its rows 0 to 7 and their second bytes in
// rows 8 to 15, so that a thread gets both sums of a score, exact, and score = (256 hi + lo) * (top / top') * key scale * scale.
// The value's codes become float16 (a byte b of 0 to 255 behind the byte 0x64 is 1,024 + b) for products of 16 x 8 x 16 with the weights
// w_j = 2^15 p_j t_j / T, where t_j is the value's scale and T a power of two above all scales that the warp has met: w_j is below
// 2^15, and float16 holds what is 2^-29 of the largest weight to its full 11 bits.  bfloat16: eight more queries in rows 8 to 15.
// float32: what float16 has left of the weights there, so that a weight has 22 bits.  Maxima, sums and outputs are float32.
//
// Any order of a head's values serves the first product and any order of positions the second, so a thread's part of every fragment lies
// side by side in shared memory as the copies bring it: a thread of the key product holds bytes [t D / 4, (t + 1) D / 4) of a
// position's row, of the value product bytes [g D / 8, (g + 1) D / 8) of positions 4 t to 4 t + 3 (g = lane / 4, t = lane % 4).
//
// A CTA: four warps, (run of rows with one sequence, key/value head, tile of queries, slice of positions); a warp takes every fourth piece
// of 32 positions of the slice through a ring of its own, filled by bulk copies, so that nothing meets before the slice's end.  Slices are of a
// fixed number of pieces, so sequences of all lengths are cut into equal pieces; the slice that ends last joins them.
#include <float.h>
#include <string.h>

#include <cuda_fp16.h>

#include "async_copy.cuh"
#include "int8_rows.cuh"
#include "attention_int8.cuh"

namespace nnis {

constexpr int kPage8 = 64, kPiece8 = 32, kWarps8 = 4;  // positions of a page, and of what a warp takes at a time

__host__ __device__ constexpr int stage_bytes8(int d) { return 2 * kPiece8 * d + 2 * kPiece8 * 4; }

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
    constexpr float kMost = F32 ? 8323072.f : 32512.f;  // 127 * 65,536, 127 * 256
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

template <int D, bool F32, int MT>
__global__ void __launch_bounds__(kWarps8 * 32) attn_int8_mma_kernel(const __grid_constant__ Attend8 p) {
    using T = std::conditional_t<F32, float, bf16>;
    constexpr int kStage = stage_bytes8(D), kTile = 8 * MT, kSteps = D / 32, kWords = D / 16, kValueWords = D / 32, kCols = D / 8;
    constexpr int kOuts = F32 ? MT : (MT + 1) / 2;  // products of the weights per step of 16 positions
    constexpr int kStages = stages8(D), kScores = kPiece8 / 4;  // (a lane's positions of a piece: 16 s + 4 t + 0 to 3)
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[kWarps8][kStages];
    __shared__ int joins, piece_in[kWarps8][kStages];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {  // (a warp's barriers are its own)
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();

    const int per = p.nq / p.nkv, slice = blockIdx.y;
    int unit = blockIdx.x;
    const int tile = unit % p.tiles;
    unit /= p.tiles;
    const int hk = unit % p.nkv, row_first = unit / p.nkv * p.rows_at_once, row_end = min(p.n, row_first + p.rows_at_once);
    unsigned char* ring = smem + (size_t)warp * kStages * kStage;
    int filled = 0, used = 0;  // pieces asked for and met, over all runs

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
        // ---- the run, its keys and this slice's part of them (the same for every thread of the CTA)
        const int seq = p.token_seq[r0];
        int top_pos = -1, low = INT_MAX, low_pos = INT_MAX, top_low = 0;
        for (r1 = r0; r1 < row_end && p.token_seq[r1] == seq; ++r1) {
            const int pos = p.token_pos[r1];
            if (pos < 0) continue;
            const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            top_pos = max(top_pos, pos);
            low_pos = min(low_pos, pos);
            low = min(low, lo);
            top_low = max(top_low, lo);
        }
        const int entries = (r1 - r0) * per;
        if (e0 >= entries) continue;
        const bool known = seq >= 0 && seq < p.table_rows && top_pos >= 0;
        const int* table = p.page_table + (size_t)(known ? seq : 0) * p.table_cols;
        constexpr int kHalves = kPage8 / kPiece8;
        const int piece_low = known ? low / kPiece8 : 0, piece_top = known ? (int)min((long long)top_pos / kPiece8 + 1, (long long)kHalves * p.table_cols) : 0;
        const int slices = max(1, (piece_top - piece_low + p.slice_pieces - 1) / p.slice_pieces);
        if (slice >= slices) continue;
        const int first = piece_low + slice * p.slice_pieces, last = min(piece_top, first + p.slice_pieces);

        // ---- copies: this warp's pieces are first + warp, + 4, ...; those of pages outside the store are passed over
        // (the next piece's page is asked for as a piece is filled, and looked at when its turn comes)
        int next = first + warp, page = next < last ? table[next / kHalves] : -1;
        auto fill = [&]() {
            while (next < last && (unsigned)page >= (unsigned)p.pages) {
                next += kWarps8;
                page = next < last ? table[next / kHalves] : -1;
            }
            if (next >= last) return;
            if (lane < 4) {  // (keys, values and the scales of each: one copy a lane)
                unsigned char* at = ring + (filled % kStages) * kStage;
                uint64_t* bar = &full[warp][filled % kStages];
                const size_t row = ((size_t)page * p.nkv + hk) * kPage8 + next % kHalves * kPiece8;
                if (lane == 0) {
                    mbar_expect_tx(bar, kStage);
                    piece_in[warp][filled % kStages] = next;
                }
                const void* from = lane < 2 ? (const void*)((lane == 0 ? p.k : p.v) + row * D) : (const void*)((lane == 2 ? p.k_scales : p.v_scales) + row);
                bulk_load(at + (lane < 2 ? lane * kPiece8 * D : 2 * kPiece8 * D + (lane - 2) * kPiece8 * 4), from,
                          lane < 2 ? kPiece8 * D : kPiece8 * 4, bar);
            }
            ++filled;
            next += kWarps8;
            page = next < last ? table[next / kHalves] : -1;
        };
#pragma unroll 1
        for (int s = 0; s < kStages; ++s) fill();
        __syncwarp();

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
        while (used < filled) {
            const int piece = piece_in[warp][used % kStages];
            const unsigned char* at = ring + (used % kStages) * kStage;
            if (!mbar_wait(&full[warp][used % kStages], (uint32_t)(used / kStages) & 1u)) {
                if (lane == 0) atomicExch(p.status, 1);
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
                int acc[MT][2][4] = {}, acl[F32 ? MT : 1][2][4] = {};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t w[kWords];
                    load_words<kWords>(w, at + (16 * s + 4 * (g >> 1) + 2 * j + (g & 1)) * D + t * (D / 4));
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            mma_s8(acc[i][j], qa[i][k], w[2 * k], w[2 * k + 1]);
                            if constexpr (F32) {
                                const uint32_t a[4] = {ql[i][k][0], 0u, ql[i][k][1], 0u};
                                mma_s8(acl[i][j], a, w[2 * k], w[2 * k + 1]);
                            }
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
            if (!whole) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int c = 0; c < kScores; ++c) {
                        const int key = key0 + 16 * (c >> 2) + (c & 3);
                        if (key > pos_of[i] || key < low_of[i]) sc[i][c] = -INFINITY;
                    }
            }
            // ---- T grows to a power of two above the scales of the positions that anyone sees
            float ts[kScores], t_most = 0.f;
#pragma unroll
            for (int s = 0; s < kScores / 4; ++s) {
                const float4 scales = *reinterpret_cast<const float4*>(vs + 16 * s + 4 * t);
                ts[4 * s] = scales.x; ts[4 * s + 1] = scales.y; ts[4 * s + 2] = scales.z; ts[4 * s + 3] = scales.w;
            }
#pragma unroll
            for (int c = 0; c < kScores; ++c) {
                const int key = key0 + 16 * (c >> 2) + (c & 3);
                if (whole || (key >= low && key <= top_pos)) t_most = fmaxf(t_most, ts[c]);
            }
            t_most = fmaxf(t_most, __shfl_xor_sync(0xffffffffu, t_most, 1));
            t_most = fmaxf(t_most, __shfl_xor_sync(0xffffffffu, t_most, 2));
            float grown = 1.f;
            if (t_most >= unit_t && t_most >= 0x1p-100f) {
                const uint32_t bits = min((__float_as_uint(t_most) & 0x7f800000u) + 0x00800000u, 0x7e800000u);  // (at most 2^126)
                grown = unit_t * __uint_as_float(0x7f000000u - bits);  // T before / T now
                unit_t = __uint_as_float(bits);
                inverse_t = __uint_as_float(0x7f000000u - bits) * 32768.f;
            }
            // ---- weights
            float shrink[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float most = sc[i][0];
#pragma unroll
                for (int c = 1; c < kScores; ++c) most = fmaxf(most, sc[i][c]);
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float now = fmaxf(m[i], most), base = now == -INFINITY ? 0.f : now;
                shrink[i] = ex2_8(m[i] - base);
                m[i] = now;
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < kScores; ++c) {
                    sc[i][c] = ex2_8(sc[i][c] - base);
                    sum += sc[i][c];
                }
                l[i] = l[i] * shrink[i] + sum;
                shrink[i] *= grown;
            }
            bool same = true;
#pragma unroll
            for (int i = 0; i < MT; ++i) same = same && shrink[i] == 1.f;
            if (!__all_sync(0xffffffffu, same)) {
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
            // ---- outputs
#pragma unroll
            for (int s = 0; s < kScores / 4; ++s) {
                uint32_t a[kOuts][4];
#pragma unroll
                for (int u = 0; u < kOuts; ++u)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // positions 4 t + 2 half, + 1
                        const int c = 4 * s + 2 * half;
                        float w[2][2];
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int mt = F32 ? u : 2 * u + i < MT ? 2 * u + i : 0;
                                const float weight = sc[mt][c + e];
                                // (a scale that is no number, where nobody looks, must not meet a weight of zero)
                                w[i][e] = whole || weight != 0.f ? weight * (ts[c + e] * inverse_t) : 0.f;
                            }
                        if constexpr (F32) {
                            const uint32_t h = half2_bits(w[0][0], w[0][1]);
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                            a[u][2 * half] = h;
                            a[u][2 * half + 1] = half2_bits(w[0][0] - f.x, w[0][1] - f.y);
                        } else {
                            a[u][2 * half] = half2_bits(w[0][0], w[0][1]);
                            a[u][2 * half + 1] = 2 * u + 1 < MT ? half2_bits(w[1][0], w[1][1]) : 0u;
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
            ++used;
            __syncwarp();  // every lane is done with the stage
            fill();
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
        __syncthreads();
        const int count = min(kTile, entries - e0);
        auto warp_part = [&](int w) { return reinterpret_cast<const float*>(smem + (size_t)w * kStages * kStage); };
        for (int at = threadIdx.x; at < count * (D / 4); at += kWarps8 * 32) {
            const int e = at / (D / 4), d = at % (D / 4) * 4;
            const int row = r0 + (e0 + e) / per, head = hk * per + (e0 + e) % per;
            float most = -INFINITY, total = 0.f;
            float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps8; ++w) most = fmaxf(most, warp_part(w)[kTile * D + 2 * e]);
            const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
            for (int w = 0; w < kWarps8; ++w) {
                const float* part = warp_part(w);
                const float share = ex2_8(part[kTile * D + 2 * e] - base);
                const float4 v = *reinterpret_cast<const float4*>(part + e * D + d);
                total = fmaf(share, part[kTile * D + 2 * e + 1], total);
                sum.x = fmaf(share, v.x, sum.x);
                sum.y = fmaf(share, v.y, sum.y);
                sum.z = fmaf(share, v.z, sum.z);
                sum.w = fmaf(share, v.w, sum.w);
            }
            const size_t place = (size_t)row * p.nq + head;
            if (slices == 1) {
                const float inv = total == 0.f ? 0.f : 1.f / total;
                store4(reinterpret_cast<T*>(p.out) + place * D + d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
            } else {
                float* rec = p.partial + (place * p.splits + slice) * (D + 4);
                __stcg(reinterpret_cast<float4*>(rec + 4 + d), sum);
                if (d == 0) __stcg(reinterpret_cast<float2*>(rec), make_float2(most, total));
            }
        }
        if (slices > 1) {
            // ---- the slice that ends last joins the others' records, in their order
            __threadfence();
            __syncthreads();
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
                    const size_t place = (size_t)(r0 + (e0 + e) / per) * p.nq + hk * per + (e0 + e) % per;
                    const float* rec = p.partial + place * p.splits * (D + 4);
                    float most = -INFINITY, total = 0.f;
                    float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
                    for (int s = 0; s < slices; ++s) most = fmaxf(most, __ldcg(rec + (size_t)s * (D + 4)));
                    const float base = most == -INFINITY ? 0.f : most;
#pragma unroll 8
                    for (int s = 0; s < slices; ++s) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(rec + (size_t)s * (D + 4)));
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(rec + (size_t)s * (D + 4) + 4 + d));
                        const float share = ex2_8(ml.x - base);
                        total = fmaf(share, ml.y, total);
                        sum.x = fmaf(share, v.x, sum.x);
                        sum.y = fmaf(share, v.y, sum.y);
                        sum.z = fmaf(share, v.z, sum.z);
                        sum.w = fmaf(share, v.w, sum.w);
                    }
                    const float inv = total == 0.f ? 0.f : 1.f / total;
                    store4(reinterpret_cast<T*>(p.out) + place * D + d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
                }
            }
        }
        fence_async_shared8();
        __syncthreads();  // the rings are read no more
    }
}

template <int D, bool F32, int MT>
static cudaError_t launch_mma8(const Attend8& p, unsigned units, cudaStream_t stream) {
    constexpr size_t smem = (size_t)kWarps8 * stages8(D) * stage_bytes8(D);
    static_assert(stages8(D) * stage_bytes8(D) >= 8 * MT * (D + 2) * 4, "a warp's part of the outputs fits its ring");
    auto kernel = attn_int8_mma_kernel<D, F32, MT>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(units, (unsigned)p.splits), kWarps8 * 32, smem, stream, p);
}

template <int D>
static cudaError_t launch_mma8_of(const Attend8& p, bool f32, int mt, unsigned units, cudaStream_t stream) {
    if (f32) return launch_mma8<D, true, 1>(p, units, stream);
    return mt == 1 ? launch_mma8<D, false, 1>(p, units, stream) : launch_mma8<D, false, 2>(p, units, stream);
}

cudaError_t attend_int8_mma(Attend8 p, bool f32, cudaStream_t stream) {
    const int per = p.nq / p.nkv, entries = p.rows_at_once * per, mt = f32 || entries <= 8 ? 1 : 2;
    p.tiles = (entries + 8 * mt - 1) / (8 * mt);
    const long long units = (long long)((p.n + p.rows_at_once - 1) / p.rows_at_once) * p.nkv * p.tiles;
    if (units > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    switch (p.d) {
        case 32: return launch_mma8_of<32>(p, f32, mt, (unsigned)units, stream);
        case 64: return launch_mma8_of<64>(p, f32, mt, (unsigned)units, stream);
        case 96: return launch_mma8_of<96>(p, f32, mt, (unsigned)units, stream);
        default: return launch_mma8_of<128>(p, f32, mt, (unsigned)units, stream);
    }
}

}  // namespace nnis
