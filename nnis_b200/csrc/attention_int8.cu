// Attention of single rows over the paged cache held in 8 bits, for any even head size up to 256, in float32 and bfloat16: a warp
// per (row, query head, slice of keys) with an online softmax in float32, as over the 16-bit cache.  With a key's codes c, its scale
// s and the value's codes e, scale t:
//     score_j = scale * s_j * sum_i q_i c_ji,    out = sum_j p_j t_j e_j / sum_j p_j,    p_j = exp(score_j - max).
// A position whose page the table does not name holds no key; a row that sees none, as a padding row at position -1, is zero.
#include <float.h>
#include <string.h>

#include "attention_int8.cuh"
#include "attention_merge.cuh"
#include "int8_rows.cuh"

namespace nnis {

template <typename T, int R>
__global__ void __launch_bounds__(128) attn_int8_warp_kernel(const __grid_constant__ Attend8 p) {
    extern __shared__ float q_smem[];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = blockIdx.x * 4 + warp, hq = blockIdx.y, split = blockIdx.z, d = p.d;
    if (n >= p.n) return;
    const int hk = hq / (p.nq / p.nkv), pos = p.token_pos[n], seq = p.token_seq[n];
    float* qs = q_smem + warp * d;
    float m = -FLT_MAX, l = 0.f, acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.f;
    if (pos >= 0 && seq >= 0 && seq < p.table_rows) {
        const T* qrow = reinterpret_cast<const T*>(p.q) + (size_t)n * p.q_stride + (size_t)hq * d;
        for (int i = lane; i < d; i += 32) qs[i] = to_float(qrow[i]);
        __syncwarp();
        const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const int hi = (int)min((long long)pos + 1, (long long)p.table_cols * p.page_size);
        const int per = (((hi - lo + p.splits - 1) / p.splits) + 31) & ~31;
        const int start = (int)min((long long)lo + (long long)split * per, (long long)hi), end = min(hi, start + per);
        const int* table = p.page_table + (size_t)seq * p.table_cols;
        for (int c = start; c < end; c += 32) {
            const int t = c + lane;
            const int page = t < end ? table[t / p.page_size] : -1;
            const bool valid = page >= 0 && page < p.pages;
            if (!__any_sync(0xffffffffu, valid)) continue;
            const long long row = valid ? ((long long)page * p.nkv + hk) * p.page_size + t % p.page_size : 0;
            float s = -FLT_MAX, tv = 0.f;
            if (valid) {
                const int8_t* krow = p.k + row * d;
                float dot = 0.f;
                if (d % 4 == 0)
                    for (int i = 0; i < d; i += 4) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(krow + i);
                        dot = fmaf(qs[i], code_value(w, 0), dot);
                        dot = fmaf(qs[i + 1], code_value(w, 1), dot);
                        dot = fmaf(qs[i + 2], code_value(w, 2), dot);
                        dot = fmaf(qs[i + 3], code_value(w, 3), dot);
                    }
                else
                    for (int i = 0; i < d; ++i) dot = fmaf(qs[i], (float)krow[i], dot);
                s = dot * p.k_scales[row] * p.scale;
                tv = p.v_scales[row];
            }
            // (a NaN score is not lost in the maximum: it comes back with the weight)
            const float m_new = fmaxf(m, warp_max(s));
            const float w = valid ? expf(s - m_new) : 0.f;
            const float alpha = l == 0.f ? 0.f : expf(m - m_new);
            l = l * alpha + warp_sum(w);
            m = m_new;
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] *= alpha;
            const float weight = valid ? w * tv : 0.f;
            const int count = min(32, end - c);
            for (int j = 0; j < count; ++j) {
                const float wj = __shfl_sync(0xffffffffu, weight, j);
                const long long rj = __shfl_sync(0xffffffffu, row, j);
                if (!__shfl_sync(0xffffffffu, valid, j)) continue;
                const int8_t* vrow = p.v + rj * d;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int i = lane + 32 * r;
                    if (i < d) acc[r] = fmaf(wj, (float)vrow[i], acc[r]);
                }
            }
        }
    }
    if (p.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* o = reinterpret_cast<T*>(p.out) + ((size_t)n * p.nq + hq) * d;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = lane + 32 * r;
            if (i < d) o[i] = from_float<T>(acc[r] * inv);
        }
        return;
    }
    float* rec = p.partial + (((size_t)n * p.nq + hq) * p.splits + split) * (size_t)(d + 2);
    if (lane == 0) {
        rec[0] = m;
        rec[1] = l;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = lane + 32 * r;
        if (i < d) rec[2 + i] = acc[r];
    }
}

template <typename T>
static cudaError_t launch_warps8(const Attend8& p, cudaStream_t stream) {
    auto kernel = p.d <= 32 ? attn_int8_warp_kernel<T, 1> : p.d <= 64 ? attn_int8_warp_kernel<T, 2>
                  : p.d <= 128 ? attn_int8_warp_kernel<T, 4> : attn_int8_warp_kernel<T, 8>;
    const dim3 grid((unsigned)((p.n + 3) / 4), (unsigned)p.nq, (unsigned)p.splits);
    const cudaError_t e = launch_dependent(kernel, grid, 128, 4 * (size_t)p.d * sizeof(float), stream, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_merge<T>(p.partial, (T*)p.out, (size_t)p.n * p.nq, p.d, p.splits, nullptr, stream);
}

}  // namespace nnis

// slice_pieces 0: a warp a row, head and slice, `partial` n * nq * splits * (d + 2) floats where splits > 1.  slice_pieces > 0: the tensor
// cores' kernel (heads of 32, 64, 96, 128, pages of 64): rows_at_once rows of a sequence together, slices of that many runs of 64
// positions (32 for heads of 96 and 128), the last with what is left, each shared by a cluster of 1, 2, 4 or 8 CTAs (0: a
// warp takes a unit alone), tiles of 8 or 16 queries; `partial` n * nq *
// splits * (d + 4) floats and n * nkv * (heads of rows_at_once rows / 8, rounded up) tickets where splits > 1.
struct Attend8Call {
    const void *q, *k, *v;
    const float *k_scales, *v_scales;
    const int *token_pos, *token_seq, *page_table;
    void* out;
    float* partial;
    unsigned* tickets;
    int* status;
    int q_stride, table_rows, table_cols, pages, n, nq, nkv, d, page_size, window;
    float scale;
    int splits, slice_pieces, rows_at_once, cluster, tile_eights, dtype;
    cudaStream_t stream;
};
NNIS_API int nnis_attention_int8(const void* call) {
    using namespace nnis;
    Attend8Call c;
    memcpy(&c, call, sizeof c);
    const auto [q, k, v, k_scales, v_scales, token_pos, token_seq, page_table, out, partial, tickets, status, q_stride, table_rows, table_cols, pages, n,
                nq, nkv, d, page_size, window, scale, splits, slice_pieces, rows_at_once, cluster, tile_eights, dtype, stream] = c;
    if (n <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || table_rows <= 0 || table_cols <= 0 || pages <= 0 || page_size <= 0 || window < 0 ||
        splits < 1 || (splits > 1 && !partial) || !q || !k || !v || !k_scales || !v_scales || !token_pos || !token_seq ||
        !page_table || !out)
        return NNIS_ERR_ARGUMENT;
    if (d < 2 || d % 2 || d > 256 || nq > 65535 || splits > 64) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)k | (uintptr_t)v) % 4) return NNIS_ERR_ALIGNMENT;
    const bool aligned = (uintptr_t)q % 16 == 0 && q_stride % 4 == 0;
    const Attend8 p{q, q_stride, (const int8_t*)k, (const int8_t*)v, k_scales, v_scales, token_pos, token_seq, page_table, table_rows,
                    table_cols, pages, out, partial, n, nq, nkv, d, page_size, window, scale, splits, slice_pieces, rows_at_once, 0, aligned,
                    cluster, tile_eights, 0, tickets, status};
    if (slice_pieces > 0) {
        if (page_size != 64 || (d != 32 && d != 64 && d != 96 && d != 128) || (dtype != NNIS_DTYPE_F32 && dtype != NNIS_DTYPE_BF16))
            return NNIS_ERR_UNSUPPORTED;
        if (cluster == 0 ? splits != 1 : cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) return NNIS_ERR_UNSUPPORTED;
        if (rows_at_once < 1 || tile_eights < 1 || tile_eights > 2 || !status || (splits > 1 && !tickets)) return NNIS_ERR_ARGUMENT;
        if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_scales | (uintptr_t)v_scales | (uintptr_t)out | (uintptr_t)partial) % 16)
            return NNIS_ERR_ALIGNMENT;
        return (int)attend_int8_mma(p, dtype == NNIS_DTYPE_F32, stream);
    }
    if (dtype == NNIS_DTYPE_F32) return (int)launch_warps8<float>(p, stream);
    if (dtype == NNIS_DTYPE_BF16) return (int)launch_warps8<bf16>(p, stream);
    return NNIS_ERR_UNSUPPORTED;
}
