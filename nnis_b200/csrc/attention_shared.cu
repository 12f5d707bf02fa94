// Attention of token rows that share pages of the cache, any even head size up to 256, float32 or bfloat16, on the CUDA
// cores; and the merge that all forms end with.  See attention_shared.cuh for units and records.
//
// A CTA owns a unit and a kv head: a tile of 16 or 64 entries (token row, query head) over the unit's pages.  A page of K
// comes into shared memory as float32, scores of tile x 64 keys are sums in registers (a thread: 1 or 4 entries x 4 keys),
// the softmax's running maximum and sum are a half-warp's shuffles, the weights go to shared memory and the outputs, a
// thread's 1 or 4 entries x d / 16 values, are added up in registers while the page's V replaces its K.  It is the form that is
// right for every size, not a fast one: its loads wait for its products.
#include <string.h>

#include "attention_shared.cuh"

namespace nnis {

constexpr int kAnyThreads = 256;

__device__ __forceinline__ int row_stride_any(int d) { return ((d + 3) & ~3) + 4; }

// ROWS: entries a thread (tile = 16 ROWS); NJ: runs of 16 output values
template <typename T, int ROWS, int NJ>
__global__ void __launch_bounds__(kAnyThreads)
attn_shared_any_kernel(const SharedArgs a) {
    constexpr int kTile = 16 * ROWS;
    extern __shared__ __align__(16) float smem_any[];
    const int d = a.d, ds = row_stride_any(d);
    float* q_s = smem_any;                      // [tile, ds], scaled
    float* kv_s = q_s + kTile * ds;             // [64, ds]: a page's K, then its V
    float* p_s = kv_s + kSharedPage * ds;       // [tile, 68]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const SharedUnit u = a.units[blockIdx.x];
    units_begin(a);
    const int hk = blockIdx.y, G = a.nq / a.nkv;
    const int* members = a.members + u.members;
    const int pos = u.ends ? a.token_pos[u.ends - 1] : 0x7fffffff;
    const int n_pages = min(a.table_cols, u.ends ? min(u.page_end, pos < 0 ? 0 : pos / kSharedPage + 1) : u.page_end);
    const int* table = a.page_table + (size_t)u.seq * a.table_cols;
    if (tid == 0) units_end_check(a, u, pos);
    const T* q = static_cast<const T*>(a.q);

    for (int i = tid; i < kTile * ds; i += kAnyThreads) {
        const int e = i / ds, c = i % ds;
        float x = 0.f;
        if (e < u.entries && c < d) {
            const int at = u.entry + e;
            x = to_float(q[(size_t)members[at / G] * a.q_stride + (size_t)(hk * G + at % G) * d + c]) * (a.scale * 1.4426950408889634f);
        }
        q_s[i] = x;
    }
    float o[ROWS][NJ], m_run[ROWS], l_run[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[r][j] = 0.f;
    }
    auto load = [&](const void* cache, int page, int keys) {  // rows from `keys` on are zero: what lies there may be anything
        const T* src = static_cast<const T*>(cache) + ((size_t)page * a.nkv + hk) * kSharedPage * d;
        const int half = d / 2, hs = ds / 2;
        for (int i = tid; i < kSharedPage * hs; i += kAnyThreads) {
            const int row = i / hs, c = i % hs;
            float2 x = make_float2(0.f, 0.f);
            if (row < keys && c < half) x = load2(src + (size_t)row * d + 2 * c);
            *reinterpret_cast<float2*>(kv_s + (size_t)row * ds + 2 * c) = x;
        }
    };
    for (int it = u.page_begin; it < n_pages; ++it) {
        const int page = table[it];
        if (page < 0 || page >= a.pages) continue;  // (the table's gaps hold no keys)
        const int keys = min(kSharedPage, u.ends ? pos + 1 - it * kSharedPage : kSharedPage);
        __syncthreads();
        load(a.k_cache, page, keys);
        __syncthreads();
        float s[ROWS][4];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i] = 0.f;
        for (int c = 0; c < d; c += 4) {
            float4 kk[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) kk[i] = *reinterpret_cast<const float4*>(kv_s + (size_t)(tx + 16 * i) * ds + c);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float4 qq = *reinterpret_cast<const float4*>(q_s + (size_t)(ty * ROWS + r) * ds + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[r][i] = fmaf(qq.x, kk[i].x, s[r][i]);
                    s[r][i] = fmaf(qq.y, kk[i].y, s[r][i]);
                    s[r][i] = fmaf(qq.z, kk[i].z, s[r][i]);
                    s[r][i] = fmaf(qq.w, kk[i].w, s[r][i]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (tx + 16 * i >= keys) s[r][i] = -INFINITY;
                mx = fmaxf(mx, s[r][i]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float m_new = fmaxf(m_run[r], mx), base = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = sh_ex2(m_run[r] - base);
            m_run[r] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = sh_ex2(s[r][i] - base);
                sum += p;
                p_s[(ty * ROWS + r) * 68 + tx + 16 * i] = p;
            }
            l_run[r] = l_run[r] * alpha + half_warp_sum(sum);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[r][j] *= alpha;
        }
        __syncthreads();
        load(a.v_cache, page, keys);
        __syncthreads();
#pragma unroll 4
        for (int t = 0; t < kSharedPage; ++t) {
            float p[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) p[r] = p_s[(ty * ROWS + r) * 68 + t];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const float v = kv_s[(size_t)t * ds + min(tx + 16 * j, ds - 1)];
#pragma unroll
                for (int r = 0; r < ROWS; ++r) o[r][j] = fmaf(p[r], v, o[r][j]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int e = ty * ROWS + r;
        if (e >= u.entries) continue;
        const int at = u.entry + e, row = members[at / G];
        const size_t rec = (size_t)(a.record[row] + u.slot) * a.nq + hk * G + at % G;
        if (tx == 0) reinterpret_cast<float2*>(a.sums)[rec] = make_float2(m_run[r], l_run[r]);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (tx + 16 * j < d) a.partial[rec * d + tx + 16 * j] = o[r][j];
    }
    if (a.tickets) merge_finished<T, kAnyThreads>(a, u, hk, G, reinterpret_cast<int4*>(p_s));
    units_end(a);
}

// A warp per (token row, head), AHEAD of its records asked for at once.
template <typename T, int AHEAD>
__global__ void __launch_bounds__(128)
attn_shared_merge_kernel(const float* __restrict__ partial, const float2* __restrict__ sums, const int* __restrict__ record,
                         T* __restrict__ out, int n_tokens, int nq, int d) {
    const size_t at = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (at >= (size_t)n_tokens * nq) return;
    const int row = (int)(at / nq), first = record[row];
    const int count = record[row + 1] - first;
    pdl_wait();
    pdl_launch_dependents();
    merge_row<T, AHEAD>(partial, sums, first, count, row, (int)(at % nq), nq, d, out);
}

// 32 records ahead where two CTAs an SM are all there are (8 rows of 9 heads 3.5 -> 3.1 us), 16 where registers decide how many run
// at once (51 rows of 32 heads 3.7 us, with 32 ahead 4.2; 80 rows of 32 heads of 128 5.4 and 9.4).
template <typename T>
static cudaError_t launch_merge(const SharedArgs& a, unsigned ctas, int n_tokens, cudaStream_t stream) {
    static const unsigned sms = (unsigned)device_sms();
    auto kernel = ctas <= 2 * sms ? attn_shared_merge_kernel<T, 32> : attn_shared_merge_kernel<T, 16>;
    return launch_dependent(kernel, ctas, 128, 0, stream, (const float*)a.partial, reinterpret_cast<const float2*>(a.sums), a.record,
                            static_cast<T*>(a.out), n_tokens, a.nq, a.d);
}

template <typename T, int ROWS, int NJ>
static cudaError_t launch_any(const SharedArgs& a, int n_units, cudaStream_t stream) {
    const int ds = ((a.d + 3) & ~3) + 4, tile = 16 * ROWS;
    const size_t smem = ((size_t)(tile + kSharedPage) * ds + (size_t)tile * 68) * sizeof(float);
    auto kernel = attn_shared_any_kernel<T, ROWS, NJ>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(n_units, a.nkv), kAnyThreads, smem, stream, a);
}

template <typename T, int ROWS>
static cudaError_t launch_any_size(const SharedArgs& a, int n_units, cudaStream_t stream) {
    return a.d <= 64 ? launch_any<T, ROWS, 4>(a, n_units, stream) : a.d <= 128 ? launch_any<T, ROWS, 8>(a, n_units, stream)
                                                                  : launch_any<T, ROWS, 16>(a, n_units, stream);
}

cudaError_t shared_units_any(const SharedArgs& a, int n_units, int tile, bool f32, cudaStream_t stream) {
    if (f32) return tile == 16 ? launch_any_size<float, 1>(a, n_units, stream) : launch_any_size<float, 4>(a, n_units, stream);
    return tile == 16 ? launch_any_size<bf16, 1>(a, n_units, stream) : launch_any_size<bf16, 4>(a, n_units, stream);
}

}  // namespace nnis

// units: n[0] units of the first kind, n[1] of the second, n[2] of the third.  `form` 0 (any even head size, float32 or
// bfloat16) and 2 (float32, heads of 64 and 128): at most 16, at most 64 entries, none; `form` 1 (bfloat16, heads of 64 and 128): at most 16, 32 and 128, the last
// of which cover only positions that all their rows see.  The plan (units, members, record) is the host's, made of
// page lists that the call's page table agrees with; a page id outside the store holds no keys (zeros in units of the third kind of
// form 1).  partial: records x nq x d floats,
// sums: records x nq x 2.  tickets (n_tokens x nq counters, zero, left zero): every row is merged by the CTA that completes it, and no
// merge is launched (where all units are of the second kind, or `form` is not 1); every row then has a record.
struct SharedCall {
    const void* q;
    int q_stride;
    const void *k_cache, *v_cache;
    const int *token_pos, *page_table;
    int table_cols;
    const int* units;
    int n0, n1, n2;
    const int *members, *record;
    float *partial, *sums;
    unsigned* tickets;
    void* out;
    int n_tokens, nq, nkv, d, pages, page_size;
    float scale;
    int dtype, form;
    int* status;
    cudaStream_t stream;
};
NNIS_API int nnis_attention_shared(const void* call) {
    using namespace nnis;
    SharedCall c;
    memcpy(&c, call, sizeof c);
    const auto [q, q_stride, k_cache, v_cache, token_pos, page_table, table_cols, units, n0, n1, n2, members, record, partial, sums,
                tickets, out, n_tokens, nq, nkv, d, pages, page_size, scale, dtype, form, status, stream] = c;
    if (n_tokens <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || table_cols <= 0 || n0 < 0 || n1 < 0 || n2 < 0 || pages <= 0 || !record ||
        !partial || !sums || !(scale > 0.f) || (n0 + n1 + n2 > 0 && (!units || !members)))
        return NNIS_ERR_ARGUMENT;
    if (page_size != kSharedPage || d < 2 || d > 256 || d % 2 || nkv > 65535) return NNIS_ERR_UNSUPPORTED;
    const bool f32 = dtype == NNIS_DTYPE_F32;
    if (form == 1 && (f32 || (d != 64 && d != 128))) return NNIS_ERR_UNSUPPORTED;
    if (form == 2 && (!f32 || (d != 64 && d != 128))) return NNIS_ERR_UNSUPPORTED;
    if (form < 0 || form > 2) return NNIS_ERR_ARGUMENT;
    if ((n2 && form != 1) || (tickets && (n2 || (n0 && form == 1)))) return NNIS_ERR_UNSUPPORTED;
    if ((uintptr_t)units % 16 || (uintptr_t)partial % 32 || (uintptr_t)sums % 8) return NNIS_ERR_ALIGNMENT;
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache;
    if (all % (form ? 16 : f32 ? 8 : 4) || (uintptr_t)out % (f32 ? 8 : 4) || (form && q_stride % (f32 ? 4 : 8))) return NNIS_ERR_ALIGNMENT;
    SharedArgs a = {q,       k_cache, v_cache, token_pos, page_table, reinterpret_cast<const SharedUnit*>(units), members, record,
                    partial, sums,    tickets, out,       q_stride,   table_cols, pages,   nq,     nkv, d, scale, status, 0};
    // (the large units first: the small ones end what is left of the device)
    const SharedUnit* first = a.units;
    for (int kind = 2; kind >= 0; --kind) {
        const int n = kind == 2 ? n2 : kind == 1 ? n1 : n0;
        if (!n) continue;
        a.units = first + (kind == 2 ? n0 + n1 : kind == 1 ? n0 : 0);
        const cudaError_t e = form == 0   ? shared_units_any(a, n, kind == 1 ? 64 : 16, f32, stream)
                              : form == 2 ? shared_units_f32(a, n, kind == 1 ? 64 : 16, stream)
                              : kind == 2 ? shared_units_tc(a, n, stream)
                                          : kind == 1 ? shared_units_mma(a, n, stream)
                                          : shared_units_warp(a, n, stream);
        if (e != cudaSuccess) return (int)e;
        a.beside = 1;
    }
    if (tickets) return NNIS_OK;
    const unsigned ctas = (unsigned)(((size_t)n_tokens * nq + 3) / 4);
    const cudaError_t e = f32 ? launch_merge<float>(a, ctas, n_tokens, stream) : launch_merge<bf16>(a, ctas, n_tokens, stream);
    return e == cudaSuccess ? NNIS_OK : (int)e;
}
