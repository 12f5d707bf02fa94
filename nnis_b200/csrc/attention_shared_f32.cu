// Attention over shared pages in float32, heads of 64 or 128, on the CUDA cores.  See attention_shared.cuh for units and records.
//
// A CTA of 256 threads owns a unit of at most 16 or 64 entries and a kv head.  A page of K and one of V come by 16-byte
// asynchronous copies: the next page's K while this one's softmax and outputs are made, its V under the next scores.  A thread
// has 1 or 4 entries x 4 keys of the scores (sums over four values of d at a time) and 1 or 4 entries x 4 (8) neighbouring
// values of the outputs (sums over four keys at a time), so a product of four by four takes eight loads of 16 bytes.  Rows
// beyond the last visible key are filled with zeros instead of read.  With 64 entries bound by the multiply-adds (1 us each of
// scores and outputs a page and SM at heads of 64), with 16 by shared memory; both products are true float32.  16 rows of 9 heads
// over 3 behind 2,000 tokens: 10.8 us the units of 64, 6.9 those of 16 beside them (the form for any head size: 19 and 16).
#include "attention_shared.cuh"
#include "fma_pairs.cuh"

namespace nnis {

constexpr int kF32Threads = 256;

template <int D, int ROWS>
__global__ void __launch_bounds__(kF32Threads, 2)
attn_shared_f32_kernel(const SharedArgs a) {
    constexpr int kTile = 16 * ROWS, kStride = D + 4, kPs = kSharedPage + 4, J = D / 64;
    extern __shared__ __align__(16) float smem_f32[];
    float* q_s = smem_f32;                      // [tile, D + 4], scaled
    float* k_s = q_s + kTile * kStride;         // [64, D + 4]
    float* v_s = k_s + kSharedPage * kStride;   // [64, D]
    float* p_s = v_s + kSharedPage * D;         // [tile, 68]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const SharedUnit u = a.units[blockIdx.x];
    units_begin(a);
    const int hk = blockIdx.y, G = a.nq / a.nkv;
    const int* members = a.members + u.members;
    const int* table = a.page_table + (size_t)u.seq * a.table_cols;
    const int pos = u.ends ? a.token_pos[u.ends - 1] : 0x7fffffff;
    const int n_pages = min(a.table_cols, u.ends ? min(u.page_end, pos < 0 ? 0 : pos / kSharedPage + 1) : u.page_end);
    if (tid == 0) units_end_check(a, u, pos);

    auto keys_of = [&](int it, int page) {  // keys of a page that the unit's rows see (0 where the table has a gap)
        return page < 0 || page >= a.pages ? 0 : u.ends ? min(kSharedPage, pos + 1 - it * kSharedPage) : kSharedPage;
    };
    auto load = [&](const void* cache, float* to, int stride, int it) {
        if (it < n_pages) {
            const int page = table[it], keys = keys_of(it, page);
            const float* from = static_cast<const float*>(cache) + ((size_t)(keys ? page : 0) * a.nkv + hk) * kSharedPage * D;
#pragma unroll
            for (int i = 0; i < kSharedPage * D / 4 / kF32Threads; ++i) {
                const int c = tid + i * kF32Threads, row = c / (D / 4), at = c % (D / 4);
                const bool there = row < keys;
                copy16_or_zero(to + row * stride + at * 4, from + (there ? (size_t)c * 4 : 0), there);
            }
        }
        copy_commit();
    };
    load(a.k_cache, k_s, kStride, u.page_begin);
    load(a.v_cache, v_s, D, u.page_begin);
    for (int i = tid; i < kTile * (D / 4); i += kF32Threads) {
        const int e = i / (D / 4), c = i % (D / 4) * 4, at = u.entry + e;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (e < u.entries) {
            x = load4(static_cast<const float*>(a.q) + (size_t)members[at / G] * a.q_stride + (size_t)(hk * G + at % G) * D + c);
            const float f = a.scale * 1.4426950408889634f;
            x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        }
        *reinterpret_cast<float4*>(q_s + e * kStride + c) = x;
    }
    float4 o[ROWS][J];
    float m_run[ROWS], l_run[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) o[r][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int it = u.page_begin; it < n_pages; ++it) {
        const int keys = keys_of(it, table[it]);
        copy_wait<1>();
        __syncthreads();  // K is there
        float s[ROWS][4];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i] = 0.f;
#pragma unroll 4
        for (int c = 0; c < D; c += 4) {
            float4 kk[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) kk[i] = load4(k_s + (tx + 16 * i) * kStride + c);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float4 qq = load4(q_s + (ty * ROWS + r) * kStride + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[r][i] = fmaf(qq.x, kk[i].x, s[r][i]);
                    s[r][i] = fmaf(qq.y, kk[i].y, s[r][i]);
                    s[r][i] = fmaf(qq.z, kk[i].z, s[r][i]);
                    s[r][i] = fmaf(qq.w, kk[i].w, s[r][i]);
                }
            }
        }
        __syncthreads();  // ... and read
        load(a.k_cache, k_s, kStride, it + 1);
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
                p_s[(ty * ROWS + r) * kPs + tx + 16 * i] = p;
            }
            l_run[r] = l_run[r] * alpha + half_warp_sum(sum);
#pragma unroll
            for (int j = 0; j < J; ++j) o[r][j] = make_float4(o[r][j].x * alpha, o[r][j].y * alpha, o[r][j].z * alpha, o[r][j].w * alpha);
        }
        copy_wait<1>();
        __syncthreads();  // V is there, and the weights
#pragma unroll 2
        for (int t = 0; t < kSharedPage; t += 4) {
            float4 p[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) p[r] = load4(p_s + (ty * ROWS + r) * kPs + t);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const float4 v = load4(v_s + (t + i) * D + j * 64 + tx * 4);
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const float w = i == 0 ? p[r].x : i == 1 ? p[r].y : i == 2 ? p[r].z : p[r].w;
                        o[r][j].x = fmaf(w, v.x, o[r][j].x);
                        o[r][j].y = fmaf(w, v.y, o[r][j].y);
                        o[r][j].z = fmaf(w, v.z, o[r][j].z);
                        o[r][j].w = fmaf(w, v.w, o[r][j].w);
                    }
                }
        }
        __syncthreads();  // ... and read
        load(a.v_cache, v_s, D, it + 1);
    }
    copy_wait<0>();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int e = ty * ROWS + r;
        if (e >= u.entries) continue;
        const int at = u.entry + e;
        const size_t rec = (size_t)(a.record[members[at / G]] + u.slot) * a.nq + hk * G + at % G;
        if (tx == 0) reinterpret_cast<float2*>(a.sums)[rec] = make_float2(m_run[r], l_run[r]);
#pragma unroll
        for (int j = 0; j < J; ++j) store4(a.partial + rec * D + j * 64 + tx * 4, o[r][j]);
    }
    if (a.tickets) merge_finished<float, kF32Threads>(a, u, hk, G, reinterpret_cast<int4*>(p_s));
    units_end(a);
}

template <int D, int ROWS>
static cudaError_t launch_f32(const SharedArgs& a, int n_units, cudaStream_t stream) {
    const size_t smem = ((size_t)(16 * ROWS + kSharedPage) * (D + 4) + (size_t)kSharedPage * D + (size_t)16 * ROWS * (kSharedPage + 4)) * sizeof(float);
    auto kernel = attn_shared_f32_kernel<D, ROWS>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(n_units, a.nkv), kF32Threads, smem, stream, a);
}

cudaError_t shared_units_f32(const SharedArgs& a, int n_units, int tile, cudaStream_t stream) {
    if (a.d == 64) return tile == 16 ? launch_f32<64, 1>(a, n_units, stream) : launch_f32<64, 4>(a, n_units, stream);
    return tile == 16 ? launch_f32<128, 1>(a, n_units, stream) : launch_f32<128, 4>(a, n_units, stream);
}

}  // namespace nnis
