// Attention over shared pages for units of up to 32 entries (token row, query head) on mma.sync tiles, bfloat16, heads of
// 64 or 128: what a sequence has alone, and pages that few rows share.  See attention_shared.cuh for units and records.
//
// A CTA of four warps owns a unit and a kv head.  Pages of K and V come into shared memory by 16-byte asynchronous copies,
// several ahead, rows swizzled for ldmatrix.  Each warp takes 16 keys of every page for all the unit's entries, so K and V are
// read from shared memory once, and keeps a running maximum, sum and output of its own; the warps meet at the end.
// Rows of a page beyond the last visible key are filled with zeros instead of read: what lies there may be no number.
// Bound by the bytes of K and V where units are many (three CTAs an SM, pages of three more ahead each), by a unit's trips to memory
// (plan, page id, page, records: 3.5 us for a page) where they are few.  8 rows of 9 heads over 3 behind 4,032 tokens: 8.5 us, the
// merge 3.3 more; 24 rows of 32 heads behind each of two prompts of 4,001 tokens (65 MB): 24.0 us.
// P is rounded to bfloat16 for the tensor cores (up to 2^-8 of a weight, of either sign), sums are of the 32-bit weights.
#include "attention_shared.cuh"
#include "fma_pairs.cuh"
#include "mma_helpers.cuh"

namespace nnis {

constexpr int kSmWarps = 4, kSmThreads = kSmWarps * 32;

template <int D>
constexpr int sm_stages() { return D == 64 ? 4 : 3; }

template <int D>
__global__ void __launch_bounds__(kSmThreads, D == 64 ? 3 : 2)
attn_shared_mma_kernel(const SharedArgs a) {
    constexpr int CH = D / 8, NT = D / 8, KS = D / 16, STAGES = sm_stages<D>(), MT = 2, kSmEntries = 16 * MT;  // (MT tiles of 16 entries)
    extern __shared__ __align__(128) unsigned char smem_raw[];
    bf16* q_s = reinterpret_cast<bf16*>(smem_raw);  // [32, D] swizzled
    bf16* tiles = q_s + kSmEntries * D;             // stages x (K [64, D], V [64, D])
    __shared__ float sm_ml[kSmWarps][kSmEntries][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const SharedUnit u = a.units[blockIdx.x];  // (the plan comes from the host: it is asked for ahead of the wait)
    units_begin(a);
    const int hk = blockIdx.y, G = a.nq / a.nkv;
    const int* members = a.members + u.members;
    const int* table = a.page_table + (size_t)u.seq * a.table_cols + u.page_begin;
    const int some = min(u.page_end, a.table_cols) - u.page_begin;  // (a tail may be given room to grow)
    const int ids = lane < some ? table[lane] : -1;  // a lane a page, up to 32 of them
    const int pos = u.ends ? a.token_pos[u.ends - 1] : 0x7fffffff;
    const int n_pages = u.ends ? min(some, pos < 0 ? 0 : pos / kSharedPage + 1 - u.page_begin) : some;
    if (tid == 0) units_end_check(a, u, pos);
    const bool two = u.entries > 16;  // the second tile of 16 entries holds any
    const bf16 *k_cache = static_cast<const bf16*>(a.k_cache), *v_cache = static_cast<const bf16*>(a.v_cache);
    constexpr size_t kTile = (size_t)kSharedPage * D;

    auto page_of = [&](int it) { return it < 32 ? __shfl_sync(0xffffffffu, ids, it) : table[it]; };
    // keys of page `it` that the unit's rows see (0 where the table has a gap)
    auto keys_of = [&](int it, int page) {
        return page < 0 || page >= a.pages ? 0 : u.ends ? min(kSharedPage, pos + 1 - (u.page_begin + it) * kSharedPage) : kSharedPage;
    };
    auto load_page = [&](int it) {
        if (it < n_pages) {
            const int page = page_of(it), keys = keys_of(it, page);
            const size_t from = (size_t)((keys ? page : 0) * (long long)a.nkv + hk) * kTile;
            bf16* kd = tiles + (size_t)(it % STAGES) * 2 * kTile;
            bf16* vd = kd + kTile;
#pragma unroll
            for (int i = 0; i < kSharedPage * CH / kSmThreads; ++i) {
                const int c = tid + i * kSmThreads, row = c / CH, chunk = c % CH;
                const bool there = row < keys;
                copy16_or_zero(kd + swz<D>(row, chunk), k_cache + from + (there ? (size_t)c * 8 : 0), there);
                copy16_or_zero(vd + swz<D>(row, chunk), v_cache + from + (there ? (size_t)c * 8 : 0), there);
            }
        }
        cp_async_commit();
    };
    for (int it = 0; it < STAGES - 1; ++it) load_page(it);

    for (int c = tid; c < kSmEntries * CH; c += kSmThreads) {
        const int e = c / CH, chunk = c % CH, at = u.entry + e;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (e < u.entries)
            x = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.q) + (size_t)members[at / G] * a.q_stride +
                                                (size_t)(hk * G + at % G) * D + chunk * 8);
        *reinterpret_cast<uint4*>(q_s + swz<D>(e, chunk)) = x;
    }
    const int r_lo = lane >> 2, c_lo = (lane & 3) * 2;
    float o[MT][NT][4], m_run[MT][2], l_run[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
        m_run[t][0] = m_run[t][1] = -INFINITY;
        l_run[t][0] = l_run[t][1] = 0.f;
    }
    const float sc = a.scale * kLog2e;
    const int key0 = warp * 16;
    for (int it = 0; it < n_pages; ++it) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();  // page `it` has landed for everyone; the stage of the page before is free
        load_page(it + STAGES - 1);
        const bf16* kt = tiles + (size_t)(it % STAGES) * 2 * kTile;
        const bf16* vt = kt + kTile;
        const int keys = keys_of(it, page_of(it));
        uint32_t pa[MT][4];
        float alpha[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (t && !two) break;
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; kk += 2) {
                uint32_t qa[2][4];
                ldmatrix_x4(qa[0], q_s + swz<D>(t * 16 + (lane & 15), kk * 2 + (lane >> 4)));
                ldmatrix_x4(qa[1], q_s + swz<D>(t * 16 + (lane & 15), kk * 2 + 2 + (lane >> 4)));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t kb[4];
                    ldmatrix_x4(kb, kt + swz<D>(key0 + j * 8 + (lane & 7), kk * 2 + (lane >> 3)));
                    mma_bf16(s[j], qa[0], kb[0], kb[1]);
                    mma_bf16(s[j], qa[1], kb[2], kb[3]);
                }
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = key0 + j * 8 + c_lo + (e & 1) < keys ? s[j][e] * sc : -INFINITY;
                    s[j][e] = x;
                    mx[e >> 1] = fmaxf(mx[e >> 1], x);
                }
            float base[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float mn = fmaxf(m_run[t][r], mx[r]);
                base[r] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: no inf - inf
                alpha[t][r] = sh_ex2(m_run[t][r] - base[r]);
                m_run[t][r] = mn;
            }
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float p0 = sh_ex2(s[j][0] - base[0]), p1 = sh_ex2(s[j][1] - base[0]);
                const float p2 = sh_ex2(s[j][2] - base[1]), p3 = sh_ex2(s[j][3] - base[1]);
                sum[0] += p0 + p1;
                sum[1] += p2 + p3;
                pa[t][j * 2] = pack_bf16(p0, p1);
                pa[t][j * 2 + 1] = pack_bf16(p2, p3);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) l_run[t][r] = l_run[t][r] * alpha[t][r] + sum[r];
            if (__any_sync(0xffffffffu, alpha[t][0] != 1.f || alpha[t][1] != 1.f)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][j][e] *= alpha[t][e >> 1];
            }
        }
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
            uint32_t vb[4];
            ldmatrix_x4_trans(vb, vt + swz<D>(key0 + (lane & 15), j + (lane >> 4)));
            mma_bf16(o[0][j], pa[0], vb[0], vb[1]);
            mma_bf16(o[0][j + 1], pa[0], vb[2], vb[3]);
            if (two) {
                mma_bf16(o[MT - 1][j], pa[MT - 1], vb[0], vb[1]);
                mma_bf16(o[MT - 1][j + 1], pa[MT - 1], vb[2], vb[3]);
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();  // everyone is done with the tiles: the warps' outputs meet there
    float* o_s = reinterpret_cast<float*>(smem_raw);  // [warps, 16, D], one tile of entries after the other
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t && !two) break;
        if (t) __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l_run[t][r] += __shfl_xor_sync(0xffffffffu, l_run[t][r], 1);
            l_run[t][r] += __shfl_xor_sync(0xffffffffu, l_run[t][r], 2);
            if ((lane & 3) == 0) {
                sm_ml[warp][t * 16 + r_lo + 8 * r][0] = m_run[t][r];
                sm_ml[warp][t * 16 + r_lo + 8 * r][1] = l_run[t][r];
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float* at = o_s + ((size_t)warp * 16 + r_lo) * D + j * 8 + c_lo;
            *reinterpret_cast<float2*>(at) = make_float2(o[t][j][0], o[t][j][1]);
            *reinterpret_cast<float2*>(at + 8 * D) = make_float2(o[t][j][2], o[t][j][3]);
        }
        __syncthreads();
        for (int item = tid; item < 16 * (D / 4); item += kSmThreads) {
            const int row = item / (D / 4), c = item % (D / 4), e = t * 16 + row;
            if (e >= u.entries) continue;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kSmWarps; ++w) mm = fmaxf(mm, sm_ml[w][e][0]);
            const float base = mm == -INFINITY ? 0.f : mm;  // (sums of weights that are no number stay that)
            float l = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kSmWarps; ++w) {
                const float f = exp2f(sm_ml[w][e][0] - base);
                l += sm_ml[w][e][1] * f;
                const float4 y = *reinterpret_cast<const float4*>(o_s + ((size_t)w * 16 + row) * D + c * 4);
                x.x = fmaf(y.x, f, x.x);
                x.y = fmaf(y.y, f, x.y);
                x.z = fmaf(y.z, f, x.z);
                x.w = fmaf(y.w, f, x.w);
            }
            const int at = u.entry + e;
            const size_t rec = (size_t)(a.record[members[at / G]] + u.slot) * a.nq + hk * G + at % G;
            if (c == 0) reinterpret_cast<float2*>(a.sums)[rec] = make_float2(mm, l);
            *reinterpret_cast<float4*>(a.partial + rec * D + c * 4) = x;
        }
    }
    if (a.tickets) merge_finished<bf16, kSmThreads>(a, u, hk, G, reinterpret_cast<int4*>(tiles + 4 * kTile));
    units_end(a);
}

template <int D>
static cudaError_t launch_small(const SharedArgs& a, int n_units, cudaStream_t stream) {
    const size_t tiles = (32 * D + sm_stages<D>() * 2 * (size_t)kSharedPage * D) * sizeof(bf16);
    auto kernel = attn_shared_mma_kernel<D>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, tiles, held);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(n_units, a.nkv), kSmThreads, tiles, stream, a);
}

cudaError_t shared_units_mma(const SharedArgs& a, int n_units, cudaStream_t stream) {
    return a.d == 64 ? launch_small<64>(a, n_units, stream) : launch_small<128>(a, n_units, stream);
}

}  // namespace nnis
