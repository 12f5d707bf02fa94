// Attention over shared pages for many small units (up to 16 entries: token row, query head), bfloat16, heads of 64 or 128: the
// tails of a large batch, a page or three each.  See attention_shared.cuh for units and records.
//
// Such units are over before a CTA of their own has come into its stride (start, plan, page id, page, records: four trips to
// memory, 3.5 us for one page, and 2,048 of them 12 us).  So a warp takes units one after another, (unit, kv head) by (unit, kv
// head): the next one's plan and page ids come while this one is worked, its first page while this one's last is.  A page's K and
// V [64 keys, D] come by TMA into two places of the warp's own, each asked for again as soon as it has been read: with a dozen
// (six at 128 values) warps an SM that is 192 KB on its way.  Scores and outputs are mma.sync products, a warp has all keys of
// its page, and nothing is shared among warps.  Bound by the bytes of K and V: 51 rows of 32 heads, tails of one to five pages and three
// long ones (188 MB), 37 us, 5.1 TB/s.
// P is rounded to bfloat16 for the tensor cores (up to 2^-8 of a weight, of either sign), sums are of the 32-bit weights.
// Every wait is bounded; a warp whose wait runs out sets the status word and leaves.
#include "attention_shared.cuh"
#include "mma_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace nnis {

template <int D>
constexpr int wp_warps() { return D == 64 ? 12 : 6; }

template <int D>
__global__ void __launch_bounds__(wp_warps<D>() * 32, 1)
attn_shared_warp_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedArgs a,
                        int n_items) {
    constexpr int C = D / 64, NT = D / 8, KS = D / 16, W = wp_warps<D>();
    constexpr uint32_t kBytes = kSharedPage * D * 2, kChunk = kSharedPage * 128;  // of a page's K or V, of 64 columns of it
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[W][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* k_s = shared_1024(smem_raw) + warp * 2 * kBytes;
    unsigned char* v_s = k_s + kBytes;
    uint64_t *k_bar = &bars[warp][0], *v_bar = &bars[warp][1];
    if (lane == 0) {
        if (warp == 0) {
            prefetch_tensormap(&map_k);
            prefetch_tensormap(&map_v);
        }
        mbar_init(k_bar, 1);
        mbar_init(v_bar, 1);
        mbar_fence_init();
    }
    __syncwarp();
    const int G = a.nq / a.nkv, stride = gridDim.x * W;
    const int r_lo = lane >> 2, c_lo = (lane & 3) * 2;
    const float sc = a.scale * kLog2e;

    // What is known of an item ahead of its turn.
    struct Item {
        SharedUnit u;
        int hk, ids, pos, pages;
    };
    auto unit_of = [&](int i) { return i < n_items ? a.units[i / a.nkv] : SharedUnit{}; };
    auto look = [&](const SharedUnit& u, int i) {  // asks for its ids and position
        Item t;
        t.u = u;
        t.hk = i % a.nkv;
        const int some = min(u.page_end, a.table_cols) - u.page_begin;
        t.ids = i < n_items && lane < some ? a.page_table[(size_t)u.seq * a.table_cols + u.page_begin + lane] : -1;
        t.pos = i < n_items && u.ends ? a.token_pos[u.ends - 1] : 0x7fffffff;
        t.pages = some;
        return t;
    };
    auto pages_of = [&](const Item& t) {
        return t.u.ends ? min(t.pages, t.pos < 0 ? 0 : t.pos / kSharedPage + 1 - t.u.page_begin) : t.pages;
    };
    auto id_of = [&](const Item& t, int it) {
        return it < 32 ? __shfl_sync(0xffffffffu, t.ids, it) : a.page_table[(size_t)t.u.seq * a.table_cols + t.u.page_begin + it];
    };
    auto fetch = [&](const CUtensorMap* map, unsigned char* to, uint64_t* bar, int page, int hk) {
        if (lane == 0) {
            mbar_expect_tx(bar, kBytes);
            const int row = (page * a.nkv + hk) * kSharedPage;  // (outside the store: zeros)
#pragma unroll
            for (int c = 0; c < C; ++c) tma_load_2d(to + c * kChunk, map, c * 64, row, bar);
        }
    };
    // an element of a page's tile: 16-byte chunk `chunk` of row `row`, 128-byte rows of 64 columns, swizzled
    auto at = [&](unsigned char* tile, int row, int chunk) { return tile + (chunk >> 3) * kChunk + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); };

    int i = warp * gridDim.x + blockIdx.x;  // (neighbouring items go to different SMs)
    const SharedUnit u_first = unit_of(i);  // (the plan comes from the host: it is asked for ahead of the wait)
    SharedUnit u_next = unit_of(i + stride);
    units_begin(a);
    Item now = look(u_first, i);
    uint32_t k_turn = 0, v_turn = 0;
    int n_pages = i < n_items ? pages_of(now) : 0;
    bool ok = true, asked = false;  // whether this item's first page is on its way
    for (; i < n_items && ok; i += stride) {
        const Item next = look(u_next, i + stride);
        u_next = unit_of(i + 2 * stride);
        const int next_pages = i + stride < n_items ? pages_of(next) : 0;
        if (lane == 0) units_end_check(a, now.u, now.pos);
        const int* members = a.members + now.u.members;
        if (n_pages > 0 && !asked) {
            const int page = id_of(now, 0);
            fetch(&map_k, k_s, k_bar, page, now.hk);
            fetch(&map_v, v_s, v_bar, page, now.hk);
        }
        // the queries as the products' left operand: rows r_lo and r_lo + 8
        uint32_t qa[KS][4];
        {
            const bf16* q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int e = r_lo + 8 * h, place = now.u.entry + e;
                q[h] = e < now.u.entries ? static_cast<const bf16*>(a.q) + (size_t)members[place / G] * a.q_stride +
                                               (size_t)(now.hk * G + place % G) * D + c_lo
                                         : nullptr;
            }
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    qa[kk][h] = q[h & 1] ? *reinterpret_cast<const uint32_t*>(q[h & 1] + kk * 16 + (h >> 1) * 8) : 0u;
        }
        float o[NT][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        asked = false;
        for (int it = 0; it < n_pages; ++it) {
            const int page = id_of(now, it);
            const int keys = page < 0 || page >= a.pages ? 0 : now.u.ends ? min(kSharedPage, now.pos + 1 - (now.u.page_begin + it) * kSharedPage) : kSharedPage;
            const bool more = it + 1 < n_pages, other = !more && next_pages > 0;
            const int page_next = more ? id_of(now, it + 1) : other ? id_of(next, 0) : 0, hk_next = more ? now.hk : next.hk;
            ok = __all_sync(0xffffffffu, mbar_wait(k_bar, k_turn));
            if (!ok) break;
            k_turn ^= 1u;
            float s[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; kk += 2)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t kb[4];
                    ldmatrix_x4(kb, at(k_s, j * 8 + (lane & 7), kk * 2 + (lane >> 3)));
                    mma_bf16(s[j], qa[kk], kb[0], kb[1]);
                    mma_bf16(s[j], qa[kk + 1], kb[2], kb[3]);
                }
            __syncwarp();
            if (more || other) fetch(&map_k, k_s, k_bar, page_next, hk_next);
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = j * 8 + c_lo + (e & 1) < keys ? s[j][e] * sc : -INFINITY;
                    s[j][e] = x;
                    mx[e >> 1] = fmaxf(mx[e >> 1], x);
                }
            float base[2], alpha[2], sum[2] = {0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float mn = fmaxf(m_run[r], mx[r]);
                base[r] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: no inf - inf
                alpha[r] = sh_ex2(m_run[r] - base[r]);
                m_run[r] = mn;
            }
            uint32_t pa[4][4];  // four k-steps of 16 keys
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p0 = sh_ex2(s[j][0] - base[0]), p1 = sh_ex2(s[j][1] - base[0]);
                const float p2 = sh_ex2(s[j][2] - base[1]), p3 = sh_ex2(s[j][3] - base[1]);
                sum[0] += p0 + p1;
                sum[1] += p2 + p3;
                pa[j >> 1][(j & 1) * 2] = pack_bf16(p0, p1);
                pa[j >> 1][(j & 1) * 2 + 1] = pack_bf16(p2, p3);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) l_run[r] = l_run[r] * alpha[r] + sum[r];
            ok = __all_sync(0xffffffffu, mbar_wait(v_bar, v_turn));
            if (!ok) break;
            v_turn ^= 1u;
            if (keys < kSharedPage) {  // what lies behind the last visible key may be no number: zeros
                for (int c = lane; c < (kSharedPage - keys) * C * 8; c += 32)
                    *reinterpret_cast<uint4*>(at(v_s, keys + c / (C * 8), c % (C * 8))) = make_uint4(0, 0, 0, 0);
                fence_async_shared();  // (the next page comes by the other proxy)
                __syncwarp();
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e >> 1];
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t vb[4];
                    ldmatrix_x4_trans(vb, at(v_s, ks * 16 + (lane & 15), j + (lane >> 4)));
                    mma_bf16(o[j], pa[ks], vb[0], vb[1]);
                    mma_bf16(o[j + 1], pa[ks], vb[2], vb[3]);
                }
            __syncwarp();
            if (more || other) fetch(&map_v, v_s, v_bar, page_next, hk_next);
            asked = other;
        }
        if (!ok) break;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
            const int e = r_lo + 8 * r, place = now.u.entry + e;
            if (e < now.u.entries) {
                const size_t rec = (size_t)(a.record[members[place / G]] + now.u.slot) * a.nq + now.hk * G + place % G;
                if ((lane & 3) == 0) reinterpret_cast<float2*>(a.sums)[rec] = make_float2(m_run[r], l_run[r]);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    *reinterpret_cast<float2*>(a.partial + rec * D + j * 8 + c_lo) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
            }
        }
        now = next;
        n_pages = next_pages;
    }
    if (!ok) {  // no copy may land after the CTA has left
        mbar_wait(k_bar, k_turn);
        mbar_wait(v_bar, v_turn);
        if (lane == 0 && a.status) atomicExch(a.status, 1);
    }
    __syncthreads();
    units_end(a);
}

template <int D>
static cudaError_t launch_warp(const SharedArgs& a, int n_units, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    const long long rows = (long long)a.pages * a.nkv * kSharedPage;
    if (!make_map(&map_k, a.k_cache, rows, D, kSharedPage) || !make_map(&map_v, a.v_cache, rows, D, kSharedPage))
        return cudaErrorInvalidValue;
    constexpr int W = wp_warps<D>();
    const size_t smem = 1024 + (size_t)W * 2 * kSharedPage * D * 2;
    auto kernel = attn_shared_warp_kernel<D>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    const int items = n_units * a.nkv, sms = device_sms();
    return launch_dependent(kernel, dim3(items < sms ? items : sms), W * 32, smem, stream, map_k, map_v, a, items);
}

cudaError_t shared_units_warp(const SharedArgs& a, int n_units, cudaStream_t stream) {
    return a.d == 64 ? launch_warp<64>(a, n_units, stream) : launch_warp<128>(a, n_units, stream);
}

}  // namespace nnis
