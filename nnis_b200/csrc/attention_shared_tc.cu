// Attention over shared pages on the fifth-generation tensor cores: units of up to 128 entries (token row, query head),
// bfloat16, heads of 64 or 128.  See attention_shared.cuh for units and records.
//
// A CTA owns a unit and a kv head; all its entries see all keys of its pages, so nothing is masked.  Eleven warps:
//   warp 0     one lane issues TMA loads: a page of K and of V [64 keys, D] per step into rings of their own (K is done with as
//              soon as its scores are, V a softmax later);
//   warp 1     allocates tensor memory and issues S[128, 64] = Q K^T (two buffers), the next pages' while this one's
//              softmax runs;
//   warp 2     issues O[128, D] += P V, P from tensor memory;
//   warps 3-10 stack the entries' queries into shared memory (they lie rows apart, G heads together), then softmax: two
//              warps per quarter of the rows, a thread has one row and half of a page's keys.  The halves tell each
//              other their maximum through shared memory, so that one accumulator O serves both, and write P
//              (bfloat16) into tensor memory: with 64 values into columns of its own, so that a buffer takes its next scores as
//              soon as the last have been read; with 128, where O takes those columns, over the scores.
// P is rounded to bfloat16 because the tensor cores take it so (up to 2^-8 of a weight, of either sign); sums are of the 32-bit
// weights.  O stays in tensor memory; the maximum that P is taken against is only raised when a page exceeds it by
// more than 8 (a factor 256, harmless in both types), then the warps wait for the products so far and multiply O.  So the largest
// weight is not the 1 that it is against the running maximum, and is rounded too: 0.0023 of the outputs' norm from 64 bits, where the
// mma.sync units' are 0.0017 to 0.0019 and the outputs' own rounding is 0.0017.
// Every wait is bounded; one that runs out raises an abort flag, all warps meet at the end and tensor memory is freed.
//
// Two CTAs an SM, so that one's softmax runs under the other's waits.  A page of 128 entries takes 1,095 clocks of an SM (2,190
// with two CTAs), of which its 8,192 exponentials are 512; the tensor pipe is busy a fifth of the time.  To that come 5 to 8 us
// a launch: set-up, queries from all over, the first page, records.  64 rows of 15 heads over 5 behind 16,384 tokens
// (bytes 3.3 us, exponentials 3.4): 17.6 us; 16 sequences of 5 tokens, 32 heads of 128 over 8, behind 8,190: 23.9 us.  Tried and slower: one CTA an
// SM with two tiles (256 entries) and 128 keys a step, 23.6 us where this took 20.2, 36 where it took 30.
#include "attention_shared.cuh"
#include "fma_pairs.cuh"
#include "tcgen05_helpers.cuh"

namespace nnis {

constexpr int kShRows = 128, kShThreads = 352;
constexpr uint32_t kShChunkQ = kShRows * 128, kShChunkK = kSharedPage * 128;  // bytes of 64 columns of the queries, of a page
constexpr float kShRaise = 8.0f;

template <int D>
constexpr int sh_stages() { return D == 64 ? 4 : 2; }

__device__ __forceinline__ bool sh_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

__device__ __forceinline__ void sh_store16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
    tmem_store_wait();
}

// 32 bytes, a whole sector, at once: a lane's row is far from its neighbours'.
__device__ __forceinline__ void store_sector(float* to, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// The two warps of a quarter of the rows meet.  A warp that gives up raises the abort flag and then arrives once, so that its
// partner, wherever it is, comes through its next meeting, sees the flag there and gives up too: no meeting waits for good.
__device__ __forceinline__ void quarter_meet(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }
__device__ __forceinline__ void quarter_leave(int quarter) { asm volatile("bar.arrive %0, 64;" ::"r"(1 + quarter) : "memory"); }

// V as loaded ([64 keys] by chunks of 64 values, rows of 128 bytes, 128-byte swizzle) as the MN-major B operand: chunks lie
// 8 KB apart (leading byte offset), groups of 8 keys 1,024 bytes (stride byte offset).
__device__ __forceinline__ uint64_t sh_desc_v(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(kShChunkK >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

template <int D>
__global__ void __launch_bounds__(kShThreads, 2)
attn_shared_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedArgs a) {
    constexpr int C = D / 64, kStages = sh_stages<D>();
    constexpr uint32_t kPageBytes = C * kShChunkK, kCols = 256;
    // tensor memory: S, two buffers of 64 columns; P, 32 columns a buffer; O
    constexpr bool kOwnP = D == 64;
    constexpr uint32_t kP = kOwnP ? 128 : 0, kStrideP = kOwnP ? 32 : 64, kColsO = kOwnP ? 192 : 128;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* q_s = shared_1024(smem_raw);           // C x [128, 64] swizzled
    unsigned char* k_s = q_s + C * kShChunkQ;             // stages x C x [64, 64]
    unsigned char* v_s = k_s + kStages * kPageBytes;
    __shared__ __align__(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    __shared__ __align__(8) uint64_t q_ready, s_full[2], s_free[2], p_ready[2], pv_done[2];
    __shared__ float half_max[2][2][kShRows], half_sum[kShRows];
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        mbar_init(&q_ready, 8);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&s_free[b], 8);  // the softmax warps
            mbar_init(&p_ready[b], 8);
            mbar_init(&pv_done[b], 1);
        }
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    const SharedUnit u = a.units[blockIdx.x];
    const int hk = blockIdx.y, G = a.nq / a.nkv;
    const int n_pages = u.entries > 0 ? u.page_end - u.page_begin : 0;
    units_begin(a);  // (queries, keys and values come from the kernel before; the set-up above ran under it)

    if (n_pages <= 0) {
    } else if (warp == 0) {
        if (lane == 0) {
            const int* table = a.page_table + (size_t)u.seq * a.table_cols + u.page_begin;
            int i = 0, i_v = 0;  // pages whose K, whose V has been asked for
            while (i < n_pages) {
                const int s = i % kStages;
                const uint32_t turn = (uint32_t)(i / kStages - 1) & 1u;
                const int row = (table[i] * a.nkv + hk) * kSharedPage;
                if (i >= kStages && !mbar_wait(&k_empty[s], turn)) abort_flag = 1;
                if (abort_flag) break;
                mbar_expect_tx(&k_full[s], kPageBytes);
#pragma unroll
                for (int c = 0; c < C; ++c) tma_load_2d(k_s + s * kPageBytes + c * kShChunkK, &map_k, c * 64, row, &k_full[s]);
                if (i++ >= kStages && !mbar_wait(&v_empty[s], turn)) abort_flag = 1;
                if (abort_flag) break;
                mbar_expect_tx(&v_full[s], kPageBytes);
#pragma unroll
                for (int c = 0; c < C; ++c) tma_load_2d(v_s + s * kPageBytes + c * kShChunkK, &map_v, c * 64, row, &v_full[s]);
                ++i_v;
            }
            // no copy may land after the CTA has left, whatever the others do
            for (int j = max(0, i - kStages); j < i; ++j) mbar_wait(&k_full[j % kStages], (uint32_t)(j / kStages) & 1u);
            for (int j = max(0, i_v - kStages); j < i_v; ++j) mbar_wait(&v_full[j % kStages], (uint32_t)(j / kStages) & 1u);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = instr_desc(kShRows, kSharedPage);
        const uint64_t desc_q = smem_desc_k128(smem_addr(q_s)), desc_k0 = smem_desc_k128(smem_addr(k_s));
        bool ok = sh_wait(&q_ready, 0);
        for (int i = 0; ok && i < n_pages; ++i) {
            const int s = i % kStages, b = i & 1;
            ok = sh_wait(&k_full[s], (uint32_t)(i / kStages) & 1u) && !__any_sync(0xffffffffu, abort_flag);
            // (the buffer's scores of two pages ago have been read, or the product that read P over them is over)
            if (ok && i >= 2) ok = sh_wait(kOwnP ? &s_free[b] : &pv_done[b], (uint32_t)((i >> 1) - 1) & 1u);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    warp_mma(tmem + b * 64, desc_advance(desc_q, c * kShChunkQ + k * 32),
                             desc_advance(desc_k0, (uint32_t)s * kPageBytes + c * kShChunkK + k * 32), idesc, (c | k) != 0);
            warp_commit(&s_full[b]);
            warp_commit(&k_empty[s]);
        }
        if (!ok && lane == 0) abort_flag = 1;
    } else if (warp == 2) {
        constexpr uint32_t idesc = instr_desc(kShRows, D) | (1u << 16);  // (V: MN-major)
        const uint64_t desc_v0 = sh_desc_v(smem_addr(v_s));
        bool ok = true;
        for (int i = 0; ok && i < n_pages; ++i) {
            const int s = i % kStages, b = i & 1;
            ok = sh_wait(&v_full[s], (uint32_t)(i / kStages) & 1u) && sh_wait(&p_ready[b], (uint32_t)(i >> 1) & 1u) &&
                 !__any_sync(0xffffffffu, abort_flag);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
                warp_mma_ts(tmem + kColsO, tmem + kP + b * kStrideP + k * 8, desc_advance(desc_v0, (uint32_t)s * kPageBytes + k * 2048),
                            idesc, (i | k) != 0);
            warp_commit(&pv_done[b]);
            warp_commit(&v_empty[s]);
        }
        if (!ok && lane == 0) abort_flag = 1;
    } else {
        const int quarter = warp & 3, half = (warp - 3) >> 2;
        const int row = quarter * 32 + lane;
        const int* members = a.members + u.members;
        {   // the queries: eight warps, a row of 128 bytes by eight lanes, all of a thread's on their way together
            constexpr int kPer = kShRows * C * 8 / 256;
            const bf16* q = static_cast<const bf16*>(a.q);
            uint4 x[kPer];
#pragma unroll
            for (int n = 0; n < kPer; ++n) {
                const int i = threadIdx.x - 96 + n * 256, e = i / (C * 8), c = i % (C * 8), at = u.entry + e;
                x[n] = make_uint4(0, 0, 0, 0);
                if (e < u.entries)
                    x[n] = __ldg(reinterpret_cast<const uint4*>(q + (size_t)__ldg(members + at / G) * a.q_stride + (size_t)(hk * G + at % G) * D + c * 8));
            }
#pragma unroll
            for (int n = 0; n < kPer; ++n) {
                const int i = threadIdx.x - 96 + n * 256, e = i / (C * 8), c = i % (C * 8);
                *reinterpret_cast<uint4*>(q_s + (c >> 3) * kShChunkQ + e * 128 + (((c & 7) ^ (e & 7)) << 4)) = x[n];
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready);
        }
        int rec = -1;  // this row's record
        if (row < u.entries) {
            const int at = u.entry + row;
            rec = (a.record[members[at / G]] + u.slot) * a.nq + hk * G + at % G;
        }
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const float sc = a.scale * 1.4426950408889634f;
        const bool idle = quarter * 32 >= u.entries;  // rows of no entry: their P may be anything
        float m_run = -INFINITY, l_run = 0.f;         // maximum in use (scaled, log2 units), this half's sum against it
        bool ok = true;
        // Where the next scores come before a product is over, a page's P (and a warp's word that it is there) waits for that of
        // two pages ago.
        auto last_over = [&](int i) { return !kOwnP || i < 2 || sh_wait(&pv_done[i & 1], (uint32_t)((i >> 1) - 1) & 1u); };
        for (int i = 0; i < n_pages; ++i) {
            const int b = i & 1;
            ok = sh_wait(&s_full[b], (uint32_t)(i >> 1) & 1u);
            if (!ok) break;
            if (idle) {
                if (kOwnP && lane == 0) mbar_arrive(&s_free[b]);
                ok = last_over(i);
                if (!ok) break;
                if (lane == 0) mbar_arrive(&p_ready[b]);
                continue;
            }
            tc_fence_after();
            uint32_t sv[32];
            tmem_load32(tmem + b * 64 + half * 32 + lane_base, sv);
            if (kOwnP) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[b]);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 32; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sv[c + 2 * e]), __uint_as_float(sv[c + 2 * e + 1]));
            const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            half_max[b][half][row] = mine;
            tc_fence_before();
            quarter_meet(quarter);  // (both halves have read their scores, too)
            ok = !__any_sync(0xffffffffu, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const float m_new = fmaxf(m_run, fmaxf(mine, half_max[b][half ^ 1][row]) * sc);
            const bool raise = m_run != -INFINITY && m_new > m_run + kShRaise;
            if (m_run == -INFINITY) m_run = m_new;  // nothing summed yet: this row of O is zero, or not begun
            if (i > 0 && __any_sync(0xffffffffu, raise)) {
                ok = sh_wait(&pv_done[b ^ 1], (uint32_t)((i - 1) >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const float alpha = m_run == -INFINITY ? 1.f : exp2f(m_run - m_new);
#pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t ov[16];
                    tmem_load16_issue(tmem + kColsO + half * (D / 2) + h * 16 + lane_base, ov);
                    tmem_load_wait();
#pragma unroll
                    for (int c = 0; c < 16; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
                    sh_store16(tmem + kColsO + half * (D / 2) + h * 16 + lane_base, ov);
                }
                l_run *= alpha;
                m_run = m_new;
            }
            const unsigned long long neg_base = both(m_run == -INFINITY ? 0.f : -m_run);
            unsigned long long ps[2] = {0ull, 0ull};
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                unsigned long long at = neg_base;
                fma2(at, pair_of(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), both(sc));
                const float p0 = sh_ex2(halves(at).x), p1 = sh_ex2(halves(at).y);
                ps[e & 1] = add2(ps[e & 1], pair_of(p0, p1));
                __nv_bfloat162 pk = __floats2bfloat162_rn(p0, p1);
                w[e] = *reinterpret_cast<uint32_t*>(&pk);
            }
            const float2 s0 = halves(ps[0]), s1 = halves(ps[1]);
            l_run += (s0.x + s0.y) + (s1.x + s1.y);
            ok = last_over(i);
            if (!ok) break;
            if (kOwnP) tc_fence_after();
            sh_store16(tmem + kP + b * kStrideP + half * 16 + lane_base, w);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[b]);
        }
        if (!ok) {
            abort_flag = 1;
            __syncwarp();
            quarter_leave(quarter);
        } else if (!idle) {
            if (half) half_sum[row] = l_run;
            quarter_meet(quarter);
            const int last = n_pages - 1;
            ok = sh_wait(&pv_done[last & 1], (uint32_t)(last >> 1) & 1u) && !__any_sync(0xffffffffu, abort_flag);
            if (!ok) {
                abort_flag = 1;
            } else {
                tc_fence_after();
                const bool real = rec >= 0;
                if (real && !half) reinterpret_cast<float2*>(a.sums)[rec] = make_float2(m_run, l_run + half_sum[row]);
                float* dst = a.partial + (size_t)rec * D + half * (D / 2);
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    uint32_t ov[32];
                    tmem_load32(tmem + kColsO + half * (D / 2) + h * 32 + lane_base, ov);
                    if (real) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8) store_sector(dst + h * 32 + c, ov + c);
                    }
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (abort_flag && threadIdx.x == 0 && a.status) atomicExch(a.status, 1);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kCols);
    }
}

template <int D>
static cudaError_t launch_tc(const SharedArgs& a, int n_units, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    const long long rows = (long long)a.pages * a.nkv * kSharedPage;
    if (!make_map(&map_k, a.k_cache, rows, D, kSharedPage) || !make_map(&map_v, a.v_cache, rows, D, kSharedPage))
        return cudaErrorInvalidValue;
    const size_t smem = 1024 + (D / 64) * (size_t)kShChunkQ + 2 * sh_stages<D>() * (size_t)(D / 64) * kShChunkK;
    auto kernel = attn_shared_tc_kernel<D>;
    static std::atomic<int> held[16];
    const cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3(n_units, a.nkv), kShThreads, smem, stream, map_k, map_v, a);
}

cudaError_t shared_units_tc(const SharedArgs& a, int n_units, cudaStream_t stream) {
    return a.d == 64 ? launch_tc<64>(a, n_units, stream) : launch_tc<128>(a, n_units, stream);
}

}  // namespace nnis
