// Products of 8-bit codes with many rows on the fifth-generation tensor cores: sums of products of signed bytes in 32 bits (tcgen05.mma,
// kind::i8), exact, in tensor memory; the epilogue multiplies each by its token's and its channel's scale.
//
// Roles as in the bfloat16 product: lane 0 of warp 0 loads tiles of x, lane 0 of warp 2 tiles of W (128 places of K, a row of the 128-byte
// swizzle, a stage), one lane of warp 1 issues the products, warps 2 to 9 read tensor memory, scale, and send boxes of 32 rows x
// 128 bytes out by TMA.  A byte is a place of K, so a stage of as many bytes carries twice the products of bfloat16's at twice the rate:
// the same bytes a cycle are asked of L2, 64 for each SM of a pair of CTAs that share a tile of 256 x 256 (gated: 128 gate and the 128
// up columns), 128 for a CTA of its own with a tile of 128 x 128 (gated: 64 and 64), which is for products of fewer tiles.
// Where tiles are fewer than half of the SMs (some hundred rows at most), a cluster of up to eight CTAs shares a tile's K; their sums,
// whole numbers, are added through the cluster's shared memory (64 rows through 1.7B's down projection, 16 tiles: 26.2 -> 11.5 us).
// Every wait is bounded; a wait that runs out sets the status word, and all warps still meet at the end and free tensor memory.
#include "fma_pairs.cuh"
#include "linear_int8.cuh"
#include "tcgen05_helpers.cuh"

namespace nnis {

constexpr int kRows8 = 128, kSlice8 = 128, kThreads8 = 320, kEpilogueWarps8 = 8;
constexpr int kSumsRow8 = 132;  // of a tile's sums in shared memory: a row of 128 and a gap that keeps rows off one another's banks
constexpr uint32_t kTileBytes8 = kRows8 * kSlice8;  // x's tile, and W's: 128 rows in either form

// The addresses of the cluster's CTAs' copies of a place in shared memory, and four sums there
__device__ __forceinline__ int4 peer_sums(const int* p, int rank) {
    uint32_t at;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// Two sums as float32, times their token's scale, times their channels'
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(b));
    return a;
}
__device__ __forceinline__ unsigned long long scaled_pair(uint32_t a, uint32_t b, unsigned long long xs, unsigned long long ws) {
    return mul2(mul2(pair_of((float)(int)a, (float)(int)b), xs), ws);
}
// silu_gate of two
__device__ __forceinline__ unsigned long long silu_pair(unsigned long long gate, unsigned long long up) {
    const float2 x = halves(mul2(gate, both(-1.4426950408889634f)));
    float a, b, ra, rb;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(x.y));
    const float2 d = halves(add2(pair_of(a, b), both(1.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ra) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rb) : "f"(d.y));
    return mul2(mul2(gate, pair_of(ra, rb)), up);
}

// T: the output's type; ADD: into float32; SPLIT: gridDim.z CTAs of a cluster share a tile's K.  BN: columns of a tile's products, gate and up together.
template <typename T, bool ADD, bool GATED, bool PAIR, int STAGES, bool SPLIT = false>
__global__ void __launch_bounds__(kThreads8, STAGES <= 3 ? 2 : 1)
linear_int8_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ CUtensorMap map_out, const __grid_constant__ Linear8 p) {
    constexpr int BN = PAIR ? 256 : 128, kOutCols = GATED ? BN / 2 : BN;  // columns of the output that the tile makes
    constexpr int kLoads = GATED ? 2 : 1, kLoadRows = 128 / kLoads;       // of W, by each CTA: 128 rows in one or two boxes
    constexpr uint32_t kTmemCols = BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = shared_1024(smem_raw);
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], done;
    __shared__ uint32_t tmem_s;
    __shared__ volatile int abort_flag;
    __shared__ __align__(16) float scales[BN], biases[BN];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const int m0 = blockIdx.x * kRows8, n0 = blockIdx.y * kOutCols;
    const int all_slices = (p.kp + kSlice8 - 1) / kSlice8, per_cta = SPLIT ? (all_slices + (int)gridDim.z - 1) / (int)gridDim.z : all_slices;
    const int first_slice = SPLIT ? (int)blockIdx.z * per_cta : 0, slices = SPLIT ? min(per_cta, all_slices - first_slice) : all_slices;
    if (threadIdx.x == 32) {
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_w);
        if (p.out_by_tma) prefetch_tensormap(&map_out);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) pair_tmem_alloc(&tmem_s, kTmemCols);
        else tmem_alloc(&tmem_s, kTmemCols);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_meet();
    tc_fence_after();
    const uint32_t tmem = tmem_s;

    // Each CTA of a pair loads its 128 rows of x and half of the tile's rows of W; the bytes of both count on the first one's barrier.
    auto load = [&](bool of_x, int i) {
        const int s = i % STAGES, slice = first_slice + i;
        unsigned char* to = base + (size_t)s * 2 * kTileBytes8 + (of_x ? 0 : kTileBytes8);
        const int w_row = n0 + (int)rank * kLoadRows;
        if constexpr (PAIR) {
            const uint32_t bar = leader_addr(&full[s]);
            if (rank == 0) mbar_expect_tx(&full[s], 2 * kTileBytes8);
            if (of_x) pair_load_2d(to, &map_x, slice * kSlice8, m0, bar);
            else
#pragma unroll
                for (int h = 0; h < kLoads; ++h) pair_load_2d(to + h * kLoadRows * kSlice8, &map_w, slice * kSlice8, h * p.n + w_row, bar);
        } else {
            mbar_expect_tx(&full[s], kTileBytes8);
            if (of_x) tma_load_2d(to, &map_x, slice * kSlice8, m0, &full[s]);
            else
#pragma unroll
                for (int h = 0; h < kLoads; ++h) tma_load_2d(to + h * kLoadRows * kSlice8, &map_w, slice * kSlice8, h * p.n + w_row, &full[s]);
        }
    };
    // W does not depend on the kernel before: its first stages are asked for ahead of the wait
    int ahead = 0;
    if (warp == 2 && lane == 0)
        for (; ahead < slices && ahead < STAGES; ++ahead) load(false, ahead);
    pdl_wait();
    pdl_launch_dependents();

    int issued = warp == 0 ? 0 : ahead;
    if (lane == 0 && (warp == 0 || warp == 2)) {
        for (int& i = issued; i < slices; ++i) {
            if (i >= STAGES && !mbar_wait(&empty[i % STAGES], (uint32_t)(i / STAGES - 1) & 1u)) {
                abort_flag = 1;
                break;
            }
            if (abort_flag) break;
            load(warp == 0, i);
        }
    }
    __syncwarp();
    if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = instr_desc_i8(PAIR ? 256 : 128, BN);
            const uint64_t desc_x = smem_desc_k128(smem_addr(base)), desc_w = smem_desc_k128(smem_addr(base + kTileBytes8));
            bool ok = true;
            for (int i = 0; i < slices; ++i) {
                const int s = i % STAGES;
                if (!mbar_wait(&full[s], (uint32_t)(i / STAGES) & 1u) || abort_flag) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // 32 places of K each
                    const uint64_t a = desc_advance(desc_x, s * 2 * kTileBytes8 + k * 32), b = desc_advance(desc_w, s * 2 * kTileBytes8 + k * 32);
                    if constexpr (PAIR) pair_mma_i8(tmem, a, b, idesc, (i | k) != 0);
                    else tc_mma_i8(tmem, a, b, idesc, (i | k) != 0);
                }
                if constexpr (PAIR) pair_commit(&empty[s]);
                else tc_commit(&empty[s]);
            }
            if (!ok) {
                abort_flag = 1;
                if constexpr (PAIR) follower_set(&abort_flag, 1);
            }
            if constexpr (PAIR) pair_commit(&done);
            else tc_commit(&done);
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane, m = m0 + row;
        // the tile's scales and biases, in the order of its products' columns: of a pair's gate and up, the first CTA's gate and up
        // rows, then the second's
        for (int c = threadIdx.x - 64; c < BN; c += kEpilogueWarps8 * 32) {
            int col = c, up = 0;
            if (GATED) {
                up = c / kLoadRows % 2;
                col = c / (2 * kLoadRows) * kLoadRows + c % kLoadRows;
            }
            const bool in = n0 + col < p.n;
            scales[c] = in ? p.ws[(size_t)up * p.n + n0 + col] : 0.f;
            biases[c] = in && p.bias ? p.bias[(size_t)up * p.n + n0 + col] : 0.f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps8 * 32) : "memory");
        const unsigned long long xs2 = both(m < p.m ? p.xs[m] : 0.f);
        const bool biased = p.bias != nullptr;
        bool ok = mbar_wait(&done, 0);
        ok = __all_sync(0xffffffffu, ok) && !abort_flag;
        if (!ok) {
            abort_flag = 1;
        } else {
            tc_fence_after();
            constexpr int kBoxCols = 128 / (int)sizeof(T), kSlots = 2;
            const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
            unsigned char* boxes = base + (size_t)(warp - 2) * (kSlots * 4096);
            // (a tile's rows beyond the last: nothing to send)
            const bool sends = !SPLIT && m0 + quarter * 32 < p.m;
            if constexpr (SPLIT) {  // this CTA's sums to its own shared memory
                int* mine = reinterpret_cast<int*>(base) + (size_t)row * kSumsRow8;
#pragma unroll 1
                for (int c0 = group * 32; c0 < BN; c0 += 64) {
                    uint32_t v[32];
                    tmem_load32(lanes + (uint32_t)c0, v);
                    if (m < p.m)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<int4*>(mine + c0 + 4 * j) = make_int4((int)v[4 * j], (int)v[4 * j + 1], (int)v[4 * j + 2], (int)v[4 * j + 3]);
                }
            }
#pragma unroll 1
            for (int b = group, i = 0; b < kOutCols / kBoxCols && n0 + b * kBoxCols < p.n && sends; b += 2, ++i) {
                unsigned char* box = boxes + (i % kSlots) * 4096;
                if (p.out_by_tma && i >= kSlots) {
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kSlots - 1) : "memory");
                    __syncwarp();
                }
#pragma unroll 1
                for (int c0 = b * kBoxCols; c0 < (b + 1) * kBoxCols; c0 += 32) {
                    uint32_t v[32], u[32];
                    const int at = GATED ? c0 / kLoadRows * 2 * kLoadRows + c0 % kLoadRows : c0;
                    tmem_load32_issue(lanes + (uint32_t)at, v);
                    if constexpr (GATED) tmem_load32_issue(lanes + (uint32_t)(at + kLoadRows), u);
                    tmem_load_wait();
                    // (two columns an instruction: a third of the gated epilogue's instructions less)
                    float y[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(scales + at + j);
                        unsigned long long lo = scaled_pair(v[j], v[j + 1], xs2, s4.x), hi = scaled_pair(v[j + 2], v[j + 3], xs2, s4.y);
                        if (biased) {
                            const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(biases + at + j);
                            lo = add2(lo, b4.x);
                            hi = add2(hi, b4.y);
                        }
                        if constexpr (GATED) {
                            const ulonglong2 t4 = *reinterpret_cast<const ulonglong2*>(scales + at + kLoadRows + j);
                            unsigned long long up_lo = scaled_pair(u[j], u[j + 1], xs2, t4.x), up_hi = scaled_pair(u[j + 2], u[j + 3], xs2, t4.y);
                            if (biased) {
                                const ulonglong2 c4 = *reinterpret_cast<const ulonglong2*>(biases + at + kLoadRows + j);
                                up_lo = add2(up_lo, c4.x);
                                up_hi = add2(up_hi, c4.y);
                            }
                            lo = silu_pair(lo, up_lo);
                            hi = silu_pair(hi, up_hi);
                        }
                        const float2 l = halves(lo), h = halves(hi);
                        y[j] = l.x;
                        y[j + 1] = l.y;
                        y[j + 2] = h.x;
                        y[j + 3] = h.y;
                    }
                    if constexpr (sizeof(T) == 2) {
                        const int unit = c0 % 64 / 8;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                __nv_bfloat162 two = __floats2bfloat162_rn(y[8 * j + 2 * e], y[8 * j + 2 * e + 1]);
                                w[e] = *reinterpret_cast<uint32_t*>(&two);
                            }
                            *reinterpret_cast<uint4*>(box + lane * 128 + (((unit + j) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                                make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                    }
                }
                if (p.out_by_tma) {
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        if (ADD) tma_add_2d(&map_out, n0 + b * kBoxCols, m0 + quarter * 32, box);
                        else tma_store_2d(&map_out, n0 + b * kBoxCols, m0 + quarter * 32, box);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    // (rows that TMA cannot write: eight at a time, lanes side by side.  us by lanes with a row each / so: 4,096 rows 961 x 1,024
                    // bfloat16 48 / 9.6, 4,001 x 2,048 added into float32 495 / 69)
                    __syncwarp();
                    constexpr int kUnit = 16 / (int)sizeof(T), kRowsAtOnce = 8;
                    const int rows = min(32, p.m - m0 - quarter * 32);
                    T* out = reinterpret_cast<T*>(p.out) + (size_t)(m0 + quarter * 32) * p.n + n0 + b * kBoxCols;
                    for (int r0 = 0; r0 < rows; r0 += kRowsAtOnce)
#pragma unroll
                        for (int c = lane; c < kBoxCols; c += 32) {
                            T y[kRowsAtOnce];
                            const bool in = n0 + b * kBoxCols + c < p.n;
#pragma unroll
                            for (int i = 0; i < kRowsAtOnce; ++i) {
                                const int r = r0 + i;
                                y[i] = *reinterpret_cast<const T*>(box + r * 128 + ((c / kUnit ^ (r & 7)) << 4) + c % kUnit * (int)sizeof(T));
                                if (ADD && in && r < rows) y[i] = from_float<T>(to_float(y[i]) + to_float(out[(size_t)r * p.n + c]));
                            }
#pragma unroll
                            for (int i = 0; i < kRowsAtOnce; ++i)
                                if (in && r0 + i < rows) out[(size_t)(r0 + i) * p.n + c] = y[i];
                        }
                    __syncwarp();
                }
            }
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
    }
    if constexpr (SPLIT) {
        cluster_meet();  // every CTA's sums are there (whether or not a wait ran out: the status word says so)
        constexpr int kQuads = kOutCols / 4;
        const int rows = min(kRows8, p.m - m0), parts = (int)gridDim.z;
        for (int at = (int)blockIdx.z * kThreads8 + threadIdx.x; at < rows * kQuads; at += parts * kThreads8) {
            const int r = at / kQuads, c = at % kQuads * 4;
            if (n0 + c >= p.n) continue;
            const int* from = reinterpret_cast<const int*>(base) + (size_t)r * kSumsRow8 + c;
            int4 v = {0, 0, 0, 0}, u = {0, 0, 0, 0};
            for (int z = 0; z < parts; ++z) {
                const int4 a = peer_sums(from, z);
                v = make_int4(v.x + a.x, v.y + a.y, v.z + a.z, v.w + a.w);
                if (GATED) {
                    const int4 b = peer_sums(from + kLoadRows, z);
                    u = make_int4(u.x + b.x, u.y + b.y, u.z + b.z, u.w + b.w);
                }
            }
            const float xs = p.xs[m0 + r];
            const int vs[4] = {v.x, v.y, v.z, v.w}, us[4] = {u.x, u.y, u.z, u.w};
            T* out = reinterpret_cast<T*>(p.out) + (size_t)(m0 + r) * p.n + n0 + c;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n0 + c + j >= p.n) break;
                float y = (float)vs[j] * xs * scales[c + j] + biases[c + j];
                if (GATED) y = silu_gate(y, (float)us[j] * xs * scales[kLoadRows + c + j] + biases[kLoadRows + c + j]);
                out[j] = from_float<T>(ADD ? to_float(out[j]) + y : y);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && rank == 0 && abort_flag)  // (copies that are on their way, of both CTAs of a pair, do not outlive them)
        for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i) mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u);
    if constexpr (PAIR || SPLIT) cluster_meet();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) pair_tmem_dealloc(tmem, kTmemCols);
        else tmem_dealloc(tmem, kTmemCols);
    }
    if constexpr (PAIR) cluster_meet();
    if (threadIdx.x == 0 && abort_flag && p.status) atomicExch(p.status, 3);
}

template <typename T, bool ADD, bool GATED, bool PAIR, int STAGES, bool SPLIT = false>
static cudaError_t launch_tc8(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mo, const Linear8& p, cudaStream_t stream,
                              int parts = 1) {
    constexpr size_t smem = (size_t)STAGES * 2 * kTileBytes8 + 1024;
    static_assert(STAGES * 2 * kTileBytes8 >= kEpilogueWarps8 * 2 * 4096, "the epilogue's boxes fit the ring");
    static_assert(!SPLIT || STAGES * 2 * kTileBytes8 >= kRows8 * kSumsRow8 * 4, "a tile's sums fit the ring");
    auto kernel = linear_int8_tc_kernel<T, ADD, GATED, PAIR, STAGES, SPLIT>;
    static std::atomic<int> held[16];
    cudaError_t e = allow_shared(kernel, smem, held);
    if (e != cudaSuccess) return e;
    constexpr int kOutCols = (PAIR ? 256 : 128) / (GATED ? 2 : 1);
    const unsigned tiles = (unsigned)((p.m + kRows8 - 1) / kRows8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(PAIR ? (tiles + 1) / 2 * 2 : tiles, (unsigned)((p.n + kOutCols - 1) / kOutCols), (unsigned)parts);
    cfg.blockDim = dim3(kThreads8);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int attrs = 0;
    if (PAIR || SPLIT) {
        attr[attrs].id = cudaLaunchAttributeClusterDimension;
        attr[attrs].val.clusterDim.x = PAIR ? 2 : 1;
        attr[attrs].val.clusterDim.y = 1;
        attr[attrs++].val.clusterDim.z = (unsigned)parts;
    }
    if (dependent_launches()) {
        attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[attrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = attrs;
    return cudaLaunchKernelEx(&cfg, kernel, mx, mw, mo, p);
}

// Three stages let two CTAs share an SM, so that one's epilogue runs under the other's products; six where there are no more CTAs than SMs.
template <typename T, bool ADD, bool GATED>
static cudaError_t launch_tc8_of(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mo, const Linear8& p, bool pair, bool alone,
                                 int parts, cudaStream_t stream) {
    if (parts > 1) return launch_tc8<T, ADD, GATED, false, 6, true>(mx, mw, mo, p, stream, parts);
    if (pair) return alone ? launch_tc8<T, ADD, GATED, true, 6>(mx, mw, mo, p, stream) : launch_tc8<T, ADD, GATED, true, 3>(mx, mw, mo, p, stream);
    return alone ? launch_tc8<T, ADD, GATED, false, 6>(mx, mw, mo, p, stream) : launch_tc8<T, ADD, GATED, false, 3>(mx, mw, mo, p, stream);
}

int linear_int8_tc(Linear8 p, int mode, bool f32, int sms, cudaStream_t stream) {
    const bool gated = mode == INT8_GATED, wide = f32 || mode == INT8_STORE_F32 || mode == INT8_ADD_F32;
    const long tiles = (p.m + 127) / 128, pair_cols = gated ? 128 : 256, single_cols = gated ? 64 : 128;
    const long pairs = (tiles + 1) / 2 * 2 * ((p.n + pair_cols - 1) / pair_cols), singles = tiles * ((p.n + single_cols - 1) / single_cols);
    const bool pair = 5 * pairs >= 3 * sms;
    if ((p.n + single_cols - 1) / single_cols > 65535) return NNIS_ERR_UNSUPPORTED;
    CUtensorMap mx, mw, mo;
    const int bytes = wide ? 4 : 2;
    if (!make_map(&mx, p.x, p.m, p.kp, kRows8, 0, 1) || !make_map(&mw, p.w, (gated ? 2LL : 1LL) * p.n, p.kp, gated ? 64 : 128, 0, 1))
        return NNIS_ERR_UNSUPPORTED;
    p.out_by_tma = (uintptr_t)p.out % 16 == 0 && (long long)p.n * bytes % 16 == 0 && make_map(&mo, p.out, p.m, p.n, 32, 0, bytes);
    if (!p.out_by_tma) mo = mx;
    const bool alone = (pair ? pairs : singles) <= sms;
    // CTAs that share a tile's K, two runs of 128 places each at least, none of them empty, where that saves a CTA six runs (eight beyond 64
    // rows, which are more to add up): a run takes 0.33 us, sharing 2 to 2.6.  Clusters have to find their SMs side by side, and where they
    // would fill the device some wait for a second turn.  us with 1, 2, 3, 4, 8: 16 tiles (64 x 2,048 x 2,048) 8.4, 8.2, 7.0, 5.9, 9.8;
    // x 8,192 24.6, 16.6, 12.7, 10.4, 14.5; 32 tiles (256 x 2,048 x 8,192) 25.6, 20.6, 16.2, 13.2, 27.7; 44 tiles (1,400 x 512 x 4,096) 14.2,
    // 12.0, 10.5, 16.3, 21.8; 48 tiles (64 x 6,144 x 2,048) 8.2, 7.5, 12.5; 1 tile (128 x 128 x 2,555) 9.5, 8.8, 7.7, 6.3, 6.0; 10 tiles of 5
    // runs (239 x 576 x 576) 4.5, 6.5; 64 of 8 (911 x 960 x 960) 6.4, 7.4; 8 of 8 (64 x 960 x 960) 5.2, 5.5, 5.3, 4.4.
    const int slices = (p.kp + kSlice8 - 1) / kSlice8;
    int parts = pair ? 1 : 16 * singles <= sms ? 8 : 32 * singles <= 7 * sms ? 4 : 30 * singles <= 9 * sms ? 3 : 16 * singles <= 7 * sms ? 2 : 1;
    if (parts > slices / 2) parts = slices / 2;
    if (parts > 1) {
        const int each = (slices + parts - 1) / parts;
        parts = slices - each < (p.m <= 64 ? 6 : 8) ? 1 : (slices + each - 1) / each;
    }
    if (gated)
        return (int)(f32 ? launch_tc8_of<float, false, true>(mx, mw, mo, p, pair, alone, parts, stream)
                         : launch_tc8_of<bf16, false, true>(mx, mw, mo, p, pair, alone, parts, stream));
    if (mode == INT8_ADD_F32) return (int)launch_tc8_of<float, true, false>(mx, mw, mo, p, pair, alone, parts, stream);
    return (int)(wide ? launch_tc8_of<float, false, false>(mx, mw, mo, p, pair, alone, parts, stream)
                      : launch_tc8_of<bf16, false, false>(mx, mw, mo, p, pair, alone, parts, stream));
}

}  // namespace nnis
