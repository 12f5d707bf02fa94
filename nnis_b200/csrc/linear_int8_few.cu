// Products of 8-bit codes with few rows (decode steps), bound by the bytes of W: a CTA's eight warps share 16 rows of W (gated: 8 gate
// and the 8 up rows), each takes every eighth run of 64 places of K straight into registers, and multiplies them (mma.sync, signed
// bytes, W as the 16-row operand) with up to 32 rows of x; the eight sums, whole numbers, are added in shared memory.
//
// Any order of K serves a sum: a lane holds 16 bytes of a row that lie side by side, so that a warp's load of 8 rows takes whole
// 64-byte runs and no byte is moved afterwards.  The first loads of W go out ahead of the wait for the kernel that makes x's codes.
//
// One or two rows are put into codes by every CTA for itself, in shared memory, while its first loads of W are on their way, where every
// CTA has an SM of its own: a kernel less to launch and to wait for.  us with a kernel for the codes / without: one row 960 x 576
// 3.4 / 3.1, 2,048 x 2,048 3.6 / 3.7, two 3.4 / 3.1 and 3.8 / 3.7; four 3.4 / 3.6, 3.9 / 4.0; one row in 1,024 CTAs (gate and up of
// 1.7B) 9.3 / 11.7.
#include <type_traits>

#include "async_copy.cuh"
#include "int8_rows.cuh"
#include "linear_int8.cuh"

namespace nnis {


__device__ __forceinline__ uint4 load_w(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void few_mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kFusedRows = 2, kFewRows = 32;
// NT: tiles of 8 rows of x; kFewWarps: 8, or 16 where there are fewer CTAs than SMs and a long K.
// X: the type of x where its rows are still values (fused), int8_t where they are codes.
// (up to eight rows of codes: registers for three CTAs an SM, which is asked for: 80 where the compiler takes 70 by itself and keeps fewer loads
// ahead.  8 rows, us without / with: gate and up 16,384 x 2,048 10.2 / 9.8, 576 x 1,536 3.5 / 3.1, 32,768 x 2,048 16.0 / 15.2.  A CTA that walks
// over tiles with the next one's loads ahead: 10.9, 3.6, 16.8)
template <typename T, bool ADD, bool GATED, int NT, int kFewWarps, typename X = int8_t>
__global__ void __launch_bounds__(kFewWarps * 32, kFewWarps == 8 && NT == 1 && std::is_same<X, int8_t>::value ? 3 : 0) linear_int8_few_kernel(const __grid_constant__ Linear8 p) {
    constexpr int kAhead = 4, kOut = GATED ? 8 : 16;  // runs of K that a lane has asked for; outputs of a CTA and row of x
    constexpr bool kFused = !std::is_same<X, int8_t>::value;
    __shared__ int sums[kFewWarps][NT * 128];
    __shared__ uint32_t tops[kFused ? kFewWarps : 1];
    __shared__ float row_scales[kFused ? kFusedRows : 1];
    extern __shared__ __align__(16) int8_t coded[];  // fused: m rows of `coded_row` codes
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kOut, runs = (p.kp + 63) / 64;
    const uint4 none = {0u, 0u, 0u, 0u};
    // row g of the operand's 16, and row g + 8: of a gated product the same output's gate and up
    const int8_t* rows[2] = {p.w + (size_t)(n0 + g) * p.kp, p.w + ((size_t)n0 + g + (GATED ? p.n : 8)) * p.kp};
    const bool in[2] = {n0 + g < p.n, n0 + g + (GATED ? 0 : 8) < p.n};
    uint4 w[kAhead][2];
    auto load = [&](int i, int run) {
        const int k = run * 64 + 16 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) w[i][h] = k < p.kp && in[h] ? load_w(rows[h] + k) : none;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(i, warp + i * kFewWarps);
    pdl_wait();
    pdl_launch_dependents();
    // (rows lie an odd number of 64 bytes apart: two rows' 64 bytes are on all 32 banks)
    const int coded_row = (runs | 1) * 64;
    if constexpr (kFused) {
        const int share = kFewWarps / p.m;  // warps of a row
        const int row = warp / share, at = warp % share * 32 + lane;
        const X* x = reinterpret_cast<const X*>(p.values) + (size_t)row * p.x_stride;
        uint32_t top = 0;
        if (row < p.m)
            for (int i = at * 8; i < p.k; i += share * 256) {
                const float4 a = load4(x + i), b = load4(x + i + 4);
                top = max(top, max(max(magnitude_bits(a.x), magnitude_bits(a.y)), max(magnitude_bits(a.z), magnitude_bits(a.w))));
                top = max(top, max(max(magnitude_bits(b.x), magnitude_bits(b.y)), max(magnitude_bits(b.z), magnitude_bits(b.w))));
            }
        top = group_max<32>(top);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
        if (row < p.m) {
            for (int v = 0; v < share; ++v) top = max(top, tops[row * share + v]);
            const RowScale s = row_scale(top);
            const uint32_t good = good_row(s.scale);
            if (at == 0) row_scales[row] = s.scale;
            for (int i = at * 8; i < runs * 64; i += share * 256) {
                uint2 codes = {0u, 0u};
                if (i < p.k) {
                    const float4 a = load4(x + i), b = load4(x + i + 4);
                    codes = make_uint2(code_word(a.x, a.y, a.z, a.w, s.inverse, good), code_word(b.x, b.y, b.z, b.w, s.inverse, good));
                }
                *reinterpret_cast<uint2*>(coded + (size_t)row * coded_row + i) = codes;
            }
        }
        __syncthreads();
    }
    int acc[NT][4] = {};
    for (int first = warp; first < runs; first += kAhead * kFewWarps) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int k = (first + i * kFewWarps) * 64 + 16 * t;
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const int m = 8 * c + g;
                uint4 x = none;
                if (k < p.kp && m < p.m)
                    x = *reinterpret_cast<const uint4*>(kFused ? coded + (size_t)m * coded_row + k : p.x + (size_t)m * p.kp + k);
                few_mma(acc[c], w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, x.x, x.y);
                few_mma(acc[c], w[i][0].z, w[i][1].z, w[i][0].w, w[i][1].w, x.z, x.w);
            }
            load(i, first + (i + kAhead) * kFewWarps);
        }
    }
    // sums[token][row of W]: a lane's are rows g and g + 8, tokens 2 t and 2 t + 1 of each tile
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][(c * 8 + 2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[c][i];
    __syncthreads();
    auto value = [&](int m, int row_in, size_t row) {
        int sum = 0;
#pragma unroll
        for (int v = 0; v < kFewWarps; ++v) sum += sums[v][m * 16 + row_in];
        return (float)sum * (kFused ? row_scales[m] : p.xs[m]) * p.ws[row] + (p.bias ? p.bias[row] : 0.f);
    };
    for (int at = threadIdx.x; at < NT * 8 * kOut; at += kFewWarps * 32) {
        const int m = at / kOut, c = at % kOut, n = n0 + c;
        if (m >= p.m || n >= p.n) continue;
        float y = value(m, c, (size_t)n);
        if (GATED) y = silu_gate(y, value(m, 8 + c, (size_t)p.n + n));
        T* out = reinterpret_cast<T*>(p.out) + (size_t)m * p.n + n;
        *out = from_float<T>(ADD ? to_float(*out) + y : y);
    }
}

// Warps of a CTA: 16 where there are fewer CTAs than SMs and a long K.
static bool few_wide(unsigned ctas, const Linear8& p, int sms) { return ctas <= (unsigned)sms && p.kp >= 2048 && p.m <= 16; }

template <typename T, bool ADD, bool GATED>
static cudaError_t launch_few(const Linear8& p, int sms, cudaStream_t stream) {
    const unsigned ctas = (unsigned)((p.n + (GATED ? 7 : 15)) / (GATED ? 8 : 16));
    if (few_wide(ctas, p, sms)) {
        auto kernel = p.m <= 8 ? linear_int8_few_kernel<T, ADD, GATED, 1, 16> : linear_int8_few_kernel<T, ADD, GATED, 2, 16>;
        return launch_dependent(kernel, ctas, 512, 0, stream, p);
    }
    auto kernel = p.m <= 8 ? linear_int8_few_kernel<T, ADD, GATED, 1, 8> : p.m <= 16 ? linear_int8_few_kernel<T, ADD, GATED, 2, 8>
                  : linear_int8_few_kernel<T, ADD, GATED, 4, 8>;
    return launch_dependent(kernel, ctas, 256, 0, stream, p);
}

template <typename T, bool ADD, bool GATED, typename X>
static cudaError_t launch_fused(const Linear8& p, int sms, cudaStream_t stream) {
    const unsigned ctas = (unsigned)((p.n + (GATED ? 7 : 15)) / (GATED ? 8 : 16));
    const size_t smem = (size_t)p.m * (((p.kp + 63) / 64) | 1) * 64;
    if (few_wide(ctas, p, sms)) return launch_dependent(linear_int8_few_kernel<T, ADD, GATED, 1, 16, X>, ctas, 512, smem, stream, p);
    return launch_dependent(linear_int8_few_kernel<T, ADD, GATED, 1, 8, X>, ctas, 256, smem, stream, p);
}

bool linear_int8_may_fuse(const Linear8& p, bool f32) {
    return p.m <= kFusedRows && p.kp <= 16384 && p.k % 8 == 0 && p.x_stride % 8 == 0 && (uintptr_t)p.values % (f32 ? 16 : 8) == 0;
}

cudaError_t linear_int8_few(const Linear8& p, int mode, bool f32, bool fused, int sms, cudaStream_t stream) {
    if (p.m > (fused ? kFusedRows : kFewRows)) return cudaErrorInvalidValue;
    if (fused) {
        if (mode == INT8_GATED) return f32 ? launch_fused<float, false, true, float>(p, sms, stream) : launch_fused<bf16, false, true, bf16>(p, sms, stream);
        if (mode == INT8_ADD_F32) return f32 ? launch_fused<float, true, false, float>(p, sms, stream) : launch_fused<float, true, false, bf16>(p, sms, stream);
        if (mode == INT8_STORE_F32)
            return f32 ? launch_fused<float, false, false, float>(p, sms, stream) : launch_fused<float, false, false, bf16>(p, sms, stream);
        return f32 ? launch_fused<float, false, false, float>(p, sms, stream) : launch_fused<bf16, false, false, bf16>(p, sms, stream);
    }
    if (mode == INT8_GATED) return f32 ? launch_few<float, false, true>(p, sms, stream) : launch_few<bf16, false, true>(p, sms, stream);
    if (mode == INT8_ADD_F32) return launch_few<float, true, false>(p, sms, stream);
    return f32 || mode == INT8_STORE_F32 ? launch_few<float, false, false>(p, sms, stream) : launch_few<bf16, false, false>(p, sms, stream);
}

}  // namespace nnis
