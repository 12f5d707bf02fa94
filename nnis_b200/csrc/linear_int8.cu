// Products of whole numbers: C[m, n] (op)= (sum_k xc[m, k] wc[n, k]) * xs[m] * ws[n] + bias[n], rows x put into codes with a scale for
// every token, the matrix held in codes with a scale for every row of it (int8_rows.cuh).  The sum of products of codes is exact
// in 32 bits up to k = 133,143; one float32 product with each scale follows.  Rows of codes take a multiple of 16 bytes, zero
// behind the row's end.
#include <string.h>

#include "async_copy.cuh"
#include "int8_rows.cuh"
#include "linear_int8.cuh"

namespace nnis {

struct Quantize8 {
    const void* x;
    long long x_stride;
    int8_t* codes;
    float* scales;
    int rows, k, kp;
};

// WARPS warps a row, its values in registers between the two looks at them: CHUNKS runs of eight a lane.
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    pdl_launch_dependents();
    constexpr int kLanes = WARPS * 32;
    const int row = blockIdx.x * (4 / WARPS) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const T* x = reinterpret_cast<const T*>(p.x) + (size_t)row * p.x_stride;
    float v[CHUNKS][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * kLanes + lane) * 8;
        if (row < p.rows && i < p.k) {
            const float4 a = load4(x + i), b = load4(x + i + 4);
            v[c][0] = a.x; v[c][1] = a.y; v[c][2] = a.z; v[c][3] = a.w;
            v[c][4] = b.x; v[c][5] = b.y; v[c][6] = b.z; v[c][7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
        }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude_bits(v[c][e]));
    top = group_max<32>(top);
    if (WARPS > 1) {
        if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    if (row >= p.rows) return;
    const RowScale r = row_scale(top);
    const uint32_t good = good_row(r.scale);
    int8_t* codes = p.codes + (size_t)row * p.kp;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * kLanes + lane) * 8;
        if (i >= p.kp) continue;
        *reinterpret_cast<uint2*>(codes + i) = make_uint2(code_word(v[c][0], v[c][1], v[c][2], v[c][3], r.inverse, good),
                                                          code_word(v[c][4], v[c][5], v[c][6], v[c][7], r.inverse, good));
    }
    if (lane == 0) p.scales[row] = r.scale;
}

// Any row: a CTA each, read twice.
template <typename T>
__global__ void __launch_bounds__(128) quantize_rows_any_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    pdl_launch_dependents();
    const T* x = reinterpret_cast<const T*>(p.x) + (size_t)blockIdx.x * p.x_stride;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < p.k; i += 128) top = max(top, magnitude_bits(to_float(x[i])));
    top = group_max<32>(top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const RowScale r = row_scale(top);
    int8_t* codes = p.codes + (size_t)blockIdx.x * p.kp;
    for (int i = threadIdx.x * 4; i < p.kp; i += 512) {
        int c[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < p.k) c[j] = row_code(to_float(x[i + j]), r.inverse);
        *reinterpret_cast<uint32_t*>(codes + i) = pack_codes(c[0], c[1], c[2], c[3]);
    }
    if (threadIdx.x == 0) p.scales[blockIdx.x] = r.scale;
}

template <typename T>
static cudaError_t launch_quantize(const Quantize8& p, cudaStream_t stream) {
    const bool eights = p.k % 8 == 0 && p.x_stride % 8 == 0 && (uintptr_t)p.x % (4 * sizeof(T)) == 0;
    if (!eights || p.kp > 8192) return launch_dependent(quantize_rows_any_kernel<T>, (unsigned)p.rows, 128, 0, stream, p);
    // (a warp a row up to 1,024 values, and up to 2,048 where rows are many)
    if (p.kp <= 1024 || (p.kp <= 2048 && p.rows >= 1024)) {
        auto kernel = p.kp <= 512 ? quantize_rows_kernel<T, 1, 2> : p.kp <= 1024 ? quantize_rows_kernel<T, 1, 4> : quantize_rows_kernel<T, 1, 8>;
        return launch_dependent(kernel, (unsigned)((p.rows + 3) / 4), 128, 0, stream, p);
    }
    auto kernel = p.kp <= 2048 ? quantize_rows_kernel<T, 4, 2> : p.kp <= 4096 ? quantize_rows_kernel<T, 4, 4> : quantize_rows_kernel<T, 4, 8>;
    return launch_dependent(kernel, (unsigned)p.rows, 128, 0, stream, p);
}

}  // namespace nnis

// codes [rows, kp], kp = k rounded up to a multiple of 16; scales [rows]
struct Quantize8Call {
    const void* x;
    void* codes;
    float* scales;
    int x_stride, dtype, rows, k;
    cudaStream_t stream;
};
NNIS_API int nnis_quantize_rows(const void* call) {
    using namespace nnis;
    Quantize8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, codes, scales, x_stride, dtype, rows, k, stream] = c;
    if (!x || !codes || !scales || rows <= 0 || k <= 0 || k > 0x7ffffff0 || x_stride < k) return NNIS_ERR_ARGUMENT;
    if ((uintptr_t)codes % 16) return NNIS_ERR_ALIGNMENT;
    const Quantize8 p{x, x_stride, (int8_t*)codes, scales, rows, k, (k + 15) / 16 * 16};
    if (dtype == NNIS_DTYPE_F32) return (int)launch_quantize<float>(p, stream);
    if (dtype == NNIS_DTYPE_BF16) return (int)launch_quantize<bf16>(p, stream);
    return NNIS_ERR_UNSUPPORTED;
}

// x [m, k] (rows `x_stride` apart) is put into `codes` [m, kp] and `scales` [m] (or, one row or two, into shared memory), w [n (gated: 2
// n), kp] codes, ws their scales, bias float32 like ws or null, out [m, n]: `dtype` (x's) in the modes 0 (store) and 3 (gated: silu(first half of w's rows) * the
// second), float32 in 1 (store) and 2 (add).
struct Linear8Call {
    const void *x, *w;
    const float *ws, *bias;
    void *out, *codes;
    float* scales;
    int* status;
    int x_stride, m, n, k, mode, dtype, sms, padding;
    cudaStream_t stream;
};
NNIS_API int nnis_linear_int8(const void* call) {
    using namespace nnis;
    Linear8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, w, ws, bias, out, codes, scales, status, x_stride, m, n, k, mode, dtype, sms, padding, stream] = c;
    (void)padding;
    const int kp = (k + 15) / 16 * 16;
    if (!x || !w || !ws || !out || !codes || !scales || m <= 0 || n <= 0 || k <= 0 || x_stride < k || mode < 0 || mode > 3)
        return NNIS_ERR_ARGUMENT;
    if (k > 133136 || (dtype != NNIS_DTYPE_F32 && dtype != NNIS_DTYPE_BF16)) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)codes | (uintptr_t)w) % 16) return NNIS_ERR_ALIGNMENT;
    const bool f32 = dtype == NNIS_DTYPE_F32;
    const Linear8 p{(const int8_t*)codes, (const int8_t*)w, scales, ws, bias, out, m, n, kp, status, 0, x, x_stride, k};
    const int held = sms > 0 ? sms : 148;
    if (linear_int8_fuses(p, mode == INT8_GATED, f32, held)) return (int)linear_int8_few(p, mode, f32, true, stream);
    const Quantize8 q{x, x_stride, (int8_t*)codes, scales, m, k, kp};
    const cudaError_t e = f32 ? launch_quantize<float>(q, stream) : launch_quantize<bf16>(q, stream);
    if (e != cudaSuccess) return (int)e;
    // us by few rows' kernel / by tcgen05: 16 rows 16,384 x 2,048 13.2 / 13.7, 2,048 x 8,192 8.8 / 11; 32 rows 960 x 576 4.5 / 5.9,
    // 2,048 x 2,048 6.1 / 6.4, 6,144 x 2,048 9.1 / 8.2, 2,048 x 8,192 14.4 / 11.1, 16,384 x 2,048 18.0 / 13.5
    const long long bytes = (long long)(mode == INT8_GATED ? 2 : 1) * n * kp;
    if (m <= 16 || (m <= 32 && bytes < 8 << 20)) return (int)linear_int8_few(p, mode, f32, false, stream);
    return linear_int8_tc(p, mode, f32, held, stream);
}
