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
    int matrix;  // 1: the rows may be a matrix's, which products ask for ahead of their wait
};

// A product's kernel loads codes of its matrix before it waits for the kernel ahead of it.  So a kernel that may make a matrix lets nothing
// start before its end, by when its codes are out; one that makes a product's own x lets the product start at once.
__device__ __forceinline__ void release_early(const Quantize8& p) {
    if (!p.matrix) pdl_launch_dependents();
}
__device__ __forceinline__ void release_late(const Quantize8& p) {
    if (p.matrix) __threadfence();
}

// WARPS warps a row, its values in registers between the two looks at them: CHUNKS runs of eight a lane.
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    release_early(p);
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
    release_late(p);
}

// Rows of odd lengths or at odd addresses: a CTA each, the row's values in registers, CHUNKS runs of four a thread.
template <typename T, int CHUNKS>
__global__ void __launch_bounds__(128) quantize_rows_odd_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    release_early(p);
    const T* x = reinterpret_cast<const T*>(p.x) + (size_t)blockIdx.x * p.x_stride;
    float v[CHUNKS][4];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = (c * 128 + threadIdx.x) * 4 + j;
            v[c][j] = i < p.k ? to_float(x[i]) : 0.f;
        }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, magnitude_bits(v[c][j]));
    top = group_max<32>(top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const RowScale r = row_scale(top);
    const uint32_t good = good_row(r.scale);
    int8_t* codes = p.codes + (size_t)blockIdx.x * p.kp;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * 128 + threadIdx.x) * 4;
        if (i < p.kp) *reinterpret_cast<uint32_t*>(codes + i) = code_word(v[c][0], v[c][1], v[c][2], v[c][3], r.inverse, good);
    }
    if (threadIdx.x == 0) p.scales[blockIdx.x] = r.scale;
    release_late(p);
}

// Any row: a CTA each, read twice.
template <typename T>
__global__ void __launch_bounds__(128) quantize_rows_any_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    release_early(p);
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
    release_late(p);
}

// A norm's rows put into codes: y = x / sqrt(mean(x^2) + eps) * w, rounded to T as the norm by itself would be, its codes and scale.  A CTA a
// row, the row and the weights in registers.
template <typename T, int Q>
__global__ void __launch_bounds__(256)
rmsnorm_int8_kernel(const float* __restrict__ x, const float* __restrict__ w, int8_t* __restrict__ codes, float* __restrict__ scales,
                    int width, int kp, float eps) {
    __shared__ float partial[8];
    __shared__ uint32_t tops[8];
    const int tid = threadIdx.x, n4 = width >> 2;
    float4 g[Q], v[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) g[j] = tid + 256 * j < n4 ? load4(w + 4 * (tid + 256 * j)) : make_float4(0.f, 0.f, 0.f, 0.f);
    pdl_wait();  // (the weights depend on no kernel)
    pdl_launch_dependents();
    const float* in = x + (size_t)blockIdx.x * width;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        v[j] = tid + 256 * j < n4 ? load4(in + 4 * (tid + 256 * j)) : make_float4(0.f, 0.f, 0.f, 0.f);
        ss = fmaf(v[j].x, v[j].x, fmaf(v[j].y, v[j].y, fmaf(v[j].z, v[j].z, fmaf(v[j].w, v[j].w, ss))));
    }
    ss = warp_sum(ss);
    if ((tid & 31) == 0) partial[tid >> 5] = ss;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) total += partial[k];
    const float s = 1.0f / sqrtf(total * (1.0f / (float)width) + eps);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        v[j] = make_float4(to_float(from_float<T>((v[j].x * s) * g[j].x)), to_float(from_float<T>((v[j].y * s) * g[j].y)),
                           to_float(from_float<T>((v[j].z * s) * g[j].z)), to_float(from_float<T>((v[j].w * s) * g[j].w)));
        top = max(top, max(max(magnitude_bits(v[j].x), magnitude_bits(v[j].y)), max(magnitude_bits(v[j].z), magnitude_bits(v[j].w))));
    }
    top = group_max<32>(top);
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, tops[k]);
    const RowScale r = row_scale(top);
    const uint32_t good = good_row(r.scale);
    int8_t* out = codes + (size_t)blockIdx.x * kp;
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        const int i = 4 * (tid + 256 * j);
        if (i < kp) *reinterpret_cast<uint32_t*>(out + i) = i < width ? code_word(v[j].x, v[j].y, v[j].z, v[j].w, r.inverse, good) : 0u;
    }
    if (tid == 0) scales[blockIdx.x] = r.scale;
}

template <typename T>
static cudaError_t launch_rmsnorm8(const float* x, const float* w, int8_t* codes, float* scales, int rows, int width, int kp, float eps,
                                   cudaStream_t stream) {
    auto kernel = kp <= 1024 ? rmsnorm_int8_kernel<T, 1> : kp <= 2048 ? rmsnorm_int8_kernel<T, 2> : kp <= 4096 ? rmsnorm_int8_kernel<T, 4>
                  : rmsnorm_int8_kernel<T, 8>;
    return launch_dependent(kernel, (unsigned)rows, 256, 0, stream, x, w, codes, scales, width, kp, eps);
}

template <typename T>
static cudaError_t launch_quantize(const Quantize8& p, cudaStream_t stream) {
    const bool eights = p.k % 8 == 0 && p.x_stride % 8 == 0 && (uintptr_t)p.x % (4 * sizeof(T)) == 0;
    if (!eights && p.kp <= 4096) {
        auto kernel = p.kp <= 1024 ? quantize_rows_odd_kernel<T, 2> : p.kp <= 2048 ? quantize_rows_odd_kernel<T, 4>
                      : quantize_rows_odd_kernel<T, 8>;
        return launch_dependent(kernel, (unsigned)p.rows, 128, 0, stream, p);
    }
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

// codes [rows, kp], kp = k rounded up to a multiple of 16; scales [rows].  Rows of x lie `x_stride` elements apart, 0 or less than k where they
// share memory.
struct Quantize8Call {
    const void* x;
    void* codes;
    float* scales;
    long long x_stride;
    int dtype, rows, k;
    cudaStream_t stream;
};
NNIS_API int nnis_quantize_rows(const void* call) {
    using namespace nnis;
    Quantize8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, codes, scales, x_stride, dtype, rows, k, stream] = c;
    if (!x || !codes || !scales || rows <= 0 || k <= 0 || k > 0x7ffffff0 || x_stride < 0) return NNIS_ERR_ARGUMENT;
    if ((uintptr_t)codes % 16) return NNIS_ERR_ALIGNMENT;
    const Quantize8 p{x, x_stride, (int8_t*)codes, scales, rows, k, (k + 15) / 16 * 16, 1};
    if (dtype == NNIS_DTYPE_F32) return (int)launch_quantize<float>(p, stream);
    if (dtype == NNIS_DTYPE_BF16) return (int)launch_quantize<bf16>(p, stream);
    return NNIS_ERR_UNSUPPORTED;
}

// Rows x [rows, width] float32 through an RMS norm with `weight`, rounded to `dtype`, as codes [rows, kp] and scales [rows].
struct Rmsnorm8Call {
    const float *x, *weight;
    void* codes;
    float* scales;
    int rows, width, dtype;
    float eps;
    cudaStream_t stream;
};
NNIS_API int nnis_rmsnorm_int8(const void* call) {
    using namespace nnis;
    Rmsnorm8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, weight, codes, scales, rows, width, dtype, eps, stream] = c;
    if (!x || !weight || !codes || !scales || rows <= 0 || width <= 0 || !(eps > 0.f)) return NNIS_ERR_ARGUMENT;
    if (width % 4 || width > 8192) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)x | (uintptr_t)weight | (uintptr_t)codes) % 16) return NNIS_ERR_ALIGNMENT;
    const int kp = (width + 15) / 16 * 16;
    if (dtype == NNIS_DTYPE_F32) return (int)launch_rmsnorm8<float>(x, weight, (int8_t*)codes, scales, rows, width, kp, eps, stream);
    if (dtype == NNIS_DTYPE_BF16) return (int)launch_rmsnorm8<bf16>(x, weight, (int8_t*)codes, scales, rows, width, kp, eps, stream);
    return NNIS_ERR_UNSUPPORTED;
}

// x [m, k] (rows `x_stride` apart) is put into `codes` [m, kp] and `scales` [m] (or, one row or two, into shared memory), w [n (gated: 2
// n), kp] codes, ws their scales, bias float32 like ws or null, out [m, n]: `dtype` (x's) in the modes 0 (store) and 3 (gated: silu(first half of w's rows) * the
// second), float32 in 1 (store) and 2 (add).  `coded`:
// `codes` and `scales` are there already.  Both are null where the caller wants rows put into shared memory.
struct Linear8Call {
    const void *x, *w;
    const float *ws, *bias;
    void *out, *codes;
    float* scales;
    int* status;
    long long x_stride;
    int m, n, k, mode, dtype, sms, coded;
    cudaStream_t stream;
};
NNIS_API int nnis_linear_int8(const void* call) {
    using namespace nnis;
    Linear8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, w, ws, bias, out, codes, scales, status, x_stride, m, n, k, mode, dtype, sms, coded, stream] = c;
    const int kp = (k + 15) / 16 * 16;
    if ((!x && !coded) || !w || !ws || !out || (coded && (!codes || !scales)) || m <= 0 || n <= 0 || k <= 0 || (!coded && x_stride < 0) || mode < 0 || mode > 3)
        return NNIS_ERR_ARGUMENT;
    if (k > 133136 || (dtype != NNIS_DTYPE_F32 && dtype != NNIS_DTYPE_BF16)) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)codes | (uintptr_t)w) % 16) return NNIS_ERR_ALIGNMENT;
    const bool f32 = dtype == NNIS_DTYPE_F32;
    const Linear8 p{(const int8_t*)codes, (const int8_t*)w, scales, ws, bias, out, status, x, x_stride, m, n, kp, k, 0};
    const int held = sms > 0 ? sms : device_sms();
    if (!codes && !scales && linear_int8_may_fuse(p, f32)) return (int)linear_int8_few(p, mode, f32, true, held, stream);
    if (!codes || !scales) return NNIS_ERR_ARGUMENT;
    const Quantize8 q{x, x_stride, (int8_t*)codes, scales, m, k, kp, 0};
    const cudaError_t e = coded ? cudaSuccess : f32 ? launch_quantize<float>(q, stream) : launch_quantize<bf16>(q, stream);
    if (e != cudaSuccess) return (int)e;
    // us by few rows' kernel / by tcgen05: 16 rows 16,384 x 2,048 13.2 / 13.7, 2,048 x 8,192 8.8 / 11; 32 rows 960 x 576 4.5 / 5.9,
    // 2,048 x 2,048 6.1 / 6.4, 6,144 x 2,048 9.1 / 8.2, 2,048 x 8,192 14.4 / 11.1, 16,384 x 2,048 18.0 / 13.5
    const long long bytes = (long long)(mode == INT8_GATED ? 2 : 1) * n * kp;
    if (m <= 16 || (m <= 32 && bytes < 8 << 20)) return (int)linear_int8_few(p, mode, f32, false, held, stream);
    return linear_int8_tc(p, mode, f32, held, stream);
}
