// Products of whole numbers: C[m, n] (op)= (sum_k xc[m, k] wc[n, k]) * xs[m] * ws[n] + bias[n], rows x put into codes with a scale for
// every token, the matrix held in codes with a scale for every row of it (int8_rows.cuh).  The sum of products of codes is exact
// in 32 bits up to k = 133,143; one float32 product with each scale follows.  Rows of codes take a multiple of 16 bytes, zero
// behind the row's end.
#include <string.h>

#include "async_copy.cuh"
#include "int8_rows.cuh"

namespace nnis {

enum { INT8_STORE = 0, INT8_STORE_F32 = 1, INT8_ADD_F32 = 2, INT8_GATED = 3 };

struct Quantize8 {
    const void* x;
    long long x_stride;
    int8_t* codes;
    float* scales;
    int rows, k, kp;
};

// A CTA a row.
template <typename T, bool QUADS>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const __grid_constant__ Quantize8 p) {
    __shared__ uint32_t tops[4];
    pdl_wait();
    pdl_launch_dependents();
    const T* x = reinterpret_cast<const T*>(p.x) + (size_t)blockIdx.x * p.x_stride;
    uint32_t top = 0;
    if (QUADS) {
        for (int i = threadIdx.x * 4; i < p.k; i += 512) {
            const float4 v = load4(x + i);
            top = max(top, max(max(magnitude_bits(v.x), magnitude_bits(v.y)), max(magnitude_bits(v.z), magnitude_bits(v.w))));
        }
    } else {
        for (int i = threadIdx.x; i < p.k; i += 128) top = max(top, magnitude_bits(to_float(x[i])));
    }
    top = group_max<32>(top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const RowScale r = row_scale(top);
    int8_t* codes = p.codes + (size_t)blockIdx.x * p.kp;
    for (int i = threadIdx.x * 4; i < p.kp; i += 512) {
        int c[4] = {0, 0, 0, 0};
        if (QUADS) {
            if (i < p.k) {
                const float4 v = load4(x + i);
                c[0] = row_code(v.x, r.inverse);
                c[1] = row_code(v.y, r.inverse);
                c[2] = row_code(v.z, r.inverse);
                c[3] = row_code(v.w, r.inverse);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < p.k) c[j] = row_code(to_float(x[i + j]), r.inverse);
        }
        *reinterpret_cast<uint32_t*>(codes + i) = pack_codes(c[0], c[1], c[2], c[3]);
    }
    if (threadIdx.x == 0) p.scales[blockIdx.x] = r.scale;
}

struct Linear8 {
    const int8_t *x, *w;
    const float *xs, *ws, *bias;
    void* out;
    int m, n, kp;  // n: columns of the output; a gated product's w has 2 n rows, gate before up
};

__device__ __forceinline__ float silu_gate(float gate, float up) { return __fdividef(gate, 1.0f + __expf(-gate)) * up; }

template <typename T, int MODE>
__device__ __forceinline__ void put_value(void* out, size_t at, float y) {
    if (MODE == INT8_STORE || MODE == INT8_GATED) reinterpret_cast<T*>(out)[at] = from_float<T>(y);
    else if (MODE == INT8_STORE_F32) reinterpret_cast<float*>(out)[at] = y;
    else reinterpret_cast<float*>(out)[at] += y;
}

// Tiles of 64 x 64 outputs on the CUDA cores, four codes a product.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) linear_int8_dots_kernel(const __grid_constant__ Linear8 p) {
    constexpr int NB = MODE == INT8_GATED ? 2 : 1;
    __shared__ uint32_t xs[64][17], ws[NB][64][17];
    pdl_wait();
    pdl_launch_dependents();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    int acc[NB][4][4] = {};
    for (int k0 = 0; k0 < p.kp; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i >> 4, c = i & 15;
            const bool in = k0 + c * 4 < p.kp;
            xs[r][c] = in && m0 + r < p.m ? *reinterpret_cast<const uint32_t*>(p.x + (size_t)(m0 + r) * p.kp + k0 + c * 4) : 0u;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                ws[b][r][c] = in && n0 + r < p.n
                    ? *reinterpret_cast<const uint32_t*>(p.w + ((size_t)b * p.n + n0 + r) * p.kp + k0 + c * 4) : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[b][i][j] = __dp4a((int)xs[ty * 4 + i][c], (int)ws[b][tx + 16 * j][c], acc[b][i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m >= p.m || n >= p.n) continue;
            float y[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const size_t row = (size_t)b * p.n + n;
                y[b] = (float)acc[b][i][j] * p.xs[m] * p.ws[row] + (p.bias ? p.bias[row] : 0.f);
            }
            put_value<T, MODE>(p.out, (size_t)m * p.n + n, NB == 2 ? silu_gate(y[0], y[NB - 1]) : y[0]);
        }
}

template <typename T>
static cudaError_t launch_dots(const Linear8& p, int mode, cudaStream_t stream) {
    const dim3 grid((unsigned)((p.n + 63) / 64), (unsigned)((p.m + 63) / 64));
    auto kernel = mode == INT8_STORE ? linear_int8_dots_kernel<T, INT8_STORE>
                  : mode == INT8_STORE_F32 ? linear_int8_dots_kernel<T, INT8_STORE_F32>
                  : mode == INT8_ADD_F32 ? linear_int8_dots_kernel<T, INT8_ADD_F32> : linear_int8_dots_kernel<T, INT8_GATED>;
    return launch_dependent(kernel, grid, 256, 0, stream, p);
}

template <typename T>
static cudaError_t launch_quantize(const Quantize8& p, cudaStream_t stream) {
    const bool quads = p.k % 4 == 0 && p.x_stride % 4 == 0 && (uintptr_t)p.x % (4 * sizeof(T)) == 0;
    return launch_dependent(quads ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, (unsigned)p.rows, 128, 0, stream, p);
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

// x [m, k] (rows `x_stride` apart) is put into `codes` [m, kp] and `scales` [m], w [n (gated: 2 n), kp] codes, ws their scales, bias
// float32 like ws or null, out [m, n]: `dtype` (x's) in the modes 0 (store) and 3 (gated: silu(first half of w's rows) * the
// second), float32 in 1 (store) and 2 (add).
struct Linear8Call {
    const void *x, *w;
    const float *ws, *bias;
    void *out, *codes;
    float* scales;
    int x_stride, m, n, k, mode, dtype;
    cudaStream_t stream;
};
NNIS_API int nnis_linear_int8(const void* call) {
    using namespace nnis;
    Linear8Call c;
    memcpy(&c, call, sizeof c);
    const auto [x, w, ws, bias, out, codes, scales, x_stride, m, n, k, mode, dtype, stream] = c;
    const int kp = (k + 15) / 16 * 16;
    if (!x || !w || !ws || !out || !codes || !scales || m <= 0 || n <= 0 || k <= 0 || x_stride < k || mode < 0 || mode > 3)
        return NNIS_ERR_ARGUMENT;
    if (k > 133136 || (m + 63) / 64 > 65535 || (dtype != NNIS_DTYPE_F32 && dtype != NNIS_DTYPE_BF16)) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)codes | (uintptr_t)w) % 16) return NNIS_ERR_ALIGNMENT;
    const Quantize8 q{x, x_stride, (int8_t*)codes, scales, m, k, kp};
    const cudaError_t e = dtype == NNIS_DTYPE_F32 ? launch_quantize<float>(q, stream) : launch_quantize<bf16>(q, stream);
    if (e != cudaSuccess) return (int)e;
    const Linear8 p{(const int8_t*)codes, (const int8_t*)w, scales, ws, bias, out, m, n, kp};
    return (int)(dtype == NNIS_DTYPE_F32 ? launch_dots<float>(p, mode, stream) : launch_dots<bf16>(p, mode, stream));
}
