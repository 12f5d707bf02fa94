// The cache of keys and values held in 8 bits: written as the step's rows are rotated, and read back.
//
// Codes lie as the 16-bit cache's values do, [pages, kv_heads, page_size, d], and every position of a page's head has a scale,
// [pages, kv_heads, page_size] float32 (int8_rows.cuh).  A scale per position, not per block of positions: a block's scale is
// known when its last position is, so the positions before would have to be coded again whenever a larger one comes, and a
// position's codes would depend on what was written (and perhaps taken back) after it.  This way a sequence's cache is the
// same however its tokens were dealt to steps, forked, drafted or truncated; it costs 4 bytes beside 64 or 128.
#include <string.h>

#include "async_copy.cuh"
#include "int8_rows.cuh"

namespace nnis {

struct RopeStore8 {
    const void* qkv;       // [n, (nq + 2 nkv) d]
    void* q;               // [n, nq d]: the rotated queries
    const int *token_pos, *token_seq, *page_table;
    int table_rows, table_cols;
    const float *cos_t, *sin_t;  // [angle_rows, d / 2], or null: nothing is rotated
    int angle_rows;
    int8_t *k, *v;
    float *k_scales, *v_scales;
    int pages, n, nq, nkv, d, page_size;
};

// A pair of values that turn together, each product and sum rounded by itself (no contraction: what is rounded to 8 bits
// next would otherwise hang on the compiler's choice).
__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// The place of a token's row in the store (without the head), or -1 where it has none.
__device__ __forceinline__ long long store_page(const RopeStore8& p, int n, int pos) {
    const int seq = p.token_seq[n], col = pos / p.page_size;
    if (seq < 0 || seq >= p.table_rows || col >= p.table_cols) return -1;
    const int page = p.page_table[(size_t)seq * p.table_cols + col];
    return page >= 0 && page < p.pages ? page : -1;
}

// G lanes a (token, head): a lane four values of the head's first half and the four that turn with them.  Heads of a multiple
// of 8 values.
template <typename T, int G>
__global__ void __launch_bounds__(256) rope_store_int8_kernel(const __grid_constant__ RopeStore8 p) {
    pdl_wait();
    pdl_launch_dependents();
    const int heads = p.nq + 2 * p.nkv, half = p.d >> 1;
    const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    const int j = (threadIdx.x % G) * 4;
    const int n = (int)(unit / heads), head = (int)(unit - (long long)n * heads);
    const int pos = n < p.n ? p.token_pos[n] : -1;
    const bool lives = pos >= 0 && !(p.cos_t && pos >= p.angle_rows), mine = lives && j < half;
    float4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (mine) {
        const T* row = reinterpret_cast<const T*>(p.qkv) + ((size_t)n * heads + head) * p.d + j;
        a = load4(row);
        b = load4(row + half);
        if (p.cos_t && head < p.nq + p.nkv) {
            const float4 c = load4(p.cos_t + (size_t)pos * half + j), s = load4(p.sin_t + (size_t)pos * half + j);
            rotate_pair(a.x, b.x, c.x, s.x);
            rotate_pair(a.y, b.y, c.y, s.y);
            rotate_pair(a.z, b.z, c.z, s.z);
            rotate_pair(a.w, b.w, c.w, s.w);
        }
    }
    if (mine && head < p.nq) {
        T* out = reinterpret_cast<T*>(p.q) + ((size_t)n * p.nq + head) * p.d + j;
        store4(out, a);
        store4(out + half, b);
    }
    // (a warp may hold heads of q and of k: all its lanes take part in the maximum)
    float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = to_float(from_float<T>(x[i]));  // (as a cache of the operands' type holds it)
        top = max(top, magnitude_bits(x[i]));
    }
    top = group_max<G>(top);
    if (!lives || head < p.nq) return;
    const long long page = store_page(p, n, pos);
    if (page < 0 || !mine) return;
    const RowScale r = row_scale(top);
    const bool value = head >= p.nq + p.nkv;
    const size_t at = ((size_t)page * p.nkv + (head - p.nq - (value ? p.nkv : 0))) * p.page_size + pos % p.page_size;
    int8_t* codes = (value ? p.v : p.k) + at * p.d + j;
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = row_code(x[i], r.inverse);
    *reinterpret_cast<uint32_t*>(codes) = pack_codes(c[0], c[1], c[2], c[3]);
    *reinterpret_cast<uint32_t*>(codes + half) = pack_codes(c[4], c[5], c[6], c[7]);
    if (j == 0) (value ? p.v_scales : p.k_scales)[at] = r.scale;
}

// The same for any even head size up to 256: a warp a (token, head), a value and the one that turns with it at a time.
template <typename T>
__global__ void __launch_bounds__(256) rope_store_int8_any_kernel(const __grid_constant__ RopeStore8 p) {
    pdl_wait();
    pdl_launch_dependents();
    const int heads = p.nq + 2 * p.nkv, half = p.d >> 1, lane = threadIdx.x & 31;
    const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
    const int n = (int)(unit / heads), head = (int)(unit - (long long)n * heads);
    const int pos = n < p.n ? p.token_pos[n] : -1;
    if (pos < 0 || (p.cos_t && pos >= p.angle_rows)) return;  // (whole warps)
    const T* row = reinterpret_cast<const T*>(p.qkv) + ((size_t)n * heads + head) * p.d;
    float a[4], b[4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = lane + 32 * i;
        a[i] = b[i] = 0.f;
        if (j >= half) continue;
        a[i] = to_float(row[j]);
        b[i] = to_float(row[j + half]);
        if (p.cos_t && head < p.nq + p.nkv)
            rotate_pair(a[i], b[i], p.cos_t[(size_t)pos * half + j], p.sin_t[(size_t)pos * half + j]);
        if (head < p.nq) {
            T* out = reinterpret_cast<T*>(p.q) + ((size_t)n * p.nq + head) * p.d + j;
            out[0] = from_float<T>(a[i]);
            out[half] = from_float<T>(b[i]);
        }
        a[i] = to_float(from_float<T>(a[i]));
        b[i] = to_float(from_float<T>(b[i]));
        top = max(top, max(magnitude_bits(a[i]), magnitude_bits(b[i])));
    }
    if (head < p.nq) return;
    top = group_max<32>(top);
    const long long page = store_page(p, n, pos);
    if (page < 0) return;
    const RowScale r = row_scale(top);
    const bool value = head >= p.nq + p.nkv;
    const size_t at = ((size_t)page * p.nkv + (head - p.nq - (value ? p.nkv : 0))) * p.page_size + pos % p.page_size;
    int8_t* codes = (value ? p.v : p.k) + at * p.d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = lane + 32 * i;
        if (j >= half) continue;
        codes[j] = (int8_t)row_code(a[i], r.inverse);
        codes[j + half] = (int8_t)row_code(b[i], r.inverse);
    }
    if (lane == 0) (value ? p.v_scales : p.k_scales)[at] = r.scale;
}

struct ReadPages8 {
    const int8_t *k, *v;
    const float *k_scales, *v_scales;
    const int *page_table, *local_table;
    int table_cols, local_cols;
    void *k_out, *v_out;  // [out_pages, kv_heads, page_size, d]
    int pages, out_pages, kv_heads, page_size, d;
};

// A CTA a page's head, of keys or of values: blockIdx.x = entry of the local table, y = head, z = which.
template <typename T, bool QUADS>
__global__ void __launch_bounds__(256) read_pages_int8_kernel(const __grid_constant__ ReadPages8 p) {
    pdl_wait();
    pdl_launch_dependents();
    const int seq = blockIdx.x / p.local_cols, col = blockIdx.x - seq * p.local_cols;
    const int to = p.local_table[blockIdx.x];
    if (to < 0 || to >= p.out_pages || col >= p.table_cols) return;
    const int page = p.page_table[(size_t)seq * p.table_cols + col];
    if (page < 0 || page >= p.pages) return;
    const size_t from = ((size_t)page * p.kv_heads + blockIdx.y) * p.page_size;
    const int8_t* codes = (blockIdx.z ? p.v : p.k) + from * p.d;
    const float* scales = (blockIdx.z ? p.v_scales : p.k_scales) + from;
    T* out = reinterpret_cast<T*>(blockIdx.z ? p.v_out : p.k_out) + ((size_t)to * p.kv_heads + blockIdx.y) * p.page_size * p.d;
    const int count = p.page_size * p.d;
    if (QUADS) {  // (four values lie in one row)
        for (int i = threadIdx.x * 4; i < count; i += 1024) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + i);
            const float s = scales[i / p.d];
            store4(out + i, make_float4(code_value(w, 0) * s, code_value(w, 1) * s, code_value(w, 2) * s, code_value(w, 3) * s));
        }
    } else {
        for (int i = threadIdx.x; i < count; i += 256) out[i] = from_float<T>((float)codes[i] * scales[i / p.d]);
    }
}

template <typename T>
static cudaError_t launch_rope_store8(const RopeStore8& p, cudaStream_t stream) {
    const long long units = (long long)p.n * (p.nq + 2 * p.nkv);
    const int half = p.d / 2;
    const bool quads = p.d % 8 == 0;
    int g = 1;
    while (g * 4 < half) g *= 2;
    const long long blocks = (units * (quads ? g : 32) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    auto kernel = !quads ? rope_store_int8_any_kernel<T>
                  : g == 1 ? rope_store_int8_kernel<T, 1> : g == 2 ? rope_store_int8_kernel<T, 2>
                  : g == 4 ? rope_store_int8_kernel<T, 4> : g == 8 ? rope_store_int8_kernel<T, 8>
                  : g == 16 ? rope_store_int8_kernel<T, 16> : rope_store_int8_kernel<T, 32>;
    return launch_dependent(kernel, (unsigned)blocks, 256, 0, stream, p);
}

}  // namespace nnis

// Rows of q, k and v: q and k rotated (cos_t null: as they are), q to `q`, k and v into the store as codes and scales.  A row at
// position -1 (padding), or beyond the angles, writes nothing; one whose page the table does not name stores nothing.
struct RopeStore8Call {
    const void* qkv;
    void* q;
    const int *token_pos, *token_seq, *page_table;
    const float *cos_t, *sin_t;
    void *k, *v;
    float *k_scales, *v_scales;
    int dtype, table_rows, table_cols, angle_rows, pages, n, nq, nkv, d, page_size;
    cudaStream_t stream;
};
NNIS_API int nnis_rope_store_int8(const void* call) {
    using namespace nnis;
    RopeStore8Call c;
    memcpy(&c, call, sizeof c);
    const auto [qkv, q, token_pos, token_seq, page_table, cos_t, sin_t, k, v, k_scales, v_scales, dtype, table_rows, table_cols,
                angle_rows, pages, n, nq, nkv, d, page_size, stream] = c;
    if (n <= 0 || nq <= 0 || nkv <= 0 || table_rows <= 0 || table_cols <= 0 || pages <= 0 || page_size <= 0 || !qkv || !q || !k ||
        !v || !k_scales || !v_scales || !page_table || !cos_t != !sin_t)
        return NNIS_ERR_ARGUMENT;
    if (d < 2 || d % 2 || d > 256) return NNIS_ERR_UNSUPPORTED;
    const uintptr_t rows = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)cos_t | (uintptr_t)sin_t, codes = (uintptr_t)k | (uintptr_t)v;
    if (rows % 16 || codes % 4) return NNIS_ERR_ALIGNMENT;
    const RopeStore8 p{qkv, q, token_pos, token_seq, page_table, table_rows, table_cols, cos_t, sin_t, angle_rows,
                       (int8_t*)k, (int8_t*)v, k_scales, v_scales, pages, n, nq, nkv, d, page_size};
    if (dtype == NNIS_DTYPE_F32) return (int)launch_rope_store8<float>(p, stream);
    if (dtype == NNIS_DTYPE_BF16) return (int)launch_rope_store8<bf16>(p, stream);
    return NNIS_ERR_UNSUPPORTED;
}

// Pages read back: for every sequence (row) and column of `local_table` that names a place, that page of the outputs becomes
// the values of the page that `page_table` names in the same row and column.
struct ReadPages8Call {
    const void *k, *v;
    const float *k_scales, *v_scales;
    const int *page_table, *local_table;
    void *k_out, *v_out;
    int table_cols, seqs, local_cols, dtype, pages, out_pages, kv_heads, page_size, d;
    cudaStream_t stream;
};
NNIS_API int nnis_read_pages_int8(const void* call) {
    using namespace nnis;
    ReadPages8Call c;
    memcpy(&c, call, sizeof c);
    const auto [k, v, k_scales, v_scales, page_table, local_table, k_out, v_out, table_cols, seqs, local_cols, dtype, pages, out_pages,
                kv_heads, page_size, d, stream] = c;
    if (!k || !v || !k_scales || !v_scales || !page_table || !local_table || !k_out || !v_out || seqs <= 0 || table_cols <= 0 ||
        local_cols <= 0 || pages <= 0 || out_pages <= 0 || kv_heads <= 0 || page_size <= 0 || d <= 0)
        return NNIS_ERR_ARGUMENT;
    if (kv_heads > 65535 || (long long)seqs * local_cols > 0x7fffffffLL || (long long)page_size * d > 0x3fffffff)
        return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)k | (uintptr_t)v) % 16) return NNIS_ERR_ALIGNMENT;
    const ReadPages8 p{(const int8_t*)k, (const int8_t*)v, k_scales, v_scales, page_table, local_table, table_cols, local_cols,
                       k_out, v_out, pages, out_pages, kv_heads, page_size, d};
    const dim3 grid((unsigned)(seqs * local_cols), (unsigned)kv_heads, 2);
    const bool quads = d % 4 == 0;
    if (dtype == NNIS_DTYPE_F32)
        return (int)launch_dependent(quads ? read_pages_int8_kernel<float, true> : read_pages_int8_kernel<float, false>, grid, 256, 0,
                                     stream, p);
    if (dtype == NNIS_DTYPE_BF16)
        return (int)launch_dependent(quads ? read_pages_int8_kernel<bf16, true> : read_pages_int8_kernel<bf16, false>, grid, 256, 0,
                                     stream, p);
    return NNIS_ERR_UNSUPPORTED;
}
