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

// The page of a position in the store, or -1 where it has none.
__device__ __forceinline__ long long store_page(const RopeStore8& p, int seq, int pos) {
    const int col = pos / p.page_size;
    if (seq < 0 || seq >= p.table_rows || col >= p.table_cols) return -1;
    const int page = p.page_table[(size_t)seq * p.table_cols + col];
    return page >= 0 && page < p.pages ? page : -1;
}

// Eight consecutive values of a head as they are held: bfloat16 in pairs.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float x[8];
    __device__ __forceinline__ void load(const float* p) {
        const float4 a = load4(p), b = load4(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    __device__ __forceinline__ void store(float* p) const {
        store4(p, make_float4(x[0], x[1], x[2], x[3]));
        store4(p + 4, make_float4(x[4], x[5], x[6], x[7]));
    }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ void set_pair(int i, float a, float b) { x[2 * i] = a; x[2 * i + 1] = b; }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t = max(t, magnitude_bits(x[i]));
        return t;
    }
};
template <> struct Eight<bf16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const bf16* p) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
    __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
    __device__ __forceinline__ void set_pair(int i, float a, float b) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(a, b);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    __device__ __forceinline__ uint32_t top() const {  // (the largest of each half, then of the two)
        const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        return max(m & 0xffff0000u, m << 16);
    }
};

// Heads of a multiple of 16 values, bound by bytes: G lanes take H heads of a token, a lane eight values of a head's first half and the eight
// that turn with them, and keep the position's angles for all of them; lane i of the G divides for head i.  H = 4 where rows are
// many, 1 where the launch's own time counts.  6,022 rows of 96 heads of 64, bfloat16: 26.4 us for 19.0 of bytes; with as many CTAs an SM as 84
// registers leave 28.5, with 64 registers 26.9.
template <typename T, int G, int H>
__global__ void __launch_bounds__(128, sizeof(T) == 2 && H == 4 ? 7 : 1) rope_store_int8_kernel(const __grid_constant__ RopeStore8 p) {
    pdl_wait();
    pdl_launch_dependents();
    const int heads = p.nq + 2 * p.nkv, half = p.d >> 1, runs = (heads + H - 1) / H;
    const unsigned unit = blockIdx.x * (128u / G) + threadIdx.x / G;
    const int sub = threadIdx.x % G, j = sub * 8;
    const int n = (int)(unit / (unsigned)runs), first = (int)(unit - (unsigned)n * runs) * H;
    // (the row's values, its position and its sequence are asked for together; angles and page when those are there)
    const bool there = n < p.n;
    const int pos = there ? p.token_pos[n] : -1, seq = there ? p.token_seq[n] : -1;
    Eight<T> a[H], b[H];
    const T* row = reinterpret_cast<const T*>(p.qkv) + ((size_t)n * heads + first) * p.d + j;
#pragma unroll
    for (int i = 0; i < H; ++i) {
        a[i] = {};
        b[i] = {};
        if (there && j < half && first + i < heads) {
            a[i].load(row + (size_t)i * p.d);
            b[i].load(row + (size_t)i * p.d + half);
        }
    }
    const bool lives = pos >= 0 && !(p.cos_t && pos >= p.angle_rows), mine = lives && j < half;
    const long long page = lives && first + H > p.nq ? store_page(p, seq, pos) : -1;
    if (mine && p.cos_t && first < p.nq + p.nkv) {
        Eight<float> c, s;
        c.load(p.cos_t + (size_t)pos * half + j);
        s.load(p.sin_t + (size_t)pos * half + j);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (first + i >= p.nq + p.nkv) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x0 = a[i].get(2 * e), y0 = b[i].get(2 * e), x1 = a[i].get(2 * e + 1), y1 = b[i].get(2 * e + 1);
                rotate_pair(x0, y0, c.x[2 * e], s.x[2 * e]);
                rotate_pair(x1, y1, c.x[2 * e + 1], s.x[2 * e + 1]);
                a[i].set_pair(e, x0, x1);  // (rounded as a cache of the operands' type holds it)
                b[i].set_pair(e, y0, y1);
            }
        }
    }
    if (mine) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (first + i >= p.nq) break;
            T* out = reinterpret_cast<T*>(p.q) + ((size_t)n * p.nq + first + i) * p.d + j;
            a[i].store(out);
            b[i].store(out + half);
        }
    }
    if (!__any_sync(0xffffffffu, page >= 0)) return;
    uint32_t my_top = 0;
#pragma unroll
    for (int i = 0; i < H; ++i) {
        // (all lanes of a warp take part in the maximum, whatever heads they hold)
        const uint32_t top = group_max<G>(max(a[i].top(), b[i].top()));
        if (i == sub) my_top = top;
    }
    const RowScale r = row_scale(my_top);
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const int head = first + i;
        const float inverse = __shfl_sync(0xffffffffu, r.inverse, i % G, G), scale = __shfl_sync(0xffffffffu, r.scale, i % G, G);
        if (!mine || head >= heads || head < p.nq || page < 0) continue;
        const bool value = head >= p.nq + p.nkv;
        const size_t at = ((size_t)page * p.nkv + (head - p.nq - (value ? p.nkv : 0))) * p.page_size + pos % p.page_size;
        int8_t* codes = (value ? p.v : p.k) + at * p.d + j;
        const uint32_t good = good_row(scale);
        *reinterpret_cast<uint2*>(codes) =
            make_uint2(code_word(a[i].get(0), a[i].get(1), a[i].get(2), a[i].get(3), inverse, good),
                       code_word(a[i].get(4), a[i].get(5), a[i].get(6), a[i].get(7), inverse, good));
        *reinterpret_cast<uint2*>(codes + half) =
            make_uint2(code_word(b[i].get(0), b[i].get(1), b[i].get(2), b[i].get(3), inverse, good),
                       code_word(b[i].get(4), b[i].get(5), b[i].get(6), b[i].get(7), inverse, good));
        if (sub == 0) (value ? p.v_scales : p.k_scales)[at] = scale;
    }
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
    const long long page = store_page(p, p.token_seq[n], pos);
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

// A page's codes lie in one run over its heads, and so do its values.  blockIdx.x = entry of the local table, y = a share of the page, z =
// keys or values.  WIDE: heads of a multiple of 16 values; a thread takes as many codes of a row as are 16 bytes of values, so that a
// warp's loads and stores are runs without gaps.
constexpr int kReadAhead = 8;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(128) read_pages_int8_kernel(const __grid_constant__ ReadPages8 p) {
    pdl_wait();
    pdl_launch_dependents();
    const int seq = blockIdx.x / p.local_cols, col = blockIdx.x - seq * p.local_cols;
    // (both asked for at once)
    const int to = p.local_table[blockIdx.x], page = col < p.table_cols ? p.page_table[(size_t)seq * p.table_cols + col] : -1;
    if (to < 0 || to >= p.out_pages || page < 0 || page >= p.pages) return;
    const int rows = p.kv_heads * p.page_size;
    const int8_t* codes = (blockIdx.z ? p.v : p.k) + (size_t)page * rows * p.d;
    const float* scales = (blockIdx.z ? p.v_scales : p.k_scales) + (size_t)page * rows;
    T* out = reinterpret_cast<T*>(blockIdx.z ? p.v_out : p.k_out) + (size_t)to * rows * p.d;
    if (WIDE) {
        constexpr int kCodes = 16 / sizeof(T);
        const unsigned per = (unsigned)p.d / kCodes, count = (unsigned)rows * per, step = gridDim.y * 128u;
        for (unsigned at = blockIdx.y * 128u + threadIdx.x; at < count; at += kReadAhead * step) {
            uint2 w[kReadAhead];
            float s[kReadAhead];
#pragma unroll
            for (int i = 0; i < kReadAhead; ++i)
                if (at + i * step < count) {
                    const int8_t* from = codes + (size_t)(at + i * step) * kCodes;
                    w[i].x = *reinterpret_cast<const uint32_t*>(from);
                    if constexpr (kCodes == 8) w[i] = *reinterpret_cast<const uint2*>(from);
                    s[i] = scales[(at + i * step) / per];
                }
#pragma unroll
            for (int i = 0; i < kReadAhead; ++i)
                if (at + i * step < count) {
                    T* to_out = out + (size_t)(at + i * step) * kCodes;
                    if constexpr (kCodes == 8) {
                        Eight<bf16> v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t word = e < 2 ? w[i].x : w[i].y;
                            v.set_pair(e, code_value(word, 2 * e % 4) * s[i], code_value(word, 2 * e % 4 + 1) * s[i]);
                        }
                        v.store(to_out);
                    } else {
                        store4(to_out, make_float4(code_value(w[i].x, 0) * s[i], code_value(w[i].x, 1) * s[i], code_value(w[i].x, 2) * s[i],
                                                   code_value(w[i].x, 3) * s[i]));
                    }
                }
        }
    } else {
        const unsigned count = (unsigned)rows * p.d;
        for (unsigned i = blockIdx.y * 128u + threadIdx.x; i < count; i += gridDim.y * 128u)
            out[i] = from_float<T>((float)codes[i] * scales[i / (unsigned)p.d]);
    }
}

template <typename T, int H>
static cudaError_t launch_rope_heads8(const RopeStore8& p, cudaStream_t stream) {
    const int heads = p.nq + 2 * p.nkv, half = p.d / 2;
    int g = H;  // (a lane for each head's division)
    while (g * 8 < half) g *= 2;
    const long long units = (long long)p.n * ((heads + H - 1) / H), blocks = (units * g + 127) / 128;
    if (units >= 1LL << 32 || blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if constexpr (H == 1) {
        if (g == 1) return launch_dependent(rope_store_int8_kernel<T, 1, 1>, (unsigned)blocks, 128, 0, stream, p);
        if (g == 2) return launch_dependent(rope_store_int8_kernel<T, 2, 1>, (unsigned)blocks, 128, 0, stream, p);
    }
    auto kernel = g == 4 ? rope_store_int8_kernel<T, 4, H> : g == 8 ? rope_store_int8_kernel<T, 8, H> : rope_store_int8_kernel<T, 16, H>;
    return launch_dependent(kernel, (unsigned)blocks, 128, 0, stream, p);
}

template <typename T>
static cudaError_t launch_rope_store8(const RopeStore8& p, cudaStream_t stream) {
    const int heads = p.nq + 2 * p.nkv;
    if (p.d % 16 == 0)
        return (long long)p.n * heads * p.d >= 1 << 21 ? launch_rope_heads8<T, 4>(p, stream) : launch_rope_heads8<T, 1>(p, stream);
    const long long blocks = ((long long)p.n * heads * 32 + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    auto kernel = rope_store_int8_any_kernel<T>;
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
        !v || !k_scales || !v_scales || !token_pos || !token_seq || !page_table || !cos_t != !sin_t)
        return NNIS_ERR_ARGUMENT;
    if (d < 2 || d % 2 || d > 256) return NNIS_ERR_UNSUPPORTED;
    const uintptr_t rows = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)cos_t | (uintptr_t)sin_t, codes = (uintptr_t)k | (uintptr_t)v;
    if (rows % 16 || codes % 16) return NNIS_ERR_ALIGNMENT;
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
    if ((long long)seqs * local_cols > 0x7fffffffLL || (long long)kv_heads * page_size * d > 0x3fffffff) return NNIS_ERR_UNSUPPORTED;
    if (((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)k | (uintptr_t)v) % 16) return NNIS_ERR_ALIGNMENT;
    const ReadPages8 p{(const int8_t*)k, (const int8_t*)v, k_scales, v_scales, page_table, local_table, table_cols, local_cols,
                       k_out, v_out, pages, out_pages, kv_heads, page_size, d};
    // (a CTA 8,192 codes of bfloat16, and fewer where there are few pages)
    const bool wide = d % 16 == 0;
    const long long codes = (long long)kv_heads * page_size * d;
    const int run = (dtype == NNIS_DTYPE_F32 ? 4 : 8) * 128;
    long long share = (codes + run * kReadAhead - 1) / (run * kReadAhead);
    const long long fill = (8LL * device_sms() + 2LL * seqs * local_cols - 1) / (2LL * seqs * local_cols), most = (codes + run - 1) / run;
    if (share < fill) share = fill < most ? fill : most;
    if (share > 65535) share = 65535;
    const dim3 grid((unsigned)(seqs * local_cols), (unsigned)share, 2);
    if (dtype == NNIS_DTYPE_F32)
        return (int)launch_dependent(wide ? read_pages_int8_kernel<float, true> : read_pages_int8_kernel<float, false>, grid, 128, 0,
                                     stream, p);
    if (dtype == NNIS_DTYPE_BF16)
        return (int)launch_dependent(wide ? read_pages_int8_kernel<bf16, true> : read_pages_int8_kernel<bf16, false>, grid, 128, 0,
                                     stream, p);
    return NNIS_ERR_UNSUPPORTED;
}
