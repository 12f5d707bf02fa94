// What the products of 8-bit codes are given, and what becomes of their sums.
#pragma once

#include "common.cuh"

namespace nnis {

enum { INT8_STORE = 0, INT8_STORE_F32 = 1, INT8_ADD_F32 = 2, INT8_GATED = 3 };

struct Linear8 {
    const int8_t *x, *w;
    const float *xs, *ws, *bias;
    void* out;
    int* status;
    const void* values;  // x before it is put into codes, rows `x_stride` apart, k values each
    long long x_stride;
    int m, n, kp;  // n: columns of the output; a gated product's w has 2 n rows, gate before up
    int k, out_by_tma;
};
// (a single row's call takes the host 3.5 us with 96 bytes of arguments, 3.9 with 104)
static_assert(sizeof(Linear8) <= 96, "a launch's arguments");

// silu(gate) * up with the two approximate instructions (2^x and 1 / x, relative error about 1e-7 each)
__device__ __forceinline__ float silu_gate(float gate, float up) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(gate * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return gate * r * up;
}

// The product of few rows (`fused`: rows that are still values, where the kernel takes them as such); of many (tcgen05).  `f32`: the operands'
// type is float32.
bool linear_int8_may_fuse(const Linear8& p, bool f32);
cudaError_t linear_int8_few(const Linear8& p, int mode, bool f32, bool fused, int sms, cudaStream_t stream);
int linear_int8_tc(Linear8 p, int mode, bool f32, int sms, cudaStream_t stream);

}  // namespace nnis
