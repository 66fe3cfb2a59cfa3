// What the products with 4-bit matrices share: operands, and what becomes of a sum.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(4))) float floatx4_t;
typedef __attribute__((ext_vector_type(16))) float floatx16_t;
typedef __attribute__((ext_vector_type(4))) unsigned int uintx4_t;
typedef __attribute__((ext_vector_type(8))) int intx8_t;

enum { X_BF16 = 0, X_F32 = 1, X_FP4 = 2 };
enum { TAIL_STORE = 0, TAIL_ADD = 1, TAIL_SILU = 2 };

// Eight codes with their block's scale as eight bfloat16.
__device__ __forceinline__ bf16x8_t fp4_to_bf16(uint32_t c, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
    bf16x8_t r;
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = d[0]; r[5] = d[1]; r[6] = e[0]; r[7] = e[1];
    return r;
}

// v = hi + mid + lo, each of at most 8 significant bits (cut, not rounded: nothing overflows); an infinity or a NaN stays in hi alone.
__device__ __forceinline__ void cut_in_three(float v, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
    const uint32_t b = __float_as_uint(v);
    hi = (uint16_t)(b >> 16);
    mid = lo = 0;
    if ((b & 0x7f800000u) == 0x7f800000u) {
        if (b & 0x007fffffu) hi = 0x7fc0;
        return;
    }
    const float r = v - __uint_as_float(b & 0xffff0000u);
    const uint32_t c = __float_as_uint(r);
    mid = (uint16_t)(c >> 16);
    lo = (uint16_t)(__float_as_uint(r - __uint_as_float(c & 0xffff0000u)) >> 16);
}

// The codes of a block of which only the first n numbers count (n < 32): the others 0.
__device__ __forceinline__ uintx4_t first_codes(uintx4_t c, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int here = n - 8 * j;
        if (here < 8) c[j] &= here <= 0 ? 0u : (1u << (4 * here)) - 1u;
    }
    return c;
}

struct Fp4Args {
    const void* x;                  // rows of x (X_FP4: their codes)
    const unsigned char* xs;        // X_FP4: their scales
    const unsigned char* codes;     // [N, blocks * 16]
    const unsigned char* scales;    // [N, blocks]
    const float* bias;              // [N] or null
    void* out;
    int M, N, K, blocks;            // blocks = ceil(K / 32)
    int out_f32;
};

// What becomes of a sum: row m, column n (silu: gate and up of column n of N / 2).
template <int TAIL>
__device__ __forceinline__ void fp4_store(const Fp4Args& a, long m, int n, float v, float up) {
    if (a.bias) {
        v += a.bias[n];
        if constexpr (TAIL == TAIL_SILU) up += a.bias[a.N / 2 + n];
    }
    const long at = m * (TAIL == TAIL_SILU ? a.N / 2 : a.N) + n;
    if constexpr (TAIL == TAIL_SILU) v = v / (1.f + expf(-v)) * up;
    if constexpr (TAIL == TAIL_ADD) ((float*)a.out)[at] += v;
    else if (a.out_f32) ((float*)a.out)[at] = v;
    else ((bf16_t*)a.out)[at] = float_to_bf16(v);
}

// gemm_mxfp4_tiles.hip: the products of many rows of 16 or 32 bits; the bytes of workspace that these sizes take
bool fp4_tiles_take(int M, int N, int K, int x_kind);
long fp4_tiles_workspace(int M, int N, int K, int x_kind, bool aligned);
int fp4_tiles(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream);
