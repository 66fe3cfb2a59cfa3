// Microscaled 4-bit floating point: a row is cut into blocks of 32 numbers, a block is one scale 2^(s - 127) (a byte s) and 32
// codes of 4 bits: sign, two bits of exponent, one of mantissa, for 0, 1/2, 1, 3/2, 2, 3, 4, 6.  Two codes lie in a byte, the first in
// its low half; a row takes ceil(K / 32) blocks of 16 bytes, what is behind K is code 0.
//
//   e = floor(log2(max |x|)),  s = max(e - 2, -127) + 127,  code = the nearest of x / 2^(s - 127), ties to the even code, beyond 6: 6
//
// (2 is the exponent of the largest code.)  A block of zeros has s = 0; a block with an infinity or a NaN has s = 255, which makes
// all its numbers NaN.  The division is exact and the conversion instruction's rounding is the one above, so that the codes do not
// depend on how this is computed.
//
// Bound by memory: a lane takes eight numbers, four lanes a block; the largest is found by two exchanges among the four.  24576 rows of 4096
// bfloat16 numbers, 201 MB, take 43 to 50 us to codes (5.1 to 5.9 TB/s) and 36 to 42 us back; 77 rows of 2570 a launch's 3 us each way.  Rows that are not
// whole blocks go number by number: 24576 of 4098 119 us to codes and 134 back in bfloat16, 170 and 252 in float32 (2.7 to 1.8 TB/s).
#include "common.h"

// The scale's byte of a block whose largest magnitude has these bits (sign cleared).
__device__ __forceinline__ int mxfp4_scale_of(uint32_t bits) {
    if (bits >= 0x7f800000u) return 255;
    int e = (int)(bits >> 23);                                      // biased exponent; the numbers below 2^-126 have 0
    return e > 2 ? e - 2 : 0;                                       // (floor(log2) - 2 is below -127 for all with e <= 2: 2^(2 - 127) gives 0 too)
}

// Eight numbers of one lane to eight codes, the first in the lowest bits; the block is the four lanes 4 i .. 4 i + 3.
__device__ __forceinline__ uint32_t mxfp4_encode(const float (&v)[8], int& s) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    s = mxfp4_scale_of(top);
    if (s == 255) return 0;
    const float scale = __uint_as_float((uint32_t)s << 23);         // (the instruction takes the exponent's byte: 0 stands for 2^-127)
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    return c;
}

// WHOLE: K is a multiple of 32 and x begins at a whole 16-byte piece: the rows' blocks lie side by side throughout.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, uint32_t* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, long units, int K, unsigned per_row) {
    const long u = (long)blockIdx.x * 256 + threadIdx.x;            // eight numbers of a block
    if (u >= units) return;                                         // (units is a multiple of 4: a block's lanes leave together)
    float v[8];
    if constexpr (WHOLE) {
        float a[4], b[4];
        Vec4<T>::load(x + u * 8, a);
        Vec4<T>::load(x + u * 8 + 4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        const unsigned row = (unsigned)u / per_row;
        const int k = (int)((unsigned)u - row * per_row) * 8;
        const T* p = x + (long)row * K + k;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? Elem<T>::load(p + i) : 0.f;
    }
    int s;
    codes[u] = mxfp4_encode(v, s);
    if ((u & 3) == 0) scales[u >> 2] = (unsigned char)s;
}

// x [T, K] -> codes [T, ceil(K / 32) * 16] bytes, scales [T, ceil(K / 32)] bytes
extern "C" int qe_mxfp4_quantize(const void* x, void* codes, void* scales, int T, int K, int dtype, hipStream_t stream) {
    QE_REQUIRE(T >= 0 && K > 0, "mxfp4_quantize: bad sizes T=%d K=%d", T, K);
    QE_REQUIRE(dtype == QE_F32 || dtype == QE_BF16, "mxfp4_quantize: unknown element type %d", dtype);
    QE_REQUIRE(((uintptr_t)codes & 3) == 0, "mxfp4_quantize: the codes do not begin at a whole word");
    if (T == 0) return 0;
    const unsigned per_row = (unsigned)((K + 31L) / 32) * 4;
    const long units = (long)T * per_row;
    QE_REQUIRE(units < (1L << 32) - 256, "mxfp4_quantize: %d rows of %d numbers are too many", T, K);
    const bool whole = K % 32 == 0 && ((uintptr_t)x & 15) == 0;
    const unsigned blocks = (unsigned)((units + 255) / 256);
#define QE_GO(T_, W_) mxfp4_quantize_kernel<T_, W_><<<blocks, 256, 0, stream>>>((const T_*)x, (uint32_t*)codes, (unsigned char*)scales, units, K, per_row)
    if (dtype == QE_F32) { if (whole) QE_GO(float, true); else QE_GO(float, false); }
    else { if (whole) QE_GO(bf16_t, true); else QE_GO(bf16_t, false); }
#undef QE_GO
    QE_LAUNCH_CHECK();
    return 0;
}

// The numbers that eight codes stand for.
__device__ __forceinline__ void mxfp4_decode(uint32_t c, int s, float (&v)[8]) {
    typedef __attribute__((ext_vector_type(2))) float float2_t;
    const float scale = __uint_as_float((uint32_t)s << 23);         // (255: the conversion gives NaN)
    const float2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
    const float2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void mxfp4_values_kernel(const uint32_t* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                           T* __restrict__ out, long units, int K, unsigned per_row) {
    const long u = (long)blockIdx.x * 256 + threadIdx.x;
    if (u >= units) return;
    float v[8];
    mxfp4_decode(codes[u], scales[u >> 2], v);
    if constexpr (WHOLE) {
        const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
        Vec4<T>::store(out + u * 8, a);
        Vec4<T>::store(out + u * 8 + 4, b);
    } else {
        const unsigned row = (unsigned)u / per_row;
        const int k = (int)((unsigned)u - row * per_row) * 8;
        T* p = out + (long)row * K + k;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) Elem<T>::store(p + i, v[i]);
    }
}

// codes, scales as above -> out [T, K]
extern "C" int qe_mxfp4_values(const void* codes, const void* scales, void* out, int T, int K, int dtype, hipStream_t stream) {
    QE_REQUIRE(T >= 0 && K > 0, "mxfp4_values: bad sizes T=%d K=%d", T, K);
    QE_REQUIRE(dtype == QE_F32 || dtype == QE_BF16, "mxfp4_values: unknown element type %d", dtype);
    QE_REQUIRE(((uintptr_t)codes & 3) == 0, "mxfp4_values: the codes do not begin at a whole word");
    if (T == 0) return 0;
    const unsigned per_row = (unsigned)((K + 31L) / 32) * 4;
    const long units = (long)T * per_row;
    QE_REQUIRE(units < (1L << 32) - 256, "mxfp4_values: %d rows of %d numbers are too many", T, K);
    const bool whole = K % 32 == 0 && ((uintptr_t)out & 15) == 0;
    const unsigned blocks = (unsigned)((units + 255) / 256);
#define QE_GO(T_, W_) mxfp4_values_kernel<T_, W_><<<blocks, 256, 0, stream>>>((const uint32_t*)codes, (const unsigned char*)scales, (T_*)out, units, K, per_row)
    if (dtype == QE_F32) { if (whole) QE_GO(float, true); else QE_GO(float, false); }
    else { if (whole) QE_GO(bf16_t, true); else QE_GO(bf16_t, false); }
#undef QE_GO
    QE_LAUNCH_CHECK();
    return 0;
}
