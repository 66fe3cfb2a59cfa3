// Matrix product with a 4-bit matrix: out[M, N] = x[M, K] . V[N, K]^T (+ bias), V the numbers that codes and scales stand for
// (see mxfp4.hip: blocks of 32 along K).  x is bfloat16, float32 or itself in 4 bits.
//
// A lane of the matrix instruction takes a whole block of a row of V, 16 bytes of codes with their scale, and the same block of a row
// of x.  The numbers of a block are products of at most two significant bits with a power of two, so they are exact in bfloat16: with
// bfloat16 x the codes become bfloat16 in registers (an instruction for two of them, the scale included) and v_mfma_f32_16x16x32_bf16
// sums in 32-bit.  Numbers of 32-bit x are cut into three bfloat16 (8 + 8 + 8 bits, exact) and multiplied by three instructions.  With
// both sides in 4 bits the codes go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are.
#include "mxfp4.h"

// A block of NW waves: MT tiles of 16 rows of x against 16 columns (silu: 16 of gate and the same 16 of up).  Its waves take steps of
// four blocks of K in turn and their sums are added in the order of the waves.
template <int X, int TAIL, int MT, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW) void fp4_rows_kernel(Fp4Args a) {
    constexpr int NT = TAIL == TAIL_SILU ? 2 : 1;
    __shared__ float sums[NW][NT][MT * 16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const int n = blockIdx.x * 16 + r;
    const long m0 = (long)blockIdx.y * MT * 16;
    const unsigned char *codes[NT], *scales[NT];
    bool have_n = n < wide;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const long row = have_n ? n + (long)t * wide : 0;
        codes[t] = a.codes + row * a.blocks * 16;
        scales[t] = a.scales + row * a.blocks;
    }
    floatx4_t acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = {0.f, 0.f, 0.f, 0.f};
    for (int step = wave; step * 4 < a.blocks; step += NW) {
        const int b = step * 4 + g;                     // this lane's block of K
        const bool have = b < a.blocks;
        uintx4_t c[NT];
        float scale[NT];
        int sbyte[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            c[t] = {0u, 0u, 0u, 0u};
            sbyte[t] = 0;
            if (have && have_n) {
                c[t] = *(const uintx4_t*)(codes[t] + (long)b * 16);
                sbyte[t] = scales[t][b];
            }
            scale[t] = __uint_as_float((uint32_t)sbyte[t] << 23);
        }
        if constexpr (X == X_FP4) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const long m = m0 + i * 16 + r;
                uintx4_t xc = {0u, 0u, 0u, 0u};
                int xs = 0;
                if (have && m < a.M) {
                    xc = *(const uintx4_t*)((const unsigned char*)a.x + (m * a.blocks + b) * 16);
                    xs = a.xs[m * a.blocks + b];
                    if constexpr (!WHOLE) if (a.K - b * 32 < 32) xc = first_codes(xc, a.K - b * 32);
                }
                const intx8_t xa = {(int)xc[0], (int)xc[1], (int)xc[2], (int)xc[3], 0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const intx8_t wb = {(int)c[t][0], (int)c[t][1], (int)c[t][2], (int)c[t][3], 0, 0, 0, 0};
                    acc[t][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t][i], 4, 4, 0, xs, 0, sbyte[t]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16x8_t w[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) w[t] = fp4_to_bf16(c[t][j], scale[t]);
                const int k = b * 32 + j * 8;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const long m = m0 + i * 16 + r;
                    if constexpr (X == X_BF16) {
                        union { bf16x8_t v; uintx4_t q; uint16_t e[8]; } xv;
                        xv.q = {0u, 0u, 0u, 0u};
                        const uint16_t* p = (const uint16_t*)a.x + m * a.K + k;
                        if (have && m < a.M) {
                            if constexpr (WHOLE) xv.q = *(const uintx4_t*)p;
                            else
#pragma unroll
                                for (int e = 0; e < 8; ++e) if (k + e < a.K) xv.e[e] = p[e];
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv.v, w[t], acc[t][i], 0, 0, 0);
                    } else {
                        union { bf16x8_t v; uint16_t e[8]; } hi, mid, lo;
                        float f[8];
                        const float* p = (const float*)a.x + m * a.K + k;
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = 0.f;
                        if (have && m < a.M) {
                            if constexpr (WHOLE) {
                                const floatx4_t u = *(const floatx4_t*)p, v = *(const floatx4_t*)(p + 4);
#pragma unroll
                                for (int e = 0; e < 4; ++e) { f[e] = u[e]; f[4 + e] = v[e]; }
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e) if (k + e < a.K) f[e] = p[e];
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) cut_in_three(f[e], hi.e[e], mid.e[e], lo.e[e]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, w[t], acc[t][i], 0, 0, 0);
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mid.v, w[t], acc[t][i], 0, 0, 0);
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, w[t], acc[t][i], 0, 0, 0);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][t][i * 16 + g * 4 + e][r] = acc[t][i][e];
    __syncthreads();
    for (int at = threadIdx.x; at < MT * 256; at += 64 * NW) {
        const int row = at >> 4, col = at & 15;
        const long m = m0 + row;
        const int nn = blockIdx.x * 16 + col;
        if (m >= a.M || nn >= wide) continue;
        float v = 0.f, up = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            v += sums[w][0][row][col];
            if constexpr (NT == 2) up += sums[w][1][row][col];
        }
        fp4_store<TAIL>(a, m, nn, v, up);
    }
}

template <int X, int TAIL, int MT, bool WHOLE>
static void fp4_rows_launch(const Fp4Args& a, hipStream_t stream) {
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const dim3 grid(qe_cdiv(wide, 16), qe_cdiv(a.M, MT * 16));
    fp4_rows_kernel<X, TAIL, MT, 4, WHOLE><<<grid, 256, 0, stream>>>(a);
}

template <int X, int TAIL, bool WHOLE>
static void fp4_launch(const Fp4Args& a, hipStream_t stream) {
    if (a.M <= 16) fp4_rows_launch<X, TAIL, 1, WHOLE>(a, stream);
    else if (a.M <= 32) fp4_rows_launch<X, TAIL, 2, WHOLE>(a, stream);
    else fp4_rows_launch<X, TAIL, 4, WHOLE>(a, stream);
}

// More rows than this go by tiles.
#define FP4_ROWS 64

static bool fp4_by_tiles(int M, int N, int K, int x_kind) {
    return M > FP4_ROWS && (x_kind == X_FP4 ? fp4_both_take(M, N, K) : fp4_tiles_take(M, N, K, x_kind));
}

// Bytes of workspace that qe_gemm_mxfp4 needs for these operands.
extern "C" long qe_gemm_mxfp4_workspace_bytes(const void* x, const void* x_scales, const void* scales, int M, int N, int K, int x_kind) {
    if (M <= 0 || N <= 0 || K <= 0 || !fp4_by_tiles(M, N, K, x_kind)) return 0;
    if (x_kind == X_FP4) return fp4_both_workspace(M, N, K, x_scales, scales);
    return fp4_tiles_workspace(M, N, K, x_kind, (((uintptr_t)x & 15) | ((uintptr_t)scales & 3)) == 0);
}

// x: [M, K] bfloat16 (x_kind 0) or float32 (1), or the codes of x in 4 bits with their scales x_scales (2); codes [N, ceil(K / 32) * 16],
// scales [N, ceil(K / 32)]; out [M, N] (silu: [M, N / 2], gate rows of the matrix first, then up rows); tail: 0 store, 1 add into out
// (float32), 2 silu(gate) * up.
extern "C" int qe_gemm_mxfp4(const void* x, const void* x_scales, const void* codes, const void* scales, const float* bias, void* out,
                             int M, int N, int K, int x_kind, int out_dtype, int tail, void* workspace, long workspace_bytes,
                             hipStream_t stream) {
    QE_REQUIRE(M >= 0 && N > 0 && K > 0, "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
    QE_REQUIRE(x_kind >= 0 && x_kind <= 2 && tail >= 0 && tail <= 2, "gemm_mxfp4: unknown form");
    QE_REQUIRE(out_dtype == QE_F32 || out_dtype == QE_BF16, "gemm_mxfp4: unknown element type %d", out_dtype);
    QE_REQUIRE(tail != TAIL_ADD || out_dtype == QE_F32, "gemm_mxfp4: the stream to add into is float32");
    QE_REQUIRE(tail != TAIL_SILU || N % 2 == 0, "gemm_mxfp4: gate|up of an odd number of rows");
    QE_REQUIRE(((uintptr_t)codes & 15) == 0, "gemm_mxfp4: the codes do not begin at a whole 16-byte piece");
    QE_REQUIRE(x_kind != X_FP4 || ((uintptr_t)x & 15) == 0, "gemm_mxfp4: the codes of x do not begin at a whole 16-byte piece");
    QE_REQUIRE(M <= 65535 * 64, "gemm_mxfp4: %d rows are too many", M);
    if (M == 0) return 0;
    const Fp4Args a{x, (const unsigned char*)x_scales, (const unsigned char*)codes, (const unsigned char*)scales, bias, out, M, N, K,
                    qe_cdiv(K, 32), out_dtype == QE_F32};
    const long need = qe_gemm_mxfp4_workspace_bytes(x, x_scales, scales, M, N, K, x_kind);
    QE_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need), "gemm_mxfp4: workspace too small");
    if (fp4_by_tiles(M, N, K, x_kind)) return x_kind == X_FP4 ? fp4_both(a, tail, workspace, stream) : fp4_tiles(a, x_kind, tail, workspace, stream);
    // whole blocks of 16-byte pieces of x
    const bool whole = K % 32 == 0 && ((uintptr_t)x & 15) == 0;
#define QE_TAILS(X_, W_)                                                          \
    do {                                                                          \
        if (tail == TAIL_STORE) fp4_launch<X_, TAIL_STORE, W_>(a, stream);        \
        else if (tail == TAIL_ADD) fp4_launch<X_, TAIL_ADD, W_>(a, stream);       \
        else fp4_launch<X_, TAIL_SILU, W_>(a, stream);                            \
    } while (0)
    if (x_kind == X_FP4) { if (whole) QE_TAILS(X_FP4, true); else QE_TAILS(X_FP4, false); }
    else if (x_kind == X_BF16) { if (whole) QE_TAILS(X_BF16, true); else QE_TAILS(X_BF16, false); }
    else { if (whole) QE_TAILS(X_F32, true); else QE_TAILS(X_F32, false); }
#undef QE_TAILS
    QE_LAUNCH_CHECK();
    return 0;
}
