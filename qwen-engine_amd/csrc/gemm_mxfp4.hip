// Matrix product with a 4-bit matrix: out[M, N] = x[M, K] . V[N, K]^T (+ bias), V the numbers that codes and scales stand for
// (see mxfp4.hip: blocks of 32 along K).  x is bfloat16, float32 or itself in 4 bits.
//
// A lane of the matrix instruction takes a whole block of a row of V, 16 bytes of codes with their scale, and the same block of a row
// of x.  The numbers of a block are products of at most two significant bits with a power of two, so they are exact in bfloat16: with
// bfloat16 x the codes become bfloat16 in registers (an instruction for two of them, the scale included) and v_mfma_f32_16x16x32_bf16
// sums in 32-bit.  Numbers of 32-bit x are cut into three bfloat16 (8 + 8 + 8 bits, exact) and multiplied by three instructions.  With
// both sides in 4 bits the codes go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are.
#include "mxfp4.h"

// What the other kernels do not take (very wide rows; more bytes than 32-bit places reach): rows of any width at any place, 16 at a time.  A block of up to 16 waves
// multiplies them with NT tiles of 16 columns (silu: the second is the up rows of the first's gate rows).  Its waves take steps of four blocks
// of K in turn, and their sums are added in the order of the waves.  A wave asks for everything that the next U steps multiply before it
// multiplies (of bfloat16 rows and one tile two steps: the 16 waves leave 128 registers each, and with four 67 of them went to scratch memory;
// 3 rows of 400000 numbers against 1024 1.48 -> 1.12 ms, 1 against 4096 2.23 -> 0.94).
template <int X, int NT>
__global__ __launch_bounds__(NT == 1 ? 1024 : 512) void fp4_rows_kernel(Fp4Args a, int tail) {
    constexpr int U = X == X_F32 ? 1 : X == X_BF16 && NT == 1 ? 2 : 4;
    constexpr int XP = X == X_FP4 ? 1 : X == X_BF16 ? 4 : 8;           // 16-byte pieces of a block of x
    extern __shared__ float sums[];                                    // [waves][NT][16][16]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, waves = blockDim.x >> 6;
    const bool silu = tail == TAIL_SILU;
    const int wide = silu ? a.N / 2 : a.N, cols = silu ? NT * 8 : NT * 16;
    const int n0 = blockIdx.x * cols;
    const long m0 = (long)blockIdx.y * 16;
    // (columns and rows beyond the matrices are read as the last ones and not stored; blocks beyond K become zeros below: a branch around a
    // load would make the next one wait for it)
    const unsigned char *codes[NT], *scales[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const bool up = silu && t >= NT / 2;
        const int n = min(n0 + (up ? t - NT / 2 : t) * 16 + r, wide - 1);
        const long row = n + (up ? (long)wide : 0);
        codes[t] = a.codes + row * a.blocks * 16;
        scales[t] = a.scales + row * a.blocks;
    }
    const long x_row = m0 + r < a.M ? m0 + r : a.M - 1;
    floatx4_t acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = {0.f, 0.f, 0.f, 0.f};
    for (int step0 = wave; step0 * 4 < a.blocks; step0 += waves * U) {
        uintx4_t c[U][NT], xp[U][XP];
        int sc[U][NT], xs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = min((step0 + u * waves) * 4 + g, a.blocks - 1);      // this lane's block of K
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                c[u][t] = *(const uintx4_t*)(codes[t] + (long)b * 16);
                sc[u][t] = scales[t][b];
            }
            xs[u] = 0;
            if constexpr (X == X_FP4) {
                xp[u][0] = *(const uintx4_t*)((const unsigned char*)a.x + (x_row * a.blocks + b) * 16);
                xs[u] = a.xs[x_row * a.blocks + b];
            } else {
#pragma unroll
                for (int e = 0; e < XP; ++e) xp[u][e] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const bool there = b * 32 + e < a.K;
                    const long at = x_row * a.K + (there ? b * 32 + e : 0);
                    if constexpr (X == X_BF16) xp[u][e / 8][e / 2 % 4] |= there ? (uint32_t)((const uint16_t*)a.x)[at] << (16 * (e & 1)) : 0u;
                    else xp[u][e / 4][e % 4] = there ? ((const uint32_t*)a.x)[at] : 0u;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = (step0 + u * waves) * 4 + g;
            if (b >= a.blocks) {                       // (codes 0 of scale 2^-127 on both sides: x beyond K may be anything that a row holds)
#pragma unroll
                for (int t = 0; t < NT; ++t) { c[u][t] = {0u, 0u, 0u, 0u}; sc[u][t] = 0; }
#pragma unroll
                for (int e = 0; e < XP; ++e) xp[u][e] = {0u, 0u, 0u, 0u};
                xs[u] = 0;
            } else if constexpr (X == X_FP4) {
                if (a.K - b * 32 < 32) xp[u][0] = first_codes(xp[u][0], a.K - b * 32);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (X == X_FP4) {
                const uintx4_t& x = xp[u][0];
                const intx8_t xa = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const intx8_t wb = {(int)c[u][t][0], (int)c[u][t][1], (int)c[u][t][2], (int)c[u][t][3], 0, 0, 0, 0};
                    acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t], 4, 4, 0, xs[u], 0, sc[u][t]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bf16x8_t w[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) w[t] = fp4_to_bf16(c[u][t][j], __uint_as_float((uint32_t)sc[u][t] << 23));
                    if constexpr (X == X_BF16) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, xp[u][j]), w[t], acc[t], 0, 0, 0);
                    } else {
                        union { bf16x8_t v; uint16_t e[8]; } hi, mid, lo;
#pragma unroll
                        for (int e = 0; e < 8; ++e) cut_in_three(__uint_as_float(xp[u][2 * j + e / 4][e % 4]), hi.e[e], mid.e[e], lo.e[e]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, w[t], acc[t], 0, 0, 0);
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mid.v, w[t], acc[t], 0, 0, 0);
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, w[t], acc[t], 0, 0, 0);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[((wave * NT + t) * 16 + g * 4 + e) * 16 + r] = acc[t][e];
    __syncthreads();
    const int out_tiles = silu ? NT / 2 : NT;
    for (int at = threadIdx.x; at < out_tiles * 256; at += blockDim.x) {
        const int t = at >> 8, row = at >> 4 & 15, col = at & 15;
        const long m = m0 + row;
        const int n = n0 + t * 16 + col;
        if (m >= a.M || n >= wide) continue;
        float v = 0.f, up = 0.f;
        for (int w = 0; w < waves; ++w) {
            v += sums[((w * NT + t) * 16 + row) * 16 + col];
            if (silu) up += sums[((w * NT + t + NT / 2) * 16 + row) * 16 + col];
        }
        if (tail == TAIL_STORE) fp4_store<TAIL_STORE>(a, m, n, v, up);
        else if (tail == TAIL_ADD) fp4_store<TAIL_ADD>(a, m, n, v, up);
        else fp4_store<TAIL_SILU>(a, m, n, v, up);
    }
}

template <int X>
static int fp4_rows(const Fp4Args& a, int tail, hipStream_t stream) {
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N;
    // about four steps a wave: what it asks for at once
    const int steps = qe_cdiv(a.blocks, 4);
    int waves = steps >= 48 ? 16 : steps >= 12 ? 8 : steps >= 4 ? 4 : 2;
    if (tail == TAIL_SILU && waves > 8) waves = 8;
    // (as many rows a launch as a grid's second axis holds)
    for (long m = 0; m < a.M; m += 65535 * 16) {
        Fp4Args s = a;
        s.M = (int)(a.M - m < 65535 * 16 ? a.M - m : 65535 * 16);
        s.x = (const unsigned char*)a.x + m * (X == X_FP4 ? a.blocks * 16L : a.K * (X == X_BF16 ? 2L : 4L));
        if (X == X_FP4) s.xs = a.xs + m * a.blocks;
        s.out = (unsigned char*)a.out + m * wide * (a.out_f32 ? 4L : 2L);
        const dim3 grid(qe_cdiv(wide, 16), qe_cdiv(s.M, 16));
        if (tail == TAIL_SILU) fp4_rows_kernel<X, 2><<<grid, 64 * waves, waves * 2048, stream>>>(s, tail);
        else fp4_rows_kernel<X, 1><<<grid, 64 * waves, waves * 1024, stream>>>(s, tail);
    }
    return 0;
}

// The kernel for these operands: fp4_few (gemm_mxfp4_rows.hip), by tiles, or fp4_rows.
enum { BY_FEW, BY_TILES, BY_ROWS };
static int fp4_way(int M, int N, int K, int x_kind, int tail) {
    if (fp4_few_takes(M, N, K, x_kind, tail)) return BY_FEW;
    return M > (x_kind == X_F32 ? 8 : 16) && (x_kind == X_FP4 ? fp4_both_take(M, N, K) : fp4_tiles_take(M, N, K, x_kind)) ? BY_TILES : BY_ROWS;
}

// Bytes of workspace that qe_gemm_mxfp4 needs for these operands.
extern "C" long qe_gemm_mxfp4_workspace_bytes(const void* x, const void* x_scales, const void* scales, int M, int N, int K, int x_kind, int tail) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int way = fp4_way(M, N, K, x_kind, tail);
    if (way == BY_FEW) return fp4_few_workspace(x, M, K, x_kind);
    if (way == BY_ROWS) return 0;
    return x_kind == X_FP4 ? fp4_both_workspace(M, N, K, x_scales, scales) : fp4_tiles_workspace(M, N, K, x_kind, x, scales);
}

// x: [M, K] bfloat16 (x_kind 0) or float32 (1), or the codes of x in 4 bits with their scales x_scales (2); codes [N, ceil(K / 32) * 16],
// scales [N, ceil(K / 32)]; out [M, N] (silu: [M, N / 2], gate rows of the matrix first, then up rows); tail: 0 store, 1 add into out
// (float32), 2 silu(gate) * up.
extern "C" int qe_gemm_mxfp4(const void* x, const void* x_scales, const void* codes, const void* scales, const float* bias, void* out,
                             int M, int N, int K, int x_kind, int out_dtype, int tail, void* workspace, long workspace_bytes,
                             hipStream_t stream) {
    QE_REQUIRE(M >= 0 && N > 0 && K > 0 && K < (1 << 30), "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
    QE_REQUIRE(x_kind >= 0 && x_kind <= 2 && tail >= 0 && tail <= 2, "gemm_mxfp4: unknown form");
    QE_REQUIRE(out_dtype == QE_F32 || out_dtype == QE_BF16, "gemm_mxfp4: unknown element type %d", out_dtype);
    QE_REQUIRE(tail != TAIL_ADD || out_dtype == QE_F32, "gemm_mxfp4: the stream to add into is float32");
    QE_REQUIRE(tail != TAIL_SILU || N % 2 == 0, "gemm_mxfp4: gate|up of an odd number of rows");
    QE_REQUIRE(((uintptr_t)codes & 15) == 0, "gemm_mxfp4: the codes do not begin at a whole 16-byte piece");
    QE_REQUIRE(x_kind != X_FP4 || ((uintptr_t)x & 15) == 0, "gemm_mxfp4: the codes of x do not begin at a whole 16-byte piece");
    QE_REQUIRE(M <= (1 << 30), "gemm_mxfp4: %d rows are too many", M);
    if (M == 0) return 0;
    const Fp4Args a{x, (const unsigned char*)x_scales, (const unsigned char*)codes, (const unsigned char*)scales, bias, out, M, N, K,
                    qe_cdiv(K, 32), out_dtype == QE_F32};
    const int way = fp4_way(M, N, K, x_kind, tail);
    const long need = qe_gemm_mxfp4_workspace_bytes(x, x_scales, scales, M, N, K, x_kind, tail);
    QE_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need), "gemm_mxfp4: workspace too small");
    int rc;
    if (way == BY_FEW) rc = fp4_few(a, x_kind, tail, workspace, stream);
    else if (way == BY_TILES) rc = x_kind == X_FP4 ? fp4_both(a, tail, workspace, stream) : fp4_tiles(a, x_kind, tail, workspace, stream);
    else rc = x_kind == X_FP4 ? fp4_rows<X_FP4>(a, tail, stream) : x_kind == X_BF16 ? fp4_rows<X_BF16>(a, tail, stream) : fp4_rows<X_F32>(a, tail, stream);
    if (rc) return rc;
    QE_LAUNCH_CHECK();
    return 0;
}
