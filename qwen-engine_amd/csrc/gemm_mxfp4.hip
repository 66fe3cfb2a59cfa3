// Matrix product with a 4-bit matrix: out[M, N] = x[M, K] . V[N, K]^T (+ bias), V the numbers that codes and scales stand for
// (see mxfp4.hip: blocks of 32 along K).  x is bfloat16, float32 or itself in 4 bits.
//
// A lane of the matrix instruction takes a whole block of a row of V, 16 bytes of codes with their scale, and the same block of a row
// of x.  The numbers of a block are products of at most two significant bits with a power of two, so they are exact in bfloat16: with
// bfloat16 x the codes become bfloat16 in registers (an instruction for two of them, the scale included) and v_mfma_f32_16x16x32_bf16
// sums in 32-bit.  Numbers of 32-bit x are cut into three bfloat16 (8 + 8 + 8 bits, exact) and multiplied by three instructions.  With
// both sides in 4 bits the codes go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are.
#include "mxfp4.h"

// Few rows: a block of up to 16 waves multiplies MT tiles of 16 rows of x with NT tiles of 16 columns (silu: the second half of the tiles
// are the up rows of the first half's gate rows).  Its waves take steps of four blocks of K in turn, and their sums are added in the order
// of the waves.
//
// Bound by the matrix's bytes on their way from memory: a wave asks for everything that the next U steps multiply before it multiplies.
template <int X, int MT, int NT, bool WHOLE>
__global__ __launch_bounds__(MT * NT == 1 ? 1024 : 512) void fp4_rows_kernel(Fp4Args a, int tail) {
    constexpr int U = MT == 1 && NT <= 2 && X != X_F32 ? 4 : MT <= 2 && X != X_F32 ? 2 : 1;
    constexpr int XP = X == X_FP4 ? 1 : X == X_BF16 ? 4 : 8;           // 16-byte pieces of a block of x
    extern __shared__ float sums[];                                    // [waves][NT][MT * 16][16]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, waves = blockDim.x >> 6;
    const bool silu = tail == TAIL_SILU;
    const int wide = silu ? a.N / 2 : a.N, cols = silu ? NT * 8 : NT * 16;
    const int n0 = blockIdx.x * cols;
    const long m0 = (long)blockIdx.y * MT * 16;
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
    long x_row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long m = m0 + i * 16 + r;
        x_row[i] = m < a.M ? m : a.M - 1;
    }
    floatx4_t acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = {0.f, 0.f, 0.f, 0.f};
    for (int step0 = wave; step0 * 4 < a.blocks; step0 += waves * U) {
        uintx4_t c[U][NT], xp[U][MT][XP];
        int sc[U][NT], xs[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = min((step0 + u * waves) * 4 + g, a.blocks - 1);      // this lane's block of K
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                c[u][t] = *(const uintx4_t*)(codes[t] + (long)b * 16);
                sc[u][t] = scales[t][b];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (X == X_FP4) {
                    xp[u][i][0] = *(const uintx4_t*)((const unsigned char*)a.x + (x_row[i] * a.blocks + b) * 16);
                    xs[u][i] = a.xs[x_row[i] * a.blocks + b];
                } else if constexpr (WHOLE) {
                    const uintx4_t* p = (const uintx4_t*)((const unsigned char*)a.x + (x_row[i] * a.K + b * 32) * (X == X_BF16 ? 2 : 4));
#pragma unroll
                    for (int e = 0; e < XP; ++e) xp[u][i][e] = p[e];
                } else {
#pragma unroll
                    for (int e = 0; e < XP; ++e) xp[u][i][e] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const bool there = b * 32 + e < a.K;
                        const long at = x_row[i] * a.K + (there ? b * 32 + e : 0);
                        if constexpr (X == X_BF16) xp[u][i][e / 8][e / 2 % 4] |= there ? (uint32_t)((const uint16_t*)a.x)[at] << (16 * (e & 1)) : 0u;
                        else xp[u][i][e / 4][e % 4] = there ? ((const uint32_t*)a.x)[at] : 0u;
                    }
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
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int e = 0; e < XP; ++e) xp[u][i][e] = {0u, 0u, 0u, 0u};
                    if constexpr (X == X_FP4) xs[u][i] = 0;
                }
            } else if constexpr (X == X_FP4 && !WHOLE) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (a.K - b * 32 < 32) xp[u][i][0] = first_codes(xp[u][i][0], a.K - b * 32);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (X == X_FP4) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uintx4_t& x = xp[u][i][0];
                    const intx8_t xa = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const intx8_t wb = {(int)c[u][t][0], (int)c[u][t][1], (int)c[u][t][2], (int)c[u][t][3], 0, 0, 0, 0};
                        acc[t][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t][i], 4, 4, 0, xs[u][i], 0, sc[u][t]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bf16x8_t w[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) w[t] = fp4_to_bf16(c[u][t][j], __uint_as_float((uint32_t)sc[u][t] << 23));
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if constexpr (X == X_BF16) {
                            const bf16x8_t x = __builtin_bit_cast(bf16x8_t, xp[u][i][j]);
#pragma unroll
                            for (int t = 0; t < NT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w[t], acc[t][i], 0, 0, 0);
                        } else {
                            union { bf16x8_t v; uint16_t e[8]; } hi, mid, lo;
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                cut_in_three(__uint_as_float(xp[u][i][2 * j + e / 4][e % 4]), hi.e[e], mid.e[e], lo.e[e]);
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
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[((wave * NT + t) * MT * 16 + i * 16 + g * 4 + e) * 16 + r] = acc[t][i][e];
    __syncthreads();
    const int out_tiles = silu ? NT / 2 : NT;
    for (int at = threadIdx.x; at < out_tiles * MT * 256; at += blockDim.x) {
        const int t = at / (MT * 256), row = at / 16 % (MT * 16), col = at & 15;
        const long m = m0 + row;
        const int n = n0 + t * 16 + col;
        if (m >= a.M || n >= wide) continue;
        float v = 0.f, up = 0.f;
        for (int w = 0; w < waves; ++w) {
            v += sums[((w * NT + t) * MT * 16 + row) * 16 + col];
            if (silu) up += sums[((w * NT + t + NT / 2) * MT * 16 + row) * 16 + col];
        }
        if (tail == TAIL_STORE) fp4_store<TAIL_STORE>(a, m, n, v, up);
        else if (tail == TAIL_ADD) fp4_store<TAIL_ADD>(a, m, n, v, up);
        else fp4_store<TAIL_SILU>(a, m, n, v, up);
    }
}

template <int X, int MT, int NT, bool WHOLE>
static int fp4_rows_launch(const Fp4Args& a, int tail, hipStream_t stream) {
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N, cols = tail == TAIL_SILU ? NT * 8 : NT * 16;
    const int steps = qe_cdiv(a.blocks, 4), most = MT * NT == 1 ? 16 : MT * NT <= 8 ? 8 : 4;       // (4: 64 KB of sums at most)
    // about four steps a wave: what it asks for at once
    int waves = steps >= 48 ? 16 : steps >= 12 ? 8 : steps >= 4 ? 4 : 2;
    if (waves > most) waves = most;
    const size_t shared = (size_t)waves * NT * MT * 1024;
    const dim3 grid(qe_cdiv(wide, cols), qe_cdiv(a.M, MT * 16));
    fp4_rows_kernel<X, MT, NT, WHOLE><<<grid, 64 * waves, shared, stream>>>(a, tail);
    return 0;
}

template <int X, bool WHOLE>
static int fp4_rows(const Fp4Args& a, int tail, hipStream_t stream) {
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N;
    // Four tiles of columns a block where that leaves two blocks a compute unit: every block reads all of x.
    const bool many = wide >= 2 * 256 * (tail == TAIL_SILU ? 32 : 64);
    if (a.M <= 16) return many ? fp4_rows_launch<X, 1, 4, WHOLE>(a, tail, stream)
                          : tail == TAIL_SILU ? fp4_rows_launch<X, 1, 2, WHOLE>(a, tail, stream) : fp4_rows_launch<X, 1, 1, WHOLE>(a, tail, stream);
    if (a.M <= 32) return many ? fp4_rows_launch<X, 2, 4, WHOLE>(a, tail, stream) : fp4_rows_launch<X, 2, 2, WHOLE>(a, tail, stream);
    if (a.M <= 48) return many ? fp4_rows_launch<X, 3, 4, WHOLE>(a, tail, stream) : fp4_rows_launch<X, 3, 2, WHOLE>(a, tail, stream);
    return many && X != X_F32 ? fp4_rows_launch<X, 4, X == X_F32 ? 2 : 4, WHOLE>(a, tail, stream) : fp4_rows_launch<X, 4, 2, WHOLE>(a, tail, stream);
}

static bool fp4_by_tiles(int M, int N, int K, int x_kind) {
    return M > (x_kind == X_FP4 ? 64 : 16) && (x_kind == X_FP4 ? fp4_both_take(M, N, K) : fp4_tiles_take(M, N, K, x_kind));
}

// Bytes of workspace that qe_gemm_mxfp4 needs for these operands.
extern "C" long qe_gemm_mxfp4_workspace_bytes(const void* x, const void* x_scales, const void* scales, int M, int N, int K, int x_kind) {
    if (M <= 0 || N <= 0 || K <= 0 || !fp4_by_tiles(M, N, K, x_kind)) return 0;
    if (x_kind == X_FP4) return fp4_both_workspace(M, N, K, x_scales, scales);
    return fp4_tiles_workspace(M, N, K, x_kind, x, scales);
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
    int rc;
    if (fp4_few_takes(x, M, N, K, x_kind, tail)) rc = fp4_few(a, x_kind, tail, stream);
    else if (x_kind == X_FP4) rc = whole ? fp4_rows<X_FP4, true>(a, tail, stream) : fp4_rows<X_FP4, false>(a, tail, stream);
    else if (x_kind == X_BF16) rc = whole ? fp4_rows<X_BF16, true>(a, tail, stream) : fp4_rows<X_BF16, false>(a, tail, stream);
    else rc = whole ? fp4_rows<X_F32, true>(a, tail, stream) : fp4_rows<X_F32, false>(a, tail, stream);
    if (rc) return rc;
    QE_LAUNCH_CHECK();
    return 0;
}
