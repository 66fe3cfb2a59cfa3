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
enum { TAIL_STORE = 0, TAIL_ADD = 1, TAIL_SILU = 2, TAIL_PARTIAL = 3 };      // (PARTIAL: a cut of K, summed by fp4_join)

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

// Every eighth block goes to the same XCD, which has an L2 of its own: it takes an eighth of a walk through the tiles in bands of 8 tile rows,
// column by column, so that what it runs at a time shares rows of x and of the matrix.  false: a block beyond the tiles.
__device__ __forceinline__ bool fp4_tile_of(int block, int tiles_m, int tiles_n, int& tile_m, int& tile_n) {
    const int all = tiles_m * tiles_n, each = all / 8, over = all % 8, xcd = block % 8;
    int local = block / 8;
    if (local >= each + (xcd < over)) return false;
    local += xcd * each + min(xcd, over);
    const int band = local / (8 * tiles_n), within = local - band * 8 * tiles_n, rows = min(8, tiles_m - band * 8);
    tile_m = band * 8 + within % rows;
    tile_n = within / rows;
    return true;
}

// The row of the matrix behind column i of the tile that begins at column n0 (-1: none); silu: 16 of gate and their 16 of up in turn.
template <int TAIL>
__device__ __forceinline__ int fp4_matrix_row(int n0, int i, int wide) {
    if constexpr (TAIL == TAIL_SILU) {
        const int n = n0 / 2 + (i >> 5) * 16 + (i & 15);
        return n < wide ? ((i >> 4) & 1) * wide + n : -1;
    } else {
        return n0 + i < wide ? n0 + i : -1;
    }
}

// The sums of a wave's tiles of 32 x 32, from row m0 and column n0 of the whole product on: lane (r, h) = (lane % 32, lane / 32) has column
// r of a tile and its rows 8 b + 4 h + e.  Stored from there, an instruction would write 2 rows of 64 or 128 bytes, two or four bytes a
// lane (a tile of 256 x 256 took 20 us to store); so a strip of 32 rows at a time is turned round in the wave's own piece of shared
// memory, and a lane stores four columns.  Silu: of 32 columns of a tile 16 are gates and 16 their ups.
template <int NJ> constexpr int fp4_strip_bytes() { return 32 * (NJ * 32 + 8) * 4; }     // (8: the rows that two halves of a wave write lie in other banks)

template <int TAIL, int MI, int NJ>
__device__ __forceinline__ void fp4_store_tiles(const Fp4Args& a, const floatx16_t (&acc)[MI][NJ], int m0, int n0, unsigned char* strip_at) {
    constexpr int ROW = NJ * 32 + 8, COLS = TAIL == TAIL_SILU ? NJ * 16 : NJ * 32, LANES = COLS / 4, ROWS = 64 / LANES;      // lanes of a row, rows of an instruction
    float* strip = (float*)strip_at;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5, wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const int col = lane % LANES * 4, from = TAIL == TAIL_SILU ? col / 16 * 32 + col % 16 : col;
    const int n = (TAIL == TAIL_SILU ? n0 / 2 : n0) + col;
    const bool four = wide % 4 == 0 && ((unsigned long)a.out & 15) == 0 && n + 4 <= wide;
    float bias[4] = {0.f, 0.f, 0.f, 0.f}, bias_up[4] = {0.f, 0.f, 0.f, 0.f};
    if (TAIL != TAIL_PARTIAL && a.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < wide) {
                bias[e] = a.bias[n + e];
                if constexpr (TAIL == TAIL_SILU) bias_up[e] = a.bias[wide + n + e];
            }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) strip[(8 * (e / 4) + 4 * h + e % 4) * ROW + j * 32 + r] = acc[i][j][e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 4
        for (int k = 0; k < 32 / ROWS; ++k) {
            const int row = k * ROWS + lane / LANES;
            const long m = m0 + i * 32 + row;
            if (m >= a.M || n >= wide) continue;
            const floatx4_t s = *(const floatx4_t*)(strip + row * ROW + from);
            floatx4_t u = {0.f, 0.f, 0.f, 0.f};
            if constexpr (TAIL == TAIL_SILU) u = *(const floatx4_t*)(strip + row * ROW + from + 16);
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = s[e] + bias[e];
                if constexpr (TAIL == TAIL_SILU) v[e] = v[e] / (1.f + expf(-v[e])) * (u[e] + bias_up[e]);
            }
            const long at = m * wide + n;
            if (four) {
                if (TAIL == TAIL_ADD) {
                    float old[4];
                    Vec4<float>::load((const float*)a.out + at, old);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += old[e];
                }
                if (TAIL == TAIL_ADD || TAIL == TAIL_PARTIAL || a.out_f32) Vec4<float>::store((float*)a.out + at, v);
                else Vec4<bf16_t>::store((bf16_t*)a.out + at, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n + e >= wide) break;
                    if (TAIL == TAIL_ADD) ((float*)a.out)[at + e] += v[e];
                    else if (TAIL == TAIL_PARTIAL || a.out_f32) ((float*)a.out)[at + e] = v[e];
                    else ((bf16_t*)a.out)[at + e] = float_to_bf16(v[e]);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");      // the reads before the next strip's writes
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// A lane's offset of a buffer load that is beyond every buffer: it arrives as zero.
constexpr int FP4_OUT = 0x7fffffff;

// One descriptor of a buffer of so many bytes, the same in every lane.
__device__ __forceinline__ uintx4_t fp4_buffer(const void* p, unsigned bytes) {
    uintx4_t d;
    d[0] = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)p);
    d[1] = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long)p >> 32) & 0xffffu);
    d[2] = __builtin_amdgcn_readfirstlane(bytes);
    d[3] = 0x00020000u;
    return d;
}

// Scales travel 16 at a time, those of FP4_SPAN numbers of a row, from any whole word on.  Of a row's last span some may be another row's or lie
// beyond the matrix (a word there arrives as zero): they belong to no stage if the row is whole stages.  Other rows are copied, zeros
// behind (a launch, 5 us of a product of 100 rows against 5120 x 2560 that takes 17).
#define FP4_SPAN 512
inline bool fp4_scales_whole(int K, const void* scales, int stage) { return K % 128 == 0 && K % stage == 0 && ((uintptr_t)scales & 3) == 0; }
inline int fp4_scales_row(int K, bool whole) { return whole ? K / 32 : qe_cdiv(K, FP4_SPAN) * (FP4_SPAN / 32); }      // bytes from a row to the next
inline long fp4_scales_bytes(int rows, int K) { return (long)rows * fp4_scales_row(K, false); }                       // of a copy

// partial products [splits][M][N] -> a.out, summed in their order, with the tail
int fp4_join(const Fp4Args& a, const float* parts, int splits, int tail, hipStream_t stream);

// Rows of bfloat16 as the loads take them: at whole 16-byte pieces, plane after plane (or rows of codes).
struct Fp4Rows {
    const void* data;
    int row_bytes, planes;
};
// gemm_mxfp4_tiles.hip: rows copied so (out null: they are not), 32-bit ones in three planes of bfloat16 (low, middle, high), zeros from K to whole
// stages; and scales of so many rows in whole spans (scales_out null: they are not)
long fp4_planes_bytes(int M, int K, int x_kind);
Fp4Rows fp4_copies(const void* x, int M, int K, int x_kind, void* out, const unsigned char* scales, int rows, void* scales_out, hipStream_t stream);

// gemm_mxfp4_rows.hip: few rows
bool fp4_few_takes(int M, int N, int K, int x_kind, int tail);
long fp4_few_workspace(const void* x, int M, int K, int x_kind);
int fp4_few(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream);
// gemm_mxfp4_tiles.hip: the products of many rows of 16 or 32 bits; the bytes of workspace that these sizes take
bool fp4_tiles_take(int M, int N, int K, int x_kind);
long fp4_tiles_workspace(int M, int N, int K, int x_kind, const void* x, const void* scales);
int fp4_tiles(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream);
// gemm_mxfp4_both.hip: many rows that are in 4 bits themselves
bool fp4_both_take(int M, int N, int K);
long fp4_both_workspace(int M, int N, int K, const void* xs, const void* scales);
int fp4_both(const Fp4Args& a, int tail, void* workspace, hipStream_t stream);
