// Products of many rows of 16-bit or 32-bit numbers with a 4-bit matrix (see mxfp4.h): out[M, N] = x[M, K] . V[N, K]^T.
//
// A block of four waves computes BM rows by BN columns.  K is walked in stages of 128 or 64 through a ring in shared memory: of 128, 256 bytes of a
// row of x and 64 of codes of a row of the matrix, and for 512 of K 16 of its scales, brought by loads that write to shared memory directly.  A
// wave multiplies its part in tiles of 32 x 32 with v_mfma_f32_32x32x16_bf16: lane (r, h) = (lane % 32, lane / 32) takes, of row r,
// block 2 b + h of the stage, so that a 16-byte piece of codes with one scale gives four matrix instructions' operands, eight numbers
// each, by four conversions each.  The conversions for the next k step stand between the matrix instructions of this one.
//
// Rows of 32-bit numbers come as three planes of bfloat16 (cut_in_three), made by a launch of their own, which also fills K up to whole
// stages.  They are walked one after the other, the smallest first, against the same matrix; or a tile has 32 rows of all three, so that the
// codes are loaded and converted once (130 rows of 2568 numbers against 5120 24 us, walked three times 30).
//
// 2048 rows against 24576 x 4096 take 319 us (1.29 PFLOP/s): the matrix units are 65 % busy at the clock that the power leaves.  64 rows against that take 23.4 us:
// they are 34 % busy, the one wave of a SIMD issues half of its time (conversions, fragments, loads and their places, one after
// the other) and waits for 30 %; a ring of six stages instead of three changes nothing.
#include "mxfp4.h"

#define FP4_STAGE 128      // numbers of K

// What the loads cannot take as it is, in one launch.  Blocks 0 .. x_blocks - 1: x [M, K] float32 -> planes [3][M][Kp] (low, middle, high) of
// bfloat16, zeros from K on, or bfloat16 -> [M][Kp]; `whole`: K is a multiple of four and x lies at a whole four numbers.  The others:
// scales [rows, blocks] -> [rows, words * 4], zeros behind.
struct Fp4Copies {
    const void* x;
    uint16_t* planes;
    int M, K, Kp;
    unsigned x_blocks, per;             // blocks of a row of x
    const unsigned char* scales;
    uint32_t* scales_out;
    unsigned all_words, words;          // of all rows, of a row
    int blocks;
    bool whole;
};

template <typename T>
__global__ __launch_bounds__(256) void fp4_copies_kernel(Fp4Copies p) {
    if (blockIdx.x >= p.x_blocks) {
        const unsigned at = (blockIdx.x - p.x_blocks) * 256 + threadIdx.x, row = at / p.words;
        if (at >= p.all_words) return;
        const int b = (int)(at - row * p.words) * 4;
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (b + e < p.blocks) v |= (uint32_t)p.scales[(long)row * p.blocks + b + e] << (8 * e);
        p.scales_out[at] = v;
        return;
    }
    const unsigned row = blockIdx.x / p.per;
    const int k = (int)((blockIdx.x - row * p.per) * 256 + threadIdx.x) * 4;
    if (k >= p.Kp) return;
    const T* x = (const T*)p.x + (long)row * p.K + k;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.whole) {
        if (k < p.K) Vec4<T>::load(x, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < p.K) v[e] = Elem<T>::load(x + e);
    }
    uint16_t* to = p.planes + (long)row * p.Kp + k;
    uint16_t hi[4], mid[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) cut_in_three(v[e], hi[e], mid[e], lo[e]);
        else hi[e] = (uint16_t)(__float_as_uint(v[e]) >> 16);
    }
    if constexpr (sizeof(T) == 4) {
        const long plane = (long)p.M * p.Kp;
        *(ushort4*)to = make_ushort4(lo[0], lo[1], lo[2], lo[3]);
        *(ushort4*)(to + plane) = make_ushort4(mid[0], mid[1], mid[2], mid[3]);
        *(ushort4*)(to + 2 * plane) = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
    } else {
        *(ushort4*)to = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
    }
}

static int padded(int K) { return qe_cdiv(K, FP4_STAGE) * FP4_STAGE; }

long fp4_planes_bytes(int M, int K, int x_kind) { return (x_kind == X_F32 ? 6L : 2L) * M * padded(K); }

Fp4Rows fp4_copies(const void* x, int M, int K, int x_kind, void* out, const unsigned char* scales, int rows, void* scales_out, hipStream_t stream) {
    Fp4Copies p{};
    p.x = x;
    p.planes = (uint16_t*)out;
    p.M = M;
    p.K = K;
    p.Kp = padded(K);
    p.per = qe_cdiv(p.Kp, 1024);
    p.x_blocks = out ? (unsigned)M * p.per : 0;
    p.scales = scales;
    p.scales_out = (uint32_t*)scales_out;
    p.words = (unsigned)(fp4_scales_bytes(1, K) / 4);
    p.all_words = scales_out ? (unsigned)rows * p.words : 0;      // (below 2^31 / 16: fp4_tiles_take)
    p.blocks = qe_cdiv(K, 32);
    p.whole = K % 4 == 0 && ((uintptr_t)x & (x_kind == X_F32 ? 15 : 7)) == 0;
    const unsigned grid = p.x_blocks + qe_cdiv(p.all_words, 256);
    if (x_kind == X_F32) fp4_copies_kernel<float><<<grid, 256, 0, stream>>>(p);
    else fp4_copies_kernel<bf16_t><<<grid, 256, 0, stream>>>(p);
    return {out, p.Kp * 2, x_kind == X_F32 ? 3 : 1};
}

struct Fp4Tiles {
    Fp4Args a;
    const uint16_t* planes;     // rows of x, row_bytes apart, plane after plane
    unsigned row_bytes, plane_bytes, x_bytes;      // (x_bytes: of all planes)
    const unsigned char* scales;
    int scale_bytes;            // from a row to the next
    int num_planes, nk, k_in_row;                  // (numbers of K that a row holds: K, or whole stages where it is a plane's)
    int tiles_m, tiles_n;
    int per_split;              // stages of a cut: block (., y) sums the stages from y * per_split on
};

// The sum of the cuts' products, and what becomes of it: a thread four columns.
template <int TAIL>
__global__ __launch_bounds__(256) void fp4_join_kernel(Fp4Args a, const float* __restrict__ parts, int splits) {
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= wide) return;
    const long size = (long)a.M * a.N;
    for (long m = blockIdx.y; m < a.M; m += gridDim.y) {
        float v[4] = {0.f, 0.f, 0.f, 0.f}, up[4] = {0.f, 0.f, 0.f, 0.f};
        const float* p = parts + m * a.N + n;
        for (int s = 0; s < splits; ++s, p += size) {
            if (a.N % 4 == 0 && wide % 4 == 0) {
                const floatx4_t q = *(const floatx4_t*)p;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += q[e];
                if constexpr (TAIL == TAIL_SILU) {
                    const floatx4_t u = *(const floatx4_t*)(p + wide);
#pragma unroll
                    for (int e = 0; e < 4; ++e) up[e] += u[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < wide) {
                        v[e] += p[e];
                        if constexpr (TAIL == TAIL_SILU) up[e] += p[wide + e];
                    }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < wide) fp4_store<TAIL>(a, m, n + e, v[e], up[e]);
    }
}

int fp4_join(const Fp4Args& a, const float* parts, int splits, int tail, hipStream_t stream) {
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N;
    const dim3 grid(qe_cdiv(wide, 1024), a.M < 65535 ? a.M : 65535);
    if (tail == TAIL_STORE) fp4_join_kernel<TAIL_STORE><<<grid, 256, 0, stream>>>(a, parts, splits);
    else if (tail == TAIL_ADD) fp4_join_kernel<TAIL_ADD><<<grid, 256, 0, stream>>>(a, parts, splits);
    else fp4_join_kernel<TAIL_SILU><<<grid, 256, 0, stream>>>(a, parts, splits);
    return 0;
}

// BM x BN: the tile; WR x WC: the waves; SK: numbers of K of a stage, 128 or 64 (whole lines of x either way); RING: stages in shared memory;
// PLANES: 3: the tile's rows are those of x in each of the three planes, whose sums are added at the end, the smallest first
template <int TAIL, int BM, int BN, int WR, int WC, int SK, int RING, int PLANES>
__global__ __launch_bounds__(64 * WR * WC, 1) void fp4_tiles_kernel(Fp4Tiles t) {
    constexpr int NW = WR * WC, WM = BM / WR, WN = BN / WC, MI = WM / 32, NJ = WN / 32, QS = SK / 16, BL = SK / 32;
    constexpr int LDA = BM * SK / (512 * NW), LDB = BN * SK / (2048 * NW), LD = LDA + LDB;      // a wave's loads of a stage: x, codes
    constexpr int SPAN = FP4_SPAN / SK, SLOADS = BN / (64 * NW) > 0 ? BN / (64 * NW) : 1, SROWS = BN / (NW * SLOADS);      // stages of a span of scales; a wave's loads of it, of so many rows
    constexpr int B_AT = BM * SK * 2, STAGE = B_AT + BN * SK / 2, S_AT = RING * STAGE, S_BYTES = BN * 16;
    static_assert(NW == 4 && (SK == 128 || SK == 64) && BM * SK % (512 * NW) == 0 && SROWS * NW * SLOADS == BN, "whole loads of every wave");
    constexpr int PER = MI * NJ, PER_STEP = (LD + QS / 2 - 1) / (QS / 2) < PER ? (LD + QS / 2 - 1) / (QS / 2) : PER, HEAD = 2 * PER_STEP < LD ? 2 * PER_STEP : LD;      // loads of a k step; of the two steps behind the barrier
    static_assert((RING - 2) * LD + HEAD < 64 && LD <= 16 && MI <= PER && PER_STEP * QS >= LD, "the loads in flight can be counted");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Fp4Args& a = t.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);

    int tile_m, tile_n;
    if (!fp4_tile_of(blockIdx.x, t.tiles_m, t.tiles_n, tile_m, tile_n)) return;
    const int m0 = tile_m * (BM / PLANES), n0 = tile_n * BN;
    const int wm = (wave / WC) * WM, wn = (wave % WC) * WN;
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;

    // The loads: per lane the bytes within x (from row m0), the codes and the scales; beyond the matrix: out of range, which arrives as zero.
    // The pieces of a row (of x), of two or four rows that are a line (of the codes), are exchanged by the row's or line's number, so that what
    // 16 lanes read at a time lies in distinct banks.
    int va[LDA], vb[LDB], vs[SLOADS];
    constexpr int AP = SK / 8, AR = 64 / AP;               // pieces of a row of x, rows of a load
    const int a_row = wave * AR + lane / AP;
    const int a_piece = SK == 128 ? (lane & 15) ^ (a_row & 15) : (lane & 7) ^ ((a_row >> 1) & 7);
#pragma unroll
    for (int i = 0; i < LDA; ++i) {
        const int row = i * NW * AR + a_row, plane = row / (BM / PLANES), of_plane = row % (BM / PLANES);
        va[i] = m0 + of_plane < a.M ? plane * (int)t.plane_bytes + of_plane * (int)t.row_bytes + a_piece * 16 : FP4_OUT;
    }
    const int line = lane >> 3, idx = (lane & 7) ^ ((line >> 1) & (SK == 128 ? 3 : 1)), b_piece = idx & (BL - 1);      // (a load is eight lines)
#pragma unroll
    for (int i = 0; i < LDB; ++i) {
        const int row = fp4_matrix_row<TAIL>(n0, ((i * NW + wave) * 8 + line) * (8 / BL) + idx / BL, wide);
        vb[i] = row >= 0 ? row * (a.blocks * 16) + b_piece * 16 : FP4_OUT;
    }
#pragma unroll
    for (int i = 0; i < SLOADS; ++i) {
        const int row = lane < SROWS ? fp4_matrix_row<TAIL>(n0, (i * NW + wave) * SROWS + lane, wide) : -1;
        vs[i] = row >= 0 ? row * t.scale_bytes : FP4_OUT;
    }
    uintx4_t rsrc_a = fp4_buffer((const unsigned char*)t.planes + (unsigned long)m0 * t.row_bytes, t.x_bytes - (unsigned)m0 * t.row_bytes);
    uintx4_t rsrc_b = fp4_buffer(a.codes, (unsigned)((long)a.N * a.blocks * 16)), rsrc_s = fp4_buffer(t.scales, (unsigned)((long)a.N * t.scale_bytes));
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem;
    // The stage that is being asked for: its place in the ring, its step along K, its bytes within x, and the stages left.  The scales of a span of
    // stages come with its first one (or the first of all) into a ring of their own, of one span more than stages are on their way.
    const int first_stage = blockIdx.y * t.per_split, stages = min(t.nk * t.num_planes - first_stage, t.per_split);
    int ask_k = __builtin_amdgcn_readfirstlane(first_stage % t.nk), ask_left = __builtin_amdgcn_readfirstlane(stages);
    unsigned ask_plane = __builtin_amdgcn_readfirstlane(first_stage / t.nk) * t.plane_bytes, ask_at = lds0, ask_span = lds0 + S_AT;
    // (K is no whole stages: of the last one's pieces some lie beyond the row; a lane's offset is then made one that is out of range)
    const int x_left = t.k_in_row - (t.nk - 1) * SK, blocks_left = a.blocks - (t.nk - 1) * BL;
    const int a_off = a_piece * 8 < x_left ? 0 : FP4_OUT, b_off = b_piece < blocks_left ? 0 : FP4_OUT;
    int a_not = t.nk == ask_k + 1 ? a_off : 0, b_not = t.nk == ask_k + 1 ? b_off : 0;
    if constexpr (TAIL == TAIL_PARTIAL) t.a.out = (float*)t.a.out + (long)blockIdx.y * a.M * a.N;
#define LOAD_PIECE(i_)                                                                                                    \
    {                                                                                                                     \
        if ((i_) < LDA) {                                                                                                 \
            constexpr int n_ = (i_) < LDA ? (i_) : 0;                                                                     \
            QE_LOAD_TO_SHARED(ask_at + (n_ * NW + wave_s) * 1024, va[n_] | a_not, rsrc_a, ask_plane + ask_k * (SK * 2), "0", ""); \
        } else {                                                                                                          \
            constexpr int n_ = (i_) < LDA ? 0 : (i_) < LD ? (i_) - LDA : 0;                                               \
            QE_LOAD_TO_SHARED(ask_at + B_AT + (n_ * NW + wave_s) * 1024, vb[n_] | b_not, rsrc_b, ask_k * (SK / 2), "0", ""); \
        }                                                                                                                 \
    }
#define LOAD_SPAN()                                                                                                       \
    {                                                                                                                     \
        if (SROWS == 64 || lane < SROWS) {                                                                                \
            _Pragma("unroll") for (int i = 0; i < SLOADS; ++i)                                                            \
                QE_LOAD_TO_SHARED(ask_span + (i * NW + wave_s) * (SROWS * 16), vs[i], rsrc_s, ask_k / SPAN * 16, "0", ""); \
        }                                                                                                                 \
        ask_span = ask_span + S_BYTES == lds0 + S_AT + (RING + 1) * S_BYTES ? lds0 + S_AT : ask_span + S_BYTES;           \
    }
    // (beyond the last stage every load is out of range: the buffers have no bytes)
#define ASKED()                                                                                                           \
    {                                                                                                                     \
        ask_at = ask_at + STAGE == lds0 + RING * STAGE ? lds0 : ask_at + STAGE;                                           \
        if (++ask_k == t.nk) { ask_k = 0; ask_plane += t.plane_bytes; }                                                   \
        if (--ask_left <= 0) { rsrc_a[2] = 0; rsrc_b[2] = 0; rsrc_s[2] = 0; ask_k = 0; ask_plane = 0; }                   \
        const int ends_ = ask_k + 1 == t.nk ? -1 : 0;                                                                     \
        a_not = a_off & ends_; b_not = b_off & ends_;                                                                     \
    }
    // waits until at most younger_ loads of the wave are in flight and its reads of shared memory are done, then for the other waves
#define MEET(younger_) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(younger_) : "memory");

    // where a lane reads: of x its piece of k step q, of the codes its block of pair b
    int fa_at[QS], fb_at[BL / 2];
#pragma unroll
    for (int q = 0; q < QS; ++q)
        fa_at[q] = SK == 128 ? (wm + r) * 256 + ((((q >> 2) * 8 + (q & 3)) ^ (h * 4) ^ (r & 15)) * 16) : (wm + r) * 128 + ((q ^ (h * 4) ^ ((r >> 1) & 7)) * 16);
#pragma unroll
    for (int b = 0; b < BL / 2; ++b)
        fb_at[b] = B_AT + (SK == 128 ? (wn + r) / 2 * 128 + ((((r & 1) * 4 + 2 * b + h) ^ ((r >> 2) & 3)) * 16)
                                     : (wn + r) / 4 * 128 + ((((r & 3) * 2 + h) ^ ((r >> 3) & 1)) * 16));
    const int fs_at = S_AT + (wn + r) * 16 + h;
    // of the stage that is read from: its step along K and the place of its span
    int read_k = ask_k, read_span = 0;
#define READ_ON()                                                                                                         \
    {                                                                                                                     \
        if (++read_k == t.nk) read_k = 0;                                                                                 \
        if (read_k % SPAN == 0) read_span = read_span + S_BYTES == (RING + 1) * S_BYTES ? 0 : read_span + S_BYTES;        \
    }
    floatx16_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    bf16x8_t fa[4][MI], fb[2][NJ];
    uintx4_t code[2][NJ];                                  // stages of 128: of pairs 0 and 1; of 64: of this stage and of the next
    uint32_t word[2][NJ];
#define READ_A(q_, place_, i_) fa[(q_) & 3][i_] = *(const bf16x8_t*)(smem + (place_) + fa_at[(q_) & (QS - 1)] + (i_) * (SK * 64));
#define READ_CODES(to_, b_, place_, j_)                                                                                   \
    {                                                                                                                     \
        code[to_][j_] = *(const uintx4_t*)(smem + (place_) + fb_at[(b_) < BL / 2 ? (b_) : 0] + (j_) * (SK * 16));         \
        word[to_][j_] = smem[read_span + read_k % SPAN * BL + fs_at + (b_) * 2 + (j_) * 512];                             \
    }
    // the eight numbers of k step q_, of the codes that are in registers
#define EXPAND(q_, j_)                                                                                                    \
    {                                                                                                                     \
        constexpr int of_ = SK == 128 ? ((q_) >> 2) & 1 : 0;                                                              \
        fb[(q_) & 1][j_] = fp4_to_bf16(code[of_][j_][(q_) & 3], __uint_as_float(word[of_][j_] << 23));                    \
    }
    // k step q_: between its matrix instructions the fragments of x of the step after the next are read, the next step's codes expanded, and the
    // loads of the stage that is being asked for go out, from the step behind the barrier on
#define K_STEP(q_, place_, next_)                                                                                         \
    {                                                                                                                     \
        if (SK == 64 && (q_) == QS - 1) {                                                                                 \
            _Pragma("unroll") for (int j = 0; j < NJ; ++j) { code[0][j] = code[1][j]; word[0][j] = word[1][j]; }          \
        }                                                                                                                 \
        if ((q_) == QS - 2) READ_ON()                                                                                     \
        _Pragma("unroll") for (int sl = 0; sl < PER; ++sl) {                                                              \
            if (sl < MI) { if ((q_) < QS - 2) { READ_A((q_) + 2, place_, sl < MI ? sl : 0) } else { READ_A((q_) + 2 - QS, next_, sl < MI ? sl : 0) } } \
            if (sl < NJ) {                                                                                                \
                if (SK == 128 && (q_) == 1) READ_CODES(1, 1, place_, sl < NJ ? sl : 0)                                    \
                if ((q_) == QS - 2) READ_CODES(SK == 128 ? 0 : 1, 0, next_, sl < NJ ? sl : 0)                             \
            }                                                                                                             \
            acc[sl % MI][sl / MI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[(q_) & 3][sl % MI], fb[(q_) & 1][sl / MI], acc[sl % MI][sl / MI], 0, 0, 0); \
            if (sl % MI == 0) { EXPAND(((q_) + 1) & (QS - 1), sl / MI) }                                                  \
            _Pragma("unroll") for (int l = 0; l < PER_STEP; ++l)                                                          \
                if (l * PER / PER_STEP == sl) LOADS_OF((((q_) + 2) & (QS - 1)) * PER_STEP + l)                            \
            __builtin_amdgcn_sched_barrier(0);                                                                            \
        }                                                                                                                 \
        if ((q_) == QS - 3) { ASKED() MEET((RING - 2) * LD) if (ask_left > 0 && ask_k % SPAN == 0) LOAD_SPAN() }          \
    }
#define LOADS_OF(n_)                                                                                                      \
    switch (n_) {                                                                                                         \
        case 0: LOAD_CASE(0) case 1: LOAD_CASE(1) case 2: LOAD_CASE(2) case 3: LOAD_CASE(3) case 4: LOAD_CASE(4)          \
        case 5: LOAD_CASE(5) case 6: LOAD_CASE(6) case 7: LOAD_CASE(7) case 8: LOAD_CASE(8) case 9: LOAD_CASE(9)          \
        case 10: LOAD_CASE(10) case 11: LOAD_CASE(11) case 12: LOAD_CASE(12) case 13: LOAD_CASE(13) case 14: LOAD_CASE(14) \
        case 15: LOAD_CASE(15) default: break;                                                                            \
    }
#define LOAD_CASE(i_) if constexpr ((i_) < LD) LOAD_PIECE(i_) break;

    // (the scales come before their stages' codes, and a stage is waited for by the loads behind it: with more of those than are counted,
    // where a span lies between, the wait is only longer)
    LOAD_SPAN()
#pragma unroll
    for (int s = 0; s < RING; ++s) {
        if (s > 0 && ask_left > 0 && ask_k % SPAN == 0) LOAD_SPAN()
#pragma unroll
        for (int i = 0; i < LD; ++i)
            if (s + 1 < RING || i < HEAD) { LOADS_OF(i) }
        if (s + 1 < RING) ASKED()
    }
    MEET((RING - 2) * LD + HEAD)
#pragma unroll
    for (int j = 0; j < NJ; ++j) READ_CODES(0, 0, 0, j)
#pragma unroll
    for (int i = 0; i < MI; ++i) { READ_A(0, 0, i) READ_A(1, 0, i) }
#pragma unroll
    for (int j = 0; j < NJ; ++j) EXPAND(0, j)
    int at = 0;
    for (int st = 0; st < stages; ++st) {
        const int next = at + STAGE == RING * STAGE ? 0 : at + STAGE;
        K_STEP(0, at, next)
        K_STEP(1, at, next)
        K_STEP(2, at, next)
        K_STEP(3, at, next)
        if constexpr (SK == 128) {
            K_STEP(4, at, next)
            K_STEP(5, at, next)
            K_STEP(6, at, next)
            K_STEP(7, at, next)
        }
        at = next;
    }
    MEET(0)                                                // (what was asked for beyond the end has arrived)
#undef K_STEP
#undef LOADS_OF
#undef LOAD_CASE
#undef LOAD_PIECE
#undef LOAD_SPAN
#undef READ_ON
#undef ASKED
#undef MEET
#undef READ_A
#undef READ_CODES
#undef EXPAND
    static_assert(4 * fp4_strip_bytes<NJ>() <= S_AT, "the waves' strips must fit the ring");
    if constexpr (PLANES == 3) {
        static_assert(MI == 3 && WR == 1, "a plane is a wave's 32 rows");
        floatx16_t sum[1][NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) sum[0][j] = acc[0][j] + acc[1][j] + acc[2][j];
        fp4_store_tiles<TAIL, 1, NJ>(a, sum, m0, n0 + wn, smem + wave * fp4_strip_bytes<NJ>());
    } else {
        fp4_store_tiles<TAIL, MI, NJ>(a, acc, m0 + wm, n0 + wn, smem + wave * fp4_strip_bytes<NJ>());
    }
}

template <int TAIL, int BM, int BN, int WR, int WC, int SK, int RING, int PLANES = 1>
static int fp4_tiles_launch(Fp4Tiles t, int splits, hipStream_t stream) {
    constexpr int SHARED = RING * (BM * SK * 2 + BN * SK / 2) + (RING + 1) * BN * 16;
    static_assert(SHARED <= 160 * 1024, "the ring must fit a compute unit");
    t.tiles_m = qe_cdiv(t.a.M, BM / PLANES);
    t.tiles_n = qe_cdiv(t.a.N, BN);
    const long blocks = ((long)t.tiles_m * t.tiles_n + 7) / 8 * 8;
    QE_REQUIRE(blocks <= 2147483647L, "gemm_mxfp4: too many tiles");
    QE_RAISE_SHARED((fp4_tiles_kernel<TAIL, BM, BN, WR, WC, SK, RING, PLANES>), SHARED);
    fp4_tiles_kernel<TAIL, BM, BN, WR, WC, SK, RING, PLANES><<<dim3((unsigned)blocks, (unsigned)splits), 256, SHARED, stream>>>(t);
    return 0;
}

// The kernel's 32-bit places reach all of the operands.
bool fp4_tiles_take(int M, int N, int K, int x_kind) {
    return (long)N * padded(K) / 2 < (1L << 31) && (long)M * padded(K) * 2 * (x_kind == X_F32 ? 3 : 1) < (1L << 31);
}

// The rows of x of a tile (32: of three planes), the numbers of K of its stages, and in how many cuts of K the tiles fill the chip.
struct Fp4Shape {
    int bm, sk, per_split, splits;
};

// A round of tiles of so many rows (one a unit) takes `round` us and `stage` us for 128 of K, as measured (with rounds of them: 4096 x 24576, 12288, 6144;
// 1024 x 40000, 3000; 12288 x 4096; 65 to 2048 rows).  Of 64 rows two share a unit, 1.04 us a stage; alone there, 0.62.
struct Fp4TileCost {
    int bm;
    double round, stage;
};
static const Fp4TileCost fp4_tile_costs[] = {{32, 4.1, 0.68}, {64, 3.4, 1.04}, {96, 4.1, 0.68}, {128, 4.6, 0.80}, {160, 6.0, 0.93}, {256, 12.8, 2.27}};

// The tiles that are done first by these times: what counts is how many rounds the units make and how many of a tile's rows are idle (65 rows
// against 24576 x 4096 by 96 rows 27.5 us, by 64 36.4; 160 rows by 160 37.4, by 64 51.8; 256 rows by 64 58.8, by 160 71; 700 against
// 6144 x 4096 by 160 39, by 128 60; 512 against 24576 x 4096 by 256 92, by 128 103).  Over 53 sizes the choice is 0.6 % slower than the best one on the
// average, 9 % at the most.
// K in cuts where that leaves a block a unit at the most and a cut eight stages, at the price of the join (64 rows against 4096 x 4096 in four cuts
// 13.9 us, eight 16.0; against 4096 x 12288 in eight 18.1, four 21.0; against 24576 x 4096, 192 tiles, uncut 24.1, two 26.2).
static Fp4Shape fp4_tiles_shape(int M, int N, int K, int x_kind) {
    Fp4Shape best{};
    double least = 0.0;
    for (const Fp4TileCost& c : fp4_tile_costs) {
        if (c.bm == 32 && x_kind != X_F32) continue;
        Fp4Shape s;
        s.bm = c.bm;
        s.sk = c.bm == 256 ? 64 : 128;
        const int planes = x_kind == X_F32 && c.bm != 32 ? 3 : 1, stages = qe_cdiv(K, s.sk) * planes;
        const long tiles = (long)qe_cdiv(M, s.bm) * qe_cdiv(N, s.bm == 256 ? 256 : 128);
        long splits = s.bm == 256 ? 1 : 256 / tiles;
        if (splits > stages / 8) splits = stages / 8;
        if (splits < 1) splits = 1;
        s.per_split = qe_cdiv(stages, (int)splits);
        s.splits = qe_cdiv(stages, s.per_split);
        const double walk = (double)s.per_split * s.sk / 128;      // in stages of 128
        const long blocks = tiles * s.splits;
        double time = (double)qe_cdiv(blocks, 256) * (c.round + c.stage * walk);
        if (s.bm == 64) {
            const long rest = blocks % 512;
            time = (double)(blocks / 512 + (rest > 256)) * (c.round + c.stage * walk) + (rest > 0 && rest <= 256 ? 3.0 + 0.62 * walk : 0.0);
        }
        if (s.splits > 1) time += 3.0 + 2e-6 * s.splits * (double)M * N;
        if (best.bm == 0 || time < least) { best = s; least = time; }
    }
    return best;
}

long fp4_tiles_workspace(int M, int N, int K, int x_kind, const void* x, const void* scales) {
    const bool aligned = ((uintptr_t)x & 15) == 0;
    const Fp4Shape s = fp4_tiles_shape(M, N, K, x_kind);
    long bytes = s.splits > 1 ? (4L * s.splits * M * N + 15) / 16 * 16 : 0;
    if (x_kind == X_F32 || K % 8 || !aligned) bytes += fp4_planes_bytes(M, K, x_kind);
    return bytes + (fp4_scales_whole(K, scales, s.sk) ? 0 : fp4_scales_bytes(N, K));
}

int fp4_tiles(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream) {
    const Fp4Shape s = fp4_tiles_shape(a.M, a.N, a.K, x_kind);
    Fp4Tiles t{};
    t.a = a;
    t.nk = qe_cdiv(a.K, s.sk);
    t.per_split = s.per_split;
    // the workspace: the cuts' products, then what is made of x, then of the scales
    float* parts = (float*)workspace;
    unsigned char* ws = (unsigned char*)workspace + (s.splits > 1 ? (4L * s.splits * a.M * a.N + 15) / 16 * 16 : 0);
    const bool copy_x = x_kind == X_F32 || a.K % 8 || ((uintptr_t)a.x & 15), copy_scales = !fp4_scales_whole(a.K, a.scales, s.sk);
    unsigned char* const scales_at = ws + (copy_x ? fp4_planes_bytes(a.M, a.K, x_kind) : 0);
    Fp4Rows x{a.x, a.K * 2, 1};
    if (copy_x || copy_scales) {
        const Fp4Rows copied = fp4_copies(a.x, a.M, a.K, x_kind, copy_x ? ws : nullptr, a.scales, a.N, copy_scales ? scales_at : nullptr, stream);
        if (copy_x) x = copied;
    }
    t.planes = (const uint16_t*)x.data;
    t.num_planes = s.bm == 32 ? 1 : x.planes;          // (that are walked)
    t.row_bytes = (unsigned)x.row_bytes;
    t.k_in_row = x.row_bytes / 2;
    t.plane_bytes = t.row_bytes * (unsigned)a.M;
    t.x_bytes = t.plane_bytes * x.planes;
    t.scales = copy_scales ? scales_at : a.scales;
    t.scale_bytes = fp4_scales_row(a.K, !copy_scales);
    if (s.splits > 1) t.a.out = parts;
    int rc;
#define QE_GO(T_)                                                                            \
    rc = s.bm == 256   ? fp4_tiles_launch<T_, 256, 256, 2, 2, 64, 3>(t, s.splits, stream)     \
         : s.bm == 160 ? fp4_tiles_launch<T_, 160, 128, 1, 4, 128, 3>(t, s.splits, stream)    \
         : s.bm == 128 ? fp4_tiles_launch<T_, 128, 128, 2, 2, 128, 3>(t, s.splits, stream)    \
         : s.bm == 96  ? fp4_tiles_launch<T_, 96, 128, 1, 4, 128, 3>(t, s.splits, stream)     \
         : s.bm == 32  ? fp4_tiles_launch<T_, 96, 128, 1, 4, 128, 3, 3>(t, s.splits, stream)  \
                       : fp4_tiles_launch<T_, 64, 128, 1, 4, 128, 3>(t, s.splits, stream)
    if (s.splits > 1)
        rc = s.bm == 160   ? fp4_tiles_launch<TAIL_PARTIAL, 160, 128, 1, 4, 128, 3>(t, s.splits, stream)
             : s.bm == 128 ? fp4_tiles_launch<TAIL_PARTIAL, 128, 128, 2, 2, 128, 3>(t, s.splits, stream)
             : s.bm == 96  ? fp4_tiles_launch<TAIL_PARTIAL, 96, 128, 1, 4, 128, 3>(t, s.splits, stream)
             : s.bm == 32  ? fp4_tiles_launch<TAIL_PARTIAL, 96, 128, 1, 4, 128, 3, 3>(t, s.splits, stream)
                           : fp4_tiles_launch<TAIL_PARTIAL, 64, 128, 1, 4, 128, 3>(t, s.splits, stream);
    else if (tail == TAIL_STORE) QE_GO(TAIL_STORE);
    else if (tail == TAIL_ADD) QE_GO(TAIL_ADD);
    else QE_GO(TAIL_SILU);
#undef QE_GO
    if (rc) return rc;
    if (s.splits > 1 && (rc = fp4_join(a, parts, s.splits, tail, stream))) return rc;
    QE_LAUNCH_CHECK();
    return 0;
}
