// Products of many rows of 16-bit or 32-bit numbers with a 4-bit matrix (see mxfp4.h): out[M, N] = x[M, K] . V[N, K]^T.
//
// A block of WR x WC waves computes BM rows by BN columns.  K is walked in stages of 128 through a ring in shared memory: 256 bytes of a
// row of x, 64 of codes and 4 of scales of a row of the matrix, brought by loads that write to shared memory directly.  A
// wave multiplies its part in tiles of 32 x 32 with v_mfma_f32_32x32x16_bf16: lane (r, h) = (lane % 32, lane / 32) takes, of row r,
// block 2 b + h of the stage's four, so that a 16-byte piece of codes with one scale gives four matrix instructions' operands, eight numbers
// each, by four conversions each.  The conversions for the next k step stand between the matrix instructions of this one.
//
// Rows of 32-bit numbers come as three planes of bfloat16 (cut_in_three) that are walked one after the other, the smallest
// first, against the same matrix; they are made by a launch of their own, which also fills K up to whole stages.
#include "mxfp4.h"

#define FP4_STAGE 128      // numbers of K

// x [M, K] float32 -> planes [3][M][Kp] (low, middle, high) of bfloat16, zeros from K on; bfloat16 -> [M][Kp]
template <typename T>
__global__ __launch_bounds__(256) void fp4_planes_kernel(const T* __restrict__ x, uint16_t* __restrict__ planes, int M, int K, int Kp) {
    const long plane = (long)M * Kp;
    for (long row = blockIdx.y; row < M; row += gridDim.y) {
        const int k = (blockIdx.x * 256 + threadIdx.x) * 4;
        if (k >= Kp) return;
        uint16_t hi[4], mid[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool have = k + e < K;
            if constexpr (sizeof(T) == 4) cut_in_three(have ? x[row * K + k + e] : 0.f, hi[e], mid[e], lo[e]);
            else hi[e] = have ? x[row * K + k + e].bits : 0;
        }
        uint16_t* to = planes + row * Kp + k;
        if constexpr (sizeof(T) == 4) {
            *(ushort4*)to = make_ushort4(lo[0], lo[1], lo[2], lo[3]);
            *(ushort4*)(to + plane) = make_ushort4(mid[0], mid[1], mid[2], mid[3]);
            *(ushort4*)(to + 2 * plane) = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
        } else {
            *(ushort4*)to = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
        }
    }
}

// scales [N, blocks] -> [N, padded], zeros behind
__global__ __launch_bounds__(256) void fp4_scales_kernel(const unsigned char* __restrict__ scales, uint32_t* __restrict__ out, int N,
                                                         int blocks, int words) {
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long)N * words) return;
    const long row = at / words;
    const int b = (int)(at - row * words) * 4;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (b + e < blocks) v |= (uint32_t)scales[row * blocks + b + e] << (8 * e);
    out[at] = v;
}

void fp4_pad_scales(const unsigned char* scales, uint32_t* words, int rows, int blocks, int num_words, hipStream_t stream) {
    fp4_scales_kernel<<<qe_cdiv((long)rows * num_words, 256), 256, 0, stream>>>(scales, words, rows, blocks, num_words);
}

struct Fp4Tiles {
    Fp4Args a;
    const uint16_t* planes;     // rows of x, row_bytes apart, plane after plane
    const uint32_t* words;      // the scales, `words` words a row
    unsigned row_bytes, plane_bytes, x_bytes;      // (x_bytes: of all planes)
    int num_planes, nk, num_words;
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

template <int TAIL, int BM, int BN, int WR, int WC, int RING>
__global__ __launch_bounds__(64 * WR * WC, 1) void fp4_tiles_kernel(Fp4Tiles t) {
    constexpr int NW = WR * WC, WM = BM / WR, WN = BN / WC, MI = WM / 32, NJ = WN / 32;
    constexpr int LDA = BM / (4 * NW), LDB = BN / (16 * NW), LD = LDA + LDB + 1, SROWS = BN / NW;
    constexpr int B_AT = BM * 256, S_AT = B_AT + BN * 64, STAGE = S_AT + NW * 256;
    static_assert(BM % (4 * NW) == 0 && BN % (16 * NW) == 0 && SROWS <= 64 && (RING - 1) * LD + 4 < 64 && MI * NJ >= 2, "whole loads of every wave");
    static_assert(TAIL != TAIL_SILU || NJ % 2 == 0, "a wave has the gate and the up of its columns");
    constexpr int PER_STEP = (LD + 7) / 8;                 // loads of a k step
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Fp4Args& a = t.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);

    int tile_m, tile_n;
    if (!fp4_tile_of(blockIdx.x, t.tiles_m, t.tiles_n, tile_m, tile_n)) return;
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int wm = (wave / WC) * WM, wn = (wave % WC) * WN;
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;

    // the loads: per lane the bytes within x (from row m0), the codes and the scales; beyond the matrix: out of range, which arrives as zero
    int va[LDA], vb[LDB], vs;
#pragma unroll
    for (int i = 0; i < LDA; ++i) {
        const int row = (i * NW + wave) * 4 + (lane >> 4);
        va[i] = m0 + row < a.M ? row * (int)t.row_bytes + ((lane & 15) ^ (row & 15)) * 16 : FP4_OUT;
    }
    int piece[LDB];                                        // the block of the stage that this lane brings
#pragma unroll
    for (int i = 0; i < LDB; ++i) {
        const int line = (i * NW + wave) * 8 + (lane >> 3), idx = (lane & 7) ^ (line & 7);
        const int row = fp4_matrix_row<TAIL>(n0, line * 2 + (idx >> 2), wide);
        piece[i] = row >= 0 ? idx & 3 : 1 << 28;
        vb[i] = row * (a.blocks * 16) + (idx & 3) * 16;
    }
    {
        const int row = lane < SROWS ? fp4_matrix_row<TAIL>(n0, wave * SROWS + lane, wide) : -1;
        vs = row >= 0 ? row * (t.num_words * 4) : FP4_OUT;
    }
    const uintx4_t rsrc_a = fp4_buffer((const unsigned char*)t.planes + (unsigned long)m0 * t.row_bytes, t.x_bytes - (unsigned)m0 * t.row_bytes);
    const uintx4_t rsrc_b = fp4_buffer(a.codes, (unsigned)((long)a.N * a.blocks * 16)), rsrc_s = fp4_buffer(t.words, (unsigned)((long)a.N * t.num_words * 4));
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem;
    // the stage that is being asked for: its place in the ring, its plane's bytes, its step along K, and the stages left
    const int first_stage = blockIdx.y * t.per_split, stages = min(t.nk * t.num_planes - first_stage, t.per_split);
    int ask_k = first_stage % t.nk, ask_left = stages;
    unsigned ask_x = (unsigned)(first_stage / t.nk) * t.plane_bytes, ask_at = lds0;
    if constexpr (TAIL == TAIL_PARTIAL) t.a.out = (float*)t.a.out + (long)blockIdx.y * a.M * a.N;
#define LOAD_PIECE(i_)                                                                                                    \
    {                                                                                                                     \
        const bool there = ask_left > 0;                                                                                  \
        if ((i_) < LDA) {                                                                                                 \
            const int v_ = there ? va[(i_) < LDA ? (i_) : 0] : FP4_OUT;                                                       \
            QE_LOAD_TO_SHARED(ask_at + ((i_) * NW + wave_s) * 1024, v_, rsrc_a, there ? ask_x + ask_k * 256 : 0, "0", ""); \
        } else if ((i_) < LDA + LDB) {                                                                                    \
            constexpr int b_ = (i_) < LDA ? 0 : (i_) < LDA + LDB ? (i_) - LDA : 0;                                        \
            const int v_ = there && ask_k * 4 + piece[b_] < a.blocks ? vb[b_] : FP4_OUT;                                      \
            QE_LOAD_TO_SHARED(ask_at + B_AT + (b_ * NW + wave_s) * 1024, v_, rsrc_b, there ? ask_k * 64 : 0, "0", "");   \
        } else {                                                                                                          \
            const int v_ = there ? vs : FP4_OUT;                                                                              \
            QE_LOAD_WORD_TO_SHARED(ask_at + S_AT + wave_s * 256, v_, rsrc_s, there ? ask_k * 4 : 0);                      \
        }                                                                                                                 \
    }
#define ASKED()                                                                                                           \
    {                                                                                                                     \
        ask_at = ask_at + STAGE == lds0 + RING * STAGE ? lds0 : ask_at + STAGE;                                           \
        --ask_left;                                                                                                       \
        if (++ask_k == t.nk) { ask_k = 0; ask_x += t.plane_bytes; }                                                       \
    }
    // waits until at most younger_ loads of the wave are in flight and its reads of shared memory are done, then for the other waves
#define MEET(younger_) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(younger_) : "memory");

    // where a lane reads: of x its piece of k step q, of the codes its block of pair b, of the scales its row's word
    int fa_at[8], fb_at[2], fs_at;
#pragma unroll
    for (int q = 0; q < 8; ++q) fa_at[q] = (wm + r) * 256 + ((((q >> 2) * 8 + (q & 3)) ^ (h * 4) ^ (r & 15)) * 16);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int row = wn + r, line = row >> 1;
        fb_at[b] = B_AT + line * 128 + ((((row & 1) * 4 + 2 * b + h) ^ (line & 7)) * 16);
    }
    floatx16_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    bf16x8_t fa[4][MI], fb[2][NJ];
    uintx4_t code[2][NJ];
    uint32_t word[NJ], word_next[NJ];
#define READ_A(q_, place_) _Pragma("unroll") for (int i = 0; i < MI; ++i) fa[(q_) & 3][i] = *(const bf16x8_t*)(smem + (place_) + fa_at[(q_) & 7] + i * 8192);
#define READ_CODES(b_, place_) _Pragma("unroll") for (int j = 0; j < NJ; ++j) code[b_][j] = *(const uintx4_t*)(smem + (place_) + fb_at[b_] + j * 2048);
#define READ_SCALES(place_)                                                                                               \
    _Pragma("unroll") for (int j = 0; j < NJ; ++j) {                                                                      \
        const int row = wn + j * 32 + r;                                                                                  \
        word_next[j] = *(const uint32_t*)(smem + (place_) + S_AT + (row / SROWS) * 256 + (row % SROWS) * 4);              \
    }
#define EXPAND(q_, j_) fb[(q_) & 1][j_] = fp4_to_bf16(code[((q_) >> 2) & 1][j_][(q_) & 3], __uint_as_float((word[j_] >> (((((q_) >> 2) & 1) * 2 + h) * 8) & 255u) << 23));
    // k step q_: between its matrix instructions the fragments of x of the step after the next are read, the next step's codes expanded, and the
    // loads of the stage that is being asked for go out, from the step behind the barrier on
#define K_STEP(q_, place_, next_)                                                                                         \
    {                                                                                                                     \
        if ((q_) < 6) { READ_A((q_) + 2, place_) } else { READ_A((q_) - 6, next_) }                                       \
        if ((q_) == 1) { READ_CODES(1, place_) }                                                                          \
        if ((q_) == 6) { READ_CODES(0, next_) READ_SCALES(next_) }                                                        \
        if ((q_) == 7) { _Pragma("unroll") for (int j = 0; j < NJ; ++j) word[j] = word_next[j]; }                         \
        _Pragma("unroll") for (int sl = 0; sl < MI * NJ; ++sl) {                                                          \
            acc[sl % MI][sl / MI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[(q_) & 3][sl % MI], fb[(q_) & 1][sl / MI], acc[sl % MI][sl / MI], 0, 0, 0); \
            if (sl % MI == 0) { EXPAND(((q_) + 1) & 7, sl / MI) }                                                         \
            if (sl < PER_STEP) LOADS_OF((((q_) + 2) & 7) * PER_STEP + sl)                                                 \
            __builtin_amdgcn_sched_barrier(0);                                                                            \
        }                                                                                                                 \
        if ((q_) == 5) { ASKED() MEET((RING - 2) * LD) }                                                                  \
    }
#define LOADS_OF(n_)                                                                                                      \
    switch (n_) {                                                                                                         \
        case 0: LOAD_CASE(0) case 1: LOAD_CASE(1) case 2: LOAD_CASE(2) case 3: LOAD_CASE(3) case 4: LOAD_CASE(4)          \
        case 5: LOAD_CASE(5) case 6: LOAD_CASE(6) case 7: LOAD_CASE(7) case 8: LOAD_CASE(8) case 9: LOAD_CASE(9)          \
        case 10: LOAD_CASE(10) case 11: LOAD_CASE(11) case 12: LOAD_CASE(12) case 13: LOAD_CASE(13) case 14: LOAD_CASE(14) \
        case 15: LOAD_CASE(15) default: break;                                                                            \
    }
#define LOAD_CASE(i_) if constexpr ((i_) < LD) LOAD_PIECE(i_) break;
    static_assert(LD <= 16 && PER_STEP <= MI * NJ, "a case for every load, a slot for every load of a step");

    constexpr int HEAD = 2 * PER_STEP < LD ? 2 * PER_STEP : LD;          // of a stage's loads, those that go out in the two steps behind the barrier
#pragma unroll
    for (int s = 0; s < RING; ++s) {
#pragma unroll
        for (int i = 0; i < LD; ++i)
            if (s + 1 < RING || i < HEAD) { LOADS_OF(i) }
        if (s + 1 < RING) ASKED()
    }
    MEET((RING - 2) * LD + HEAD)
    READ_CODES(0, 0)
    READ_SCALES(0)
    READ_A(0, 0)
    READ_A(1, 0)
#pragma unroll
    for (int j = 0; j < NJ; ++j) word[j] = word_next[j];
#pragma unroll
    for (int j = 0; j < NJ; ++j) { EXPAND(0, j) }
    int at = 0;
    for (int st = 0; st < stages; ++st) {
        const int next = at + STAGE == RING * STAGE ? 0 : at + STAGE;
        K_STEP(0, at, next)
        K_STEP(1, at, next)
        K_STEP(2, at, next)
        K_STEP(3, at, next)
        K_STEP(4, at, next)
        K_STEP(5, at, next)
        K_STEP(6, at, next)
        K_STEP(7, at, next)
        at = next;
    }
    MEET(0)                                                // (what was asked for beyond the end has arrived)
#undef K_STEP
#undef LOADS_OF
#undef LOAD_CASE
#undef LOAD_PIECE
#undef ASKED
#undef MEET
#undef READ_A
#undef READ_CODES
#undef READ_SCALES
#undef EXPAND

    fp4_store_tiles<TAIL, MI, NJ>(a, acc, m0 + wm, n0 + wn);
}

template <int TAIL, int BM, int BN, int WR, int WC, int RING>
static int fp4_tiles_launch(Fp4Tiles t, int splits, hipStream_t stream) {
    constexpr int NW = WR * WC, SHARED = RING * (BM * 256 + BN * 64 + NW * 256);
    t.tiles_m = qe_cdiv(t.a.M, BM);
    t.tiles_n = qe_cdiv(t.a.N, BN);
    const long blocks = ((long)t.tiles_m * t.tiles_n + 7) / 8 * 8;
    QE_REQUIRE(blocks <= 2147483647L, "gemm_mxfp4: too many tiles");
    QE_RAISE_SHARED((fp4_tiles_kernel<TAIL, BM, BN, WR, WC, RING>), SHARED);
    fp4_tiles_kernel<TAIL, BM, BN, WR, WC, RING><<<dim3((unsigned)blocks, (unsigned)splits), 64 * NW, SHARED, stream>>>(t);
    return 0;
}

static int padded(int K) { return qe_cdiv(K, FP4_STAGE) * FP4_STAGE; }

// The kernel's 32-bit places reach all of the operands.
bool fp4_tiles_take(int M, int N, int K, int x_kind) {
    return (long)N * padded(K) / 2 < (1L << 31) && (long)M * padded(K) * 2 * (x_kind == X_F32 ? 3 : 1) < (1L << 31);
}

// The rows of a tile, and in how many cuts of K the tiles fill the chip.
static int fp4_tiles_shape(int M, int N, int K, int x_kind, int* per_split) {
    const int stages = padded(K) / FP4_STAGE * (x_kind == X_F32 ? 3 : 1);
    const long rows64 = qe_cdiv(M, 64) * 64L, rows128 = qe_cdiv(M, 128) * 128L;
    const int bm = M <= 64 || (M <= 512 && rows128 * 100 > rows64 * 115) ? 64 : 128;
    const long tiles = (long)qe_cdiv(M, bm) * qe_cdiv(N, 128), slots = bm == 64 ? 512 : 256;
    long splits = slots / tiles;
    if (splits > stages / 4) splits = stages / 4;
    if (splits < 1) splits = 1;
    *per_split = qe_cdiv(stages, (int)splits);
    return bm;
}

long fp4_tiles_workspace(int M, int N, int K, int x_kind, bool aligned) {
    int per_split;
    fp4_tiles_shape(M, N, K, x_kind, &per_split);
    const int splits = qe_cdiv(padded(K) / FP4_STAGE * (x_kind == X_F32 ? 3 : 1), per_split);
    long bytes = splits > 1 ? 4L * splits * M * N : 0;
    bytes = (bytes + 15) / 16 * 16;
    if (x_kind == X_F32) bytes += 6L * M * padded(K);
    else if (K % FP4_STAGE || !aligned) bytes += 2L * M * padded(K);
    if (K % FP4_STAGE || !aligned) bytes += (long)N * (padded(K) / 32);
    return bytes;
}

int fp4_tiles(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream) {
    Fp4Tiles t{};
    t.a = a;
    const int Kp = padded(a.K);
    t.nk = Kp / FP4_STAGE;
    t.num_words = Kp / FP4_STAGE;
    t.num_planes = x_kind == X_F32 ? 3 : 1;
    t.row_bytes = (unsigned)Kp * 2;
    t.plane_bytes = (unsigned)((long)a.M * Kp * 2);
    t.x_bytes = t.plane_bytes * t.num_planes;
    // the workspace: the cuts' products, then what is made of x and of the scales
    float* parts = (float*)workspace;
    unsigned char* ws = (unsigned char*)workspace;
    {
        int per_split;
        fp4_tiles_shape(a.M, a.N, a.K, x_kind, &per_split);
        const int cuts = qe_cdiv(t.nk * t.num_planes, per_split);
        if (cuts > 1) ws += (4L * cuts * a.M * a.N + 15) / 16 * 16;
    }
    const dim3 grid(qe_cdiv(Kp, 1024), a.M < 65535 ? a.M : 65535);
    if (x_kind == X_F32) {
        fp4_planes_kernel<float><<<grid, 256, 0, stream>>>((const float*)a.x, (uint16_t*)ws, a.M, a.K, Kp);
        t.planes = (const uint16_t*)ws;
        ws += t.x_bytes;
    } else if (a.K % FP4_STAGE || ((uintptr_t)a.x & 15)) {
        fp4_planes_kernel<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)a.x, (uint16_t*)ws, a.M, a.K, Kp);
        t.planes = (const uint16_t*)ws;
        ws += t.x_bytes;
    } else {
        t.planes = (const uint16_t*)a.x;
    }
    if (a.K % FP4_STAGE || ((uintptr_t)a.scales & 3)) {
        fp4_pad_scales(a.scales, (uint32_t*)ws, a.N, a.blocks, t.num_words, stream);
        t.words = (const uint32_t*)ws;
    } else {
        t.words = (const uint32_t*)a.scales;
    }
    const int bm = fp4_tiles_shape(a.M, a.N, a.K, x_kind, &t.per_split);
    const int splits = qe_cdiv(t.nk * t.num_planes, t.per_split);
    if (splits > 1) t.a.out = parts;
    int rc;
#define QE_GO(T_) rc = bm == 64 ? fp4_tiles_launch<T_, 64, 128, 2, 2, 3>(t, splits, stream) : fp4_tiles_launch<T_, 128, 128, 2, 2, 3>(t, splits, stream)
    if (splits > 1) QE_GO(TAIL_PARTIAL);
    else if (tail == TAIL_STORE) QE_GO(TAIL_STORE);
    else if (tail == TAIL_ADD) QE_GO(TAIL_ADD);
    else QE_GO(TAIL_SILU);
#undef QE_GO
    if (rc) return rc;
    if (splits > 1 && (rc = fp4_join(a, parts, splits, tail, stream))) return rc;
    QE_LAUNCH_CHECK();
    return 0;
}
