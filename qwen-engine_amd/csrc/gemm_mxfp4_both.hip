// Products of many rows in 4 bits with a 4-bit matrix (see mxfp4.h): out[M, N] = sum_k x[m, k] v[n, k], by
// v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies codes with their blocks' scales.
//
// A block of 2 x 2 waves computes 128 rows by 128 columns (256 by 256: the second kernel).  K is walked in stages of 128 through a ring
// of four in shared memory: 64 bytes of codes a row, of both sides alike, and for every four stages 16 of scales, brought by loads that
// write to shared memory directly.  Two rows are a line of 128 bytes there, its eight pieces exchanged by the line's number (so that what 16 lanes read at a time lies in distinct banks).  Lane (r, h) =
// (lane % 32, lane / 32) takes blocks 2 h and 2 h + 1 of row r, one in each of the stage's two k steps; the fragments of a step are
// read while the step before is multiplied.
//
// 4096 rows against 4096 x 12288 take 98 us, 4.2 PFLOP/s of the 6.65 that the instruction reaches alone; 512 rows against 4096 x 4096 19 us with their quantisation.
#include "mxfp4.h"

#define FP4_STAGE 128      // numbers of K
#define FP4_RING 4

// What the loads cannot take as it is, in one launch: the codes of x with nothing behind K in a row's last block (where K is no whole
// blocks), and the scales of x and of the matrix in rows of whole spans, zeros behind.
struct Fp4Prepare {
    const uintx4_t* codes;
    uintx4_t* codes_out;
    const unsigned char *xs, *scales;
    uint32_t *xs_out, *scales_out;
    unsigned pieces, x_words, words;    // numbers of 16-byte pieces and of words to write, 0: none
    unsigned blocks, num_words;
    int K;
};

__global__ __launch_bounds__(256) void fp4_prepare_kernel(Fp4Prepare p) {
    unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at < p.pieces) {
        const int left = p.K - (int)(at % p.blocks) * 32;
        const uintx4_t c = p.codes[at];
        p.codes_out[at] = left < 32 ? first_codes(c, left) : c;
        return;
    }
    at -= p.pieces;
    const unsigned char* from = p.xs;
    uint32_t* to = p.xs_out;
    if (at >= p.x_words) {
        at -= p.x_words;
        if (at >= p.words) return;
        from = p.scales;
        to = p.scales_out;
    }
    const long row = at / p.num_words;
    const int b = (int)(at % p.num_words) * 4;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (b + e < (int)p.blocks) v |= (uint32_t)from[row * p.blocks + b + e] << (8 * e);
    to[at] = v;
}

struct Fp4Both {
    Fp4Args a;
    const unsigned char* x;     // codes, nothing behind K
    const unsigned char *xs, *scales;   // of x and of the matrix, so many bytes from a row to the next
    int x_scale_bytes, scale_bytes;
    int nk, tiles_m, tiles_n;
    int per_split;                      // stages of a cut of K, whole spans: block (., y) sums those from y * per_split on
};

template <int TAIL>
__global__ __launch_bounds__(256, 2) void fp4_both_kernel(Fp4Both t) {
    constexpr int BM = 128, BN = 128, RING = FP4_RING, WM = BM / 2, WN = BN / 2, MI = WM / 32, NJ = WN / 32;
    constexpr int LDA = BM / 64, LDB = BN / 64, LD = LDA + LDB, LDS = (BM + BN) / 256;       // a wave's loads of a stage: codes of x, of the matrix; of a span: scales
    constexpr int SPAN = FP4_SPAN / FP4_STAGE, SPANS = 3, B_AT = BM * 64, STAGE = B_AT + BN * 64, S_AT = RING * STAGE, S_BYTES = (BM + BN) * 16;
    static_assert((RING - 1) * LD < 63, "the loads in flight can be counted");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Fp4Args& a = t.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    int tile_m, tile_n;
    if (!fp4_tile_of(blockIdx.x, t.tiles_m, t.tiles_n, tile_m, tile_n)) return;
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const int row_bytes = a.blocks * 16;

    // the loads: per lane its bytes within the codes and the scales; beyond the matrices: out of range
    int va[LDA], vb[LDB], vs[LDS];
    const int idx = (lane & 7) ^ ((lane >> 4) & 3), piece = idx & 3;      // (a load is eight lines: line / 2 % 4 is lane / 16)
#pragma unroll
    for (int i = 0; i < LDA; ++i) {
        const int row = m0 + ((i * 4 + wave) * 8 + (lane >> 3)) * 2 + (idx >> 2);
        va[i] = row < a.M ? row * row_bytes + piece * 16 : FP4_OUT;
    }
#pragma unroll
    for (int i = 0; i < LDB; ++i) {
        const int row = fp4_matrix_row<TAIL>(n0, ((i * 4 + wave) * 8 + (lane >> 3)) * 2 + (idx >> 2), wide);
        vb[i] = row >= 0 ? row * row_bytes + piece * 16 : FP4_OUT;
    }
    uintx4_t rsrc_a = fp4_buffer(t.x, (unsigned)((long)a.M * row_bytes)), rsrc_b = fp4_buffer(a.codes, (unsigned)((long)a.N * row_bytes));
    // scales: loads of 64 rows, those of x first
    uintx4_t rsrc_s[LDS];
#pragma unroll
    for (int i = 0; i < LDS; ++i) {
        const int part = i * 4 + wave_s;
        const bool of_x = part < BM / 64;
        const int row = of_x ? (m0 + part * 64 + lane < a.M ? m0 + part * 64 + lane : -1)
                             : fp4_matrix_row<TAIL>(n0, (part - BM / 64) * 64 + lane, wide);
        const int scale_bytes = of_x ? t.x_scale_bytes : t.scale_bytes;
        vs[i] = row >= 0 ? row * scale_bytes : FP4_OUT;
        rsrc_s[i] = fp4_buffer(of_x ? t.xs : t.scales, (unsigned)((long)(of_x ? a.M : a.N) * scale_bytes));
    }
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem;
    const int first_stage = blockIdx.y * t.per_split, stages = min(t.nk - first_stage, t.per_split);
    int ask_k = first_stage;                               // the stage that is being asked for, and its place in the ring
    if constexpr (TAIL == TAIL_PARTIAL) t.a.out = (float*)t.a.out + (long)blockIdx.y * a.M * a.N;
    unsigned ask_at = lds0, ask_span = lds0 + S_AT;
    // (blocks of the last stage that lie beyond the row: a lane's offset is then made one that is out of range)
    const int off = piece < a.blocks - (t.nk - 1) * 4 ? 0 : FP4_OUT;
    int piece_not = ask_k + 1 == t.nk ? off : 0;
#define LOAD_PIECE(i_)                                                                                                    \
    {                                                                                                                     \
        if ((i_) < LDA) {                                                                                                 \
            constexpr int n_ = (i_) < LDA ? (i_) : 0;                                                                     \
            QE_LOAD_TO_SHARED(ask_at + (n_ * 4 + wave_s) * 1024, va[n_] | piece_not, rsrc_a, ask_k * 64, "0", "");        \
        } else {                                                                                                          \
            constexpr int n_ = (i_) < LDA ? 0 : (i_) < LD ? (i_) - LDA : 0;                                               \
            QE_LOAD_TO_SHARED(ask_at + B_AT + (n_ * 4 + wave_s) * 1024, vb[n_] | piece_not, rsrc_b, ask_k * 64, "0", ""); \
        }                                                                                                                 \
    }
    // the scales of a span of stages come with its first stage into a ring of their own
#define LOAD_SPAN()                                                                                                       \
    {                                                                                                                     \
        _Pragma("unroll") for (int i = 0; i < LDS; ++i)                                                                   \
            QE_LOAD_TO_SHARED(ask_span + (i * 4 + wave_s) * 1024, vs[i], rsrc_s[i], ask_k / SPAN * 16, "0", "");          \
        ask_span = ask_span + S_BYTES == lds0 + S_AT + SPANS * S_BYTES ? lds0 + S_AT : ask_span + S_BYTES;                \
    }
#define LOAD_CASE(i_) case i_: if constexpr ((i_) < LD) LOAD_PIECE(i_) break;
#define LOADS_OF(n_)                                                                                                      \
    switch (n_) {                                                                                                         \
        LOAD_CASE(0) LOAD_CASE(1) LOAD_CASE(2) LOAD_CASE(3) LOAD_CASE(4) LOAD_CASE(5) LOAD_CASE(6) LOAD_CASE(7)                           \
        default: break;                                                                                                   \
    }
    static_assert(LD <= 8, "a case for every load");
    // (beyond the last stage every load is out of range: the buffers have no bytes)
    int ask_left = stages;
#define ASKED()                                                                                                           \
    {                                                                                                                     \
        ask_at = ask_at + STAGE == lds0 + RING * STAGE ? lds0 : ask_at + STAGE;                                           \
        ++ask_k;                                                                                                          \
        if (--ask_left <= 0) {                                                                                            \
            rsrc_a[2] = 0; rsrc_b[2] = 0; ask_k = 0;                                                                      \
            _Pragma("unroll") for (int i = 0; i < LDS; ++i) rsrc_s[i][2] = 0;                                             \
        }                                                                                                                 \
        piece_not = off & (ask_k + 1 == t.nk ? -1 : 0);                                                                   \
    }
    // waits until at most younger_ loads of the wave are in flight and its reads of shared memory are done, then for the other waves
#define MEET(younger_) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(younger_) : "memory");

    int fa_at[2], fb_at[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int ra = wm + r, rb = wn + r;
        fa_at[q] = (ra >> 1) * 128 + ((((ra & 1) * 4 + 2 * h + q) ^ ((ra >> 2) & 3)) * 16);
        fb_at[q] = B_AT + (rb >> 1) * 128 + ((((rb & 1) * 4 + 2 * h + q) ^ ((rb >> 2) & 3)) * 16);
    }
    const int sa_at = S_AT + (wm + r) * 16 + 2 * h, sb_at = S_AT + (BM + wn + r) * 16 + 2 * h;
    int read_k = ask_k, read_span = 0;                        // the stage whose scales are read, and the place of its span
    floatx16_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    uintx4_t fa[2][MI], fb[2][NJ];
    uint32_t sa[2][MI], sb[2][NJ];                         // (by the stage's parity: a stage's last step multiplies while the next one's arrive)
    // fragment p_ of step q_ (those of x and of the matrix in turn as they are wanted), scale p_
#define READ_FRAG(q_, place_, p_)                                                                                         \
    {                                                                                                                     \
        if ((p_) < MI) fa[q_][(p_) < MI ? (p_) : 0] = *(const uintx4_t*)(smem + (place_) + fa_at[q_] + (p_) * 2048);      \
        else fb[q_][(p_) < MI ? 0 : (p_) - MI] = *(const uintx4_t*)(smem + (place_) + fb_at[q_] + ((p_) - MI) * 2048);    \
    }
#define READ_SCALE(par_, p_)                                                                                              \
    {                                                                                                                     \
        const int at_ = read_span + read_k % SPAN * 4;                                                                    \
        if ((p_) < MI) sa[par_][(p_) < MI ? (p_) : 0] = *(const uint16_t*)(smem + at_ + sa_at + (p_) * 512);              \
        else sb[par_][(p_) < MI ? 0 : (p_) - MI] = *(const uint16_t*)(smem + at_ + sb_at + ((p_) - MI) * 512);            \
    }
#define READ_ON()                                                                                                         \
    {                                                                                                                     \
        if (++read_k % SPAN == 0) read_span = read_span + S_BYTES == SPANS * S_BYTES ? 0 : read_span + S_BYTES;           \
    }
    constexpr int R = MI + NJ, PER = MI * NJ;
    // step q_ of a stage of parity par_: between its matrix instructions the fragments of the next step are read from place from_ (for step 0 of
    // the next stage with its scales); in step 1, behind the barrier, the loads of the stage that is being asked for go out
#define K_STEP(q_, par_, from_)                                                                                           \
    _Pragma("unroll") for (int sl = 0; sl < PER; ++sl) {                                                                  \
        _Pragma("unroll") for (int p = 0; p < R; ++p)                                                                     \
            if (p * PER / (2 * R) == sl) {                                                                                \
                READ_FRAG((q_) ^ 1, from_, p)                                                                             \
                if ((q_) == 1) READ_SCALE((par_) ^ 1, p)                                                                  \
            }                                                                                                             \
        const int i = sl / NJ, j = sl % NJ;                                                                               \
        const intx8_t xa = {(int)fa[q_][i][0], (int)fa[q_][i][1], (int)fa[q_][i][2], (int)fa[q_][i][3], 0, 0, 0, 0};      \
        const intx8_t wb = {(int)fb[q_][j][0], (int)fb[q_][j][1], (int)fb[q_][j][2], (int)fb[q_][j][3], 0, 0, 0, 0};      \
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xa, wb, acc[i][j], 4, 4, q_, sa[par_][i], q_, sb[par_][j]); \
        _Pragma("unroll") for (int l = 0; l < LD; ++l)                                                                    \
            if ((q_) == 1 && l * PER / LD == sl) { LOADS_OF(l) }                                                          \
        __builtin_amdgcn_sched_barrier(0);                                                                                \
    }
    // (the scales come before their stages' codes, and a stage is waited for by the loads behind it: with more of those than are counted,
    // where a span lies between, the wait is only longer)
#pragma unroll
    for (int s = 0; s < RING; ++s) {
        if (ask_left > 0 && ask_k % SPAN == 0) LOAD_SPAN()
#pragma unroll
        for (int i = 0; i < LD; ++i) { LOADS_OF(i) }
        if (s + 1 < RING) ASKED()
    }
    MEET((RING - 1) * LD)
#pragma unroll
    for (int p = 0; p < R; ++p) {
        READ_FRAG(0, 0, p)
        READ_SCALE(0, p)
    }
    // behind the barrier in the middle of a stage nothing of its place is read any more, and the next stage has arrived
#define STAGE_OF(par_)                                                                                                    \
    {                                                                                                                     \
        const int next = at + STAGE == RING * STAGE ? 0 : at + STAGE;                                                     \
        K_STEP(0, par_, at)                                                                                               \
        ASKED()                                                                                                           \
        MEET((RING - 2) * LD)                                                                                             \
        if (ask_left > 0 && ask_k % SPAN == 0) LOAD_SPAN()                                                                \
        READ_ON()                                                                                                         \
        K_STEP(1, par_, next)                                                                                             \
        at = next;                                                                                                        \
    }
    int at = 0, st = 0;
    for (; st + 1 < stages; st += 2) {
        STAGE_OF(0)
        STAGE_OF(1)
    }
    if (st < stages) STAGE_OF(0)
    MEET(0)                                                // (what was asked for beyond the end has arrived)
#undef STAGE_OF
#undef K_STEP
#undef READ_FRAG
#undef READ_SCALE
#undef LOADS_OF
#undef LOAD_CASE
#undef LOAD_PIECE
#undef LOAD_SPAN
#undef READ_ON
#undef ASKED
#undef MEET
    static_assert(4 * fp4_strip_bytes<NJ>() <= S_AT, "the waves' strips must fit the ring");
    fp4_store_tiles<TAIL, MI, NJ>(a, acc, m0 + wm, n0 + wn, smem + wave * fp4_strip_bytes<NJ>());
}

// The same in tiles of 256 x 256, a wave's part 128 x 128 with its sums in the 256 accumulation registers, and in stages of 256: whole lines of
// 128 bytes a row (a load's 64 bytes of a line cost what 128 do: from an XCD's L2 loads of whole lines bring 33 TB/s to the chip's
// shared memories, of half lines 17).  Two stages fit, so a stage is released by quarters: the halves of a wave's rows of x and of the matrix
// are four regions, each read once into registers and kept there; a quarter is a half of x with a half of the matrix (16 instructions), in
// an order in which a quarter's last operands are none of the next one's, so that each reads the region that is wanted in the next
// quarter or the one after it.  Behind the barrier at its end that region's memory takes the same rows two stages later: seven quarters
// for a load to arrive.  Even stages go x0 w0, x0 w1, x1 w1, x1 w0, odd ones x0 w1, x0 w0, x1 w0, x1 w1.  Lane (r, h) takes blocks 4 h .. 4 h + 3 of
// row r, one a k step: its four scales are a word.  (4096 rows against 4096 x 12288: 101 us, in stages of 128 by the kernel above in such tiles 114.)
template <int TAIL>
__global__ __launch_bounds__(256, 1) void fp4_both_large_kernel(Fp4Both t) {
    constexpr int SPANS = 3, S_AT = 2 * 65536, S_BYTES = 512 * 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Fp4Args& a = t.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    int tile_m, tile_n;
    if (!fp4_tile_of(blockIdx.x, t.tiles_m, t.tiles_n, tile_m, tile_n)) return;
    const int m0 = tile_m * 256, n0 = tile_n * 256;
    const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;
    const int wide = TAIL == TAIL_SILU ? a.N / 2 : a.N;
    const int row_bytes = a.blocks * 16, nk = t.nk;

    // Region g (0, 1: the halves of x; 2, 3: of the matrix) of a stage holds, for each of the two waves that read it, 64 rows: 128 rows of 128
    // bytes, the eight pieces of a row exchanged by its number.  A load is eight rows; a wave's i-th of a region: rows 32 i + 8 wave.
    const int piece = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));      // (row / 2 % 8 of row 8 wave + lane / 8)
    int va[2][4], vb[2][4], vs[2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (i / 2) * 128 + g * 64 + (i % 2) * 32 + wave * 8 + (lane >> 3);
            const int n = fp4_matrix_row<TAIL>(n0, row, wide);
            va[g][i] = m0 + row < a.M ? (m0 + row) * row_bytes + piece * 16 : FP4_OUT;
            vb[g][i] = n >= 0 ? n * row_bytes + piece * 16 : FP4_OUT;
        }
    // scales of a span of two stages: 256 rows of x with its even stage, 256 of the matrix with its odd one, 64 a wave
    vs[0] = m0 + wave * 64 + lane < a.M ? (m0 + wave * 64 + lane) * t.x_scale_bytes : FP4_OUT;
    vs[1] = fp4_matrix_row<TAIL>(n0, wave * 64 + lane, wide);
    vs[1] = vs[1] >= 0 ? vs[1] * t.scale_bytes : FP4_OUT;
    const uintx4_t rsrc_a = fp4_buffer(t.x, (unsigned)((long)a.M * row_bytes)), rsrc_b = fp4_buffer(a.codes, (unsigned)((long)a.N * row_bytes));
    const uintx4_t rsrc_x = fp4_buffer(t.xs, (unsigned)((long)a.M * t.x_scale_bytes)), rsrc_w = fp4_buffer(t.scales, (unsigned)((long)a.N * t.scale_bytes));
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem + wave_s * 1024;
    const int off = piece < a.blocks - (nk - 1) * 8 ? 0 : FP4_OUT;      // (blocks of the last stage that lie beyond the row: out of range)
#define REGION_AT(g_, par_) (((par_) * 4 + (g_)) * 16384)
#define LOAD_REGION(g_, st_, par_, i_)                                                                                    \
    {                                                                                                                     \
        const int not_ = (st_) < nk - 1 ? 0 : (st_) == nk - 1 ? off : FP4_OUT, s_ = (st_) < nk ? (st_) * 128 : 0;          \
        if ((g_) < 2) { QE_LOAD_TO_SHARED(lds0 + REGION_AT(g_, par_) + (i_) * 4096, va[(g_) & 1][i_] | not_, rsrc_a, s_, "0", ""); } \
        else { QE_LOAD_TO_SHARED(lds0 + REGION_AT(g_, par_) + (i_) * 4096, vb[(g_) & 1][i_] | not_, rsrc_b, s_, "0", ""); } \
    }
    // half_ 0: of x, 1: of the matrix; span_: its number, spans come in turn into a ring of three
#define LOAD_SPAN(half_, span_)                                                                                           \
    {                                                                                                                     \
        const bool there_ = (span_) * 2 < nk;                                                                             \
        const unsigned to_ = lds0 + S_AT + (span_) % SPANS * S_BYTES + (half_) * 4096;                                    \
        const int v_ = there_ ? vs[half_] : FP4_OUT, s_ = there_ ? (span_) * 16 : 0;                                      \
        if (half_) { QE_LOAD_TO_SHARED(to_, v_, rsrc_w, s_, "0", ""); } else { QE_LOAD_TO_SHARED(to_, v_, rsrc_x, s_, "0", ""); } \
    }
    // waits until at most younger_ loads of the wave are in flight and its reads of shared memory are done, then for the other waves
#define MEET(younger_) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(younger_) : "memory");

    floatx16_t acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    uintx4_t fa[2][2][4], fb[2][2][4];
    uint32_t sa[2][2], sb[2][2];
    const int f0 = r * 128 + (((h * 4) ^ ((r >> 1) & 7)) * 16);
    const unsigned char* const fa0 = smem + (wave >> 1) * 8192;
    const unsigned char* const fb0 = smem + (wave & 1) * 8192;
    const unsigned char* const sa0 = smem + S_AT + (wm + r) * 16 + h * 4;
    const unsigned char* const sb0 = smem + S_AT + 4096 + (wn + r) * 16 + h * 4;
    // piece p_ of region g_ of stage st_ (parity par_): fragment p_ / 2 of its tile p_ % 2, and at first the tile's word of scales
#define READ_REGION(g_, par_, st_, p_)                                                                                    \
    {                                                                                                                     \
        if ((g_) < 2) fa[(g_) & 1][(p_) & 1][(p_) >> 1] = *(const uintx4_t*)(fa0 + REGION_AT(g_, par_) + ((p_) & 1) * 4096 + (f0 ^ (((p_) >> 1) * 16))); \
        else fb[(g_) & 1][(p_) & 1][(p_) >> 1] = *(const uintx4_t*)(fb0 + REGION_AT(g_, par_) + ((p_) & 1) * 4096 + (f0 ^ (((p_) >> 1) * 16))); \
        if ((p_) < 2) {                                                                                                   \
            const int at_ = (st_) / 2 % SPANS * S_BYTES + (par_) * 8 + (g_) % 2 * 1024 + ((p_) & 1) * 512;                \
            if ((g_) < 2) sa[(g_) & 1][(p_) & 1] = *(const uint32_t*)(sa0 + at_);                                         \
            else sb[(g_) & 1][(p_) & 1] = *(const uint32_t*)(sb0 + at_);                                                  \
        }                                                                                                                 \
    }
#define MULTIPLY(ha_, hb_, i_, j_, ks_)                                                                                   \
    {                                                                                                                     \
        const uintx4_t &x_ = fa[ha_][i_][ks_], &w_ = fb[hb_][j_][ks_];                                                    \
        const intx8_t xa_ = {(int)x_[0], (int)x_[1], (int)x_[2], (int)x_[3], 0, 0, 0, 0};                                 \
        const intx8_t wb_ = {(int)w_[0], (int)w_[1], (int)w_[2], (int)w_[3], 0, 0, 0, 0};                                 \
        floatx16_t& c_ = acc[(ha_) * 2 + (i_)][(hb_) * 2 + (j_)];                                                         \
        c_ = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xa_, wb_, c_, 4, 4, ks_, sa[ha_][i_], ks_, sb[hb_][j_]);     \
    }
    // half ha_ of x with half hb_ of the matrix; meanwhile region rg_ of stage rst_ (parity rpar_) is read and region lg_ of stage lst_ (lpar_) asked for
#define QUAD(ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_)                                                                \
    {                                                                                                                     \
        QUAD_STEP(0, ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_) QUAD_STEP(1, ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_) \
        QUAD_STEP(2, ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_) QUAD_STEP(3, ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_) \
        MEET(24)                                                                                                          \
    }
    // (a k step is four of the quarter's 16 matrix instructions: beside each of the first eight a piece is read, beside every fourth a load goes out)
#define QUAD_STEP(ks_, ha_, hb_, rg_, rst_, rpar_, lg_, lst_, lpar_)                                                      \
    {                                                                                                                     \
        if constexpr ((ks_) < 2) READ_REGION(rg_, rpar_, rst_, (ks_) * 4)                                                           \
        MULTIPLY(ha_, hb_, 0, 0, ks_)                                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                                \
        if constexpr ((ks_) < 2) READ_REGION(rg_, rpar_, rst_, (ks_) * 4 + 1)                                                       \
        MULTIPLY(ha_, hb_, 0, 1, ks_)                                                                                     \
        LOAD_REGION(lg_, lst_, lpar_, ks_)                                                                                \
        __builtin_amdgcn_sched_barrier(0);                                                                                \
        if constexpr ((ks_) < 2) READ_REGION(rg_, rpar_, rst_, (ks_) * 4 + 2)                                                       \
        MULTIPLY(ha_, hb_, 1, 0, ks_)                                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                                \
        if constexpr ((ks_) < 2) READ_REGION(rg_, rpar_, rst_, (ks_) * 4 + 3)                                                       \
        MULTIPLY(ha_, hb_, 1, 1, ks_)                                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                                \
    }
    // (the scales of the span four stages on: they are older than the loads of that stage, which are waited for)
#define EVEN(st_)                                                                                                         \
    LOAD_SPAN(0, (st_) / 2 + 2)                                                                                           \
    QUAD(0, 0, 3, st_, 0, 2, (st_) + 2, 0)                                                                                \
    QUAD(0, 1, 1, st_, 0, 3, (st_) + 2, 0)                                                                                \
    QUAD(1, 1, 0, (st_) + 1, 1, 1, (st_) + 2, 0)                                                                          \
    QUAD(1, 0, 3, (st_) + 1, 1, 0, (st_) + 3, 1)
#define ODD(st_)                                                                                                          \
    LOAD_SPAN(1, (st_) / 2 + 2)                                                                                           \
    QUAD(0, 1, 2, st_, 1, 3, (st_) + 2, 1)                                                                                \
    QUAD(0, 0, 1, st_, 1, 2, (st_) + 2, 1)                                                                                \
    QUAD(1, 0, 0, (st_) + 1, 0, 1, (st_) + 2, 1)                                                                          \
    QUAD(1, 1, 2, (st_) + 1, 0, 0, (st_) + 3, 0)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        LOAD_SPAN(half, 0)
        LOAD_SPAN(half, 1)
    }
    constexpr int first[8] = {0, 2, 3, 1, 0 + 4, 3 + 4, 2 + 4, 1 + 4};      // regions in the order in which they are read (4: of the second stage)
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) LOAD_REGION(first[k] & 3, first[k] >> 2, first[k] >> 2, i)
    MEET(24)
#pragma unroll
    for (int p = 0; p < 8; ++p) READ_REGION(0, 0, 0, p)
#pragma unroll
    for (int p = 0; p < 8; ++p) READ_REGION(2, 0, 0, p)
    MEET(24)
#pragma unroll
    for (int i = 0; i < 4; ++i) LOAD_REGION(0, 2, 0, i)
    MEET(24)
    int st = 0;
    for (; st + 1 < nk; st += 2) {
        EVEN(st)
        ODD(st + 1)
    }
    if (st < nk) { EVEN(st) }
    MEET(0)                                                // (what was asked for beyond the end has arrived)
#undef EVEN
#undef ODD
#undef QUAD_STEP
#undef QUAD
#undef MULTIPLY
#undef READ_REGION
#undef MEET
#undef LOAD_SPAN
#undef LOAD_REGION
#undef REGION_AT
    static_assert(4 * fp4_strip_bytes<4>() <= S_AT, "the waves' strips must fit the stages");
    fp4_store_tiles<TAIL, 4, 4>(a, acc, m0 + wm, n0 + wn, smem + wave * fp4_strip_bytes<4>());
}

template <int TAIL>
static int fp4_both_large_launch(Fp4Both t, hipStream_t stream) {
    constexpr int SHARED = 2 * 65536 + 3 * 8192;
    t.nk = qe_cdiv(t.a.K, 256);
    t.tiles_m = qe_cdiv(t.a.M, 256);
    t.tiles_n = qe_cdiv(t.a.N, 256);
    const long blocks = ((long)t.tiles_m * t.tiles_n + 7) / 8 * 8;
    QE_REQUIRE(blocks <= 2147483647L, "gemm_mxfp4: too many tiles");
    QE_RAISE_SHARED(fp4_both_large_kernel<TAIL>, SHARED);
    fp4_both_large_kernel<TAIL><<<(unsigned)blocks, 256, SHARED, stream>>>(t);
    return 0;
}

template <int TAIL>
static int fp4_both_launch(Fp4Both t, int splits, hipStream_t stream) {
    constexpr int SHARED = 256 * (FP4_RING * 64 + 3 * 16);
    t.tiles_m = qe_cdiv(t.a.M, 128);
    t.tiles_n = qe_cdiv(t.a.N, 128);
    const long blocks = ((long)t.tiles_m * t.tiles_n + 7) / 8 * 8;
    QE_REQUIRE(blocks <= 2147483647L, "gemm_mxfp4: too many tiles");
    QE_RAISE_SHARED(fp4_both_kernel<TAIL>, SHARED);
    fp4_both_kernel<TAIL><<<dim3((unsigned)blocks, (unsigned)splits), 256, SHARED, stream>>>(t);
    return 0;
}

// The kernel's 32-bit places reach all of the operands.
bool fp4_both_take(int M, int N, int K) {
    return (long)N * qe_cdiv(K, 32) * 16 < (1L << 31) - 64 && (long)M * qe_cdiv(K, 32) * 16 < (1L << 31) - 64;
}

// 256 x 256 where its tiles keep half of the units busy, else 128 x 128 (both sides in 4 bits, quantisation included: 1024 rows against 4096 x 4096, 64
// tiles, 22 us by 128 x 128; 2048 rows, 128 tiles, 46 by 256 x 256).
static bool fp4_both_large(int M, int N) { return (long)qe_cdiv(M, 256) * qe_cdiv(N, 256) >= 128; }

// K in cuts where that leaves a block a unit at the most and a cut two spans, and what the stages left out take (half a microsecond each) is
// more than the cuts' products and their join do (130 rows against 4096 x 12288 in four cuts 22 us, uncut 36; 65 against 4096 x 4096 in four 14.9,
// 15.9; 512 against that in two 25.7, 19.4).
static int fp4_both_per_split(int M, int N, int K, int* splits) {
    const int spans = qe_cdiv(K, FP4_SPAN), stages = qe_cdiv(K, FP4_STAGE);
    long s = fp4_both_large(M, N) ? 1 : 256 / ((long)qe_cdiv(M, 128) * qe_cdiv(N, 128));
    if (s > spans / 2) s = spans / 2;
    if (s < 1 || 0.5 * stages * (double)(s - 1) / (double)s < 4.0 + 2e-6 * (double)s * M * N) s = 1;
    const int per = qe_cdiv(spans, (int)s);
    *splits = qe_cdiv(spans, per);
    return per * (FP4_SPAN / FP4_STAGE);
}

static long fp4_both_parts(int M, int N, int K) {
    int splits;
    fp4_both_per_split(M, N, K, &splits);
    return splits > 1 ? (4L * splits * M * N + 15) / 16 * 16 : 0;
}

static int fp4_both_stage(int M, int N) { return fp4_both_large(M, N) ? 2 * FP4_STAGE : FP4_STAGE; }

long fp4_both_workspace(int M, int N, int K, const void* xs, const void* scales) {
    const int stage = fp4_both_stage(M, N);
    return fp4_both_parts(M, N, K) + (K % 32 ? (long)M * qe_cdiv(K, 32) * 16 : 0) + (fp4_scales_whole(K, xs, stage) ? 0 : fp4_scales_bytes(M, K)) +
           (fp4_scales_whole(K, scales, stage) ? 0 : fp4_scales_bytes(N, K));
}

int fp4_both(const Fp4Args& a, int tail, void* workspace, hipStream_t stream) {
    Fp4Both t{};
    t.a = a;
    t.nk = qe_cdiv(a.K, FP4_STAGE);
    const int stage = fp4_both_stage(a.M, a.N);
    const bool x_whole = fp4_scales_whole(a.K, a.xs, stage), whole = fp4_scales_whole(a.K, a.scales, stage);
    t.x_scale_bytes = fp4_scales_row(a.K, x_whole);
    t.scale_bytes = fp4_scales_row(a.K, whole);
    float* parts = (float*)workspace;          // the workspace: the cuts' products, then what the loads do not take as it is
    unsigned char* ws = (unsigned char*)workspace + fp4_both_parts(a.M, a.N, a.K);
    int splits;
    t.per_split = fp4_both_per_split(a.M, a.N, a.K, &splits);
    t.x = (const unsigned char*)a.x;
    t.xs = a.xs;
    t.scales = a.scales;
    Fp4Prepare p{};
    p.blocks = a.blocks;
    p.num_words = fp4_scales_row(a.K, false) / 4;
    p.K = a.K;
    if (a.K % 32) {
        p.codes = (const uintx4_t*)a.x;
        p.codes_out = (uintx4_t*)ws;
        p.pieces = (unsigned)a.M * a.blocks;
        t.x = ws;
        ws += (long)p.pieces * 16;
    }
    if (!x_whole) {
        p.xs = a.xs;
        p.xs_out = (uint32_t*)ws;
        p.x_words = (unsigned)(fp4_scales_bytes(a.M, a.K) / 4);
        t.xs = ws;
        ws += (long)p.x_words * 4;
    }
    if (!whole) {
        p.scales = a.scales;
        p.scales_out = (uint32_t*)ws;
        p.words = (unsigned)(fp4_scales_bytes(a.N, a.K) / 4);
        t.scales = ws;
    }
    if (const long all = (long)p.pieces + p.x_words + p.words) fp4_prepare_kernel<<<qe_cdiv(all, 256), 256, 0, stream>>>(p);
    const bool large = fp4_both_large(a.M, a.N);
    if (splits > 1) t.a.out = parts;
    int rc;
#define QE_GO(T_) rc = large ? fp4_both_large_launch<T_>(t, stream) : fp4_both_launch<T_>(t, 1, stream)
    if (splits > 1) rc = fp4_both_launch<TAIL_PARTIAL>(t, splits, stream);
    else if (tail == TAIL_STORE) QE_GO(TAIL_STORE);
    else if (tail == TAIL_ADD) QE_GO(TAIL_ADD);
    else QE_GO(TAIL_SILU);
#undef QE_GO
    if (rc) return rc;
    if (splits > 1 && (rc = fp4_join(a, parts, splits, tail, stream))) return rc;
    QE_LAUNCH_CHECK();
    return 0;
}
