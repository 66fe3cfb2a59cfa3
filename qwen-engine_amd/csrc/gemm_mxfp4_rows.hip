// Products of few rows (up to 32, of 32 bits 8 or 16, in 4 bits 64) with a 4-bit matrix (see mxfp4.h): bound by the matrix's bytes on their way from memory.
// Rows of bfloat16 lie at whole words.  Up to four rows of 32-bit numbers are cut into three planes of bfloat16 where they are multiplied;
// of more the planes come from memory.  Either way the codes are read and converted once for the three.
//
// A block takes NT tiles of 16 columns, its waves chunks of 256 of K in turn, each wave by itself: it asks for a chunk of the codes (128
// bytes of a row, a line) and of x straight to its own piece of shared memory, and multiplies it when it has come.  The scales of
// the block's columns lie side by side and come as they are, once.  The sums of the waves are added in the order of the waves.
//
// What is on its way at a time is the blocks' and waves' of a unit: a second chunk a wave, asked for ahead, takes the shared memory of another
// block and is slower (16 rows against 24576 x 4096 with one chunk a wave 13.2 us, with two 14.2; 8 against gate and up of that size 12.2,
// 12.9; 16 against 4096 x 4096 5.6, 6.0; only 4-bit rows against 4096 x 12288 are a little quicker with two, 7.7 us instead of 7.9).
//
// Loads to registers would do without shared memory, but a matrix instruction's lane wants 16 bytes of a row, neighbouring lanes of
// other rows, and a load of 64 places of 64 lines takes four times the cycles of one of eight lines.
#include "mxfp4.h"

enum { X_PLANES = 3 };             // 32-bit rows as planes

// A wave's piece of shared memory: a chunk's loads of x (LX, 1 KB each: two rows of bfloat16, a row of 32-bit numbers, eight in 4 bits), of codes (2
// a tile), and the planes that are made of 32-bit rows.
template <int X, int RX, int NT> struct Fp4Slot {
    static constexpr int LX = X == X_BF16 ? RX / 2 : X == X_PLANES ? 3 * RX / 2 : X == X_F32 ? RX : (RX + 7) / 8;
    static constexpr int PLANES_AT = (LX + 2 * NT) * 1024, BYTES = PLANES_AT + (X == X_F32 ? 3 * RX * 512 : 0);
};

template <int X, int RX, int NT>
__global__ __launch_bounds__(512) void fp4_few_kernel(Fp4Args a, Fp4Rows x, int tail, int scale_bytes) {
    constexpr int MT = (RX + 15) / 16, LX = Fp4Slot<X, RX, NT>::LX, SLOT = Fp4Slot<X, RX, NT>::BYTES;        // (MT: tiles of 16 rows)
    constexpr int CHUNK = X == X_FP4 ? 128 : X == X_F32 ? 1024 : 512, NP = X == X_F32 || X == X_PLANES ? 3 : 1;      // bytes of a row of x in a chunk; planes that are multiplied
    static_assert(NP == 1 || RX <= 16, "the planes of a tile");
    static_assert(NT * MT * 1024 <= SLOT, "a wave's sums go where its slot was");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];                // scales (x's, the matrix's), then a slot a wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, r = lane & 15, g = lane >> 4;
    const bool silu = tail == TAIL_SILU;
    const int wide = silu ? a.N / 2 : a.N, halves = silu ? 2 : 1, tiles = NT / halves;  // tiles of columns that are stored
    const int n0 = blockIdx.x * tiles * 16, cols = min(tiles * 16, wide - n0);
    const int row_bytes = a.blocks * 16, chunks = (a.blocks + 7) / 8;
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem;

    // The scales: of x (in 4 bits), of the columns (silu: of the gates, of the ups).  Where a part is whole pieces of 16 bytes it is copied by
    // loads that write to shared memory directly, else byte by byte.
    const int part_bytes = tiles * 16 * a.blocks, x_part = X == X_FP4 ? (a.M * a.blocks + 15) / 16 * 16 : 0;
#pragma unroll
    for (int p = X == X_FP4 ? 0 : 1; p < 3; ++p) {
        if (p == 2 && !silu) break;
        const unsigned char* from = p == 0 ? a.xs : a.scales + ((long)(p == 2 ? wide : 0) + n0) * a.blocks;
        const int bytes = (p == 0 ? a.M : cols) * a.blocks, to = p == 0 ? 0 : x_part + (p - 1) * part_bytes;
        if (((unsigned long)from | (unsigned)bytes) % 16 == 0) {
            const uintx4_t rsrc = fp4_buffer(from, (unsigned)bytes);
            for (int at = wave * 1024; at < bytes; at += waves * 1024)
                if (at + lane * 16 < bytes) QE_LOAD_TO_SHARED(lds0 + to + at, lane * 16, rsrc, at, "4", "");      // (other lanes write nothing)
        } else {
            for (int at = threadIdx.x; at < bytes; at += blockDim.x) smem[to + at] = from[at];
        }
    }

    // the loads of a chunk: per lane the bytes within the rows of x and of a tile's columns
    const int x_row = X == X_FP4 ? lane >> 3 : X == X_F32 ? 0 : lane >> 5, plane_bytes = a.M * x.row_bytes;
    int vx[LX], px[LX], vc[2];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int row = (X == X_BF16 ? i * 2 : X == X_PLANES ? i % (RX / 2) * 2 : X == X_F32 ? i : i * 8) + x_row, plane = X == X_PLANES ? i / (RX / 2) : 0;
        px[i] = X == X_FP4 ? (lane & 7) ^ (row & 7) : X == X_F32 ? lane : (lane & 31) ^ (row & 7);
        vx[i] = row < RX && row < a.M ? plane * plane_bytes + row * x.row_bytes + px[i] * 16 : FP4_OUT;
    }
    const int pc = (lane & 7) ^ (lane >> 3);               // (a load is eight rows)
#pragma unroll
    for (int i = 0; i < 2; ++i) vc[i] = (i * 8 + (lane >> 3)) * row_bytes + pc * 16;
    const uintx4_t rsrc_x = fp4_buffer(x.data, (unsigned)(plane_bytes * x.planes));
    uintx4_t rsrc_w[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) rsrc_w[p] = fp4_buffer(a.codes + ((long)(silu && p ? wide : 0) + n0) * row_bytes, (unsigned)(cols * row_bytes));
    const int left = a.blocks - (chunks - 1) * 8, x_left = x.row_bytes - (chunks - 1) * CHUNK;      // blocks of the last chunk, bytes of its x
    unsigned char* const slot = smem + scale_bytes + wave * SLOT;
    const unsigned slot_to = lds0 + scale_bytes + wave * SLOT;
#define ASK(c_)                                                                                                      \
    {                                                                                                                \
        const int ends_ = (c_) == chunks - 1 ? -1 : 0;                                                               \
        _Pragma("unroll") for (int i = 0; i < LX; ++i) {                                                             \
            const int not_ = (px[i] * 16 < x_left ? 0 : FP4_OUT) & ends_;                                            \
            QE_LOAD_TO_SHARED(slot_to + i * 1024, vx[i] | not_, rsrc_x, (c_) * CHUNK, "4", "");                      \
        }                                                                                                            \
        const int not_ = (pc < left ? 0 : FP4_OUT) & ends_;                                                          \
        _Pragma("unroll") for (int t = 0; t < NT; ++t)                                                               \
            _Pragma("unroll") for (int i = 0; i < 2; ++i) {                                                          \
                const int in_ = silu ? t % (NT > 1 ? NT / 2 : 1) : t;        /* the tile within its half */          \
                const int v_ = (vc[i] + in_ * 16 * row_bytes) | not_;                                                \
                if (silu && t >= NT / 2) { QE_LOAD_TO_SHARED(slot_to + (LX + t * 2 + i) * 1024, v_, rsrc_w[1], (c_) * 128, "4", ""); } \
                else QE_LOAD_TO_SHARED(slot_to + (LX + t * 2 + i) * 1024, v_, rsrc_w[0], (c_) * 128, "4", "");     \
            }                                                                                                        \
    }
    floatx4_t acc[NT][MT], small[NT];                      // (small: of the low and middle planes, added at the end)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        small[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = {0.f, 0.f, 0.f, 0.f};
    }
    if (wave < chunks) ASK(wave)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");           // (the scales are there for all waves, too)

    for (int c = wave; c < chunks; c += waves) {
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        uintx4_t xv[NP][2][MT][X == X_FP4 ? 1 : 4], cv[NT][2];
        int ws[NT][2], xs[2][MT];
        unsigned char* const planes = slot + Fp4Slot<X, RX, NT>::PLANES_AT;
        if constexpr (X == X_F32) {
            // four numbers a lane of every row, none from K on, as three planes of rows as bfloat16 ones would lie
            const int left_k = a.K - (c * 256 + lane * 4);
            uintx4_t v[RX];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < RX; ++i) v[i] = *(const uintx4_t*)(slot + i * 1024 + lane * 16);
            if (c == chunks - 1) {
#pragma unroll
                for (int i = 0; i < RX; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e >= left_k) v[i][e] = 0;
            }
#pragma unroll
            for (int i = 0; i < RX; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, v[i][e] & 0x7fffffffu);
            const bool all_finite = __ballot(most >= 0x7f800000u) == 0;
#pragma unroll
            for (int i = 0; i < RX; ++i) {
                uint32_t h[3][4];                          // (the upper halves count)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[2][e] = v[i][e];
                    const float r = __uint_as_float(v[i][e]) - __uint_as_float(v[i][e] & 0xffff0000u);
                    h[1][e] = __float_as_uint(r);
                    h[0][e] = __float_as_uint(r - __uint_as_float(h[1][e] & 0xffff0000u));
                }
                if (!all_finite) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint16_t hi, mid, lo;
                        cut_in_three(__uint_as_float(v[i][e]), hi, mid, lo);
                        h[2][e] = (uint32_t)hi << 16;
                        h[1][e] = (uint32_t)mid << 16;
                        h[0][e] = (uint32_t)lo << 16;
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    typedef __attribute__((ext_vector_type(2))) uint32_t words;
                    const words two = {__builtin_amdgcn_perm(h[p][1], h[p][0], 0x07060302u), __builtin_amdgcn_perm(h[p][3], h[p][2], 0x07060302u)};
                    *(words*)(planes + p * RX * 512 + i * 512 + (((lane >> 1) ^ (i & 7)) * 16) + (lane & 1) * 8) = two;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int b = s * 4 + g, block = min(c * 8 + b, a.blocks - 1);      // (beyond the last block codes and x are zero)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int xr = (i * 16 + r) & (RX - 1);    // (a row of the tile that x does not have: another one's, and not stored)
                if constexpr (X == X_FP4) {
                    xv[0][s][i][0] = *(const uintx4_t*)(slot + xr * 128 + ((b ^ (xr & 7)) * 16));
                    xs[s][i] = smem[min(xr, a.M - 1) * a.blocks + block];
                    if (a.K % 32 && c == chunks - 1 && a.K - block * 32 < 32) xv[0][s][i][0] = first_codes(xv[0][s][i][0], a.K - block * 32);
                } else {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            xv[p][s][i][j] = *(const uintx4_t*)((X == X_F32 ? planes : slot) + p * RX * 512 + xr * 512 + (((b * 4 + j) ^ (xr & 7)) * 16));
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                cv[t][s] = *(const uintx4_t*)(slot + (LX + t * 2) * 1024 + r * 128 + ((b ^ (r & 7)) * 16));
                const int in = silu ? t % (NT > 1 ? NT / 2 : 1) : t;
                const int row = min(in * 16 + r, cols - 1);
                ws[t][s] = smem[x_part + (silu && t >= NT / 2 ? part_bytes : 0) + row * a.blocks + block];
            }
        }
        if (X == X_BF16 && a.K % 8 && c == chunks - 1) {       // (the row's last piece goes on in the next row)
            int words_left = (a.K - c * 256 + 1) / 2 - g * 16;     // (kept from the compiler: else all comparisons go in front of the loop and their results to spilled registers)
            asm volatile("" : "+v"(words_left));
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < (X == X_FP4 ? 1 : 4); ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            if (s * 64 + j * 4 + e >= words_left) xv[0][s][i][j][e] = 0;
        }
        // (the slot is read: the next chunk may come)
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        if (c + waves < chunks) ASK(c + waves)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (X != X_FP4) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bf16x8_t w = fp4_to_bf16(cv[t][s][j], __uint_as_float((uint32_t)ws[t][s] << 23));
#pragma unroll
                        for (int p = 0; p < NP - 1; ++p)
                            small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, xv[p][s][0][j]), w, small[t], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, xv[NP - 1][s][i][j]), w, acc[t][i], 0, 0, 0);
                    }
                } else {
                    const intx8_t wb = {(int)cv[t][s][0], (int)cv[t][s][1], (int)cv[t][s][2], (int)cv[t][s][3], 0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uintx4_t& q = xv[0][s][i][0];
                        const intx8_t xa = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
                        acc[t][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t][i], 4, 4, 0, xs[s][i], 0, ws[t][s]);
                    }
                }
            }
    }
#undef ASK
    if constexpr (NP == 3) {
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] += small[t];
    }
    float* sums = (float*)(smem + scale_bytes);            // of wave w from byte w SLOT on: [NT][MT * 16][16]
    constexpr int APART = SLOT / 4, TILE = MT * 256;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave * APART + t * TILE + (i * 16 + g * 4 + e) * 16 + r] = acc[t][i][e];
    __syncthreads();
    for (int at = threadIdx.x; at < tiles * TILE; at += blockDim.x) {
        const int t = at / TILE, m = at % TILE >> 4, n = n0 + t * 16 + (at & 15);
        if (m >= a.M || n >= wide) continue;
        float v = 0.f, up = 0.f;
        for (int w = 0; w < waves; ++w) {
            v += sums[w * APART + at];
            if (silu) up += sums[w * APART + at + tiles * TILE];
        }
        if (tail == TAIL_STORE) fp4_store<TAIL_STORE>(a, m, n, v, up);
        else if (tail == TAIL_ADD) fp4_store<TAIL_ADD>(a, m, n, v, up);
        else fp4_store<TAIL_SILU>(a, m, n, v, up);
    }
}

template <int X, int RX, int NT>
static int fp4_few_launch(const Fp4Args& a, const Fp4Rows& x, int tail, int waves, hipStream_t stream) {
    constexpr int SLOT = Fp4Slot<X, RX, NT>::BYTES;
    const int scale_bytes = ((X == X_FP4 ? (a.M * a.blocks + 15) / 16 * 16 : 0) + NT * 16 * a.blocks + 15) / 16 * 16;
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N, cols = tail == TAIL_SILU ? NT * 8 : NT * 16;
    QE_RAISE_SHARED((fp4_few_kernel<X, RX, NT>), 160 * 1024);
    fp4_few_kernel<X, RX, NT><<<qe_cdiv(wide, cols), 64 * waves, scale_bytes + waves * SLOT, stream>>>(a, x, tail, scale_bytes);
    return 0;
}

// Rows of 32-bit numbers that a block cuts into planes by itself, a chunk at a time, with the codes read and converted once for the three (1 row
// against 24576 x 4096 15.4 us, 3 20.5, by a launch of their own 27.7; against 4096 x 4096 6.0, 7.1 and 10.3).  Of more rows every block has too
// much to cut (8 33.5 and 26.6, 9.7 and 10.7).
#define FP4_CUT 4

// Tiles of columns and waves of a block; waves 0: not taken (the scales leave no room in shared memory).
struct Fp4Few {
    int nt, waves;
};

static Fp4Few fp4_few_shape(int M, int N, int K, int x_kind, int tail) {
    const bool cut = x_kind == X_F32 && M <= FP4_CUT;
    const int blocks = qe_cdiv(K, 32), chunks = qe_cdiv(blocks, 8);
    const int rx = M <= 2 ? 2 : cut && M <= 4 ? 4 : M <= 8 ? 8 : M <= 16 ? 16 : M <= 32 ? 32 : 64;
    Fp4Few f{};
    // Two tiles where four blocks a unit are left then: every block reads all of x (16 rows against 24576 x 4096 13.2 us, with one tile 14.7; against
    // 4096 x 4096, 128 blocks with two, 6.7 and 5.6; with four tiles 14.9 and more).
    f.nt = tail == TAIL_SILU || N >= 1024 * 16 ? 2 : 1;
    // Waves: up to a chunk each, eight where there are no more blocks than units or with one tile; with two tiles four, or two of more than 16
    // rows, which leaves room for other blocks (1 row against 6144 x 4096 with eight 5.8 us, twelve 6.1; 8 rows against gate and up
    // of 24576 x 4096 with four 12.2, eight 12.9; against 151936 x 1024, four chunks, with two 18.0, four 20.8; 17 rows against 24576 x 4096 with
    // two 16.6, three 21.4; 32 against 4096 x 4096 with eight 8.2, four 9.2).
    const int grid = qe_cdiv(tail == TAIL_SILU ? N / 2 : N, tail == TAIL_SILU ? 16 : f.nt * 16);
    const int room = 160 * 1024 - ((x_kind == X_FP4 ? M * blocks : 0) + f.nt * 16 * blocks + 32);
    const int fit = room / ((x_kind == X_FP4 ? (rx + 7) / 8 * 1024 : cut ? rx * 2560 : x_kind == X_F32 ? rx * 1536 : rx * 512) + 2 * f.nt * 1024);
    f.waves = f.nt == 1 || grid <= 256 ? (chunks < 8 ? chunks : 8) : chunks < 8 || rx > 16 ? 2 : 4;
    if (f.waves > fit) f.waves = fit;
    return f;
}

// Rows that the loads take as they are: of bfloat16, at whole words (5 rows of 2566 numbers against 5120 4.9 us; of 2567, through
// a copy, 7.4).
static bool as_it_is(const void* x, int K, int x_kind) { return x_kind == X_FP4 || (x_kind == X_BF16 && K % 2 == 0 && ((uintptr_t)x & 3) == 0); }

// (Of 32 bits 8 rows, or 16 against narrow matrices: 8 against 24576 x 4096 23.7 us, by tiles 27.6, against 4096 x 4096 10.1 and 14.6; 16 34.2, 28.6 and
// 12.6, 15.8, against 151936 x 1024 59 and 44; 24, when K was walked three times, 41.5, 28.8 and 17.3, 16.3.)
bool fp4_few_takes(int M, int N, int K, int x_kind, int tail) {
    return M <= (x_kind == X_FP4 ? 64 : x_kind == X_BF16 ? 32 : N < 16384 ? 16 : 8) && K < (1 << 20) && fp4_few_shape(M, N, K, x_kind, tail).waves > 0;
}

long fp4_few_workspace(const void* x, int M, int K, int x_kind) {
    return as_it_is(x, K, x_kind) || (x_kind == X_F32 && M <= FP4_CUT) ? 0 : fp4_planes_bytes(M, K, x_kind);
}

int fp4_few(const Fp4Args& a, int x_kind, int tail, void* workspace, hipStream_t stream) {
    const Fp4Few f = fp4_few_shape(a.M, a.N, a.K, x_kind, tail);
    const bool cut = x_kind == X_F32 && a.M <= FP4_CUT;
    Fp4Rows x{a.x, x_kind == X_FP4 ? a.blocks * 16 : cut ? a.K * 4 : a.K * 2, 1};
    if (!cut && !as_it_is(a.x, a.K, x_kind)) x = fp4_copies(a.x, a.M, a.K, x_kind, workspace, nullptr, 0, nullptr, stream);
#define QE_NT(X_, RX_) (f.nt == 1 ? fp4_few_launch<X_, RX_, 1>(a, x, tail, f.waves, stream) : fp4_few_launch<X_, RX_, 2>(a, x, tail, f.waves, stream))
#define QE_RX(X_) (a.M <= 2 ? QE_NT(X_, 2) : a.M <= 8 ? QE_NT(X_, 8) : a.M <= 16 ? QE_NT(X_, 16) : QE_NT(X_, 32))
    if (cut) return a.M <= 2 ? QE_NT(X_F32, 2) : QE_NT(X_F32, 4);
    if (x_kind == X_F32) return a.M <= 8 ? QE_NT(X_PLANES, 8) : QE_NT(X_PLANES, 16);
    if (x_kind == X_BF16) return QE_RX(X_BF16);
    return a.M > 32 ? QE_NT(X_FP4, 64) : QE_RX(X_FP4);
#undef QE_RX
#undef QE_NT
}
