// Products of up to 16 rows with a 4-bit matrix (see mxfp4.h), for rows of whole blocks: bound by the matrix's bytes on their way from memory.
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

template <int X, int RX, int NT>
__global__ __launch_bounds__(512) void fp4_few_kernel(Fp4Args a, int tail, int scale_bytes) {
    constexpr int LX = X == X_BF16 ? RX / 2 : (RX + 7) / 8, LOADS = LX + 2 * NT;        // a chunk's loads: x, codes
    constexpr int SLOT = LOADS * 1024;
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
    const int x_row = X == X_BF16 ? lane >> 5 : lane >> 3;
    int vx[LX], px[LX], vc[2];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int row = (X == X_BF16 ? i * 2 : i * 8) + x_row;
        px[i] = X == X_BF16 ? (lane & 31) ^ (row & 7) : (lane & 7) ^ (row & 7);
        vx[i] = row < RX && row < a.M ? row * (X == X_BF16 ? a.K * 2 : row_bytes) + px[i] * 16 : FP4_OUT;
    }
    const int pc = (lane & 7) ^ (lane >> 3);               // (a load is eight rows)
#pragma unroll
    for (int i = 0; i < 2; ++i) vc[i] = (i * 8 + (lane >> 3)) * row_bytes + pc * 16;
    uintx4_t rsrc_x = fp4_buffer(a.x, (unsigned)((long)a.M * (X == X_BF16 ? a.K * 2 : row_bytes))), rsrc_w[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) rsrc_w[p] = fp4_buffer(a.codes + ((long)(silu && p ? wide : 0) + n0) * row_bytes, (unsigned)(cols * row_bytes));
    const int left = a.blocks - (chunks - 1) * 8;          // blocks of the last chunk
    const unsigned char* const slot = smem + scale_bytes + wave * SLOT;
    const unsigned slot_to = lds0 + scale_bytes + wave * SLOT;
#define ASK(c_)                                                                                                      \
    {                                                                                                                \
        const int ends_ = (c_) == chunks - 1 ? -1 : 0;                                                               \
        _Pragma("unroll") for (int i = 0; i < LX; ++i) {                                                             \
            const int not_ = ((X == X_BF16 ? px[i] >> 2 : px[i]) < left ? 0 : FP4_OUT) & ends_;                      \
            QE_LOAD_TO_SHARED(slot_to + i * 1024, vx[i] | not_, rsrc_x, (c_) * (X == X_BF16 ? 512 : 128), "4", "");  \
        }                                                                                                            \
        const int not_ = (pc < left ? 0 : FP4_OUT) & ends_;                                                          \
        _Pragma("unroll") for (int t = 0; t < NT; ++t)                                                               \
            _Pragma("unroll") for (int i = 0; i < 2; ++i) {                                                          \
                const int in_ = silu ? t % (NT > 1 ? NT / 2 : 1) : t;        /* the tile within its half */          \
                const int v_ = (vc[i] + in_ * 16 * row_bytes) | not_;                                                \
                if (silu && t >= NT / 2) { QE_LOAD_TO_SHARED(slot_to + (LX + t * 2 + i) * 1024, v_, rsrc_w[1], (c_) * 128, "4", ""); } \
                else QE_LOAD_TO_SHARED(slot_to + (LX + t * 2 + i) * 1024, v_, rsrc_w[0], (c_) * 128, "4", "");       \
            }                                                                                                        \
    }
    floatx4_t acc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = {0.f, 0.f, 0.f, 0.f};
    if (wave < chunks) ASK(wave)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");           // (the scales are there for all waves, too)

    const int xr = r & (RX - 1);                           // (a row of the tile that x does not have: another one's, and not stored)
    for (int c = wave; c < chunks; c += waves) {
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        const unsigned char* at = slot;
        uintx4_t xv[2][X == X_BF16 ? 4 : 1], cv[NT][2];
        int ws[NT][2], xs[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int b = s * 4 + g, block = min(c * 8 + b, a.blocks - 1);      // (beyond the last block codes and x are zero)
            if constexpr (X == X_BF16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) xv[s][j] = *(const uintx4_t*)(at + xr * 512 + (((b * 4 + j) ^ (xr & 7)) * 16));
            } else {
                xv[s][0] = *(const uintx4_t*)(at + xr * 128 + ((b ^ (xr & 7)) * 16));
                xs[s] = smem[min(xr, a.M - 1) * a.blocks + block];
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                cv[t][s] = *(const uintx4_t*)(at + (LX + t * 2) * 1024 + r * 128 + ((b ^ (r & 7)) * 16));
                const int in = silu ? t % (NT > 1 ? NT / 2 : 1) : t;
                const int row = min(in * 16 + r, cols - 1);
                ws[t][s] = smem[x_part + (silu && t >= NT / 2 ? part_bytes : 0) + row * a.blocks + block];
            }
        }
        // (the slot is read: the next chunk may come)
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        if (c + waves < chunks) ASK(c + waves)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (X == X_BF16) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, xv[s][j]),
                                                                            fp4_to_bf16(cv[t][s][j], __uint_as_float((uint32_t)ws[t][s] << 23)), acc[t][s], 0, 0, 0);
                } else {
                    const intx8_t xa = {(int)xv[s][0][0], (int)xv[s][0][1], (int)xv[s][0][2], (int)xv[s][0][3], 0, 0, 0, 0};
                    const intx8_t wb = {(int)cv[t][s][0], (int)cv[t][s][1], (int)cv[t][s][2], (int)cv[t][s][3], 0, 0, 0, 0};
                    acc[t][s] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t][s], 4, 4, 0, xs[s], 0, ws[t][s]);
                }
            }
    }
#undef ASK
    float* sums = (float*)(smem + scale_bytes);            // of wave w from byte w SLOT on: [NT][16][16]
    constexpr int APART = SLOT / 4;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave * APART + (t * 16 + g * 4 + e) * 16 + r] = acc[t][0][e] + acc[t][1][e];
    __syncthreads();
    for (int at = threadIdx.x; at < tiles * 256; at += blockDim.x) {
        const int t = at >> 8, m = at >> 4 & 15, n = n0 + t * 16 + (at & 15);
        if (m >= a.M || n >= wide) continue;
        float v = 0.f, up = 0.f;
        for (int w = 0; w < waves; ++w) {
            v += sums[w * APART + at];
            if (silu) up += sums[w * APART + at + tiles * 256];
        }
        if (tail == TAIL_STORE) fp4_store<TAIL_STORE>(a, m, n, v, up);
        else if (tail == TAIL_ADD) fp4_store<TAIL_ADD>(a, m, n, v, up);
        else fp4_store<TAIL_SILU>(a, m, n, v, up);
    }
}

template <int X, int RX, int NT>
static int fp4_few_launch(const Fp4Args& a, int tail, int waves, hipStream_t stream) {
    constexpr int LX = X == X_BF16 ? RX / 2 : (RX + 7) / 8, SLOT = (LX + 2 * NT) * 1024;
    const int scale_bytes = ((X == X_FP4 ? (a.M * a.blocks + 15) / 16 * 16 : 0) + NT * 16 * a.blocks + 15) / 16 * 16;
    const int wide = tail == TAIL_SILU ? a.N / 2 : a.N, cols = tail == TAIL_SILU ? NT * 8 : NT * 16;
    QE_RAISE_SHARED((fp4_few_kernel<X, RX, NT>), 160 * 1024);
    fp4_few_kernel<X, RX, NT><<<qe_cdiv(wide, cols), 64 * waves, scale_bytes + waves * SLOT, stream>>>(a, tail, scale_bytes);
    return 0;
}

// Tiles of columns and waves of a block; waves 0: not taken (the scales leave no room in shared memory).
struct Fp4Few {
    int nt, waves;
};

static Fp4Few fp4_few_shape(int M, int N, int K, int x_kind, int tail) {
    const int blocks = K / 32, chunks = qe_cdiv(blocks, 8), rx = M <= 2 ? 2 : M <= 8 ? 8 : 16;
    Fp4Few f{};
    // Two tiles where four blocks a unit are left then: every block reads all of x (16 rows against 24576 x 4096 13.2 us, with one tile 14.7; against
    // 4096 x 4096, 128 blocks with two, 6.7 and 5.6; with four tiles 14.9 and more).
    f.nt = tail == TAIL_SILU || N >= 1024 * 16 ? 2 : 1;
    // Waves: up to a chunk each, eight with one tile, four with two, which leaves room for other blocks (1 row against 6144 x 4096 with eight 5.8 us,
    // twelve 6.1; 8 rows against gate and up of 24576 x 4096 with four 12.2, eight 12.9; against 151936 x 1024, four chunks, with
    // two 18.0, four 20.8).
    const int room = 160 * 1024 - ((x_kind == X_FP4 ? M * blocks : 0) + f.nt * 16 * blocks + 32);
    const int fit = room / (((x_kind == X_BF16 ? rx / 2 : (rx + 7) / 8) + 2 * f.nt) * 1024);
    f.waves = f.nt == 1 ? (chunks < 8 ? chunks : 8) : chunks < 8 ? qe_cdiv(chunks, 2) : 4;
    if (f.waves > fit) f.waves = fit;
    return f;
}

bool fp4_few_takes(const void* x, int M, int N, int K, int x_kind, int tail) {
    return M <= 16 && x_kind != X_F32 && K % 32 == 0 && K < (1 << 20) && ((uintptr_t)x & 15) == 0 && fp4_few_shape(M, N, K, x_kind, tail).waves > 0;
}

int fp4_few(const Fp4Args& a, int x_kind, int tail, hipStream_t stream) {
    const Fp4Few f = fp4_few_shape(a.M, a.N, a.K, x_kind, tail);
#define QE_NT(X_, RX_) (f.nt == 1 ? fp4_few_launch<X_, RX_, 1>(a, tail, f.waves, stream) : fp4_few_launch<X_, RX_, 2>(a, tail, f.waves, stream))
#define QE_RX(X_) (a.M <= 2 ? QE_NT(X_, 2) : a.M <= 8 ? QE_NT(X_, 8) : QE_NT(X_, 16))
    return x_kind == X_BF16 ? QE_RX(X_BF16) : QE_RX(X_FP4);
#undef QE_RX
#undef QE_NT
}
