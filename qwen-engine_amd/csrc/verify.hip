// Verification of drafted tokens.  Request r owns the rows first[r] .. first[r + 1] - 1 of the logits: n + 1 of them for n drafts, row j the
// model's logits behind j drafts.  With p_j = softmax(logits / t) and q_j the distribution that draft x_j was drawn from (softmax of
// the draft's logits at the same t, or all on x_j where there are none), draft j is accepted if u_j q_j(x_j) < p_j(x_j).  At the first that
// is not, the token comes from max(p_j - q_j, 0) over its sum; behind n accepted ones from p_n: the first token whose running sum of
// weights, in the order of the vocabulary, exceeds the request's second random number times the whole.  The tokens so given are
// distributed as if drawn from p, whatever q is.  t <= 0 (or NaN): p is all on the largest logit, the lowest index on ties.
//
// Logits of -infinity and NaN weigh nothing; infinite ones share everything.  A row where nothing weighs gives no token (-1).
//
// All weights and sums are 64-bit: a vocabulary of 150 000 has so many borders of running sums that 32-bit ones put the random number on
// the other side of one in a few per cent of the draws.
//
// Four launches: spans of 4096 logits (all rows, bound by their bytes and exponentials: of 64 requests, 425 MB, 85 to 97 us), acceptance (a block a
// request, a wave a draft, 6 to 7.5 us), the sums of pieces of 1024 of what the token is drawn from (one row a request, and its draft's, 16 to
// 19 us), the draw (5 to 6 us); the last three in one where there are few spans.
#include "common.h"

#define VERIFY_SPAN 4096        // what a block looks at; its quarters, a wave each, have sums of their own
#define VERIFY_PIECE 1024

struct VerifyArgs {
    const float* logits;        // [rows, V]
    const float* guess;         // [drafts, V] or null
    const int* first;           // [R + 1]
    const int* drafts;          // [drafts]
    const float* temperature;   // [R]
    const float* accept;        // [drafts]
    const float* draw;          // [R]
    int* tokens;                // [rows]
    int* accepted;              // [R]
    int rows, V, R, spans, pieces;
    int four;                   // the rows lie at whole 16-byte pieces
};

struct VerifyPart {             // of a span of a row: the largest logit, the lowest column that has it, its pieces' sums of exp((z - top) / t)
    double sums[4];
    float top;
    int at;
};

__device__ __forceinline__ bool verify_greedy(float t) { return !(t > 0.f); }

// A difference of logits times k is a power of two's exponent; below `least` that is -1080, which stands for nothing.
struct VerifyScale {
    double k, least;
    VerifyScale() = default;
    __device__ __forceinline__ explicit VerifyScale(float t) {
        k = verify_greedy(t) ? 1.0 : __builtin_fmax(1.4426950408889634074 / (double)t, 1e-300);      // log2(e) / t (an infinite t: all alike, but nothing stays nothing)
        least = -1080.0 / k;
    }
};

struct VerifyChoice {           // of a request: what its token is drawn from, the weights of row `row` less those of row guess_row or those of a column
    VerifyScale t;
    double p_each, q_each;      // 1 / the rows' sums; q_each 0: there is no guess_row
    float p_top, q_top;
    int row, guess_row;         // row -1: nothing is drawn
    int point;                  // the column that a draft without logits was, -1: there is none
};

// a b + c with c in scalar registers: the compiler's choice, b's product added into a copy of c, costs two more instructions a term
__device__ __forceinline__ double verify_term(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// exp((z - top) / t) in 64-bit, top the row's largest logit and not infinite: 2^y = 2^n 2^f with n = y rounded (1.5 2^52 added and taken away:
// n stands in the sum's low bits), f in [-1/2, 1/2], and 2^f by a polynomial of degree 10 through the Chebyshev points of that
// interval (off by 3.2e-16 of it at the most).  What is NaN on the way (a NaN logit; -infinity less itself) becomes 0 at the maximum, as what
// is below 2^-1080 does.
__device__ __forceinline__ double verify_power(double f) {          // 2^f
    double v = verify_term(f, 0x1.e6063f9b91935p-28, 0x1.b675bd687d9b8p-24);
    v = verify_term(v, f, 0x1.62bfd477051e0p-20);
    v = verify_term(v, f, 0x1.ffcb540541227p-17);
    v = verify_term(v, f, 0x1.430913096fcb8p-13);
    v = verify_term(v, f, 0x1.5d87fe9d7ab80p-10);
    v = verify_term(v, f, 0x1.3b2ab6fba1de1p-7);
    v = verify_term(v, f, 0x1.c6b08d703ce45p-5);
    v = verify_term(v, f, 0x1.ebfbdff82c598p-3);
    v = verify_term(v, f, 0x1.62e42fefa3a19p-1);
    return __builtin_fma(v, f, 1.0);
}
__device__ __forceinline__ double verify_finite_weight(float z, float top, const VerifyScale& t) {
    const double d = __builtin_fmax((double)z - (double)top, t.least);
    const double y = __builtin_fma(d, t.k, 0x1.8p52), f = __builtin_fma(d, t.k, -(y - 0x1.8p52));
    return __builtin_amdgcn_ldexp(verify_power(f), (int)__builtin_bit_cast(unsigned long, y));
}

// The same for a sum over many logits of a row, with fewer operations (64 requests 120 us, so 115: what counts there is how many 64-bit operations a
// logit takes, next to its bytes).  The method is the exponential by a table of 32 and a short polynomial of P. T. P. Tang (Table-driven implementation
// of the exponential function in IEEE floating-point arithmetic, ACM Transactions on Mathematical Software 15, 1989), in powers of two: 2^(z k) = 2^m 2^(j / 32) 2^f, where 32 m + j is 32 z k rounded (1.5 2^47 added) and |f| <= 1/64, so
// that a polynomial of degree 5 does (off by 1.5e-16 at the most); 2^(j / 32) comes from a table in shared memory, in 32 pairs of banks of its
// own, the nearest 64-bit numbers with their high words less j 2^15: 32 m + j, shifted by 15 and added, makes 2^m 2^(j / 32) of them.  The row's own number of the
// kind, 2^(top k), counts for the sum as a whole: its rounded exponent is taken off with the constant that rounds 32 z k, the rest
// multiplied at the end.  What is far below the top (or no number) counts as 2^-1000 of it, which the logit's 32-bit maximum with `floor` sees
// to.  Not for a top that is infinite or beyond 2^25 / k, nor where 32 bits hold no number some 1000 / k below it.
__device__ const unsigned long verify_table[32] = {
    0x3ff0000000000000ul, 0x3fefd9b0d3158574ul, 0x3fefb5586cf9890ful, 0x3fef9301d0125b51ul, 0x3fef72b83c7d517bul, 0x3fef54873168b9aaul, 0x3fef387a6e756238ul, 0x3fef1e9df51fdee1ul,
    0x3fef06fe0a31b715ul, 0x3feef1a7373aa9cbul, 0x3feedea64c123422ul, 0x3feece086061892dul, 0x3feebfdad5362a27ul, 0x3feeb42b569d4f82ul, 0x3feeab07dd485429ul, 0x3feea47eb03a5585ul,
    0x3feea09e667f3bcdul, 0x3fee9f75e8ec5f74ul, 0x3feea11473eb0187ul, 0x3feea589994cce13ul, 0x3feeace5422aa0dbul, 0x3feeb737b0cdc5e5ul, 0x3feec49182a3f090ul, 0x3feed503b23e255dul,
    0x3feee89f995ad3adul, 0x3feeff76f2fb5e47ul, 0x3fef199bdd85529cul, 0x3fef3720dcef9069ul, 0x3fef5818dcfba487ul, 0x3fef7c97337b9b5ful, 0x3fefa4afa2a490daul, 0x3fefd0765b6e4540ul};

struct VerifySum {
    double k, round;            // round: 1.5 2^47 less the top's exponent
    float floor;
    bool fits;
    __device__ __forceinline__ VerifySum(double k_, float t, float top) {
        k = k_;
        const double at = (double)top * k;
        round = 0x1.8p47 - __builtin_rint(at);
        floor = top - 693.147181f * t;             // (1000 ln 2)
        const double far = ((double)floor - (double)top) * k;
        fits = __builtin_fabs(at) < 0x1p25 && far > -1015.0 && far < -950.0;
    }
    // sum and the weight of z; table: in shared memory
    __device__ __forceinline__ double add(double sum, float z, const unsigned long* table) const {
        typedef __attribute__((ext_vector_type(2))) uint32_t words;
        const double d = (double)fmaxf(z, floor), y = __builtin_fma(d, k, round), f = __builtin_fma(d, k, -(y - round));
        const uint32_t at = __builtin_bit_cast(words, y)[0];
        words scale = __builtin_bit_cast(words, table[at & 31]);
        scale[1] += at << 15;
        double v = verify_term(f, 0x1.5d884e708e6aap-10, 0x1.3b2b1bee88b09p-7);
        v = verify_term(v, f, 0x1.c6b08d70400d0p-5);
        v = verify_term(v, f, 0x1.ebfbdff8131c3p-3);
        v = verify_term(v, f, 0x1.62e42fefa39efp-1);
        return __builtin_fma(__builtin_fma(v, f, 1.0), __builtin_bit_cast(double, scale), sum);
    }
    __device__ __forceinline__ double rest(float top) const { return verify_power(-__builtin_fma((double)top, k, -(0x1.8p47 - round))); }
};

// The same for any row: infinite logits share everything.
__device__ __forceinline__ double verify_weight(float z, float top, const VerifyScale& t) {
    return top == INFINITY ? (z == top ? 1.0 : 0.0) : verify_finite_weight(z, top, t);
}

// The rows of request r, or false where first[] holds no rows and drafts that there are.
__device__ __forceinline__ bool verify_rows(const VerifyArgs& a, int r, int& lo, int& hi) {
    lo = a.first[r];
    hi = a.first[r + 1];
    return lo >= r && hi > lo && hi <= a.rows && hi - 1 - r <= a.rows - a.R;
}

// EACH numbers of a row: four neighbours from column c on, four 256 columns on, and so on (one: column c); as 16-byte pieces where `whole` says that
// all of them are there and at such places, else one by one; beyond the row -infinity.
template <int EACH> __device__ __forceinline__ int verify_column(int c, int e) { return c + e / 4 * 256 + e % 4; }
template <int EACH>
__device__ __forceinline__ void verify_load(const float* row, int c, int V, bool whole, float (&v)[EACH]) {
    if (EACH % 4 == 0 && whole) {
#pragma unroll
        for (int e = 0; e < EACH; e += 4) {
            const float4 q = *(const float4*)(row + verify_column<EACH>(c, e));
            v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int at = verify_column<EACH>(c, e);
            v[e] = row[min(at, V - 1)];
            if (at >= V) v[e] = -INFINITY;
        }
    }
}

// Lane i's sum of the lanes up to i, each with its own: within rows of 16 lanes by shifts of a row, then the last lane of rows 0 and 2 to
// rows 1 and 3, then lane 31 to rows 2 and 3.  These moves are operands of instructions, where a shuffle is a trip through the LDS
// unit (six of them, of 64 bits, one after the other: 0.4 us).
template <int CTRL, int ROWS> __device__ __forceinline__ double verify_moved(double v) {      // 0 where no lane sends
    const unsigned long b = __builtin_bit_cast(unsigned long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, ROWS, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (unsigned long)hi << 32 | lo);
}
#define ROW_SHR(n_) (0x110 + (n_))
#define ROW_BCAST15 0x142
#define ROW_BCAST31 0x143
__device__ __forceinline__ double verify_wave_scan(double v) {
    v += verify_moved<ROW_SHR(1), 0xf>(v);
    v += verify_moved<ROW_SHR(2), 0xf>(v);
    v += verify_moved<ROW_SHR(4), 0xf>(v);
    v += verify_moved<ROW_SHR(8), 0xf>(v);
    v += verify_moved<ROW_BCAST15, 0xa>(v);
    v += verify_moved<ROW_BCAST31, 0xc>(v);
    return v;
}

// Lane `lane` of v, the same number in every lane (lane the same in every lane, too).
__device__ __forceinline__ double verify_lane(double v, int lane) {
    const unsigned long b = __builtin_bit_cast(unsigned long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
    return __builtin_bit_cast(double, (unsigned long)hi << 32 | lo);
}

__device__ __forceinline__ double verify_wave_sum(double v) { return verify_lane(verify_wave_scan(v), 63); }

// The largest of the wave and the lowest column that has it, in every lane.
__device__ __forceinline__ void verify_wave_top(float& top, int& at) {
    const float mine = top;
    top = wave_max(top);
    at = mine == top ? at : 0x7fffffff;
#define LOWER(ctrl_, rows_) at = min(at, __builtin_amdgcn_update_dpp(at, at, ctrl_, rows_, 0xf, false));
    LOWER(ROW_SHR(1), 0xf) LOWER(ROW_SHR(2), 0xf) LOWER(ROW_SHR(4), 0xf) LOWER(ROW_SHR(8), 0xf) LOWER(ROW_BCAST15, 0xa) LOWER(ROW_BCAST31, 0xc)
#undef LOWER
    at = __builtin_amdgcn_readlane(at, 63);
}

// One block a span of a row: blockIdx.y counts the rows of the logits, then those of the drafts' logits.  done[R]: whether first[] fails to rise
// somewhere, which misleads the search for a row's request; verify_accept sees to that.
__global__ __launch_bounds__(256) void verify_spans_kernel(VerifyArgs a, VerifyPart* parts, unsigned* done) {
    __shared__ float tops[4];
    __shared__ int ats[4];
    __shared__ unsigned long table[32];
    const bool is_guess = (int)blockIdx.y >= a.rows;
    const int i = is_guess ? blockIdx.y - a.rows : blockIdx.y;
    constexpr int EACH = VERIFY_PIECE / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.x * VERIFY_SPAN + wave * VERIFY_PIECE;
    float v[EACH];
    verify_load<EACH>((is_guess ? a.guess : a.logits) + (long)i * a.V, c0 + lane * 4, a.V, a.four && c0 + VERIFY_PIECE <= a.V, v);      // (on its way while the request is looked up)
    // (after the loads of what the host gives: behind a store they would not be scalar ones, 10 us for 64 requests)
    auto clear = [&] {
        if (blockIdx.x == 0 && blockIdx.y == 0) {
            for (int r = threadIdx.x; r < a.R; r += 256) done[r] = 0;
            if (wave == 0) {
                bool falls = false;
                for (int r = lane; r < a.R; r += 64) falls |= a.first[r + 1] <= a.first[r];
                const unsigned any = __ballot(falls) != 0;
                if (lane == 0) done[a.R] = any;
            }
        }
    };
    // the request: the number of first[1 .. R] (less their index, for the drafts) that are not beyond i
    int low = 0, high = a.R;
    while (low < high) {
        const int mid = (low + high) / 2;
        if ((int)((unsigned)a.first[mid + 1] - (is_guess ? mid + 1 : 0)) <= i) low = mid + 1; else high = mid;
    }
    if (low >= a.R) return clear();
    const float t = a.temperature[low];
    const bool greedy = verify_greedy(t);
    if (is_guess && greedy) return;
    const VerifyScale k(t);
    float top = -INFINITY;
    int at = 0x7fffffff;
    if (greedy) {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (v[e] > top) { top = v[e]; at = verify_column<EACH>(c0 + lane * 4, e); }      // (no NaN is larger than anything)
        verify_wave_top(top, at);
    } else {                                       // (its column is not asked for)
#pragma unroll
        for (int e = 0; e < EACH; ++e) top = fmaxf(top, v[e]);
        top = wave_max(top);
    }
    if (threadIdx.x < 32) table[threadIdx.x] = verify_table[threadIdx.x];
    if (lane == 0) { tops[wave] = top; ats[wave] = at; }
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) { top = tops[w]; at = ats[w]; }
    double sum = 0.0;
    if (!greedy) {
        const VerifySum all(k.k, t, top);
        if (all.fits) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) sum = all.add(sum, v[e], table);
            sum = verify_wave_sum(sum) * all.rest(top);
            if (sum < 0x1p-900) sum = 0.0;         // (nothing there but what counts as 2^-1000)
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) sum += verify_weight(v[e], top, k);
            sum = verify_wave_sum(sum);
        }
    }
    VerifyPart& part = parts[(long)blockIdx.y * a.spans + blockIdx.x];
    if (lane == 0) part.sums[wave] = sum;
    if (threadIdx.x == 0) { part.top = top; part.at = at; }
    clear();
}

__device__ __forceinline__ double verify_span_sum(const VerifyPart& p) { return (p.sums[0] + p.sums[1]) + (p.sums[2] + p.sums[3]); }

// The lane's span of a row's first 64.
__device__ __forceinline__ VerifyPart verify_mine(const VerifyPart* parts, int spans) {
    const int lane = threadIdx.x & 63;
    VerifyPart mine = {{0.0, 0.0, 0.0, 0.0}, -INFINITY, 0x7fffffff};
    if (lane < spans) mine = parts[lane];
    return mine;
}

// The whole row's largest logit, its column and sum, from its spans: by one wave, the same in all lanes.
__device__ __forceinline__ void verify_join(const VerifyPart* parts, const VerifyPart& mine, int spans, const VerifyScale& k, float& top, int& at, double& sum) {
    const int lane = threadIdx.x & 63;
    top = mine.top;
    at = mine.at;
    for (int s = lane + 64; s < spans; s += 64)
        if (parts[s].top > top) { top = parts[s].top; at = parts[s].at; }
    verify_wave_top(top, at);
    sum = verify_span_sum(mine) * verify_weight(mine.top, top, k);
    for (int s = lane + 64; s < spans; s += 64) sum += verify_span_sum(parts[s]) * verify_weight(parts[s].top, top, k);
    sum = verify_wave_sum(sum);
}

// The parts of request r's rows once more, where first[] falls: those that are there may be another temperature's, or none at all.  By a block of 16
// waves, a wave a span.  (In the launch that accepts in every block, a request's blocks all write the same.)
__device__ __forceinline__ void verify_redo(const VerifyArgs& a, VerifyPart* parts, int r, int lo, int n) {
    const int lane = threadIdx.x & 63;
    const float t = a.temperature[r];
    const bool greedy = verify_greedy(t);
    const VerifyScale k(t);
    const int rows = n + 1 + (a.guess && !greedy ? n : 0);
    for (int i = threadIdx.x >> 6; i < rows * a.spans; i += 16) {
        const int row = i / a.spans, c0 = i % a.spans * VERIFY_SPAN;
        const bool is_guess = row > n;
        const int at_row = is_guess ? lo - r + row - (n + 1) : lo + row;
        const float* z = (is_guess ? a.guess : a.logits) + (long)at_row * a.V;
        VerifyPart part = {{0.0, 0.0, 0.0, 0.0}, -INFINITY, 0x7fffffff};
        for (int c = c0 + lane; c < min(c0 + VERIFY_SPAN, a.V); c += 64)
            if (z[c] > part.top) { part.top = z[c]; part.at = c; }
        verify_wave_top(part.top, part.at);
        for (int q = 0; q < 4 && !greedy; ++q) {
            double sum = 0.0;
            const int from = c0 + q * VERIFY_PIECE;
            for (int c = from + lane; c < min(from + VERIFY_PIECE, a.V); c += 64) sum += verify_weight(z[c], part.top, k);
            part.sums[q] = verify_wave_sum(sum);
        }
        if (lane == 0) parts[(long)((is_guess ? a.rows : 0) + at_row) * a.spans + i % a.spans] = part;
    }
    __syncthreads();
}

// Which drafts of request r are accepted, and what its token is drawn from: by a block of 16 waves, a wave a draft, 16 at a time.  accepted: how
// many (-1: there are no such rows, or they or its drafts are not behind those of all requests before); token: the one behind them, of a request
// without temperature.  falls: whether first[] does so somewhere.
__device__ __forceinline__ VerifyChoice verify_accept(const VerifyArgs& a, VerifyPart* parts, unsigned falls, int r, int& accepted, int& token) {
    __shared__ VerifyChoice tries[16];
    __shared__ int tokens[16], stops[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo, hi;
    bool there = verify_rows(a, r, lo, hi);
    const float t = a.temperature[r];
    if (falls) {                                   // (first[k] - k: where request k's drafts begin; where none is beyond lo - r no first[k] is beyond lo)
        bool behind = true;
        for (int k = threadIdx.x; k < r; k += 1024) behind &= (long)a.first[k] - k <= (long)lo - r;
        there = __syncthreads_and(behind) && there;
        if (there) verify_redo(a, parts, r, lo, hi - lo - 1);
    }
    if (!there) {
        VerifyChoice none{};
        none.row = accepted = token = -1;
        return none;
    }
    const bool greedy = verify_greedy(t);
    const VerifyScale k(t);
    const int n = hi - lo - 1;
    int j0 = 0, stop = -1;
    for (;; j0 += 16) {
        const int j = j0 + wave;
        if (j <= n) {
            const bool guessed = !greedy && j < n && a.guess;
            const int d = lo - r + j, x = j < n ? a.drafts[d] : -1;
            const VerifyPart *parts_p = parts + (long)(lo + j) * a.spans, *parts_q = parts + (long)(a.rows + d) * a.spans;
            const VerifyPart mine_p = verify_mine(parts_p, a.spans), mine_q = verify_mine(parts_q, guessed ? a.spans : 0);
            const bool inside = x >= 0 && x < a.V;
            const float zp = inside ? a.logits[(long)(lo + j) * a.V + x] : -INFINITY;
            const float zq = inside && a.guess ? a.guess[(long)d * a.V + x] : -INFINITY;
            const float u = j < n ? a.accept[d] : 0.f;
            VerifyChoice c{};
            int at, unused;
            double p_sum, q_sum = 0.0;
            verify_join(parts_p, mine_p, a.spans, k, c.p_top, at, p_sum);
            if (guessed) verify_join(parts_q, mine_q, a.spans, k, c.q_top, unused, q_sum);
            const int largest = c.p_top > -INFINITY ? at : -1;
            c.t = k;
            c.row = greedy || !(p_sum > 0.0) ? -1 : lo + j;      // (no draw: the token is there, or there is none)
            c.p_each = p_sum > 0.0 ? 1.0 / p_sum : 0.0;
            c.q_each = q_sum > 0.0 ? 1.0 / q_sum : 0.0;
            c.guess_row = d;
            c.point = j < n && !a.guess ? x : -1;
            bool take = false;
            if (j < n && greedy) take = largest >= 0 && x == largest;
            else if (j < n) {
                const double p = verify_weight(zp, c.p_top, k) * c.p_each, q = a.guess ? verify_weight(zq, c.q_top, k) * c.q_each : 1.0;
                take = p > 0.0 && (double)u * q < p;
            }
            if (lane == 0) { tries[wave] = c; tokens[wave] = largest; stops[wave] = !take; }
        } else if (lane == 0) {
            stops[wave] = 0;
        }
        __syncthreads();
        for (int w = 15; w >= 0; --w)
            if (stops[w]) stop = w;
        if (stop >= 0) break;                      // (row n is no draft: it stops)
        __syncthreads();
    }
    accepted = j0 + stop;
    token = tokens[stop];
    return tries[stop];
}

// Writes it down: of a request whose rows are there its tokens, -1 behind them; the drawn one is left to the draw.
__device__ __forceinline__ void verify_write(const VerifyArgs& a, VerifyChoice* choices, int r, const VerifyChoice& c, int accepted, int token) {
    if (threadIdx.x == 0) {
        a.accepted[r] = accepted;
        choices[r] = c;
    }
    if (accepted < 0) return;
    const int lo = a.first[r], n = a.first[r + 1] - lo - 1;
    const bool greedy = verify_greedy(a.temperature[r]);
    for (int i = threadIdx.x; i <= n; i += 1024)
        if (lo + i != c.row) a.tokens[lo + i] = i < accepted ? a.drafts[lo - r + i] : greedy && i == accepted ? token : -1;
}

__global__ __launch_bounds__(1024) void verify_accept_kernel(VerifyArgs a, VerifyPart* parts, VerifyChoice* choices, const unsigned* done) {
    int accepted, token;
    const VerifyChoice c = verify_accept(a, parts, done[a.R], blockIdx.x, accepted, token);
    verify_write(a, choices, blockIdx.x, c, accepted, token);
}

// The weights in a draw of EACH numbers from column c on, of their logits in the model's row and in the draft's (rest: with the draft's
// distribution taken away).  The forms are told apart once, not at every number, so that the polynomials go side by side.
template <int EACH>
__device__ __forceinline__ void verify_draw_weights(const VerifyChoice& c, const float (&z)[EACH], const float (&zq)[EACH], int col, bool rest, double (&w)[EACH]) {
#pragma clang fp contract(off)                 // (both products are rounded: where p and q are alike nothing is left, not the difference of a product and its rounding)
    const bool with_q = rest && c.q_each > 0.0;
    if (c.p_top == INFINITY || (with_q && c.q_top == INFINITY)) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            w[e] = verify_weight(z[e], c.p_top, c.t) * c.p_each;
            if (with_q) w[e] = __builtin_fmax(w[e] - verify_weight(zq[e], c.q_top, c.t) * c.q_each, 0.0);
        }
    } else if (with_q) {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            w[e] = __builtin_fmax(verify_finite_weight(z[e], c.p_top, c.t) * c.p_each - verify_finite_weight(zq[e], c.q_top, c.t) * c.q_each, 0.0);
    } else {
#pragma unroll
        for (int e = 0; e < EACH; ++e) w[e] = verify_finite_weight(z[e], c.p_top, c.t) * c.p_each;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        if (rest && verify_column<EACH>(col, e) == c.point) w[e] = 0.0;
}

// A piece's weights without the draft's: summed already.
__device__ __forceinline__ double verify_plain_sum(const VerifyArgs& a, const VerifyPart* parts, const VerifyChoice& c, int piece) {
    const VerifyPart& p = parts[(long)c.row * a.spans + piece / 4];
    return p.sums[piece % 4] * verify_weight(p.top, c.p_top, c.t) * c.p_each;
}

// The draw, by the first four waves of a block.  Its piece is the first whose sum reaches beyond the random number's share of the whole (every
// wave finds it for itself, 64 pieces at a time, the first 256 side by side), then its token the first of the piece, four numbers a
// thread (with 16 waves four of a SIMD would do the search one after the other).  Where a rounding lets a piece's own sum fall short of
// the share, or the number is 1 or more, the token is the last one that weighs anything.
// The sums of the pieces go past the caches that a part of the units has for itself: other units read them in the same launch.
__device__ __forceinline__ void verify_put(double* rests, int piece, double v) {
    __hip_atomic_store((unsigned long*)rests + piece, __builtin_bit_cast(unsigned long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double verify_get(const double* rests, int piece) {
    return __builtin_bit_cast(double, __hip_atomic_load((const unsigned long*)rests + piece, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

struct VerifyFirst {                // the lane's sums of the first 256 pieces
    double v[4];
};
__device__ __forceinline__ VerifyFirst verify_first(const double* rests, int pieces) {
    VerifyFirst f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = i * 64 + (threadIdx.x & 63);
        f.v[i] = s < pieces ? verify_get(rests, s) : 0.0;
    }
    return f;
}

__device__ __forceinline__ void verify_draw(const VerifyArgs& a, const VerifyPart* parts, const VerifyChoice& c, const double* rests, VerifyFirst first, float u) {
    constexpr int EACH = VERIFY_PIECE / 256;
    __shared__ double shared[4];
    __shared__ int founds[4], lasts[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int piece = -1;
    double target = 0.0, run = 0.0, scan = 0.0, sum = 0.0, each[EACH];
    if (wave < 4) {
        double total = 0.0, scans[4];
        auto scan_all = [&](auto&& piece_sum) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                scans[i] = verify_wave_scan(first.v[i]);
                total += verify_lane(scans[i], 63);
            }
            for (int s0 = 256; s0 < a.pieces; s0 += 64) total += verify_wave_sum(piece_sum(s0 + lane));
        };
        auto rest_sum = [&](int s) { return s < a.pieces ? verify_get(rests, s) : 0.0; };
        auto plain_sum = [&](int s) { return s < a.pieces ? verify_plain_sum(a, parts, c, s) : 0.0; };
        scan_all(rest_sum);
        // (nothing left: the draft's distribution is the model's, and only a rounding or a number beyond 1 refused the draft: p alone)
        const bool rest = total > 0.0;
        if (!rest) {
            total = 0.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) first.v[i] = plain_sum(i * 64 + lane);
            scan_all(plain_sum);
        }
        target = u > 0.f ? (double)u * total : 0.0;            // (NaN: 0)
        bool reached = false;
        double before = 0.0;
        auto look = [&](double v, double scan_v, int s0) {
            const unsigned long some = __ballot(v > 0.0), over = __ballot(v > 0.0 && run + scan_v > target);
            if (some) {
                const int at = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
                piece = s0 + at;
                before = run + verify_lane(scan_v, at) - verify_lane(v, at);
            }
            run += verify_lane(scan_v, 63);
            reached = over != 0;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!reached) look(first.v[i], scans[i], i * 64);
        for (int s0 = 256; !reached && s0 < a.pieces; s0 += 64) {
            const double v = rest ? rest_sum(s0 + lane) : plain_sum(s0 + lane);
            look(v, verify_wave_scan(v), s0);
        }
        run = before;
        if (piece >= 0) {
            const int c0 = piece * VERIFY_PIECE, col = c0 + tid * EACH;
            const bool whole = a.four && c0 + VERIFY_PIECE <= a.V;
            float v[EACH], q[EACH];
            verify_load<EACH>(a.logits + (long)c.row * a.V, col, a.V, whole, v);
#pragma unroll
            for (int e = 0; e < EACH; ++e) q[e] = 0.f;
            if (rest && c.q_each > 0.0) verify_load<EACH>(a.guess + (long)c.guess_row * a.V, col, a.V, whole, q);
            verify_draw_weights<EACH>(c, v, q, col, rest, each);
#pragma unroll
            for (int e = 0; e < EACH; ++e) sum += each[e];
            scan = verify_wave_scan(sum);
            if (lane == 63) shared[wave] = scan;
        }
    }
    __syncthreads();
    if (wave < 4) {
        int found = -1, last = -1;
        if (piece >= 0) {
            const int col = piece * VERIFY_PIECE + tid * EACH;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (w < wave) run += shared[w];
            run += scan - sum;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                run += each[e];
                if (each[e] > 0.0) {
                    last = col + e;
                    if (found < 0 && run > target) found = col + e;
                }
            }
        }
        // the wave's first that reaches beyond, and its last that weighs anything, then the block's (columns rise with the threads)
        const unsigned long over = __ballot(found >= 0), some = __ballot(last >= 0);
        if (over) found = __builtin_amdgcn_readlane(found, __ffsll((unsigned long long)over) - 1);
        if (some) last = __builtin_amdgcn_readlane(last, 63 - __clzll((long long)some));
        if (lane == 0) { founds[wave] = over ? found : -1; lasts[wave] = some ? last : -1; }
    }
    __syncthreads();
    if (tid != 0) return;
    int token = -1;                            // (no weight anywhere: none)
    for (int w = 0; w < 4; ++w) {
        if (founds[w] >= 0) { token = founds[w]; break; }
        if (lasts[w] >= 0) token = lasts[w];
    }
    a.tokens[c.row] = token;
}

__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a, const VerifyPart* parts, const VerifyChoice* choices, const double* rests_all) {
    const int r = blockIdx.x;
    const double* rests = rests_all + (long)r * a.pieces;
    const VerifyFirst first = verify_first(rests, a.pieces);        // (nothing of them is used where nothing is drawn)
    const VerifyChoice c = choices[r];
    const float u = a.draw[r];
    // (all of the choice at once, with the sums, not part by part as it is wanted)
    asm volatile("" : : "s"(c.row), "s"(c.guess_row), "s"(c.point), "s"(c.p_top), "s"(c.q_top), "s"(c.p_each), "s"(c.q_each), "s"(c.t.k), "s"(c.t.least), "s"(u), "v"(first.v[0]));
    if (c.row >= 0) verify_draw(a, parts, c, rests, first, u);
}

// The sums of the weights of pieces, four numbers a thread, 256 threads a piece.  ACCEPT: the block finds the choice for itself, with its 16
// waves, and has a whole span; the request's last block to be done (`done` counts them; it waits for nothing) draws.  Else one piece.
template <bool ACCEPT>
__global__ __launch_bounds__(ACCEPT ? 1024 : 256) void verify_rest_kernel(VerifyArgs a, VerifyPart* parts, VerifyChoice* choices, double* rests, unsigned* done) {
    constexpr int EACH = VERIFY_PIECE / 256, HERE = ACCEPT ? 4 : 1;
    __shared__ double shared[4 * HERE];
    __shared__ bool is_last;
    const int r = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), piece = blockIdx.x * HERE + wave / 4;
    VerifyChoice c;
    int accepted = -1, token = -1;
    if constexpr (ACCEPT) c = verify_accept(a, parts, done[a.R], r, accepted, token);
    else c = choices[r];
    if (c.row < 0) {
        if (ACCEPT && blockIdx.x == 0) verify_write(a, choices, r, c, accepted, token);
        return;
    }
    const bool plain = c.q_each == 0.0 && (c.point < 0 || c.point / VERIFY_PIECE != piece);
    if (!plain && piece < a.pieces) {
        const int c0 = piece * VERIFY_PIECE, col = c0 + threadIdx.x % 256 * EACH;
        const bool whole = a.four && c0 + VERIFY_PIECE <= a.V;
        float v[EACH], q[EACH];
        verify_load<EACH>(a.logits + (long)c.row * a.V, col, a.V, whole, v);
#pragma unroll
        for (int e = 0; e < EACH; ++e) q[e] = 0.f;
        if (c.q_each > 0.0) verify_load<EACH>(a.guess + (long)c.guess_row * a.V, col, a.V, whole, q);
        double each[EACH], sum = 0.0;
        verify_draw_weights<EACH>(c, v, q, col, true, each);
#pragma unroll
        for (int e = 0; e < EACH; ++e) sum += each[e];
        sum = verify_wave_sum(sum);
        if (threadIdx.x % 64 == 0) shared[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x % 256 == 0 && piece < a.pieces)
        verify_put(rests + (long)r * a.pieces, piece, plain ? verify_plain_sum(a, parts, c, piece) : (shared[wave] + shared[wave + 1]) + (shared[wave + 2] + shared[wave + 3]));
    if constexpr (ACCEPT) {
        // The block's sums have arrived before it is counted, and the others' are read after all blocks have been: the stores and loads go past
        // the caches themselves, so that no fence has to write those back (with fences 25 us instead of 13.6).
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        if (threadIdx.x == 0) is_last = __hip_atomic_fetch_add(done + r, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        if (blockIdx.x == 0) verify_write(a, choices, r, c, accepted, token);
        __syncthreads();
        if (!is_last) return;
        verify_draw(a, parts, c, rests + (long)r * a.pieces, verify_first(rests + (long)r * a.pieces, a.pieces), a.draw[r]);
    }
}

extern "C" long qe_verify_drafts_workspace_bytes(int rows, int V, int R, int has_guess) {
    const long spans = qe_cdiv(V, VERIFY_SPAN), all = rows + (has_guess ? rows - R : 0);
    return all * spans * (long)sizeof(VerifyPart) + (long)R * (long)sizeof(VerifyChoice) + (long)R * (qe_cdiv(V, VERIFY_PIECE) * 8L + 4) + 4;
}

// logits float32 [rows, V], first int32 [R + 1], drafts int32 [rows - R], guess float32 [rows - R, V] or null, temperature and draw float32 [R],
// accept float32 [rows - R] -> tokens int32 [rows] (accepted drafts, the token drawn, -1), accepted int32 [R] (-1: first[] names no
// rows that there are, or none behind those of all requests before; nothing of the request is written then).
extern "C" int qe_verify_drafts(const float* logits, const int* first, const int* drafts, const float* guess, const float* temperature,
                                const float* accept, const float* draw, int* tokens, int* accepted, int rows, int V, int R,
                                void* workspace, long workspace_bytes, hipStream_t stream) {
    QE_REQUIRE(R >= 0 && V > 0 && V < (1 << 30) && rows >= R, "verify_drafts: bad sizes rows=%d V=%d R=%d", rows, V, R);
    if (R == 0) return 0;
    const int spans = qe_cdiv(V, VERIFY_SPAN), pieces = qe_cdiv(V, VERIFY_PIECE), all = rows + (guess ? rows - R : 0);
    QE_REQUIRE(all <= 65535, "verify_drafts: %d rows of logits are too many", all);
    QE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= qe_verify_drafts_workspace_bytes(rows, V, R, guess != nullptr),
               "verify_drafts: workspace too small");
    VerifyPart* parts = (VerifyPart*)workspace;
    VerifyChoice* choices = (VerifyChoice*)(parts + (long)all * spans);
    double* rests = (double*)(choices + R);
    unsigned* done = (unsigned*)(rests + (long)R * pieces);      // how many blocks of a request are done, then whether first[] falls
    const int four = V % 4 == 0 && (((uintptr_t)logits | (uintptr_t)guess) & 15) == 0;
    const VerifyArgs a{logits, guess, first, drafts, temperature, accept, draw, tokens, accepted, rows, V, R, spans, pieces, four};
    verify_spans_kernel<<<dim3(spans, all), 256, 0, stream>>>(a, parts, done);
    // Few spans: every block accepts for itself and the last one draws, in one launch instead of three (1 request of 151936, 38 spans, 13.6 us, and
    // 14.4; 8 requests, 304 spans, 25.4 and 25.9; 16 40.1 and 34.1; a program's call for 1 request 18.5 and 21.4).
    if ((long)spans * R <= 320) {
        verify_rest_kernel<true><<<dim3(spans, R), 1024, 0, stream>>>(a, parts, choices, rests, done);
    } else {
        verify_accept_kernel<<<R, 1024, 0, stream>>>(a, parts, choices, done);
        verify_rest_kernel<false><<<dim3(pieces, R), 256, 0, stream>>>(a, parts, choices, rests, done);
        verify_draw_kernel<<<R, 256, 0, stream>>>(a, parts, choices, rests);
    }
    QE_LAUNCH_CHECK();
    return 0;
}
