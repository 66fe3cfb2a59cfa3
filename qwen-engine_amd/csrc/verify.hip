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
// Up to four launches: spans of 4096 logits (all rows, bound by their bytes and exponentials), acceptance (a block a request, a wave a
// draft), the spans' sums of what the token is drawn from (one row a request, and its draft's), the draw.
#include "common.h"

#define VERIFY_SPAN 4096

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
    int rows, V, R, spans;
    int four;                   // the rows lie at whole 16-byte pieces
};

struct VerifyPart {             // of a span of a row: the largest logit, the lowest column that has it, the sum of exp((z - top) / t)
    double sum;
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
__device__ __forceinline__ double verify_finite_weight(float z, float top, const VerifyScale& t) {
    const double d = __builtin_fmax((double)z - (double)top, t.least);
    const double y = __builtin_fma(d, t.k, 0x1.8p52), f = __builtin_fma(d, t.k, -(y - 0x1.8p52));
    double v = verify_term(f, 0x1.e6063f9b91935p-28, 0x1.b675bd687d9b8p-24);
    v = verify_term(v, f, 0x1.62bfd477051e0p-20);
    v = verify_term(v, f, 0x1.ffcb540541227p-17);
    v = verify_term(v, f, 0x1.430913096fcb8p-13);
    v = verify_term(v, f, 0x1.5d87fe9d7ab80p-10);
    v = verify_term(v, f, 0x1.3b2ab6fba1de1p-7);
    v = verify_term(v, f, 0x1.c6b08d703ce45p-5);
    v = verify_term(v, f, 0x1.ebfbdff82c598p-3);
    v = verify_term(v, f, 0x1.62e42fefa3a19p-1);
    v = __builtin_fma(v, f, 1.0);
    return __builtin_amdgcn_ldexp(v, (int)__builtin_bit_cast(unsigned long, y));
}

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

// The column of number e of a thread's share of a span, THREADS threads to a block: four neighbours, four a round further on, and so on.
template <int THREADS> __device__ __forceinline__ int verify_column(int e) { return e / 4 * (4 * THREADS) + threadIdx.x * 4 + e % 4; }

// A thread's share of the span from c0 on of a row, as 16-byte pieces or one by one; beyond the row -infinity.
template <int THREADS>
__device__ __forceinline__ void verify_load(const float* row, int c0, int V, int four, float (&v)[VERIFY_SPAN / THREADS]) {
    if (four && c0 + VERIFY_SPAN <= V) {
#pragma unroll
        for (int e = 0; e < VERIFY_SPAN / THREADS; e += 4) {
            const float4 q = *(const float4*)(row + c0 + verify_column<THREADS>(e));
            v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VERIFY_SPAN / THREADS; ++e) {
            const int c = c0 + verify_column<THREADS>(e);
            v[e] = row[min(c, V - 1)];
            if (c >= V) v[e] = -INFINITY;
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

template <int THREADS>
__device__ __forceinline__ double verify_block_sum(double v, double* shared) {
    v = verify_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += shared[w];
    return v;
}

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

// One block a span of a row: blockIdx.y counts the rows of the logits, then those of the drafts' logits.
__global__ __launch_bounds__(256) void verify_spans_kernel(VerifyArgs a, VerifyPart* parts) {
    __shared__ float tops[4];
    __shared__ int ats[4];
    __shared__ double sums[4];
    const bool is_guess = (int)blockIdx.y >= a.rows;
    const int i = is_guess ? blockIdx.y - a.rows : blockIdx.y;
    constexpr int EACH = VERIFY_SPAN / 256;
    float v[EACH];
    verify_load<256>((is_guess ? a.guess : a.logits) + (long)i * a.V, blockIdx.x * VERIFY_SPAN, a.V, a.four, v);      // (on its way while the request is looked up)
    // the request: the number of first[1 .. R] (less their index, for the drafts) that are not beyond i
    int low = 0, high = a.R;
    while (low < high) {
        const int mid = (low + high) / 2;
        if (a.first[mid + 1] - (is_guess ? mid + 1 : 0) <= i) low = mid + 1; else high = mid;
    }
    if (low >= a.R) return;
    const float t = a.temperature[low];
    const bool greedy = verify_greedy(t);
    if (is_guess && greedy) return;
    const VerifyScale k(t);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float top = -INFINITY;
    int at = 0x7fffffff;
    if (greedy) {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (v[e] > top) { top = v[e]; at = blockIdx.x * VERIFY_SPAN + verify_column<256>(e); }      // (no NaN is larger than anything)
        verify_wave_top(top, at);
    } else {                                       // (its column is not asked for)
#pragma unroll
        for (int e = 0; e < EACH; ++e) top = fmaxf(top, v[e]);
        top = wave_max(top);
    }
    if (lane == 0) { tops[wave] = top; ats[wave] = at; }
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) { top = tops[w]; at = ats[w]; }
    double sum = 0.0;
    if (!greedy) {
        if (top == INFINITY) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) sum += v[e] == top ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) sum += verify_finite_weight(v[e], top, k);
        }
        sum = verify_block_sum<256>(sum, sums);
    }
    if (threadIdx.x == 0) parts[(long)blockIdx.y * a.spans + blockIdx.x] = {sum, top, at};
}

// The whole row's largest logit, its column and sum, from its spans: by one wave, the same in all lanes.
__device__ __forceinline__ void verify_join(const VerifyPart* parts, int spans, const VerifyScale& k, float& top, int& at, double& sum) {
    const int lane = threadIdx.x & 63;
    VerifyPart mine = {0.0, -INFINITY, 0x7fffffff};
    if (lane < spans) mine = parts[lane];
    top = mine.top;
    at = mine.at;
    for (int s = lane + 64; s < spans; s += 64)
        if (parts[s].top > top) { top = parts[s].top; at = parts[s].at; }
    verify_wave_top(top, at);
    sum = mine.sum * verify_weight(mine.top, top, k);
    for (int s = lane + 64; s < spans; s += 64) sum += parts[s].sum * verify_weight(parts[s].top, top, k);
    sum = verify_wave_sum(sum);
}

// Which drafts of request r are accepted, and what its token is drawn from: by a block of 16 waves, a wave a draft, 16 at a time.  One of the
// blocks that ask writes it down.
__device__ __forceinline__ VerifyChoice verify_accept(const VerifyArgs& a, const VerifyPart* parts, VerifyChoice* choices, int r, bool write) {
    __shared__ VerifyChoice tries[16];
    __shared__ int tokens[16], stops[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo, hi;
    if (!verify_rows(a, r, lo, hi)) {
        VerifyChoice none{};
        none.row = -1;
        if (write && threadIdx.x == 0) { a.accepted[r] = -1; choices[r] = none; }
        return none;
    }
    const float t = a.temperature[r];
    const bool greedy = verify_greedy(t);
    const VerifyScale k(t);
    const int n = hi - lo - 1;
    int j0 = 0, stop = -1;
    for (;; j0 += 16) {
        const int j = j0 + wave;
        if (j <= n) {
            const int d = lo - r + j, x = j < n ? a.drafts[d] : -1;
            const bool inside = x >= 0 && x < a.V;
            const float zp = inside ? a.logits[(long)(lo + j) * a.V + x] : -INFINITY;
            const float zq = inside && a.guess ? a.guess[(long)d * a.V + x] : -INFINITY;
            const float u = j < n ? a.accept[d] : 0.f;
            VerifyChoice c{};
            int at, unused;
            double p_sum, q_sum = 0.0;
            verify_join(parts + (long)(lo + j) * a.spans, a.spans, k, c.p_top, at, p_sum);
            if (!greedy && j < n && a.guess) verify_join(parts + (long)(a.rows + d) * a.spans, a.spans, k, c.q_top, unused, q_sum);
            const int token = c.p_top > -INFINITY ? at : -1;
            c.t = k;
            c.row = greedy || !(p_sum > 0.0) ? -1 : lo + j;      // (no draw: the token is there, or there is none)
            c.p_each = p_sum > 0.0 ? 1.0 / p_sum : 0.0;
            c.q_each = q_sum > 0.0 ? 1.0 / q_sum : 0.0;
            c.guess_row = d;
            c.point = j < n && !a.guess ? x : -1;
            bool take = false;
            if (j < n && greedy) take = token >= 0 && x == token;
            else if (j < n) {
                const double p = verify_weight(zp, c.p_top, k) * c.p_each, q = a.guess ? verify_weight(zq, c.q_top, k) * c.q_each : 1.0;
                take = p > 0.0 && (double)u * q < p;
            }
            if (lane == 0) { tries[wave] = c; tokens[wave] = token; stops[wave] = !take; }
        } else if (lane == 0) {
            stops[wave] = 0;
        }
        __syncthreads();
        for (int w = 15; w >= 0; --w)
            if (stops[w]) stop = w;
        if (stop >= 0) break;                      // (row n is no draft: it stops)
        __syncthreads();
    }
    if (write) {
        const int accepted = j0 + stop;
        for (int i = threadIdx.x; i <= n; i += 1024) a.tokens[lo + i] = i < accepted ? a.drafts[lo - r + i] : greedy && i == accepted ? tokens[stop] : -1;
        if (threadIdx.x == 0) {
            a.accepted[r] = accepted;
            choices[r] = tries[stop];
        }
    }
    return tries[stop];
}

__global__ __launch_bounds__(1024) void verify_accept_kernel(VerifyArgs a, const VerifyPart* parts, VerifyChoice* choices) {
    verify_accept(a, parts, choices, blockIdx.x, true);
}

// The weights in a draw of a thread's share of the span from c0 on, of the logits in the model's row and in the draft's (rest: with the draft's
// distribution taken away).  The forms are told apart once, not at every number, so that the polynomials go side by side (1 request 0.9 us less).
__device__ __forceinline__ void verify_draw_weights(const VerifyChoice& c, const float (&z)[VERIFY_SPAN / 1024], const float (&zq)[VERIFY_SPAN / 1024], int c0,
                                                    bool rest, double (&w)[VERIFY_SPAN / 1024]) {
    constexpr int EACH = VERIFY_SPAN / 1024;
    const bool with_q = rest && c.q_each > 0.0;
    if (c.p_top == INFINITY || (with_q && c.q_top == INFINITY)) {
#pragma unroll 1
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
        if (rest && c0 + verify_column<1024>(e) == c.point) w[e] = 0.0;
}

// A span's weights without the draft's: summed already.
__device__ __forceinline__ double verify_plain_sum(const VerifyArgs& a, const VerifyPart* parts, const VerifyChoice& c, int span) {
    const VerifyPart& p = parts[(long)c.row * a.spans + span];
    return p.sum * verify_weight(p.top, c.p_top, c.t) * c.p_each;
}

// The sum of the weights of a span.  ACCEPT: the block finds the choice for itself.
template <bool ACCEPT>
__global__ __launch_bounds__(1024) void verify_rest_kernel(VerifyArgs a, const VerifyPart* parts, VerifyChoice* choices, double* rests) {
    constexpr int EACH = VERIFY_SPAN / 1024;
    __shared__ double shared[16];
    const int r = blockIdx.y, span = blockIdx.x;
    VerifyChoice c;
    if constexpr (ACCEPT) c = verify_accept(a, parts, choices, r, span == 0);
    else c = choices[r];
    if (c.row < 0) return;
    double sum = 0.0;
    if (c.q_each == 0.0 && (c.point < 0 || c.point / VERIFY_SPAN != span)) {
        if (threadIdx.x != 0) return;
        sum = verify_plain_sum(a, parts, c, span);
    } else {
        float v[EACH], q[EACH];
        verify_load<1024>(a.logits + (long)c.row * a.V, span * VERIFY_SPAN, a.V, a.four, v);
#pragma unroll
        for (int e = 0; e < EACH; ++e) q[e] = 0.f;
        if (c.q_each > 0.0) verify_load<1024>(a.guess + (long)c.guess_row * a.V, span * VERIFY_SPAN, a.V, a.four, q);
        double each[EACH];
        verify_draw_weights(c, v, q, span * VERIFY_SPAN, true, each);
#pragma unroll
        for (int e = 0; e < EACH; ++e) sum += each[e];
        sum = verify_block_sum<1024>(sum, shared);
    }
    if (threadIdx.x == 0) rests[(long)r * a.spans + span] = sum;
}

// The draw: a block a request.  Its span is the first whose sum reaches beyond the random number's share of the whole (every wave finds
// it for itself, 64 spans at a time), then its token the first of the span: sums of four neighbours a thread, then a walk through
// those.  Where a rounding lets a span's own sum fall short of the share, or the number is 1 or more, the token is the last one that
// weighs anything.
__global__ __launch_bounds__(1024) void verify_draw_kernel(VerifyArgs a, const VerifyPart* parts, const VerifyChoice* choices, const double* rests_all) {
    constexpr int EACH = VERIFY_SPAN / 1024;
    __shared__ double shared[16];
    __shared__ int founds[16], lasts[16];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const double* rests = rests_all + (long)r * a.spans;
    double v0 = lane < a.spans ? rests[lane] : 0.0;        // (nothing of them is used where nothing is drawn)
    const VerifyChoice c = choices[r];
    const float u = a.draw[r];
    // (all of the choice at once, with the sums, not part by part as it is wanted)
    asm volatile("" : : "s"(c.row), "s"(c.guess_row), "s"(c.point), "s"(c.p_top), "s"(c.q_top), "s"(c.p_each), "s"(c.q_each), "s"(c.t.k), "s"(c.t.least), "s"(u), "v"(v0));
    if (c.row < 0) return;
    double scan0 = verify_wave_scan(v0), total = verify_lane(scan0, 63);
    for (int s0 = 64; s0 < a.spans; s0 += 64) total += verify_wave_sum(s0 + lane < a.spans ? rests[s0 + lane] : 0.0);
    // (nothing left: the draft's distribution is the model's, and only a rounding or a number beyond 1 refused the draft: p alone)
    const bool rest = total > 0.0;
    auto span_sum = [&](int s) { return s >= a.spans ? 0.0 : rest ? rests[s] : verify_plain_sum(a, parts, c, s); };
    if (!rest) {
        v0 = span_sum(lane);
        scan0 = verify_wave_scan(v0);
        total = 0.0;
        for (int s0 = 0; s0 < a.spans; s0 += 64) total += verify_wave_sum(span_sum(s0 + lane));
    }
    const double target = u > 0.f ? (double)u * total : 0.0;       // (NaN: 0)
    int span = -1;
    double before = 0.0, run = 0.0;
    for (int s0 = 0; s0 < a.spans; s0 += 64) {
        const double v = s0 == 0 ? v0 : span_sum(s0 + lane), scan = s0 == 0 ? scan0 : verify_wave_scan(v);
        const unsigned long some = __ballot(v > 0.0), over = __ballot(v > 0.0 && run + scan > target);
        if (some) {
            const int at = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
            span = s0 + at;
            before = run + verify_lane(scan, at) - verify_lane(v, at);
        }
        if (over) break;
        run += verify_lane(scan, 63);
    }
    if (span < 0) return;                      // (no weight anywhere)
    const int c0 = span * VERIFY_SPAN + tid * EACH;        // (a thread's share is four neighbours)
    double each[EACH], sum = 0.0;
    float v[EACH], q[EACH];
    verify_load<1024>(a.logits + (long)c.row * a.V, span * VERIFY_SPAN, a.V, a.four, v);
#pragma unroll
    for (int e = 0; e < EACH; ++e) q[e] = 0.f;
    if (rest && c.q_each > 0.0) verify_load<1024>(a.guess + (long)c.guess_row * a.V, span * VERIFY_SPAN, a.V, a.four, q);
    int last = -1;
    verify_draw_weights(c, v, q, span * VERIFY_SPAN, rest, each);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        sum += each[e];
        if (each[e] > 0.0) last = c0 + e;
    }
    const double scan = verify_wave_scan(sum);
    if (lane == 63) shared[wave] = scan;
    __syncthreads();
    run = before;
#pragma unroll
    for (int w = 0; w < 16; ++w)
        if (w < wave) run += shared[w];
    run += scan - sum;
    int found = -1;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        run += each[e];
        if (found < 0 && each[e] > 0.0 && run > target) found = c0 + e;
    }
    // the wave's first that reaches beyond, and its last that weighs anything, then the block's (columns rise with the threads)
    const unsigned long over = __ballot(found >= 0), some = __ballot(last >= 0);
    if (over) found = __builtin_amdgcn_readlane(found, __ffsll((unsigned long long)over) - 1);
    if (some) last = __builtin_amdgcn_readlane(last, 63 - __clzll((long long)some));
    if (lane == 0) { founds[wave] = over ? found : -1; lasts[wave] = some ? last : -1; }
    __syncthreads();
    if (tid != 0) return;
    int token = -1;
    for (int w = 0; w < 16; ++w) {
        if (founds[w] >= 0) { token = founds[w]; break; }
        if (lasts[w] >= 0) token = lasts[w];
    }
    a.tokens[c.row] = token;
}

extern "C" long qe_verify_drafts_workspace_bytes(int rows, int V, int R, int has_guess) {
    const long spans = qe_cdiv(V, VERIFY_SPAN), all = rows + (has_guess ? rows - R : 0);
    return all * spans * (long)sizeof(VerifyPart) + (long)R * (long)sizeof(VerifyChoice) + (long)R * spans * 8;
}

// logits float32 [rows, V], first int32 [R + 1], drafts int32 [rows - R], guess float32 [rows - R, V] or null, temperature and draw float32 [R],
// accept float32 [rows - R] -> tokens int32 [rows] (accepted drafts, the token drawn, -1), accepted int32 [R] (-1: first[] names no
// rows that there are; nothing of the request is written then).
extern "C" int qe_verify_drafts(const float* logits, const int* first, const int* drafts, const float* guess, const float* temperature,
                                const float* accept, const float* draw, int* tokens, int* accepted, int rows, int V, int R,
                                void* workspace, long workspace_bytes, hipStream_t stream) {
    QE_REQUIRE(R >= 0 && V > 0 && V < (1 << 30) && rows >= R, "verify_drafts: bad sizes rows=%d V=%d R=%d", rows, V, R);
    if (R == 0) return 0;
    const int spans = qe_cdiv(V, VERIFY_SPAN), all = rows + (guess ? rows - R : 0);
    QE_REQUIRE(all <= 65535, "verify_drafts: %d rows of logits are too many", all);
    QE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= qe_verify_drafts_workspace_bytes(rows, V, R, guess != nullptr),
               "verify_drafts: workspace too small");
    VerifyPart* parts = (VerifyPart*)workspace;
    VerifyChoice* choices = (VerifyChoice*)(parts + (long)all * spans);
    double* rests = (double*)(choices + R);
    const int four = V % 4 == 0 && (((uintptr_t)logits | (uintptr_t)guess) & 15) == 0;
    const VerifyArgs a{logits, guess, first, drafts, temperature, accept, draw, tokens, accepted, rows, V, R, spans, four};
    verify_spans_kernel<<<dim3(spans, all), 256, 0, stream>>>(a, parts);
    // Few spans: every block accepts for itself, which saves a launch (spans of 1 request of 151936 15.1 us, in two launches 16.4; of 8, 304
    // spans, 27.2 and 28.1; of 16 40.4 and 36.3).
    if ((long)spans * R <= 320) {
        verify_rest_kernel<true><<<dim3(spans, R), 1024, 0, stream>>>(a, parts, choices, rests);
    } else {
        verify_accept_kernel<<<R, 1024, 0, stream>>>(a, parts, choices);
        verify_rest_kernel<false><<<dim3(spans, R), 1024, 0, stream>>>(a, parts, choices, rests);
    }
    verify_draw_kernel<<<R, 1024, 0, stream>>>(a, parts, choices, rests);
    QE_LAUNCH_CHECK();
    return 0;
}
