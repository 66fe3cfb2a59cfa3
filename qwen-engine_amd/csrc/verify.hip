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
// Four launches: spans of 4096 logits (all rows, bound by their bytes), acceptance (a block a request, a wave a draft), the spans' sums
// of what the token is drawn from (one row a request, and its draft's), the draw.
#include "common.h"

#define VERIFY_SPAN 4096
#define VERIFY_EACH (VERIFY_SPAN / 256)        // logits of a thread

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

struct VerifyChoice {           // of a request: the row that its token is drawn from
    double p_sum, q_sum;
    float p_top, q_top;
    int row, guess_row;         // (row -1: none; guess_row -1: no draft's distribution to take away, -2: all on the draft)
    int draft, accepted;
};

__device__ __forceinline__ bool verify_greedy(float t) { return !(t > 0.f); }

// log2(e) / t, by which a difference of logits becomes a power of two's exponent
__device__ __forceinline__ double verify_scale(float t) { return 1.4426950408889634074 / (double)t; }

// exp((z - top) / t) in 64-bit, k = verify_scale(t), top the row's largest logit: 2^y = 2^n 2^f with n = y rounded, f in [-1/2, 1/2], and 2^f by a
// polynomial of degree 10 through the Chebyshev points of that interval (off by 3.2e-16 of it at the most).  What is NaN on the
// way (a NaN logit; -infinity less itself) becomes 0 at the maximum, as what is below 2^-1080 does.
__device__ __forceinline__ double verify_weight(float z, float top, double k) {
    const double y = __builtin_fmax(((double)z - (double)top) * k, -1080.0);
    const double n = __builtin_rint(y), f = y - n;
    double v = 0x1.e6063f9b91935p-28;
    v = __builtin_fma(v, f, 0x1.b675bd687d9b8p-24);
    v = __builtin_fma(v, f, 0x1.62bfd477051e0p-20);
    v = __builtin_fma(v, f, 0x1.ffcb540541227p-17);
    v = __builtin_fma(v, f, 0x1.430913096fcb8p-13);
    v = __builtin_fma(v, f, 0x1.5d87fe9d7ab80p-10);
    v = __builtin_fma(v, f, 0x1.3b2ab6fba1de1p-7);
    v = __builtin_fma(v, f, 0x1.c6b08d703ce45p-5);
    v = __builtin_fma(v, f, 0x1.ebfbdff82c598p-3);
    v = __builtin_fma(v, f, 0x1.62e42fefa3a19p-1);
    v = __builtin_fma(v, f, 1.0);
    v = __builtin_amdgcn_ldexp(v, (int)n);
    return top == INFINITY ? (z == top ? 1.0 : 0.0) : v;        // (infinite logits share everything)
}

// The rows of request r, or false where first[] holds no rows and drafts that there are.
__device__ __forceinline__ bool verify_rows(const VerifyArgs& a, int r, int& lo, int& hi) {
    lo = a.first[r];
    hi = a.first[r + 1];
    return lo >= r && hi > lo && hi <= a.rows && hi - 1 - r <= a.rows - a.R;
}

// Logits c0 + 4 tid .. + 3, c0 + 1024 + 4 tid .. and so on of a row, as 16-byte pieces or one by one; beyond the row -infinity.
__device__ __forceinline__ void verify_load(const float* row, int c0, int V, int four, float (&v)[VERIFY_EACH]) {
#pragma unroll
    for (int e = 0; e < VERIFY_EACH; e += 4) {
        const int c = c0 + e * 256 + threadIdx.x * 4;
        if (four && c + 4 <= V) {
            const float4 q = *(const float4*)(row + c);
            v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[e + i] = c + i < V ? row[c + i] : -INFINITY;
        }
    }
}

__device__ __forceinline__ double verify_wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double verify_block_sum(double v, double* shared) {       // 256 threads
    v = verify_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return shared[0] + shared[1] + shared[2] + shared[3];
}

// The largest of the wave and the lowest column that has it, in every lane.
__device__ __forceinline__ void verify_wave_top(float& top, int& at) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float other = __shfl_xor(top, o, 64);
        const int there = __shfl_xor(at, o, 64);
        if (other > top || (other == top && there < at)) { top = other; at = there; }
    }
}

// One block a span of a row: blockIdx.y counts the rows of the logits, then those of the drafts' logits.
__global__ __launch_bounds__(256) void verify_spans_kernel(VerifyArgs a, VerifyPart* parts) {
    __shared__ float tops[4];
    __shared__ int ats[4];
    __shared__ double sums[4];
    const bool is_guess = (int)blockIdx.y >= a.rows;
    const int i = is_guess ? blockIdx.y - a.rows : blockIdx.y;
    float v[VERIFY_EACH];
    verify_load((is_guess ? a.guess : a.logits) + (long)i * a.V, blockIdx.x * VERIFY_SPAN, a.V, a.four, v);      // (on its way while the request is looked up)
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
    const double k = greedy ? 0.0 : verify_scale(t);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float top = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < VERIFY_EACH; ++e)
        if (v[e] > top) { top = v[e]; at = blockIdx.x * VERIFY_SPAN + (e / 4) * 1024 + threadIdx.x * 4 + e % 4; }      // (a NaN is larger than nothing)
    verify_wave_top(top, at);
    if (lane == 0) { tops[wave] = top; ats[wave] = at; }
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) { top = tops[w]; at = ats[w]; }
    double sum = 0.0;
    if (!greedy) {
        double more = 0.0;
#pragma unroll
        for (int e = 0; e < VERIFY_EACH; e += 2) {
            sum += verify_weight(v[e], top, k);
            more += verify_weight(v[e + 1], top, k);
        }
        sum = verify_block_sum(sum + more, sums);
    }
    if (threadIdx.x == 0) parts[(long)blockIdx.y * a.spans + blockIdx.x] = {sum, top, at};
}

// The whole row's largest logit, its column and sum, from its spans: by one wave, the same in all lanes.
__device__ __forceinline__ void verify_join(const VerifyPart* parts, int spans, double k, float& top, int& at, double& sum) {
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

// A block a request, a wave a draft, 16 at a time: which drafts are accepted, and what the token is drawn from.
__global__ __launch_bounds__(1024) void verify_accept_kernel(VerifyArgs a, const VerifyPart* parts, VerifyChoice* choices) {
    __shared__ VerifyChoice tries[16];
    __shared__ int tokens[16], stops[16];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo, hi;
    if (!verify_rows(a, r, lo, hi)) {
        if (threadIdx.x == 0) { a.accepted[r] = -1; choices[r].row = -1; }
        return;
    }
    const float t = a.temperature[r];
    const bool greedy = verify_greedy(t);
    const double k = greedy ? 0.0 : verify_scale(t);
    const int n = hi - lo - 1;
    int j0 = 0, stop = -1;
    for (;; j0 += 16) {
        const int j = j0 + wave;
        if (j <= n) {
            const int d = lo - r + j, x = j < n ? a.drafts[d] : -1;
            const bool inside = x >= 0 && x < a.V;
            const float zp = inside ? a.logits[(long)(lo + j) * a.V + x] : -INFINITY;
            const float zq = inside && a.guess ? a.guess[(long)d * a.V + x] : -INFINITY;
            VerifyChoice c{};
            int at, unused;
            verify_join(parts + (long)(lo + j) * a.spans, a.spans, k, c.p_top, at, c.p_sum);
            c.row = lo + j;
            c.guess_row = j == n ? -1 : a.guess ? d : -2;
            c.draft = x;
            const int token = c.p_top > -INFINITY ? at : -1;
            bool take = false;
            if (j < n && greedy) take = token >= 0 && x == token;
            else if (j < n) {
                double q = 1.0;
                if (a.guess) {
                    verify_join(parts + (long)(a.rows + d) * a.spans, a.spans, k, c.q_top, unused, c.q_sum);
                    q = c.q_sum > 0.0 ? verify_weight(zq, c.q_top, k) / c.q_sum : 0.0;
                }
                const double p = inside && c.p_sum > 0.0 ? verify_weight(zp, c.p_top, k) / c.p_sum : 0.0;
                take = p > 0.0 && (double)a.accept[d] * q < p;
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
    const int accepted = j0 + stop;
    for (int i = threadIdx.x; i <= n; i += 1024) a.tokens[lo + i] = i < accepted ? a.drafts[lo - r + i] : greedy && i == accepted ? tokens[stop] : -1;
    if (threadIdx.x == 0) {
        a.accepted[r] = accepted;
        VerifyChoice c = tries[stop];
        c.accepted = accepted;
        if (greedy || !(c.p_sum > 0.0)) c.row = -1;      // (no draw: the token is there, or there is none)
        choices[r] = c;
    }
}

// What the weights of choice c are made of, once for a thread.
struct VerifyDraw {
    double k, p_each, q_each;          // (1 / sums; q_each 0: nothing is taken away)
    float p_top, q_top;
    int point;                         // the column that a draft without logits was, or -1
    __device__ __forceinline__ VerifyDraw(const VerifyChoice& c, float t, bool rest) {
        k = verify_scale(t);
        p_top = c.p_top;
        q_top = c.q_top;
        p_each = 1.0 / c.p_sum;
        q_each = rest && c.guess_row >= 0 && c.q_sum > 0.0 ? 1.0 / c.q_sum : 0.0;
        point = rest && c.guess_row == -2 ? c.draft : -1;
    }
    __device__ __forceinline__ double weight(float z, float zq, int i) const {
        double w = verify_weight(z, p_top, k) * p_each;
        if (q_each > 0.0) w = __builtin_fmax(w - verify_weight(zq, q_top, k) * q_each, 0.0);
        return i == point ? 0.0 : w;
    }
};

// The sum of the weights of a span.
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs a, const VerifyPart* parts, const VerifyChoice* choices, double* rests) {
    __shared__ double shared[4];
    const int r = blockIdx.y;
    const VerifyChoice c = choices[r];
    if (c.row < 0) return;
    const VerifyDraw w(c, a.temperature[r], true);
    double sum = 0.0;
    if (w.q_each == 0.0 && (w.point < 0 || w.point / VERIFY_SPAN != (int)blockIdx.x)) {     // p alone: its span is summed already
        if (threadIdx.x != 0) return;
        const VerifyPart& p = parts[(long)c.row * a.spans + blockIdx.x];
        sum = p.sum * verify_weight(p.top, c.p_top, w.k) * w.p_each;
    } else {
        float v[VERIFY_EACH], q[VERIFY_EACH];
        verify_load(a.logits + (long)c.row * a.V, blockIdx.x * VERIFY_SPAN, a.V, a.four, v);
#pragma unroll
        for (int e = 0; e < VERIFY_EACH; ++e) q[e] = 0.f;
        if (w.q_each > 0.0) verify_load(a.guess + (long)c.guess_row * a.V, blockIdx.x * VERIFY_SPAN, a.V, a.four, q);
#pragma unroll
        for (int e = 0; e < VERIFY_EACH; ++e) sum += w.weight(v[e], q[e], blockIdx.x * VERIFY_SPAN + (e / 4) * 1024 + threadIdx.x * 4 + e % 4);
        sum = verify_block_sum(sum, shared);
    }
    if (threadIdx.x == 0) rests[(long)r * a.spans + blockIdx.x] = sum;
}

// The sum of the values of the threads before this one; total: of all 256.
__device__ __forceinline__ double verify_sum_before(double v, double* shared, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double run = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double other = __shfl_up(run, o, 64);
        if (lane >= o) run += other;
    }
    __syncthreads();
    if (lane == 63) shared[wave] = run;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += shared[w];
        total += shared[w];
    }
    const double mine = __shfl_up(run, 1, 64);
    return before + (lane > 0 ? mine : 0.0);
}

// The draw: a block a request.  Its span is the first whose sum reaches beyond the random number's share of the whole, then
// its token the first of the span: sums of 16 neighbours a thread, then a walk through those.  Where a rounding lets a span's own sum
// fall short of the share, or the number is 1 or more, the token is the last one that weighs anything.
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a, const VerifyPart* parts, const VerifyChoice* choices, const double* rests_all) {
    __shared__ double shared[4];
    __shared__ int found_s, last_s;
    __shared__ double before_s;
    const int r = blockIdx.x, tid = threadIdx.x;
    const VerifyChoice c = choices[r];
    if (c.row < 0) return;
    const double* rests = rests_all + (long)r * a.spans;
    double total = 0.0, one;
    for (int s0 = 0; s0 < a.spans; s0 += 256) {
        verify_sum_before(s0 + tid < a.spans ? rests[s0 + tid] : 0.0, shared, one);
        total += one;
    }
    // (nothing left: the draft's distribution is the model's, and only a rounding or a number beyond 1 refused the draft: p alone)
    const bool rest = total > 0.0;
    const VerifyDraw w(c, a.temperature[r], rest);
    if (!rest) {
        for (int s0 = 0; s0 < a.spans; s0 += 256) {
            double v = 0.0;
            if (s0 + tid < a.spans) {
                const VerifyPart& p = parts[(long)c.row * a.spans + s0 + tid];
                v = p.sum * verify_weight(p.top, c.p_top, w.k) * w.p_each;
            }
            verify_sum_before(v, shared, one);
            total += one;
        }
    }
    const double target = a.draw[r] > 0.f ? (double)a.draw[r] * total : 0.0;     // (NaN: 0)
    if (tid == 0) { found_s = 0x7fffffff; last_s = -1; }
    double run = 0.0;
    for (int s0 = 0; s0 < a.spans; s0 += 256) {
        double v = 0.0;
        if (s0 + tid < a.spans) {
            if (rest) v = rests[s0 + tid];
            else {
                const VerifyPart& p = parts[(long)c.row * a.spans + s0 + tid];
                v = p.sum * verify_weight(p.top, c.p_top, w.k) * w.p_each;
            }
        }
        const double before = run + verify_sum_before(v, shared, one);           // (its barriers stand behind the values of found_s and last_s)
        if (v > 0.0) {
            if (before + v > target) atomicMin(&found_s, s0 + tid);
            atomicMax(&last_s, s0 + tid);
        }
        __syncthreads();
        const int span = found_s != 0x7fffffff ? found_s : last_s;
        if (span == s0 + tid) before_s = before;
        __syncthreads();
        run += one;
        if (found_s != 0x7fffffff) break;
    }
    const int span = found_s != 0x7fffffff ? found_s : last_s;
    const double before = before_s;
    if (span < 0) return;                      // (no weight anywhere)
    __syncthreads();
    if (tid == 0) { found_s = 0x7fffffff; last_s = -1; }
    const int c0 = span * VERIFY_SPAN + tid * VERIFY_EACH;
    const float* row = a.logits + (long)c.row * a.V + c0;
    const float* guess = w.q_each > 0.0 ? a.guess + (long)c.guess_row * a.V + c0 : row;
    double each[VERIFY_EACH], sum = 0.0;
    float v[VERIFY_EACH], q[VERIFY_EACH];
#pragma unroll
    for (int e = 0; e < VERIFY_EACH; e += 4) {
        if (a.four && c0 + e + 4 <= a.V) {
            const float4 x = *(const float4*)(row + e), y = *(const float4*)(guess + e);
            v[e] = x.x; v[e + 1] = x.y; v[e + 2] = x.z; v[e + 3] = x.w;
            q[e] = y.x; q[e + 1] = y.y; q[e + 2] = y.z; q[e + 3] = y.w;
        } else {
#pragma unroll
            for (int i = e; i < e + 4; ++i) {
                v[i] = q[i] = -INFINITY;
                if (c0 + i < a.V) { v[i] = row[i]; q[i] = guess[i]; }
            }
        }
    }
    int last = -1;
#pragma unroll
    for (int e = 0; e < VERIFY_EACH; ++e) {
        each[e] = w.weight(v[e], q[e], c0 + e);
        sum += each[e];
        if (each[e] > 0.0) last = c0 + e;
    }
    run = before + verify_sum_before(sum, shared, one);
    if (last >= 0) {
        int found = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < VERIFY_EACH; ++e) {
            run += each[e];
            if (found == 0x7fffffff && each[e] > 0.0 && run > target) found = c0 + e;
        }
        if (found != 0x7fffffff) atomicMin(&found_s, found);
        atomicMax(&last_s, last);
    }
    __syncthreads();
    if (tid == 0) a.tokens[c.row] = found_s != 0x7fffffff ? found_s : last_s;
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
    QE_REQUIRE(R >= 0 && V > 0 && rows >= R, "verify_drafts: bad sizes rows=%d V=%d R=%d", rows, V, R);
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
    verify_accept_kernel<<<R, 1024, 0, stream>>>(a, parts, choices);
    verify_rest_kernel<<<dim3(spans, R), 256, 0, stream>>>(a, parts, choices, rests);
    verify_draw_kernel<<<R, 256, 0, stream>>>(a, parts, choices, rests);
    QE_LAUNCH_CHECK();
    return 0;
}
