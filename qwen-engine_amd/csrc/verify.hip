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

// exp((z - top) / t), in 64-bit; top is the row's largest logit
__device__ __forceinline__ double verify_weight(float z, float top, double inv_t) {
    if (z == top) return top == -INFINITY ? 0.0 : 1.0;
    if (!(z > -INFINITY) || top == INFINITY) return 0.0;
    return exp(((double)z - (double)top) * inv_t);
}

// The rows of request r, or false where first[] holds no rows and drafts that there are.
__device__ __forceinline__ bool verify_rows(const VerifyArgs& a, int r, int& lo, int& hi) {
    lo = a.first[r];
    hi = a.first[r + 1];
    return lo >= r && hi > lo && hi <= a.rows && hi - 1 - r <= a.rows - a.R;
}

// One block a span of a row: blockIdx.y counts the rows of the logits, then those of the drafts' logits.
__global__ __launch_bounds__(256) void verify_spans_kernel(VerifyArgs a, VerifyPart* parts) {
    __shared__ float tops[4];
    __shared__ int ats[4];
    __shared__ double sums[4];
    const bool is_guess = (int)blockIdx.y >= a.rows;
    const int i = is_guess ? blockIdx.y - a.rows : blockIdx.y;
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
    const double inv_t = greedy ? 0.0 : 1.0 / (double)t;
    const float* row = (is_guess ? a.guess : a.logits) + (long)i * a.V;
    const int c0 = blockIdx.x * VERIFY_SPAN, c1 = min(a.V, c0 + VERIFY_SPAN);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float v[VERIFY_SPAN / 256];
    float top = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < VERIFY_SPAN / 256; ++e) {
        const int c = c0 + e * 256 + threadIdx.x;
        v[e] = c < c1 ? row[c] : -INFINITY;
        if (v[e] != v[e]) v[e] = -INFINITY;
        if (v[e] > top) { top = v[e]; at = c; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float other = __shfl_xor(top, o, 64);
        const int there = __shfl_xor(at, o, 64);
        if (other > top || (other == top && there < at)) { top = other; at = there; }
    }
    if (lane == 0) { tops[wave] = top; ats[wave] = at; }
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) { top = tops[w]; at = ats[w]; }
    double sum = 0.0;
    if (!greedy && top > -INFINITY) {
#pragma unroll
        for (int e = 0; e < VERIFY_SPAN / 256; ++e) sum += verify_weight(v[e], top, inv_t);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = sums[0] + sums[1] + sums[2] + sums[3];
    }
    if (threadIdx.x == 0) parts[(long)blockIdx.y * a.spans + blockIdx.x] = {sum, top, at};
}

// The whole row's largest logit, its column and sum, from its spans: by one wave, the same in all lanes.
__device__ __forceinline__ void verify_join(const VerifyPart* parts, int spans, double inv_t, float& top, int& at, double& sum) {
    const int lane = threadIdx.x & 63;
    top = -INFINITY;
    at = 0x7fffffff;
    for (int s = lane; s < spans; s += 64)
        if (parts[s].top > top) { top = parts[s].top; at = parts[s].at; }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float other = __shfl_xor(top, o, 64);
        const int there = __shfl_xor(at, o, 64);
        if (other > top || (other == top && there < at)) { top = other; at = there; }
    }
    sum = 0.0;
    for (int s = lane; s < spans; s += 64) sum += parts[s].sum * verify_weight(parts[s].top, top, inv_t);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
}

// A wave a request: which drafts are accepted, and what the token is drawn from.
__global__ __launch_bounds__(64) void verify_accept_kernel(VerifyArgs a, const VerifyPart* parts, VerifyChoice* choices) {
    const int r = blockIdx.x, lane = threadIdx.x;
    int lo, hi;
    if (!verify_rows(a, r, lo, hi)) {
        if (lane == 0) { a.accepted[r] = -1; choices[r].row = -1; }
        return;
    }
    const float t = a.temperature[r];
    const bool greedy = verify_greedy(t);
    const double inv_t = greedy ? 0.0 : 1.0 / (double)t;
    VerifyChoice c{};
    int j = 0, token = -1;
    const int n = hi - lo - 1;
    for (;; ++j) {
        int at;
        verify_join(parts + (long)(lo + j) * a.spans, a.spans, inv_t, c.p_top, at, c.p_sum);
        token = c.p_top > -INFINITY ? at : -1;
        c.row = lo + j;
        c.guess_row = -1;
        if (j == n) break;
        const int d = lo - r + j, x = a.drafts[d];
        const bool inside = x >= 0 && x < a.V;
        if (greedy) {
            if (x != token || token < 0) break;
            continue;
        }
        double p = 0.0, q = 1.0;
        if (inside && c.p_sum > 0.0) {
            const float z = a.logits[(long)(lo + j) * a.V + x];
            p = verify_weight(z, c.p_top, inv_t) / c.p_sum;
        }
        c.guess_row = -2;
        if (a.guess) {
            int unused;
            c.guess_row = d;
            verify_join(parts + (long)(a.rows + d) * a.spans, a.spans, inv_t, c.q_top, unused, c.q_sum);
            q = inside && c.q_sum > 0.0 ? verify_weight(a.guess[(long)d * a.V + x], c.q_top, inv_t) / c.q_sum : 0.0;
        }
        c.draft = x;
        if (!(p > 0.0 && (double)a.accept[d] * q < p)) break;
    }
    for (int i = lane; i <= n; i += 64) a.tokens[lo + i] = i < j ? a.drafts[lo - r + i] : greedy && i == j ? token : -1;
    if (lane == 0) {
        a.accepted[r] = j;
        c.accepted = j;
        if (greedy || !(c.p_sum > 0.0)) c.row = -1;     // (no draw: the token is there, or there is none)
        choices[r] = c;
    }
}

// The weight of column i in the draw of choice c (rest: with the draft's distribution taken away).
__device__ __forceinline__ double verify_draw_weight(const VerifyArgs& a, const VerifyChoice& c, double inv_t, int i, bool rest) {
    const double p = verify_weight(a.logits[(long)c.row * a.V + i], c.p_top, inv_t) / c.p_sum;
    if (!rest || c.guess_row == -1) return p;
    if (c.guess_row == -2) return i == c.draft ? 0.0 : p;
    const double q = c.q_sum > 0.0 ? verify_weight(a.guess[(long)c.guess_row * a.V + i], c.q_top, inv_t) / c.q_sum : 0.0;
    return p > q ? p - q : 0.0;
}

__device__ __forceinline__ double verify_block_sum(double v, double* shared) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return shared[0] + shared[1] + shared[2] + shared[3];
}

// The sum of the weights of a span, where a draft was not accepted.
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs a, const VerifyChoice* choices, double* rests) {
    __shared__ double shared[4];
    const int r = blockIdx.y;
    const VerifyChoice c = choices[r];
    if (c.row < 0) return;
    const double inv_t = 1.0 / (double)a.temperature[r];
    const int c0 = blockIdx.x * VERIFY_SPAN, c1 = min(a.V, c0 + VERIFY_SPAN);
    double sum = 0.0;
    for (int i = c0 + threadIdx.x; i < c1; i += 256) sum += verify_draw_weight(a, c, inv_t, i, true);
    sum = verify_block_sum(sum, shared);
    if (threadIdx.x == 0) rests[(long)r * a.spans + blockIdx.x] = sum;
}

// The draw: a block a request.
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a, const VerifyChoice* choices, const double* rests_all) {
    __shared__ double part[256];
    __shared__ double before_s, target_s;
    __shared__ int span_s, found_s, last_s, rest_s;
    const int r = blockIdx.x, tid = threadIdx.x;
    const VerifyChoice c = choices[r];
    if (c.row < 0) return;
    const double inv_t = 1.0 / (double)a.temperature[r];
    const double* rests = rests_all + (long)r * a.spans;
    if (tid == 0) {
        double total = 0.0;
        for (int s = 0; s < a.spans; ++s) total += rests[s];
        // (nothing left: the draft's distribution is the model's, and only a rounding or a number beyond 1 refused the draft)
        rest_s = total > 0.0;
    }
    __syncthreads();
    const bool rest = rest_s;
    if (!rest) {                          // sums of p alone, span by span
        double* mine = (double*)rests;
        for (int s = 0; s < a.spans; ++s) {
            double v = 0.0;
            for (int i = s * VERIFY_SPAN + tid; i < min(a.V, (s + 1) * VERIFY_SPAN); i += 256) v += verify_draw_weight(a, c, inv_t, i, false);
            v = verify_block_sum(v, part);
            if (tid == 0) mine[s] = v;
        }
        __syncthreads();
    }
    if (tid == 0) {
        double total = 0.0, run = 0.0;
        for (int s = 0; s < a.spans; ++s) total += rests[s];
        const double target = a.draw[r] > 0.f ? (double)a.draw[r] * total : 0.0;     // (NaN: 0)
        int span = -1, last = 0;
        double before = 0.0;
        for (int s = 0; s < a.spans; ++s) {
            if (rests[s] > 0.0) {
                if (run + rests[s] > target) { span = s; break; }
                last = s;
                before = run;
            }
            run += rests[s];
        }
        before_s = span >= 0 ? run : before;
        target_s = target;
        span_s = span >= 0 ? span : last;       // (a number of 1 or more, or the sums' rounding: the last token that weighs anything)
        found_s = last_s = -1;
    }
    __syncthreads();
    const int each = VERIFY_SPAN / 256, c0 = span_s * VERIFY_SPAN + tid * each, c1 = min(a.V, c0 + each);
    double sum = 0.0;
    int last = -1;
    for (int i = c0; i < c1; ++i) {
        const double w = verify_draw_weight(a, c, inv_t, i, rest);
        sum += w;
        if (w > 0.0) last = i;
    }
    part[tid] = sum;
    __syncthreads();
    double run = before_s;
    for (int i = 0; i < tid; ++i) run += part[i];
    if (last >= 0) {
        atomicMax(&last_s, last);
        if (run + sum > target_s && !(run > target_s)) {
            int found = last;
            for (int i = c0; i < c1; ++i) {
                const double w = verify_draw_weight(a, c, inv_t, i, rest);
                run += w;
                if (w > 0.0 && run > target_s) { found = i; break; }
            }
            atomicCAS(&found_s, -1, found);
        }
    }
    __syncthreads();
    if (tid == 0) a.tokens[c.row] = found_s >= 0 ? found_s : last_s;
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
    const VerifyArgs a{logits, guess, first, drafts, temperature, accept, draw, tokens, accepted, rows, V, R, spans};
    verify_spans_kernel<<<dim3(spans, all), 256, 0, stream>>>(a, parts);
    verify_accept_kernel<<<R, 64, 0, stream>>>(a, parts, choices);
    verify_rest_kernel<<<dim3(spans, R), 256, 0, stream>>>(a, choices, rests);
    verify_draw_kernel<<<R, 256, 0, stream>>>(a, choices, rests);
    QE_LAUNCH_CHECK();
    return 0;
}
