// vq_verify.hip -- verification of drafted tokens against the target's logits from given random numbers, and sampling of the token
// that follows them.
//
// Row j of a sequence gives p_j = softmax(l_j / T). Draft x_j is accepted while u_j q_j(x_j) < p_j(x_j); at the first refusal the
// next token comes from max(0, p_j - q_j), normalised, and after all of them from p_k, by inverse CDF: the first index whose
// cumulative weight exceeds v_j times the total. Everything from the exponent on is in 64 bits: a vocabulary of 248320 tokens
// puts the borders of the cumulative sum 4e-6 apart on average and most of them far nearer, so sums of 32 bits would pick a
// neighbour now and then, and no two orders of summation would agree.
//
// Three launches. Statistics: each row in chunks of kChunk logits, the chunk's maximum and sum of weights (one pass over the
// logits, which bounds the whole). Residual: for the row where a sequence stopped, each chunk's sum of max(0, p - q); only where
// something drafted may be refused. Pick: one workgroup per sequence finds the chunk by the chunks' sums, then the element. The
// last two decide from the statistics what was accepted, each for itself. The chunks do not depend on the batch, so neither does
// any bit of a sequence's results.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "../../include/vq.h"
#include "vq_seq.h"

namespace {

// Logits of a thread: 4 or 16 take longer (64 rows sampled: 24.4 us with 8, 28.7 and 25.0; one sequence of 4 rows: 17.5, 17.7, 21.1).
constexpr int kThreads = 256, kEach = 8, kChunk = kThreads * kEach;

struct VerSeq {
    int row0, k;  // rows row0 .. row0 + k, the first k of them followed by drafts draft0 ..
    int draft0;
    double t;
};
struct VerTable {
    int n;
    VerSeq s[VQ_MAX_SEGMENTS];
};

// What a pass reads and writes; the workspace: statistics [row][chunk], residual sums [sequence][chunk].
struct VerArgs {
    const float *logits, *probs, *u;
    const int32_t *draft;
    int32_t *tokens, *counts;
    float *logprobs;
    double2 *stats;
    double *residual;
    int vocab, chunks;
};

// A logit as it counts: NaN never wins, like -inf.
__device__ __forceinline__ float logit(float x) { return x == x ? x : -INFINITY; }
// 2^x for x <= 0: x = n + f with |f| <= 1/2, the Taylor polynomial of degree 12 in f ln 2, times 2^n. What it leaves out is at most
// (ln 2 / 2)^13 / 13! = 1.7e-16, 2.4e-16 of 2^f at f = -1/2, as much as the roundings of the evaluation. Below -1100 the result is 0
// anyway. The math library's exp, which also serves x > 0 and NaN, takes twice the instructions, and they are as many as hide behind
// the logits' loads: see verify_stats_kernel.
__device__ __forceinline__ double exp2_neg(double x) {
    constexpr double L = 0.6931471805599453;
    x = fmax(x, -1100.0);
    const double n = rint(x), f = x - n;
    double p = L * L * L * L * L * L * L * L * L * L * L * L / 479001600.0;
    p = fma(p, f, L * L * L * L * L * L * L * L * L * L * L / 39916800.0);
    p = fma(p, f, L * L * L * L * L * L * L * L * L * L / 3628800.0);
    p = fma(p, f, L * L * L * L * L * L * L * L * L / 362880.0);
    p = fma(p, f, L * L * L * L * L * L * L * L / 40320.0);
    p = fma(p, f, L * L * L * L * L * L * L / 5040.0);
    p = fma(p, f, L * L * L * L * L * L / 720.0);
    p = fma(p, f, L * L * L * L * L / 120.0);
    p = fma(p, f, L * L * L * L / 24.0);
    p = fma(p, f, L * L * L / 6.0);
    p = fma(p, f, L * L / 2.0);
    p = fma(p, f, L);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}
// exp((x - m) / T), `per` being log2(e) / T; 1 at the maximum whatever it is (all of the mass is at +inf where that is the maximum).
__device__ __forceinline__ double weight(double x, double m, double per) {
    if (m == INFINITY) return x == m ? 1.0 : 0.0;
    return x == m ? 1.0 : exp2_neg((x - m) * per);
}
// log2(e) / T, finite for the smallest T too: a zero difference times it stays zero.
__device__ __forceinline__ double per_of(double t) { return fmin(1.4426950408889634 / t, 1e300); }

// A thread's kEach neighbouring values from i on, `fill` past n.
__device__ __forceinline__ void load_each(const float *p, int i, int n, float fill, float (&x)[kEach]) {
    if (i + kEach <= n) {
        __builtin_memcpy(x, p + i, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) x[e] = i + e < n ? p[i + e] : fill;
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
// Over the workgroup's four waves, in wave order; every thread gets the result.
__device__ __forceinline__ double group_sum(double v, double *lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return ((lds[0] + lds[1]) + lds[2]) + lds[3];
}
// Inclusive sum over the threads before and at this one.
__device__ __forceinline__ double group_scan(double v, double *lds) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(v, o, 64);
        if (lane >= o) v += up;
    }
    if (lane == 63) lds[wv] = v;
    __syncthreads();
    for (int w = 0; w < wv; ++w) v += lds[w];
    return v;
}

// The least of the threads' `lo` and the largest of their `hi`, to every thread.
__device__ __forceinline__ int2 group_span(int lo, int hi, int2 *lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64)), hi = max(hi, __shfl_xor(hi, o, 64));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = int2{lo, hi};
    __syncthreads();
    int2 r = lds[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) r = int2{min(r.x, lds[w].x), max(r.y, lds[w].y)};
    return r;
}

// Workgroup (chunk, row of a sequence, sequence): (maximum, sum of weights against it), for a greedy row (maximum, its lowest index).
// Bound by the logits' bytes and by the weights' 22 instructions of 64 bits a logit, nearly equally: 64 rows of 248320 are 64 MB, 12.5
// us at the rate of a copy, and 9 us of instructions; this takes 19 (22 with an exp of 27 instructions). Workgroups of several chunks
// that load one while they compute with the one before take longer (4 chunks: 24 us): many workgroups at different points overlap the
// two better.
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerArgs a, VerTable T) {
    __shared__ float smax[4];
    __shared__ double ssum[4];
    __shared__ int2 span[4];
    const VerSeq &q = T.s[blockIdx.z];
    if (static_cast<int>(blockIdx.y) > q.k) return;
    const size_t row = static_cast<size_t>(q.row0) + blockIdx.y;
    const double t = q.t;
    const int at = blockIdx.x * kChunk + threadIdx.x * kEach;
    float x[kEach], m = -INFINITY;
    load_each(a.logits + row * a.vocab, at, a.vocab, -INFINITY, x);
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = logit(x[e]), m = fmaxf(m, x[e]);
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) smax[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    double2 *out = a.stats + row * a.chunks + blockIdx.x;
    if (t == 0.0) {
        int first = INT_MAX;
#pragma unroll
        for (int e = kEach - 1; e >= 0; --e)
            if (x[e] == m && m > -INFINITY) first = at + e;
        first = group_span(first, 0, span).x;
        if (threadIdx.x == 0) *out = double2{m, static_cast<double>(first)};
        return;
    }
    const double per = per_of(t);
    double s = 0.0;
    if (m < INFINITY) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) s += exp2_neg((static_cast<double>(x[e]) - m) * per);  // (1 at the maximum)
    } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) s += x[e] == m ? 1.0 : 0.0;
    }
    s = group_sum(m > -INFINITY ? s : 0.0, ssum);
    if (threadIdx.x == 0) *out = double2{m, s};
}

// What the statistics of a sequence's rows say: `stop`, the drafts accepted, and each row's maximum and total (greedy: its token).
struct Decision {
    int stop;
    double m[VQ_MAX_DRAFT + 1], z[VQ_MAX_DRAFT + 1];
};
// Called by a whole workgroup; each wave takes rows in turn, its lanes the row's chunks.
__device__ void decide(const VerArgs &a, const VerSeq &s, Decision &d) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const bool greedy = s.t == 0.0;
    const double per = greedy ? 0.0 : per_of(s.t);
    if (threadIdx.x == 0) d.stop = s.k;
    __syncthreads();
    for (int j = wv; j <= s.k; j += kThreads / 64) {
        const double2 *st = a.stats + static_cast<size_t>(s.row0 + j) * a.chunks;
        // The draft's own logit and probability are on their way while the statistics come together.
        int x = -1;
        float l = -INFINITY, q = 1.0f, u = 0.0f;
        if (lane == 0 && j < s.k) {
            x = a.draft[s.draft0 + j];
            u = a.u[2 * static_cast<size_t>(s.row0 + j)];
            if (x >= 0 && x < a.vocab) {
                l = logit(a.logits[static_cast<size_t>(s.row0 + j) * a.vocab + x]);
                if (a.probs) q = a.probs[static_cast<size_t>(s.draft0 + j) * a.vocab + x];
            } else {
                x = -1;
            }
        }
        // Up to kHeld of the lane's statistics stay in registers between the two passes over them.
        constexpr int kHeld = 4;
        double2 held[kHeld];
        double m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            held[i] = lane + 64 * i < a.chunks ? st[lane + 64 * i] : double2{-INFINITY, greedy ? static_cast<double>(INT_MAX) : 0.0};
            m = fmax(m, held[i].x);
        }
        for (int c = lane + 64 * kHeld; c < a.chunks; c += 64) m = fmax(m, st[c].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o, 64));
        double z = greedy ? static_cast<double>(INT_MAX) : 0.0;
        auto add = [&](const double2 &v) {
            if (!greedy) z += v.y * weight(v.x, m, per);
            else if (v.x == m) z = fmin(z, v.y);
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) add(held[i]);
        for (int c = lane + 64 * kHeld; c < a.chunks; c += 64) add(st[c]);
        if (greedy) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) z = fmin(z, __shfl_xor(z, o, 64));
        } else {
            z = wave_sum(z);
        }
        if (lane == 0) {
            d.m[j] = m;
            d.z[j] = z;
            const double given = q > 0.0f ? q : 0.0;
            const bool ok = greedy ? static_cast<double>(x) == z : z > 0.0 && static_cast<double>(u) * given * z < weight(l, m, per);
            if (j < s.k && (x < 0 || !ok)) atomicMin(&d.stop, j);
        }
    }
    __syncthreads();
}

// Weights that the token after row j's accepted drafts is drawn with: the target's, or where a draft was refused what it has over
// the draft's probabilities (a draft without probabilities: over all of the mass at the drafted token).
struct Source {
    const float *l, *q;  // q null: no draft's probabilities are taken off
    int without;         // a token left out
    double m, per, inv_z;
    __device__ __forceinline__ void each(int i, int n, double (&w)[kEach]) const {
        float x[kEach], y[kEach];
        load_each(l, i, n, -INFINITY, x);
        if (q) load_each(q, i, n, 0.0f, y);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const double p = weight(logit(x[e]), m, per) * inv_z;
            w[e] = p;
            if (q) w[e] = fmax(p - (y[e] > 0.0f ? static_cast<double>(y[e]) : 0.0), 0.0);
            if (i + e >= n || i + e == without) w[e] = 0.0;
        }
    }
};
__device__ __forceinline__ Source source_of(const VerArgs &a, const VerSeq &s, const Decision &d, bool refused) {
    const int j = d.stop;
    Source r{a.logits + static_cast<size_t>(s.row0 + j) * a.vocab, nullptr, -1, d.m[j], per_of(s.t), 1.0 / d.z[j]};
    if (refused) {
        if (a.probs) r.q = a.probs + static_cast<size_t>(s.draft0 + j) * a.vocab;
        else r.without = a.draft[s.draft0 + j];
    }
    return r;
}

// Workgroup (chunk, sequence): the chunk's sum of what is left over where a draft was refused.
__global__ __launch_bounds__(kThreads) void verify_residual_kernel(VerArgs a, VerTable T) {
    __shared__ Decision d;
    __shared__ double ssum[4];
    const VerSeq s = T.s[blockIdx.y];
    if (s.k == 0 || s.t == 0.0) return;
    decide(a, s, d);
    if (d.stop == s.k || !(d.z[d.stop] > 0.0)) return;
    double w[kEach], sum = 0.0;
    source_of(a, s, d, true).each(blockIdx.x * kChunk + threadIdx.x * kEach, a.vocab, w);
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum += w[e];
    sum = group_sum(sum, ssum);
    if (threadIdx.x == 0) a.residual[static_cast<size_t>(blockIdx.y) * a.chunks + blockIdx.x] = sum;
}

// One workgroup per sequence: the token, and what the rows give.
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerArgs a, VerTable T) {
    __shared__ Decision d;
    __shared__ double scan[4], base, total;
    __shared__ int2 span[4];
    __shared__ int token;
    const VerSeq s = T.s[blockIdx.x];
    const int tid = threadIdx.x;
    decide(a, s, d);
    const int j = d.stop;
    const bool greedy = s.t == 0.0, some = greedy ? d.z[j] < INT_MAX : d.z[j] > 0.0;
    const double inv_t = greedy ? 0.0 : 1.0 / s.t;
    if (tid == 0) token = greedy && some ? static_cast<int>(d.z[j]) : INT_MAX;
    if (!greedy && some) {
        const double2 *st = a.stats + static_cast<size_t>(s.row0 + j) * a.chunks;
        const double *left = a.residual + static_cast<size_t>(blockIdx.x) * a.chunks;
        const double v = a.u[2 * static_cast<size_t>(s.row0 + j) + 1], inv_z = 1.0 / d.z[j];
        const int per = (a.chunks + kThreads - 1) / kThreads, c0 = tid * per, c1 = min(c0 + per, a.chunks);
        bool refused = j < s.k;
        auto of_chunk = [&](int c) { return refused ? left[c] : st[c].y * weight(st[c].x, d.m[j], per_of(s.t)) * inv_z; };
        for (;;) {
            double mine = 0.0;
            for (int c = c0; c < c1; ++c) mine += of_chunk(c);
            const double upto = group_scan(mine, scan);
            if (tid == kThreads - 1) total = upto;
            __syncthreads();
            if (refused && !(total > 0.0)) {  // nothing is left over (p = q): from the target's own weights
                refused = false;
                __syncthreads();
                continue;
            }
            // The first chunk whose cumulative sum exceeds the target, else the last with any weight. One without weight is never
            // taken: a thread's `before` is the scan less its own share, which may round past the target where the thread before
            // ended at it.
            const double target = v * total;
            double before = upto - mine, mine_base = 0.0;
            int found = INT_MAX, some_at = -1;
            for (int c = c0; c < c1; ++c) {
                const double w = of_chunk(c);
                if (w > 0.0) some_at = c;
                if (w > 0.0 && before + w > target) {
                    found = c, mine_base = before;
                    break;
                }
                before += w;
            }
            const int2 at = group_span(found, some_at, span);
            const bool none = at.x == INT_MAX;
            const int chunk = none ? at.y : at.x;
            if (found == chunk) base = mine_base;
            __syncthreads();
            // The same among the chunk's elements.
            double w[kEach], in = 0.0;
            const int e0 = chunk * kChunk + tid * kEach;
            source_of(a, s, d, refused).each(e0, a.vocab, w);
#pragma unroll
            for (int e = 0; e < kEach; ++e) in += w[e];
            before = base + (group_scan(in, scan) - in);
            found = INT_MAX, some_at = -1;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (w[e] > 0.0) some_at = e0 + e;
                before += w[e];
                if (w[e] > 0.0 && before > target && found == INT_MAX) found = e0 + e;
            }
            const int2 el = group_span(found, some_at, span);
            if (tid == 0) token = !none && el.x != INT_MAX ? el.x : el.y >= 0 ? el.y : chunk * kChunk;
            break;
        }
    }
    __syncthreads();
    for (int r = tid; r <= s.k; r += kThreads) {
        const size_t row = static_cast<size_t>(s.row0) + r;
        const int x = r < j ? a.draft[s.draft0 + r] : r == j ? token : -1;
        a.tokens[row] = x;
        if (!a.logprobs) continue;
        float lp = 0.0f;
        if (r == j && !some) lp = -INFINITY;
        else if (r <= j && !greedy) {
            const float l = logit(a.logits[row * a.vocab + x]);
            lp = static_cast<float>((l == d.m[r] ? 0.0 : (l - d.m[r]) * inv_t) - log(d.z[r]));
        }
        a.logprobs[row] = lp;
    }
    if (tid == 0) a.counts[blockIdx.x] = j;
}

int make_pass(int vocab, const int32_t *drafted, const double *temperature, int nseq, VerTable &T, int &rows, int &drafts) {
    if (!drafted || nseq < 1 || nseq > VQ_MAX_SEGMENTS) return VQ_ERR_ARG;
    if (vocab < 1 || vocab > INT_MAX - 2 * kChunk) return VQ_ERR_SHAPE;
    T.n = nseq;
    rows = drafts = 0;
    for (int i = 0; i < nseq; ++i) {
        const double t = temperature ? temperature[i] : 1.0;
        if (drafted[i] < 0 || drafted[i] > VQ_MAX_DRAFT || !(t >= 0.0 && t < INFINITY)) return VQ_ERR_SHAPE;
        T.s[i] = VerSeq{rows, drafted[i], drafts, t};
        rows += drafted[i] + 1;
        drafts += drafted[i];
    }
    return VQ_OK;
}
size_t chunks_of(int vocab) { return (static_cast<size_t>(vocab) + kChunk - 1) / kChunk; }

}  // namespace

extern "C" {

size_t vq_verify_draft_workspace_bytes(int vocab, const int32_t *drafted, int nseq) {
    VerTable T;
    int rows, drafts;
    if (make_pass(vocab, drafted, nullptr, nseq, T, rows, drafts) != VQ_OK) return 0;
    return chunks_of(vocab) * (sizeof(double2) * rows + sizeof(double) * nseq);
}

int vq_verify_draft(const float *logits, const int32_t *draft, const float *probs, const float *u, int32_t *tokens, int32_t *counts,
                    float *logprobs, int vocab, const int32_t *drafted, const double *temperature, int nseq, void *workspace,
                    size_t workspace_bytes, void *stream) {
    if (!logits || !u || !tokens || !counts || !temperature) return VQ_ERR_ARG;
    VerTable T;
    int rows, drafts;
    if (const int st = make_pass(vocab, drafted, temperature, nseq, T, rows, drafts); st != VQ_OK) return st;
    if (drafts > 0 && !draft) return VQ_ERR_ARG;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < vq_verify_draft_workspace_bytes(vocab, drafted, nseq))
        return VQ_ERR_WORKSPACE;
    const size_t chunks = chunks_of(vocab);
    VerArgs a{logits, probs, u, draft, tokens, counts, logprobs, static_cast<double2 *>(workspace), nullptr, vocab,
              static_cast<int>(chunks)};
    a.residual = reinterpret_cast<double *>(a.stats + chunks * rows);
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool refusable = false;
    int most = 0;
    for (int i = 0; i < nseq; ++i) {
        refusable = refusable || (T.s[i].k > 0 && T.s[i].t > 0.0);
        most = T.s[i].k > most ? T.s[i].k : most;
    }
    verify_stats_kernel<<<dim3(chunks, most + 1, nseq), kThreads, 0, s>>>(a, T);
    if (refusable) verify_residual_kernel<<<dim3(chunks, nseq), kThreads, 0, s>>>(a, T);
    verify_pick_kernel<<<nseq, kThreads, 0, s>>>(a, T);
    return status_of(hipGetLastError());
}

}  // extern "C"
