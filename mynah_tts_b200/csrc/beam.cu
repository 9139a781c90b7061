// Beam search over a batch of requests: the selection of the best continuations of a
// request's beams, and the reordering of the beams' K/V rows that follows it.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "launch.h"

namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------- selection
//
// For beam b with cumulative log-probability s_b and logits x_b over the allowed tokens A
// (t < codebook_size, and eos_id where it is allowed) a continuation scores
//     c(b, t) = s_b + x_bt - lse_b,      lse_b = log sum_{t in A} exp(x_bt),
// and a finished beam has the one continuation (eos_id, s_b).  A request keeps its `beams`
// best, in the order (score, lower beam, higher logit, lower token).
//
// Bound by reading the logits once.  A request is one thread-block cluster, so it is one
// launch without scratch memory: the rows, or equal parts of them when there are few, are
// dealt to the CTAs, each keeps the running maximum and sum of its row and
// finds the row's best `beams` tokens, and the cluster's first CTA, into whose shared memory
// all results are stored, takes the best of at most 16 falling lists of 16.
//
// Best tokens of a part without sorting it: each of 32 groups of threads knows the largest
// logit it has seen; the K-th largest of these group maxima is a lower bound of the K-th
// largest logit, and only a few more than K tokens reach it.  They are listed as they pass.
// The bound is drawn again with 1, 2, 4, ... turns of the part seen, so about K log2(turns) tokens
// are listed in all.  A list that is full all the same (thousands of equal logits, or logits
// that rise along the vocabulary) is replaced by one pass over the part per place.
//
// The order is that of scores in 64 bits, equal ones by beam: beams differ by less than a rounding
// of a 32-bit sum often enough to change a pick.  A 64-bit exponential per logit would bind the
// kernel by its arithmetic, so a log-sum is formed of 32-bit terms, summed in 32 bits by a thread (see
// SEL_FOLD) and in 64 across them, and is off by at most sel_eps; and where a continuation
// that is picked lies within twice that of another beam's, the log-sums of those beams are formed
// again in 64 bits, in an order that goes by the tokens alone (equal rows give equal sums wherever
// they lie), and the picks are made again.  Beams farther apart than that cannot change places: a pair
// that does has been a pick and a list's head.

constexpr int SEL_CLUSTER = 8;     // portable cluster size
constexpr int SEL_SHARE = 4;       // parts of one CTA, at most
constexpr int SEL_THREADS = 512, SEL_FIT_THREADS = 256;
constexpr int SEL_HELD = 4;        // 16-byte pieces a thread takes in a turn, and holds of a short part (FIT)
constexpr int SEL_CAP = 512;       // tokens listed of a part
constexpr float SEL_SLACK = 8.0f;  // what a logit may be above its thread's base
constexpr int SEL_FOLD = 32;       // turns that a thread sums in 32 bits, or half of all
constexpr int SEL_PAD = MB_BEAM_MAX + 1;         // lists that lanes walk side by side: no common bank
constexpr int SEL_LIST = MB_BEAM_MAX * SEL_PAD;

// Long parts go through a ring in shared memory in which a thread fills and reads only its own
// places, so the copies need no barrier: SEL_DEPTH turns of SEL_HELD pieces are under way, across
// the parts of a CTA, 64 KB per CTA and two CTAs per SM.  24 requests x 16 beams x 50,000, 76.8 MB:
// loads into registers with a wait for each turn 87 us, this 30 (2.6 TB/s).  What bounds it is that
// the clusters' CTAs come in pairs on 96 of 148 SMs, each with two rows to walk one after the other
// (64 requests reach 3.7 TB/s).
constexpr int SEL_DEPTH = 2;
constexpr unsigned SEL_RING_BYTES = SEL_DEPTH * SEL_HELD * SEL_THREADS * sizeof(float4);

struct SelPart {                   // what one part of a row found
    float top;                     // maximum, -inf if no token
    float pad;
    double sum;                    // sum of exp(x - top)
    double lse;                    // top + log(sum)
    unsigned long long key[MB_BEAM_MAX];
};

struct SelScratch {                // of one part while it is worked on
    float group[32], bound;
    double wsum[SEL_THREADS / 32];
    float wtop[SEL_THREADS / 32];
    unsigned n_reach;
    unsigned long long reach[SEL_CAP], wkey[SEL_THREADS / 32];
};

struct SelSmem {
    SelPart part[MB_BEAM_MAX];     // first CTA: all parts of the request
    SelScratch work[SEL_SHARE];
    union {
        struct {                   // first CTA, at the end: the continuations of the request
            double score[SEL_LIST];
            unsigned long long order[SEL_LIST], key[SEL_LIST];
            unsigned near[SEL_LIST];       // first bits of the order of what is 2 sel_eps above the continuation
        };
        struct {                   // before: sums of turns, per thread, and their bases
            double folded[SEL_THREADS];
            float folded_base[SEL_THREADS];
        };
    };
    int taken[MB_BEAM_MAX];
    unsigned close;                // not 0: a pick may have come close to another beam's continuation
    unsigned close_beams;          // those that did
};

// Order-preserving bits of a float.
__device__ __forceinline__ unsigned sel_bits(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// Key of a logit and its token: larger logit first, then the lower token; -0 and +0 are equal.
// 0 is no key: NaN and -inf are not candidates.
__device__ __forceinline__ unsigned long long sel_key(float x, unsigned token) {
    return ((unsigned long long)sel_bits(x + 0.0f) << 32) | (0xffffffffu - token);
}
__device__ __forceinline__ float sel_logit(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned sel_token(unsigned long long key) { return 0xffffffffu - (unsigned)key; }

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// Tokens first .. last - 1 of a row as 16-byte pieces; piece v holds tokens origin + 4 v ...
struct SelRange {
    const float *row;
    const float4 *base;            // piece 0, 16-byte aligned
    int first, last, origin;
    int vecs;                      // pieces that hold the range
    int whole_from, whole_to;      // pieces that lie inside it
};

__device__ __forceinline__ SelRange sel_range(const float *row, int first, int last) {
    SelRange r;
    r.row = row;
    r.first = first;
    r.last = last;
    const int shift = (int)((reinterpret_cast<uintptr_t>(row + first) & 15u) >> 2);
    r.origin = first - shift;
    r.base = reinterpret_cast<const float4 *>(row + r.origin);
    r.vecs = last > first ? (last - r.origin + 3) >> 2 : 0;
    r.whole_from = min(r.vecs, shift ? 1 : 0);
    r.whole_to = max(r.whole_from, last > first ? (last - r.origin) >> 2 : 0);
    return r;
}
__device__ __forceinline__ float drop_nan(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ float4 drop_nan(const float4 &x) {
    return make_float4(drop_nan(x.x), drop_nan(x.y), drop_nan(x.z), drop_nan(x.w));
}
__device__ __forceinline__ float4 no_tokens() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }

// The four logits of piece v; tokens outside the range read as -inf and are not touched.
__device__ __forceinline__ float4 sel_load(const SelRange &r, int v) {
    if (v >= r.whole_from && v < r.whole_to) return r.base[v];
    const int t = r.origin + 4 * v;
    float4 x;
    x.x = t >= r.first && t < r.last ? r.row[t] : -INFINITY;
    x.y = t + 1 >= r.first && t + 1 < r.last ? r.row[t + 1] : -INFINITY;
    x.z = t + 2 >= r.first && t + 2 < r.last ? r.row[t + 2] : -INFINITY;
    x.w = t + 3 >= r.first && t + 3 < r.last ? r.row[t + 3] : -INFINITY;
    return x;
}

// exp(x - top) for x below top, or no more than SEL_SLACK above it
__device__ __forceinline__ float sel_exp(float x, float top) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__fmul_rn(__fsub_rn(x, top), 1.4426950408889634f)));
    return y;
}

// exp(x - top), 1 for nothing on both sides
__device__ __forceinline__ float sel_scale(float x, float top) { return x == top ? 1.0f : sel_exp(x, top); }

// log(s) for a positive normal s, to 1e-11: with s = 2^e f and c near 1 / f in steps of 1/256
// (64 intervals of f, Tang's table method), log s = e log 2 - log c + log(1 + r), r = f c - 1, |r| <
// 0.013.  r is formed in 64 bits; of log(1 + r) = r - r^2/2 + ... the rest is, in 32 bits, off by 9e-12.  CUDA's
// 64-bit log took 1.7 us here, which the whole cluster waits for; this takes a tenth.
__constant__ double sel_log_c[64] = {      // -log(c), c = round(256 / (1 + (i + 0.5) / 64)) / 256
    0.007843177461025893, 0.023716526617316044, 0.039845908547199674, 0.05211600113901402,
    0.06871389254805181, 0.0813456394539524, 0.09844007281325252, 0.11145544092532282,
    0.1246424452072766, 0.13800567301944372, 0.15154989812720093, 0.16528009093910292,
    0.179201429457711, 0.19331931100349597, 0.20284319251475147, 0.2173012756899814,
    0.22705745063534608, 0.24187253642048673, 0.2518726197550701, 0.26706278524904525,
    0.27731928541623435, 0.2876820724517809, 0.3034304294199201, 0.31406882762497584,
    0.32482161940123766, 0.33569129163814154, 0.3466804132137367, 0.3577916386388075,
    0.36902771190573336, 0.38039147055604844, 0.39188584998178355, 0.39768296766610944,
    0.4093790074293007, 0.42121346507630353, 0.43318965612301924, 0.4392319705789819,
    0.4514272436728001, 0.4637730794950995, 0.4700036292457356, 0.48258241145259567,
    0.4889316391312544, 0.5017523275603158, 0.5082248420659333, 0.5212969236332861,
    0.5278976076646381, 0.5345421503833068, 0.5479651707154474, 0.5547448577008262,
    0.561570822771226, 0.5753641449035618, 0.5823328142196552, 0.5893503868783018,
    0.5964175541013942, 0.6107035113488707, 0.6179237593223578, 0.6251965186514375,
    0.6325225587435105, 0.639902666041133, 0.6473376445286511, 0.6548283162578087,
    0.6623755218931916, 0.6699801212784109, 0.6776429940239801, 0.6853650401178903,
};
__device__ __forceinline__ double sel_log(double s) {
    const long long bits = __double_as_longlong(s);
    const int e = (int)(bits >> 52) - 1023, i = (int)(bits >> 46) & 63;
    const double f = __longlong_as_double((bits & 0x000fffffffffffffll) | 0x3ff0000000000000ll);
    // round(256 / (1 + (i + 0.5) / 64)) = floor((32768 + (2 i + 129) / 2) / (2 i + 129)), no ties
    const int d = 2 * i + 129, c256 = (32768 + (d >> 1)) / d;
    const double r = fma(f, (double)c256 * 0.00390625, -1.0);
    const float q = (float)r;
    const float t = q * q * fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.0f / 6.0f, 0.2f), -0.25f), 1.0f / 3.0f), -0.5f);
    return fma((double)e, 0.6931471805599453, sel_log_c[i]) + (r + (double)t);
}

struct SelP {
    const float *logits;
    size_t logits_stride;
    int requests, beams, parts, codebook, eos, has_eos;
    double near;                   // 2 sel_eps
    const int *allow_eos;
    const float *score;
    const unsigned *done, *live;
    float *score_out;
    unsigned *token, *parent, *done_out;
};

__device__ __forceinline__ void copy_async(float4 *to, const float4 *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// The tokens a thread has seen: their maximum `top` and the sum of exp(x - base).  `base` follows the
// maximum in steps above SEL_SLACK only, so a term is scaled to another base once per SEL_SLACK that it
// lies below the maximum, at most.  NaN is passed over by the maximum and shows in the sum.  `most`
// receives the pieces' maxima.  Returns what sums formed before have to be scaled by.
struct SelSeen { float top, base, sum; };
__device__ __forceinline__ SelSeen sel_none() { return SelSeen{-INFINITY, -INFINITY, 0.0f}; }

template <int N>
__device__ __forceinline__ float sel_take(const float4 (&x)[N], float (&most)[N], SelSeen &s) {
    float scaled = 1.0f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        most[u] = fmaxf(fmaxf(x[u].x, x[u].y), fmaxf(x[u].z, x[u].w));
        s.top = fmaxf(s.top, most[u]);
    }
    if (s.top > s.base + SEL_SLACK) {
        scaled = sel_exp(s.base, s.top);
        s.sum = __fmul_rn(s.sum, scaled);
        s.base = s.top;
    }
    const float ref = s.base == -INFINITY ? 0.0f : s.base;
    float part = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u)
        part += (sel_exp(x[u].x, ref) + sel_exp(x[u].y, ref)) + (sel_exp(x[u].z, ref) + sel_exp(x[u].w, ref));
    s.sum += part;
    return scaled;
}

// How far a log-sum may be off.  With u = 2^-24, per term relative to itself: the difference to a
// base or maximum, its product with log2 e and that constant are off by 2.25 u times the difference,
// ex2.approx by 4 u.  A term's factors (to its thread's base, the warp's maximum, the part's, the
// row's) are four such steps, whose differences add up to the term's distance from the row's maximum
// and twice SEL_SLACK, and 5 u for each change of the base; weighted by the terms the distance is at
// most the entropy, log(tokens).  The 32-bit sums of a turn are 7 deep, those of turns 2 more than
// there are.  Up to 2^18 tokens 2^-16.8 in all.
double sel_eps(size_t tokens) {
    const double distance = log((double)tokens + 1.0), half = (double)(tokens / (8u * SEL_HELD * SEL_THREADS)) + 1.0;
    return (2.25 * (distance + 2.0 * SEL_SLACK) + 16.0 + 5.0 * (distance / SEL_SLACK + 1.0) + 9.0 + fmin(2.0 * half, fmax(half, SEL_FOLD))) / 16777216.0;
}

// Order-preserving bits of a score, 0 for none (NaN and -inf among them).
__device__ __forceinline__ unsigned long long sel_order(double c) {
    const long long bits = __double_as_longlong(c + 0.0);
    return c > -INFINITY ? (unsigned long long)(bits < 0 ? ~bits : bits | (1ll << 63)) : 0ull;
}

// The keys of the tokens that reach the bound into the list: `most` are the pieces' maxima, piece
// u begins with token[u].
template <int N>
__device__ __forceinline__ void sel_reach(SelScratch &w, const float4 (&x)[N], const float (&most)[N], const unsigned (&token)[N],
                                          float bound) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
        if (!(most[u] >= bound)) continue;                 // nearly every piece
        const float e[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(e[j] >= bound) || e[j] == -INFINITY) continue;
            const unsigned at = atomicAdd(&w.n_reach, 1u);
            if (at < SEL_CAP) w.reach[at] = sel_key(e[j], token[u] + j);
        }
    }
}

// The bound of a part from the largest logit each thread has seen: the beams-th largest of 32
// group maxima, -inf when fewer groups have seen a token.  All threads of the CTA.
template <int NTHREADS>
__device__ __forceinline__ float sel_bound(SelScratch &w, float top, int beams) {
    constexpr int GROUP = NTHREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31;
#pragma unroll
    for (int o = GROUP >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(MB_FULL, top, o));
    if (tid % GROUP == 0) w.group[tid / GROUP] = top;
    __syncthreads();
    if (tid < 32) {
        const float mine = w.group[lane];
        int reach = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) reach += w.group[j] >= mine;
        // largest value that at least `beams` groups reach
        const unsigned best = __reduce_max_sync(MB_FULL, reach >= beams ? sel_bits(mine) : 0u);
        if (lane == 0) w.bound = sel_logit((unsigned long long)best << 32);
    }
    __syncthreads();
    return w.bound;
}

// Continuation threadIdx.x of the request, at most 16 x 16, of beam b: its score as an ordered integer.
__device__ __forceinline__ void sel_score(SelSmem &sm, int beams, int parts, int b, unsigned done, int eos, float score, double near) {
    const int part = threadIdx.x / beams, k = threadIdx.x - part * beams, to = part * SEL_PAD + k;
    unsigned long long key;
    double c;
    if (done >> b & 1u) {
        key = part == b * parts && k == 0 ? sel_key(0.0f, (unsigned)eos) : 0ull;
        c = score;
    } else {
        key = sm.part[part].key[k];
        c = (double)score + ((double)sel_logit(key) - sm.part[b * parts].lse);
    }
    sm.key[to] = key;
    sm.score[to] = c;
    sm.order[to] = key != 0ull ? sel_order(c) : 0ull;
    sm.near[to] = key != 0ull ? (unsigned)(sel_order(c + near) >> 32) : 0u;
}

// The lists fall, so the best continuation left is the best of their heads: one warp takes `beams`
// of them, a list per lane, and returns how many there are.  `close`: with LOOK the beams that come
// within `near` of a pick of another one, else the lanes whose list's head may.
template <bool LOOK>
__device__ __forceinline__ int sel_merge(SelSmem &sm, int beams, int parts, double near, unsigned &close) {
    const int lane = threadIdx.x, lists = beams * parts, last = lane * SEL_PAD + beams;    // behind a list lies a 0
    int at = lane * SEL_PAD, found = 0;
    unsigned long long head = lane < lists ? sm.order[at] : 0ull, next = lane < lists ? sm.order[at + 1] : 0ull;
    unsigned head_near = lane < lists ? sm.near[at] : 0u, next_near = lane < lists ? sm.near[at + 1] : 0u;
    bool beside = false;
    close = 0u;
    for (; found < beams; ++found) {
        const unsigned high = __reduce_max_sync(MB_FULL, (unsigned)(head >> 32));
        if (high == 0u) break;                         // nothing is left (an order's first bits are not 0)
        unsigned best = __ballot_sync(MB_FULL, (unsigned)(head >> 32) == high);
        if (best & (best - 1)) {
            const bool first = (unsigned)(head >> 32) == high;
            const unsigned low = __reduce_max_sync(MB_FULL, first ? (unsigned)head : 0u);
            best = __ballot_sync(MB_FULL, first && (unsigned)head == low);
            // equal scores: the lower beam, which is the lower list; parts of one beam by their keys
            int winner = __ffs(best) - 1;
            for (unsigned more = best & (best - 1); parts > 1 && more != 0u; more &= more - 1) {
                const int other = __ffs(more) - 1;
                const unsigned long long a = sm.key[__shfl_sync(MB_FULL, at, winner)], o = sm.key[__shfl_sync(MB_FULL, at, other)];
                if (other / parts == winner / parts && o > a) winner = other;
            }
            best = 1u << winner;
        }
        const bool won = best >> lane & 1u;
        if (LOOK) {
            const double least = sm.score[__shfl_sync(MB_FULL, at, __ffs(best) - 1)] - near;
            const unsigned who = __reduce_or_sync(MB_FULL, head != 0ull && sm.score[at] >= least ? 1u << (lane / parts) : 0u);
            if (who & (who - 1)) close |= who;
        } else {
            beside = beside || (!won && head_near >= high);
        }
        if (won) sm.taken[found] = at;
        head = won ? next : head;
        head_near = won ? next_near : head_near;
        at += won;
        next = sm.order[lane < lists ? min(at + 1, last) : 0];
        next_near = sm.near[lane < lists ? min(at + 1, last) : 0];
    }
    __syncwarp();
    if (!LOOK) close = __ballot_sync(MB_FULL, beside);
    return found;
}

// exp(d) for -700 <= d <= 0 in 64 bits, to 1e-15: with d = (64 k + j) log(2) / 64 + r, |r| < 0.0055, it is
// 2^k 2^(j/64) e^r (Tang's table method), e^r - 1 by its series to r^5.  `table` holds 2^(j/64).
constexpr int SEL_POWERS = 64;
__device__ __forceinline__ double sel_exp64(double d, const double *table) {
    constexpr double ROUND = 6755399441055744.0;       // 3 * 2^51: the sum's last bits are the rounded product
    const double t = fma(d, SEL_POWERS / 0.6931471805599453, ROUND), r = fma(t - ROUND, -0.6931471805599453 / SEL_POWERS, d);
    const int n = __double2loint(t);
    const double e = r * fma(r, fma(r, fma(r, fma(r, 1.0 / 120.0, 1.0 / 24.0), 1.0 / 6.0), 0.5), 1.0);
    const double power = table[n & (SEL_POWERS - 1)], y = fma(power, e, power);
    return __hiloint2double(__double2hiint(y) + (n >> 6 << 20), __double2loint(y));
}

struct SelRow { const float *row; size_t stride; int codebook, eos; bool allow; };

// Some pick may have come close to another beam's continuation: the log-sums of the beams that did, in
// 64 bits.  Tokens go to threads by their index, so a sum depends on the logits alone.  All threads of
// the CTA; false where none came close after all.  Bound by its 64-bit arithmetic: two rows of 2,016
// add 6 us to the call, of 50,000 33 us, sixteen 230.  With normal logits one call in 60 of 64
// requests x 8 beams x 2,016 has such a pair, and one in 20 of 24 x 16 x 50,000.
template <int NTHREADS>
__device__ __noinline__ bool sel_refine(SelSmem &sm, int beams, int parts, unsigned done, double near, SelRow q) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int SEL_BATCH = 8;
    double *wsum = sm.work[0].wsum, *table = reinterpret_cast<double *>(sm.work[0].reach);
    if (tid >= NTHREADS - SEL_POWERS) table[tid - (NTHREADS - SEL_POWERS)] = exp2((double)(tid - (NTHREADS - SEL_POWERS)) / SEL_POWERS);
    if (warp == 0) {
        unsigned close;
        sel_merge<true>(sm, beams, parts, near, close);
        if (lane == 0) sm.close_beams = close;
    }
    __syncthreads();
    const unsigned close = sm.close_beams;
    for (int b = 0; b < beams; ++b) {
        if (!((close & ~done) >> b & 1u)) continue;
        const float *row = q.row + (size_t)b * q.stride;
        SelPart *of = sm.part + b * parts;
        float m = -INFINITY;
        for (int j = 0; j < parts; ++j) m = fmaxf(m, of[j].top);
        double sum = 0.0;
        const auto take = [&](float x) {               // NaN and what is below 1e-300 add nothing
            const double d = (double)x - (double)m;
            sum += d > -690.0 ? sel_exp64(d, table) : 0.0;
        };
        if (tid == 0 && q.allow) take(row[q.eos]);
        for (int t0 = tid; t0 < q.codebook; t0 += SEL_BATCH * NTHREADS) {
            float x[SEL_BATCH];
#pragma unroll
            for (int u = 0; u < SEL_BATCH; ++u) x[u] = t0 + u * NTHREADS < q.codebook ? row[t0 + u * NTHREADS] : -INFINITY;
#pragma unroll
            for (int u = 0; u < SEL_BATCH; ++u) take(x[u]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(MB_FULL, sum, o);
        __syncthreads();                               // the sums before are read
        if (lane == 0) wsum[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < NTHREADS / 32; ++w) sum += wsum[w];
            of->lse = (double)m + log(sum);
        }
    }
    __syncthreads();
    return close != 0u;
}

// FIT: parts of at most SEL_HELD pieces per thread.
template <bool FIT>
__global__ void __launch_bounds__(FIT ? SEL_FIT_THREADS : SEL_THREADS, FIT ? 4 : 2) k_beam_select(SelP p) {
    __shared__ SelSmem sm;
    extern __shared__ float4 ring[];
    constexpr int NT = FIT ? SEL_FIT_THREADS : SEL_THREADS, WARPS = NT / 32;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();
    mb_pdl_wait();
    mb_pdl_trigger();
    const int rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
    const int request = blockIdx.x / size;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, beams = p.beams, parts = p.parts;
    const unsigned live = p.live != nullptr ? *p.live : 0xffffffffu;
    // what the first CTA needs at the end is on its way from here on
    const int n = beams * parts * beams, mine = tid < n ? tid / (parts * beams) : 0;
    const float score = p.score[request * beams + mine];
    const unsigned done = __ballot_sync(MB_FULL, p.done != nullptr && lane < beams && p.done[request * beams + lane] != 0);
    const bool allow = p.has_eos && (p.allow_eos == nullptr || p.allow_eos[request] != 0);
    if ((unsigned)request >= live) {   // the whole cluster
        cluster.barrier_wait();
        return;
    }
    if (tid < SEL_SHARE) sm.work[tid].n_reach = 0;

    const int per = (p.codebook + parts - 1) / parts;
    auto range = [&](int i) {          // of part i of the request
        const int b = i / parts, from = min((i - b * parts) * per, p.codebook);
        return sel_range(p.logits + (size_t)(request * beams + b) * p.logits_stride, from, min(from + per, p.codebook));
    };
    auto has = [&](int i) { return i < beams * parts && !(done >> (i / parts) & 1u); };
    auto has_eos = [&](int i) { return allow && tid == 0 && (i + 1) % parts == 0; };

    // what the ring is asked for next: turn f_turn of part f_part
    constexpr int TURN = SEL_HELD * NT;
    int f_part = rank, f_left = 0, f_place = 0;            // f_left: pieces of the part not yet asked for
    const float4 *f_from = nullptr;
    auto feed = [&]() {                                    // at the first part from f_part on that has pieces
        for (f_left = 0; f_part < beams * parts; f_part += size) {
            if (!has(f_part)) continue;
            const SelRange r = range(f_part);
            f_left = r.whole_to - r.whole_from;
            f_from = r.base + r.whole_from + tid;
            if (f_left > 0) return;
        }
    };
    auto ask = [&]() {
        if (f_left > 0) {
            float4 *to = ring + f_place * TURN + tid;
            if (f_left >= TURN) {
#pragma unroll
                for (int u = 0; u < SEL_HELD; ++u) copy_async(to + u * NT, f_from + u * NT);
            } else {
#pragma unroll
                for (int u = 0; u < SEL_HELD; ++u)
                    if (tid + u * NT < f_left) copy_async(to + u * NT, f_from + u * NT);
            }
            f_from += TURN;
            f_left -= TURN;
            if (f_left <= 0) {
                f_part += size;
                feed();
            }
        }
        f_place = f_place + 1 == SEL_DEPTH ? 0 : f_place + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (!FIT) {
        feed();
#pragma unroll 1
        for (int i = 0; i < SEL_DEPTH; ++i) ask();
    }

    // this CTA's parts: rank, rank + size, ... of the request's
    for (int i = rank, q = 0; i < beams * parts; i += size, ++q) {
        if (!has(i)) continue;
        SelScratch &w = sm.work[q];
        const SelRange r = range(i);
        // what lies beside the whole pieces: a ragged first or last one, which falls to one thread,
        // and the token behind the range
        const int edge = tid == 0 && r.whole_from > 0 ? 0 : tid == NT - 1 && r.whole_to < r.vecs ? r.vecs - 1 : -1;
        float4 beside[2] = {no_tokens(), no_tokens()};
        if (edge >= 0) beside[0] = drop_nan(sel_load(r, edge));
        if (has_eos(i)) beside[1].x = drop_nan(r.row[p.eos]);
        const int whole = r.whole_to - r.whole_from;
        const float4 *at = r.base + r.whole_from + tid;            // this thread's next piece
        unsigned token = (unsigned)(r.origin + 4 * (r.whole_from + tid));
        float4 x[SEL_HELD];
        float most[SEL_HELD], beside_most[2], bound;
        SelSeen seen = sel_none();
        if (FIT) {
#pragma unroll
            for (int u = 0; u < SEL_HELD; ++u) {
                x[u] = no_tokens();
                if (tid + u * NT < whole) x[u] = at[u * NT];
            }
            sel_take(x, most, seen);
            sel_take(beside, beside_most, seen);
            bound = sel_bound<NT>(w, seen.top, beams);
            const unsigned tokens[SEL_HELD] = {token, token + 4 * NT, token + 8 * NT, token + 12 * NT};
            sel_reach(w, x, most, tokens, bound);
        } else {
            sel_take(beside, beside_most, seen);
            bound = INFINITY;
            for (int turn = 0, left = whole; left > 0; ++turn, left -= TURN, token += 4 * TURN) {
                asm volatile("cp.async.wait_group %0;" ::"n"(SEL_DEPTH - 1) : "memory");
                const float4 *place = ring + f_place * TURN + tid;         // the one that is asked for next
#pragma unroll
                for (int u = 0; u < SEL_HELD; ++u) x[u] = place[u * NT];
                if (left < TURN)
#pragma unroll
                    for (int u = 0; u < SEL_HELD; ++u)
                        if (tid + u * NT >= left) x[u] = no_tokens();
                ask();
                sel_take(x, most, seen);
                if ((turn & (turn + 1)) == 0) {
                    bound = sel_bound<NT>(w, seen.top, beams);
                    if (turn >= SEL_FOLD - 1) {
                        const double before = turn >= SEL_FOLD ? sm.folded[tid] * (double)sel_scale(sm.folded_base[tid], seen.base) : 0.0;
                        sm.folded[tid] = before + (double)seen.sum;
                        sm.folded_base[tid] = seen.base;
                        seen.sum = 0.0f;
                    }
                }
                const unsigned tokens[SEL_HELD] = {token, token + 4 * NT, token + 8 * NT, token + 12 * NT};
                sel_reach(w, x, most, tokens, bound);
            }
            if (whole <= 0) bound = sel_bound<NT>(w, seen.top, beams);
        }
        const unsigned beside_tokens[2] = {(unsigned)(r.origin + 4 * edge), (unsigned)p.eos};
        sel_reach(w, beside, beside_most, beside_tokens, bound);
        double sum = (double)seen.sum;
        if (!FIT && whole > (SEL_FOLD - 1) * TURN) sum += sm.folded[tid] * (double)sel_scale(sm.folded_base[tid], seen.base);
        if (sum != sum) {              // NaN among the logits, or +inf: the sum again without NaN
            sum = 0.0;
            seen = sel_none();
            const auto add = [&](float scaled) {
                sum = sum * (double)scaled + (double)seen.sum;
                seen.sum = 0.0f;
            };
            for (int v = tid; v < whole; v += NT, at += NT) {
                const float4 y[1] = {drop_nan(*at)};
                float unused[1];
                add(sel_take(y, unused, seen));
            }
            add(sel_take(beside, beside_most, seen));
        }
        const float wtop = warp_max(seen.top);
        double wsum = seen.top == -INFINITY ? 0.0 : sum * (double)sel_scale(seen.base, wtop);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) wsum += __shfl_xor_sync(MB_FULL, wsum, o);
        if (lane == 0) { w.wtop[warp] = wtop; w.wsum[warp] = wsum; }
    }
    __syncthreads();
    cluster.barrier_wait();            // the first CTA has started: its memory may be written
    SelPart *found = cluster.map_shared_rank(sm.part, 0);
    for (int i = rank, q = 0; i < beams * parts; i += size, ++q) {
        if (!has(i)) continue;
        SelScratch &w = sm.work[q];
        SelPart *out = &found[i];
        if (warp == WARPS - 1 - q) {   // the sum of the part
            const float t = lane < WARPS ? w.wtop[lane] : -INFINITY;
            const float m = warp_max(t);
            double all = t == -INFINITY ? 0.0 : w.wsum[lane] * (double)sel_scale(t, m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(MB_FULL, all, o);
            if (lane == 0) {
                out->top = m;
                out->sum = all;
                // the largest term is 1, unless +inf is among the logits or there is no token: no distribution
                if (parts == 1) out->lse = all >= 0.5 ? (double)m + sel_log(all) : (double)NAN;
            }
        }
        const int reach = (int)w.n_reach;
        if (reach <= SEL_CAP) {
            // keys are distinct: a key's place is the number of larger ones; four threads share one
            for (int j0 = 0; j0 < reach; j0 += NT / 4) {
                const int j = j0 + (tid >> 2);
                const unsigned long long k = j < reach ? w.reach[j] : 0ull;
                int above = 0;
#pragma unroll 4
                for (int o = tid & 3; o < reach; o += 4) above += w.reach[o] > k;
                above += __shfl_xor_sync(MB_FULL, above, 1);
                above += __shfl_xor_sync(MB_FULL, above, 2);
                if (j < reach && above < beams && (tid & 3) == 0) out->key[above] = k;
            }
            if (tid >= reach && tid < beams) out->key[tid] = 0ull;
            continue;
        }
        // the largest key below the last one, once per place
        const SelRange r = range(i);
        const unsigned long long eos_key = has_eos(i) && drop_nan(r.row[p.eos]) > -INFINITY
                                               ? sel_key(r.row[p.eos], (unsigned)p.eos) : 0ull;
        unsigned long long last_key = ~0ull;
        for (int place = 0; place < beams; ++place) {
            unsigned long long k = eos_key < last_key ? eos_key : 0ull;
            for (int v = tid; v < r.vecs; v += NT) {
                const float4 x = sel_load(r, v);
                const unsigned t = (unsigned)(r.origin + 4 * v);
                const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!(e[j] > -INFINITY)) continue;
                    const unsigned long long c = sel_key(e[j], t + j);
                    if (c < last_key) k = max_u64(k, c);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) k = max_u64(k, __shfl_xor_sync(MB_FULL, k, o));
            __syncthreads();
            if (lane == 0) w.wkey[warp] = k;
            __syncthreads();
            k = 0;
            for (int v = 0; v < WARPS; ++v) k = max_u64(k, w.wkey[v]);
            if (tid == 0) out->key[place] = k;
            last_key = k;              // more than SEL_CAP keys: never 0
        }
    }
    cluster.sync();
    if (rank != 0) return;

    if (tid < beams && parts > 1 && !(done >> tid & 1u)) {
        SelPart *of = sm.part + tid * parts;
        float m = -INFINITY;
        for (int j = 0; j < parts; ++j) m = fmaxf(m, of[j].top);
        double all = 0.0;
        for (int j = 0; j < parts; ++j)
            if (of[j].top != -INFINITY) all += of[j].sum * (double)sel_scale(of[j].top, m);
        of[0].lse = all >= 0.5 ? (double)m + sel_log(all) : (double)NAN;
    }
    if (parts > 1) __syncthreads();
    if (tid < beams * parts) {
        sm.order[tid * SEL_PAD + beams] = 0ull;
        sm.near[tid * SEL_PAD + beams] = 0u;
    }
    if (tid < n) sel_score(sm, beams, parts, mine, done, p.eos, score, p.near);
    __syncthreads();
    const auto store = [&](int found_all) {            // first `beams` threads
        const int to = request * beams + tid;
        const bool alive = tid < found_all;
        const int from = alive ? sm.taken[tid] : 0;
        const unsigned t = alive ? sel_token(sm.key[from]) : 0u;
        p.score_out[to] = alive ? (float)sm.score[from] : -INFINITY;
        p.token[to] = t;
        p.parent[to] = alive ? (unsigned)(from / SEL_PAD / parts) : (unsigned)tid;         // dead: stays where it is
        if (p.done_out != nullptr) p.done_out[to] = alive && t == (unsigned)p.eos ? 1u : 0u;
    };
    unsigned close;
    if (warp == 0) {
        const int picked = sel_merge<false>(sm, beams, parts, p.near, close);
        if (tid < beams) store(picked);                // as a rule these stay
        if (tid == 0) sm.close = close;
    }
    __syncthreads();
    if (sm.close == 0u) return;
    const SelRow rows = {p.logits + (size_t)request * beams * p.logits_stride, p.logits_stride, p.codebook, p.eos, allow};
    if (!sel_refine<NT>(sm, beams, parts, done, p.near, rows)) return;
    if (tid < n) sel_score(sm, beams, parts, mine, done, p.eos, score, p.near);
    __syncthreads();
    if (warp == 0) {
        const int picked = sel_merge<false>(sm, beams, parts, p.near, close);
        if (tid < beams) store(picked);
    }
}

// ------------------------------------------------------------------------ reordering
//
// Rows 0 .. length[parent] of every beam become its parent's, in place, for all layers of K
// and V; the copies are bound by memory.  A thread owns one 16-byte column of one row in ALL
// beams of a request: it has loaded what every moved beam needs before it stores the first,
// so neither a cycle of parents nor a beam that several others follow needs a second buffer,
// and a parent's row that several beams take comes from memory once.  Beams that keep their
// own rows move nothing.  12 layers of 768 columns, 16 requests of 4 beams, f16, 332 MB: 60 us, 5.5
// TB/s; 4 requests of 8 beams, f32, 1.6 GB: 279 us, 5.75 TB/s, 85 and 89% of what a plain copy reaches; 4 of 16
// beams, f32, 1.7 GB 289 us, 5.8 TB/s.  A warp takes a row, so rows below 512 bytes leave lanes of it idle: 64
// requests of 4 beams with rows of 256 bytes 3.2 TB/s, of 64 bytes 0.9.

struct ReorderP {
    char *k, *v;
    size_t slots, capacity, row_bytes, slot_bytes, layer_bytes;
    int vecs, beams, planes;
    const unsigned *slot, *parent, *length;
    unsigned *length_out;
    const unsigned *live;
};

template <int NB, int U>
__global__ void __launch_bounds__(256) k_beam_reorder(ReorderP p) {
    __shared__ size_t s_src[MB_BEAM_MAX], s_dst[MB_BEAM_MAX];
    __shared__ unsigned s_rows[MB_BEAM_MAX];
    __shared__ int s_moved;
    mb_pdl_wait();
    mb_pdl_trigger();
    const int request = blockIdx.z, plane = blockIdx.y;
    if (p.live != nullptr && (unsigned)request >= *p.live) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == 0) {
        const int at = request * p.beams + lane;
        const bool mine = lane < p.beams;
        unsigned parent = mine ? p.parent[at] : 0u;
        const unsigned length = mine ? p.length[at] : 0u;
        const size_t slot = mine ? (p.slot != nullptr ? p.slot[at] : (size_t)at) : 0u;
        if (parent >= (unsigned)p.beams) parent = (unsigned)lane;      // not a beam: stays as it is
        const unsigned from_length = __shfl_sync(MB_FULL, length, parent & 31);
        const size_t from = __shfl_sync(MB_FULL, (unsigned long long)slot, parent & 31);
        const unsigned rows = from_length < p.capacity ? from_length : (unsigned)p.capacity;
        const bool there = slot < p.slots && from < p.slots;
        const bool moves = mine && parent != (unsigned)lane && rows > 0 && there && slot != from;
        const unsigned mask = __ballot_sync(MB_FULL, moves);
        if (moves) {
            const int i = __popc(mask & ((1u << lane) - 1u));
            s_src[i] = from * p.slot_bytes;
            s_dst[i] = slot * p.slot_bytes;
            s_rows[i] = rows;
        }
        if (lane == 0) s_moved = __popc(mask);
        if (mine && p.length_out != nullptr && plane == 0 && blockIdx.x == 0) p.length_out[at] = there ? from_length : length;
    }
    __syncthreads();
    const int moved = s_moved;
    if (moved == 0) return;
    unsigned most = 0;
    for (int i = 0; i < moved; ++i) most = max(most, s_rows[i]);
    char *base = (plane & 1 ? p.v : p.k) + (size_t)(plane >> 1) * p.layer_bytes;
    const unsigned step = gridDim.x * (blockDim.x >> 5);
    for (size_t row = blockIdx.x * (blockDim.x >> 5) + warp; row < most; row += step) {
        char *at = base + row * p.row_bytes;
        for (int c = lane; c < p.vecs; c += 32 * U) {
            float4 x[NB][U];
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (i < moved && row < s_rows[i])
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + 32 * u < p.vecs) x[i][u] = *reinterpret_cast<const float4 *>(at + s_src[i] + 16 * (size_t)(c + 32 * u));
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (i < moved && row < s_rows[i])
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + 32 * u < p.vecs) *reinterpret_cast<float4 *>(at + s_dst[i] + 16 * (size_t)(c + 32 * u)) = x[i][u];
        }
    }
}

}  // namespace

namespace {

int sel_launch(void (*kernel)(SelP), const SelP &p, size_t requests, int size, int threads, unsigned smem, cudaStream_t stream,
               int *resident) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(requests * (size_t)size));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = mb_pdl_enabled() ? 2u : 1u;
    if (resident != nullptr) {         // clusters of this size that the device holds at once
        cfg.numAttrs = 1u;
        return (int)cudaOccupancyMaxActiveClusters(resident, kernel, &cfg);
    }
    return (int)cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

extern "C" int mb_beam_init(int *clusters) {
    const int rc = (int)cudaFuncSetAttribute(k_beam_select<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_RING_BYTES);
    SelP none = {};
    for (int size = 1; rc == 0 && size <= SEL_CLUSTER; ++size) {
        const int q = sel_launch(k_beam_select<false>, none, 1, size, SEL_THREADS, SEL_RING_BYTES, 0, &clusters[size]);
        if (q != 0) return q;
        if (clusters[size] < 1) clusters[size] = 1;
    }
    return rc;
}

extern "C" int mb_beam_select(const mb_beam_select_args *a, mb_stream stream) {
    SelP p;
    p.logits = a->logits;
    p.logits_stride = a->logits_stride;
    p.requests = (int)a->requests;
    p.beams = (int)a->beams;
    p.codebook = (int)a->codebook_size;
    p.eos = (int)a->eos_id;
    p.has_eos = a->has_eos;
    p.allow_eos = a->allow_eos;
    p.score = a->score;
    p.done = a->done;
    p.live = a->live;
    p.near = 2.0 * sel_eps(a->codebook_size);
    p.score_out = a->score_out;
    p.token = a->token;
    p.parent = a->parent;
    p.done_out = a->done_out;
    // Few beams: rows are cut for the cluster's CTAs until a part fits in registers (one request of
    // one beam, 50,000 tokens: 6.2 us against 9.4 uncut, of four beams 9.0 / 9.9); one that fits is
    // not cut further (64 requests x 4 beams x 4,096: 6.0 us, in halves 7.6).
    constexpr int FITS = 4 * SEL_HELD * SEL_FIT_THREADS;
    p.parts = 1;
    while (p.beams * p.parts * 2 <= SEL_CLUSTER && p.codebook > p.parts * FITS) p.parts *= 2;
    const int pieces = p.beams * p.parts;
    // A part of at most 16 tokens per thread stays in registers: small CTAs, as many as there are (64
    // requests x 8 beams x 2,016: 8.2 us, through the ring 16.6).
    if ((p.codebook + p.parts - 1) / p.parts <= FITS) {
        const int rounds = (pieces + SEL_CLUSTER - 1) / SEL_CLUSTER, size = (pieces + rounds - 1) / rounds;
        return sel_launch(k_beam_select<true>, p, a->requests, size, SEL_FIT_THREADS, 0u, (cudaStream_t)stream, nullptr);
    }
    // Long parts: the cluster size with the fewest parts one after the other, counting the waves that
    // the device needs for all clusters (40 requests x 16 beams x 50,000: 40 us, with 8 CTAs each,
    // which are two waves, 46).
    int best = 0, least = 0;
    for (int size = SEL_CLUSTER; size >= 1; --size) {
        const int share = (pieces + size - 1) / size;
        if (share > SEL_SHARE || size > pieces) continue;
        const size_t waves = (a->requests + (size_t)a->clusters[size] - 1u) / (size_t)a->clusters[size];
        const int cost = (int)(waves > 1000000u ? 1000000u : waves) * share;
        if (best == 0 || cost < least) { best = size; least = cost; }
    }
    return sel_launch(k_beam_select<false>, p, a->requests, best, SEL_THREADS, SEL_RING_BYTES, (cudaStream_t)stream, nullptr);
}

extern "C" int mb_beam_reorder(const mb_beam_reorder_args *a, mb_stream stream) {
    const size_t size = a->cache.type == MB_F16 ? 2u : 4u;
    ReorderP p;
    p.k = (char *)a->cache.k;
    p.v = (char *)a->cache.v;
    p.slots = a->cache.slots;
    p.capacity = a->cache.capacity;
    p.row_bytes = a->cache.row_stride * size;
    p.slot_bytes = a->cache.slot_stride * size;
    p.layer_bytes = a->cache.layer_stride * size;
    p.vecs = (int)(a->cache.width * size / 16u);
    p.beams = (int)a->beams;
    p.planes = (int)(2u * a->cache.layers);
    p.slot = a->slot;
    p.parent = a->parent;
    p.length = a->length;
    p.length_out = a->length_out;
    p.live = a->live;
    // a grid of eight CTAs per SM where there is that much work, of which three, two or one are resident at a
    // time (70, 102 or 176 registers a thread for 4, 8 or 16 beams); a CTA walks its plane's rows
    const size_t want = 8u * (size_t)a->sm_count, have = (size_t)p.planes * a->requests;
    size_t x = (want + have - 1u) / have, most = (a->cache.capacity + 7u) / 8u;
    if (x > most) x = most;
    const dim3 grid((unsigned)x, (unsigned)p.planes, (unsigned)a->requests);
    // registers for as many beams as there are: with room for sixteen, 16 requests of 4 beams took 128
    // us instead of 60 and 4 requests of 8 beams 347 instead of 279
    if (a->beams <= 4) return mb_launch(k_beam_reorder<4, 2>, grid, dim3(256), 0, (cudaStream_t)stream, p);
    if (a->beams <= 8) return mb_launch(k_beam_reorder<8, 1>, grid, dim3(256), 0, (cudaStream_t)stream, p);
    return mb_launch(k_beam_reorder<16, 1>, grid, dim3(256), 0, (cudaStream_t)stream, p);
}
