// Single-token attention of a batch of lanes over a shared prefix and the lanes' own rows.
//
// Lane b has a query q, its own cached rows 0 .. n-1 and a prefix of P rows that other lanes
// may share; the new row is own row n.  With x_j = scale * q.k_j over the rows j that the lane
// sees (all of them, or with a window w the rows j < sinks and j > P + n - w of the joined
// sequence) the result is sum_j softmax(x)_j v_j.  Scores, maxima, sums and the weighted sum
// are 32-bit; K and V are f32 or f16, a new row is rounded to the cache's type once, when it
// is appended, and is attended as it was stored.
//
// Bound by reading every lane's K and V rows once.  The rows of all lanes, counted on, are cut
// into equal runs, one per resident CTA (k_lane_rows), whatever the lanes' lengths: a run that
// ends inside a lane leaves a partial result (maximum, sum, weighted sum), and k_lane_merge
// joins a lane's partials in row order, adds the new row and appends it.  A prefix of many lanes is
// read once per 128 of them (lane_prefix.cuh).
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "launch.h"
#include "tc_common.cuh"

namespace {

constexpr int WARPS_MAX = 12;      // warps of a k_lane_rows CTA
constexpr int CTAS_PER_SM = 2;

struct LaneP {
    int lanes, heads, head_width, width;
    float scale_log2;              // scale * log2(e): scores are powers of two
    const float *qkv;
    size_t qkv_stride;
    int qkv_vectors;               // rows of qkv start on 16 bytes
    char *k, *v;
    unsigned slots, capacity;
    size_t row_stride, slot_stride;               // elements
    const unsigned *slot, *length;
    const char *prefix_k, *prefix_v;
    unsigned prefixes, prefix_capacity;
    size_t prefix_row_stride, prefix_stride;      // elements
    const unsigned *prefix_length, *lane_prefix;
    unsigned window, sinks;
    const unsigned *live;
    float *out;
    size_t out_stride;
    int *status;
    unsigned polls;                // of a barrier, before a wait gives up
    // workspace
    unsigned *offset;              // [lanes + 1] rows of the lanes counted on, then the run length
    float2 *stat;                  // [part][heads] maximum, sum
    float *acc;                    // [part][heads][head_width]
    int heads_per_cta, phases;     // warps of a CTA: heads x row phases
    int step, row_bytes, row_pitch;      // rows of a step; bytes of a row's heads of a CTA, and between rows in the ring
    // the prefixes on the tensor cores (lane_prefix.cuh); 0 workers: prefix rows are walked like own rows
    int tile_workers;
    unsigned *tile_lane;           // [lanes] rank among the lanes of its prefix
    uint4 *tile_prefix;            // [prefixes]
    unsigned *tile_run;
    float2 *tile_stat;             // [partial row]
    float *tile_acc;               // [partial row][head_width]
};

// What a lane sees of its cached rows.  Prefix row i of `prefix_rows` is row i below
// prefix_head and i + prefix_jump from there on; own row i of `own_rows` lies in cache row i
// below own_head, then in own_base, own_base + 1, ... which wraps to `keep` at the capacity.
struct LaneView {
    unsigned prefix_rows, prefix_head, prefix_jump;
    unsigned own_rows, own_head, own_base, keep;
    unsigned append;               // cache row of the new row
    unsigned prefix, slot;
    bool ok;
};

// The words it is made of, loaded side by side.
struct LaneWords { unsigned live, slot, length, prefix; };

__device__ __forceinline__ LaneWords lane_words(const LaneP &p, int b) {
    LaneWords x;
    x.live = p.live != nullptr ? *p.live : 0xffffffffu;
    x.slot = p.slot != nullptr ? p.slot[b] : (unsigned)b;
    x.length = p.length[b];
    x.prefix = p.prefixes == 0 ? 0u : p.lane_prefix != nullptr ? p.lane_prefix[b] : 0u;
    return x;
}
__device__ __forceinline__ LaneView lane_view(const LaneP &p, int b, const LaneWords &x) {
    LaneView w;
    w.ok = (unsigned)b < x.live;
    w.slot = x.slot;
    w.prefix = x.prefix;
    const unsigned n = x.length;
    const unsigned P = w.prefix < p.prefixes ? min(p.prefix_length[w.prefix], p.prefix_capacity) : 0u;
    if (w.slot >= p.slots || (p.window == 0 && n >= p.capacity)) w.ok = false;
    w.keep = 0;
    if (p.window == 0) {
        w.prefix_rows = w.prefix_head = P;
        w.prefix_jump = 0;
        w.own_rows = w.own_head = n;
        w.own_base = 0;
        w.append = n;
    } else {
        // rows [0, head) and [first, P + n) of the joined sequence, head <= first
        const unsigned long long at = (unsigned long long)P + n + 1ull;
        const unsigned long long first = at > p.window ? at - p.window : 0ull;
        const unsigned head = (unsigned)(first < p.sinks ? first : p.sinks);
        const unsigned from = (unsigned)(first < P ? first : P);
        w.prefix_head = min(head, P);
        w.prefix_rows = w.prefix_head + (P - from);
        w.prefix_jump = from - w.prefix_head;
        w.keep = p.sinks > P ? p.sinks - P : 0u;
        w.own_head = head > P ? head - P : 0u;
        const unsigned own_first = first > P ? (unsigned)(first - P) : 0u;     // <= n
        const unsigned ring = p.capacity - w.keep;
        w.own_rows = w.own_head + (n - own_first);
        w.own_base = own_first < w.keep ? own_first : w.keep + (own_first - w.keep) % ring;
        w.append = n < w.keep ? n : w.keep + (n - w.keep) % ring;
    }
    if (!w.ok) w.prefix_rows = w.own_rows = 0;
    return w;
}
__device__ __forceinline__ LaneView lane_view(const LaneP &p, int b) { return lane_view(p, b, lane_words(p, b)); }

__device__ __forceinline__ unsigned own_row(const LaneP &p, const LaneView &w, unsigned i) {
    if (i < w.own_head) return i;
    const unsigned r = w.own_base + (i - w.own_head);
    return r < p.capacity ? r : r - (p.capacity - w.keep);
}

template <typename T>
struct Piece;                      // 16 bytes of a row: their elements as floats
template <>
struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4 &v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <>
struct Piece<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4 &v, float (&x)[8]) {
        const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

// 2^x, off by at most 2^-22 of itself: one instruction per row, head and thread.  A weight carries as
// much from its score, whose 32-bit sum is off by a few 2^-24 of a value of 1 to 10.
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What is left of it for k_lane_rows.
__device__ __forceinline__ LaneView lane_rows_view(const LaneP &p, int b) {
    LaneView w = lane_view(p, b);
    if (p.tile_workers > 0) w.prefix_rows = 0;
    return w;
}

// Rows of the lanes, counted on, and the length of a run: every CTA forms them (lanes <= 1024).  Few
// lanes are counted in whole runs, so that no run takes from two of them, which the whole launch
// would wait for (8 lanes of 347 rows: 9.5 us, 10.6 otherwise); `end` is where their rows end.
constexpr int FEW_LANES = 32;
__device__ __forceinline__ bool few_lanes(const LaneP &p, int workers) {
    return p.lanes > 1 && p.lanes <= FEW_LANES && 8 * p.lanes <= workers;
}

__device__ void lane_schedule(const LaneP &p, unsigned *off, unsigned *end, unsigned *run, int workers, int step) {
    __shared__ unsigned warp_sum_s[32];
    // whole steps, one at least (256 rows of one lane: 6.8 us, with two at least 7.4)
    const auto run_of = [step](unsigned rows, unsigned among) {
        return max(((rows + among - 1) / among + step - 1) / step * step, (unsigned)step);     // rows <= 2^30
    };
    const bool few = few_lanes(p, workers);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = (blockDim.x + 31) >> 5;
    unsigned carry = 0;
    if (p.lanes <= FEW_LANES) {        // one warp, one barrier
        if (warp == 0) {
            unsigned n = 0;
            if (lane < p.lanes) {
                const LaneView w = lane_rows_view(p, lane);
                n = w.prefix_rows + w.own_rows;
            }
            const unsigned rows = n;
            if (few) {
                const unsigned each = run_of(__reduce_add_sync(MB_FULL, n), workers - p.lanes);
                n = (n + each - 1) / each * each;
                if (lane == 0) *run = each;
            }
            unsigned x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(MB_FULL, x, o);
                if (lane >= o) x += y;
            }
            if (lane < p.lanes) {
                off[lane] = x - n;
                end[lane] = x - n + rows;
            }
            carry = __shfl_sync(MB_FULL, x, 31);
        }
    } else for (int b0 = 0; b0 < p.lanes; b0 += blockDim.x) {
        const int b = b0 + tid;
        unsigned n = 0;
        if (b < p.lanes) {
            const LaneView w = lane_rows_view(p, b);
            n = w.prefix_rows + w.own_rows;
        }
        unsigned x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(MB_FULL, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) warp_sum_s[warp] = x;
        __syncthreads();
        unsigned before = carry, all = 0;
        for (int w = 0; w < nwarps; ++w) {
            before += w < warp ? warp_sum_s[w] : 0u;
            all += warp_sum_s[w];
        }
        if (b < p.lanes) off[b] = before + x - n;
        carry += all;
    }
    if (tid == 0) {
        off[p.lanes] = carry;
        if (!few) *run = run_of(carry, workers);
    }
    __syncthreads();
}

// LPR lanes of a warp share a row's head (16 elements each), so a warp takes 32 / LPR rows at
// a time, U times over; a row's score is complete in its lanes after log2(LPR) exchanges, and
// every group of LPR lanes keeps its own running maximum and sum, joined once per run.  Few
// heads: `phases` warps share a head's rows and join through shared memory.
//
// A warp of its own brings the rows, all heads of a CTA in one bulk copy, into a ring of
// ROWS_DEPTH steps, across the lanes of a run: up to 100 KB per CTA, two CTAs per SM.  Rows lie
// row_pitch apart there, an odd multiple of the 16 * LPR bytes that the lanes of a row read at
// once (any 16-byte multiple for eight lanes), so that a warp's reads share no bank.
// 48 lanes x 1,029 f16 rows of 12 heads of 64, 152 MB, with the merge: loads into registers 40 us,
// 16-byte copies by every thread 34, bulk copies 32.5 (4.7 TB/s).  The rows take 21 us of it, at 7
// TB/s; the others are the schedule (2), the first rows' latency (2), uneven ends (3) and the merge
// (5).  Four steps of 8 rows instead of two of 16 save 1 us, but 8 rows at a time cost 4 to 15% wherever
// rows come from L2 or one CTA has an SM to itself.
//
// A wait that runs out (the copies take seconds: the device is in trouble) ends the launch in bounded
// time: the warp's lane is joined once more, so that no warp is missing at a barrier, and behind
// the barrier all warps of the CTA leave; without barriers each leaves alone.  A warp that has
// left empties no step, so the bringing warp and the others run out in turn.  The copies under
// way have landed, or have been waited for once more, before the CTA ends.
constexpr int ROWS_DEPTH = 2;
constexpr size_t ROWS_STAGE = 50u * 1024u;       // bytes of a step, at most

template <typename T>
constexpr int ROWS_U = sizeof(T) == 2 ? 2 : 1;   // rows of a group of lanes in a step

__device__ __forceinline__ void copy_row(unsigned to, const char *from, unsigned bytes, void *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
                 "r"(bytes), "r"(saddr(bar)) : "memory");
}
__device__ __forceinline__ void bar_arrive(void *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(bar)) : "memory");
}

// `bytes` (16 or 0) bytes, the rest of 16 zeros, by the calling thread.
__device__ __forceinline__ void copy_async(unsigned to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// FULL: the head fills all columns, LPR * 16.
template <typename T, int LPR, bool FULL>
__global__ void __maxnreg__(64) k_lane_rows(LaneP p) {
    extern __shared__ uint4 sm_rows_dyn[];
    __shared__ unsigned s_run, s_end[FEW_LANES];
    __shared__ volatile int s_lost;              // a warp's wait has run out
    __shared__ float s_acc[WARPS_MAX][MB_LANE_HEAD_WIDTH_MAX];
    __shared__ float2 s_stat[WARPS_MAX];
    __shared__ __align__(8) unsigned long long s_full[ROWS_DEPTH], s_empty[ROWS_DEPTH];
    constexpr int PER = Piece<T>::N, V = 16 / PER, U = ROWS_U<T>, GROUPS = 32 / LPR;
    unsigned *sm_off = reinterpret_cast<unsigned *>(sm_rows_dyn);
    const char *ring = reinterpret_cast<const char *>(sm_rows_dyn + (p.lanes + 1 + 3) / 4);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = p.heads_per_cta * p.phases, step = p.step;
    const unsigned plane = (unsigned)(step * p.row_pitch);       // K rows of a stage, then V rows
    if (threadIdx.x == 0) {
        s_lost = 0;
        for (int i = 0; i < ROWS_DEPTH; ++i) {
            bar_init(&s_full[i], 1u);
            bar_init(&s_empty[i], (unsigned)warps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Behind k_lane_prefix, which began when all work before it had ended, nothing has to be waited
    // for: both run side by side, and this one ends after the other (last_wait).
    if (p.tile_workers == 0) mb_pdl_wait();
    mb_pdl_trigger();
    const auto last_wait = [&]() {
        if (p.tile_workers > 0) mb_pdl_wait();
    };
    lane_schedule(p, sm_off, s_end, &s_run, gridDim.x, GROUPS * p.phases);
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int i = threadIdx.x; i <= p.lanes; i += blockDim.x) p.offset[i] = sm_off[i];
        if (threadIdx.x == 0) p.offset[p.lanes + 1] = s_run;
    }
    const auto end_of = [&](int b) { return p.lanes <= FEW_LANES ? s_end[b] : sm_off[b + 1]; };      // of lane b's rows
    const unsigned total = sm_off[p.lanes], run = s_run;
    const unsigned long long begin = (unsigned long long)blockIdx.x * run;
    if (begin >= total) { last_wait(); return; }
    const unsigned end = (unsigned)min((unsigned long long)total, begin + run);
    unsigned at = (unsigned)begin;
    int b = 0;                                   // the lane that row `at` belongs to
    for (int lo = 0, hi = p.lanes - 1; lo < hi;) {
        const int mid = (lo + hi + 1) >> 1;
        if (sm_off[mid] <= at) lo = b = mid; else hi = mid - 1;
    }
    int stage = 0;
    unsigned parity = 0;

    if (warp == warps) {                         // brings the rows
        const size_t column = (size_t)blockIdx.y * p.heads_per_cta * p.head_width * sizeof(T);
        // the last group of heads may be smaller
        const unsigned bytes = (unsigned)min((size_t)p.row_bytes, (size_t)p.width * sizeof(T) - column);
        const ptrdiff_t own_v = p.v - p.k, shared_v = p.prefix_v - p.prefix_k;      // from a row of K to its row of V
        bool fine = true;
        unsigned steps = 0;
        for (; at < end && fine; ++b) {
            if (sm_off[b + 1] <= at) continue;
            unsigned r0 = at - sm_off[b];
            const unsigned last = min(end, end_of(b)) - sm_off[b];
            const LaneView w = lane_rows_view(p, b);
            const char *own = p.k + w.slot * p.slot_stride * sizeof(T) + column;
            const char *shared = p.prefix_k + w.prefix * p.prefix_stride * sizeof(T) + column;
            at = min(end, sm_off[b + 1]);
            for (; r0 < last && fine; r0 += step) {
                if (steps >= ROWS_DEPTH) fine = __all_sync(MB_FULL, bar_wait(&s_empty[stage], parity ^ 1u, p.polls));
                if (!fine) break;
                ++steps;
                const unsigned n = min((unsigned)step, last - r0);
                if (lane == 0) bar_expect(&s_full[stage], 2u * n * bytes);
                __syncwarp();
                const unsigned to = saddr(ring) + (unsigned)stage * 2u * plane;
                for (unsigned i = lane; i < n; i += 32) {
                    const unsigned r = r0 + i;
                    const bool first = r < w.prefix_rows;
                    const size_t row = first ? (r < w.prefix_head ? r : r + w.prefix_jump) : own_row(p, w, r - w.prefix_rows);
                    const char *k = first ? shared + row * p.prefix_row_stride * sizeof(T) : own + row * p.row_stride * sizeof(T);
                    copy_row(to + i * p.row_pitch, k, bytes, &s_full[stage]);
                    copy_row(to + plane + i * p.row_pitch, k + (first ? shared_v : own_v), bytes, &s_full[stage]);
                }
                if (++stage == ROWS_DEPTH) { stage = 0; parity ^= 1u; }
            }
        }
        if (!fine && lane == 0) atomicOr(p.status, 2);
        for (unsigned i = steps - min(steps, (unsigned)ROWS_DEPTH); i < steps; ++i)       // whoever still reads them
            bar_wait(&s_full[i % ROWS_DEPTH], i / ROWS_DEPTH & 1u, TC_SPIN);
        last_wait();
        return;
    }

    // a warp without a head (of the last group) works on the last one and stores nothing
    const int wanted = blockIdx.y * p.heads_per_cta + warp % p.heads_per_cta, phase = warp / p.heads_per_cta;
    const bool has_head = wanted < p.heads;
    const int head = min(wanted, p.heads - 1), group = lane / LPR, part = lane % LPR;
    const char *mine = ring + (size_t)((head - blockIdx.y * p.heads_per_cta) * p.head_width + part * PER) * sizeof(T);
    while (at < end) {
        const unsigned first = at - sm_off[b], last = min(end, end_of(b)) - sm_off[b];
        if (last == first) { ++b; continue; }
        float q[16], acc[16], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int d = ((i / PER) * LPR + part) * PER + i % PER;
            q[i] = FULL || d < p.head_width ? p.qkv[(size_t)b * p.qkv_stride + head * p.head_width + d] * p.scale_log2 : 0.0f;
            acc[i] = 0.0f;
        }
        for (unsigned r0 = first; r0 < last; r0 += step) {
            if (!__all_sync(MB_FULL, bar_wait(&s_full[stage], parity, p.polls))) {
                if (lane == 0) {
                    atomicOr(p.status, 2);
                    s_lost = 1;
                }
                break;
            }
            const char *from = mine + (size_t)stage * 2u * plane;
            const unsigned most = min((unsigned)step, last - r0) - 1u;
            float x[U], m = top;
            const char *at_u[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned i = (phase + u * p.phases) * GROUPS + group;
                at_u[u] = from + (size_t)(min(i, most) * p.row_pitch);
                x[u] = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (!FULL && (j * LPR + part) * PER >= p.head_width) continue;
                    float k[PER];
                    Piece<T>::get(*reinterpret_cast<const uint4 *>(at_u[u] + j * LPR * 16), k);
#pragma unroll
                    for (int e = 0; e < PER; ++e) x[u] = fmaf(q[j * PER + e], k[e], x[u]);
                }
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) x[u] += __shfl_xor_sync(MB_FULL, x[u], o);
                if (i > most) x[u] = -INFINITY;
                m = fmaxf(m, x[u]);
            }
            const float ref = m == -INFINITY ? 0.0f : m;      // nothing but -inf so far: weights 0, not NaN
            const float keep = pow2(top - ref);
            top = m;
            sum *= keep;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float e = pow2(x[u] - ref);
                sum += e;
                if ((phase + u * p.phases) * GROUPS + group > most) continue;  // weight 0 times an infinity would be NaN
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (!FULL && (j * LPR + part) * PER >= p.head_width) continue;
                    float v[PER];
                    Piece<T>::get(*reinterpret_cast<const uint4 *>(at_u[u] + plane + j * LPR * 16), v);
#pragma unroll
                    for (int i = 0; i < PER; ++i) acc[j * PER + i] = fmaf(e, v[i], acc[j * PER + i]);
                }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&s_empty[stage]);
            if (++stage == ROWS_DEPTH) { stage = 0; parity ^= 1u; }
        }
        // join the groups of the warp, then its phases
        float m = top;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(MB_FULL, m, o));
        const float f = pow2(top - (m == -INFINITY ? 0.0f : m));
        sum *= f;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) sum += __shfl_xor_sync(MB_FULL, sum, o);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float a = acc[i] * f;
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1) a += __shfl_xor_sync(MB_FULL, a, o);
            acc[i] = a;
        }
        bool lost = __any_sync(MB_FULL, s_lost != 0);      // one answer for the warp
        if (p.phases > 1) {
            if (group == 0) {
                if (part == 0) s_stat[warp] = make_float2(m, sum);
#pragma unroll
                for (int i = 0; i < 16; ++i) s_acc[warp][((i / PER) * LPR + part) * PER + i % PER] = acc[i];
            }
            asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
            lost = s_lost != 0;                  // the same for all warps: it is set in front of this barrier only
            if (phase == 0) {
                float all = m;
                for (int o = 1; o < p.phases; ++o) all = fmaxf(all, s_stat[warp + o * p.heads_per_cta].x);
                const float ref = all == -INFINITY ? 0.0f : all;
                const float g = pow2(m - ref);
                sum *= g;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] *= g;
                for (int o = 1; o < p.phases; ++o) {
                    const int other = warp + o * p.heads_per_cta;
                    const float h = pow2(s_stat[other].x - ref);
                    sum = fmaf(s_stat[other].y, h, sum);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        acc[i] = fmaf(s_acc[other][((i / PER) * LPR + part) * PER + i % PER], h, acc[i]);
                }
                m = all;
            }
            asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
        }
        if (lost) break;
        if (group == 0 && phase == 0 && has_head) {
            const size_t slot = (size_t)(blockIdx.x + b) * p.heads + head;
            if (part == 0) p.stat[slot] = make_float2(m, sum);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int d = (j * LPR + part) * PER;
                if (FULL || d < p.head_width)
#pragma unroll
                    for (int i = 0; i < PER; i += 4)
                        *reinterpret_cast<float4 *>(p.acc + slot * p.head_width + d + i) =
                            make_float4(acc[j * PER + i], acc[j * PER + i + 1], acc[j * PER + i + 2], acc[j * PER + i + 3]);
            }
        }
        at = min(end, sm_off[b + 1]);
        ++b;
    }
    last_wait();
}

}  // namespace

#include "lane_prefix.cuh"

namespace {

// The new row's score, a lane's partials, the result, and the new row into the cache, for one
// head by `warps` warps: one where there are many heads of lanes, sixteen where there are few (a
// lane alone has hundreds of partials).  Four columns per thread; threads of the same columns take
// every slices-th partial, MERGE_U at a time.  A lane whose cache is full or whose slot does not
// exist is left out and sets the status word.  Bound by latency, the partials come from L2: 5 us
// behind the last rows for 48 lanes x 12 heads, of which three dependent trips to memory.
constexpr int MERGE_U = 4;

struct Merged { float top, sum; float4 acc; };

__device__ __forceinline__ void scale4(float4 &a, float f) { a.x *= f; a.y *= f; a.z *= f; a.w *= f; }
__device__ __forceinline__ void add4(float4 &a, const float4 &b, float f) {
    a.x = fmaf(b.x, f, a.x); a.y = fmaf(b.y, f, a.y); a.z = fmaf(b.z, f, a.z); a.w = fmaf(b.w, f, a.w);
}

// Joins the slices of a head; the result is in the first `columns` threads of its first warp.
template <int WARPS>
__device__ __forceinline__ Merged join_slices(Merged r, int columns, float4 (*s_acc)[32], float2 *s_stat) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = r.top;
    for (int o = columns; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(MB_FULL, m, o));
    const float f = pow2(r.top - (m == -INFINITY ? 0.0f : m));
    r.sum *= f;
    scale4(r.acc, f);
    for (int o = columns; o < 32; o <<= 1) {
        r.sum += __shfl_xor_sync(MB_FULL, r.sum, o);
        r.acc.x += __shfl_xor_sync(MB_FULL, r.acc.x, o);
        r.acc.y += __shfl_xor_sync(MB_FULL, r.acc.y, o);
        r.acc.z += __shfl_xor_sync(MB_FULL, r.acc.z, o);
        r.acc.w += __shfl_xor_sync(MB_FULL, r.acc.w, o);
    }
    r.top = m;
    if (WARPS == 1) return r;
    if (lane < columns) s_acc[warp][lane] = r.acc;
    if (lane == 0) s_stat[warp] = make_float2(m, r.sum);
    __syncthreads();
    if (warp != 0 || lane >= columns) return r;
    for (int o = 1; o < WARPS; ++o) r.top = fmaxf(r.top, s_stat[o].x);
    const float ref = r.top == -INFINITY ? 0.0f : r.top;
    r.sum = 0.0f;
    r.acc = make_float4(0, 0, 0, 0);
    for (int o = 0; o < WARPS; ++o) {
        const float g = pow2(s_stat[o].x - ref);
        r.sum = fmaf(s_stat[o].y, g, r.sum);
        add4(r.acc, s_acc[o][lane], g);
    }
    return r;
}

constexpr int MERGE_HEADS = 4;     // heads of a CTA with one warp each

template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? MERGE_HEADS * 32 : WARPS * 32) k_lane_merge(LaneP p, int columns) {
    __shared__ float4 s_acc[WARPS == 1 ? 1 : WARPS][32];
    __shared__ float2 s_stat[WARPS];
    __shared__ int s_again;
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = WARPS == 1 ? (int)blockIdx.y * MERGE_HEADS + warp : (int)blockIdx.y, tid = WARPS == 1 ? lane : (int)threadIdx.x;
    if (head >= p.heads) return;       // a warp of its own
    const int column = tid % columns, slice = tid / columns, slices = WARPS * 32 / columns;
    const int d = column * 4;
    const bool mine = d < p.head_width;
    // written before the first kernel of the call began: on their way while this one waits
    const LaneWords words = lane_words(p, b);
    const float *row = p.qkv + (size_t)b * p.qkv_stride + head * p.head_width + d;
    float q[4], kf[4], vf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[i] = mine ? row[i] : 0.0f;
        kf[i] = mine ? row[p.width + i] : 0.0f;
        vf[i] = mine ? row[2 * p.width + i] : 0.0f;
    }
    if (threadIdx.x == 0) s_again = 0;
    mb_pdl_wait();
    mb_pdl_trigger();
    const unsigned first = p.offset[b], last = p.offset[b + 1], run = p.offset[p.lanes + 1];
    if ((unsigned)b >= words.live) return;
    const LaneView w = lane_view(p, b, words);
    if (!w.ok) {
        if (tid == 0 && head == 0) atomicOr(p.status, 32);
        return;
    }
    T kt[4], vt[4];
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        kt[i] = (T)kf[i];
        vt[i] = (T)vf[i];
        q[i] *= p.scale_log2;
        x = fmaf(q[i], (float)kt[i], x);
    }
    for (int o = columns >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(MB_FULL, x, o);
    const unsigned part0 = last > first ? first / run : 0u;
    const int n_rows = last > first ? (int)((last - 1) / run - part0) + 1 : 0;
    const size_t base = (size_t)(part0 + b) * p.heads + head;
    int n = n_rows;
    size_t tile_base = 0;
    if (p.tile_workers > 0 && w.prefix_rows > 0) {
        const uint4 of = p.tile_prefix[w.prefix];
        const unsigned rank = p.tile_lane[b], tile = rank / TILE, each = *p.tile_run;
        const unsigned u0 = of.x + (tile * (unsigned)p.heads + (unsigned)head) * of.w, v0 = u0 / each;
        n += (int)((u0 + of.w - 1u) / each - v0) + 1;
        tile_base = of.y + (size_t)tile * TILE * p.heads + (size_t)head * min((unsigned)TILE, of.z - tile * TILE) +
                    (size_t)v0 * TILE + rank % TILE;
    }
    const size_t at_new = w.slot * p.slot_stride + (size_t)w.append * p.row_stride + head * p.head_width + d;
    if (slice == 0 && mine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            reinterpret_cast<T *>(p.k)[at_new + i] = kt[i];
            reinterpret_cast<T *>(p.v)[at_new + i] = vt[i];
        }
    }
    // the first slice begins with the new row, the others with nothing
    const Merged none = {-INFINITY, 0.0f, make_float4(0, 0, 0, 0)};
    const Merged own = {x, 1.0f, make_float4((float)vt[0], (float)vt[1], (float)vt[2], (float)vt[3])};
    Merged r = slice == 0 && x != -INFINITY ? own : none;
    for (int i0 = slice; i0 < n; i0 += MERGE_U * slices) {
        float2 s[MERGE_U];
        float4 a[MERGE_U];
#pragma unroll
        for (int u = 0; u < MERGE_U; ++u) {
            const int i = i0 + u * slices;
            s[u] = make_float2(-INFINITY, 0.0f);
            a[u] = make_float4(0, 0, 0, 0);
            if (i < n) {
                const bool tile = i >= n_rows;
                const size_t at = tile ? tile_base + (size_t)(i - n_rows) * TILE : base + (size_t)i * p.heads;
                s[u] = (tile ? p.tile_stat : p.stat)[at];
                if (mine) a[u] = *reinterpret_cast<const float4 *>((tile ? p.tile_acc : p.acc) + at * p.head_width + d);
            }
        }
        float m = r.top;
#pragma unroll
        for (int u = 0; u < MERGE_U; ++u) m = fmaxf(m, s[u].x);
        const float ref = m == -INFINITY ? 0.0f : m, keep = pow2(r.top - ref);
        r.top = m;
        r.sum *= keep;
        scale4(r.acc, keep);
#pragma unroll
        for (int u = 0; u < MERGE_U; ++u) {
            const float f = pow2(s[u].x - ref);
            r.sum = fmaf(s[u].y, f, r.sum);
            add4(r.acc, a[u], f);
        }
    }
    r = join_slices<WARPS>(r, columns, s_acc, s_stat);
    float *out = p.out + (size_t)b * p.out_stride + head * p.head_width + d;
    auto store = [&]() {
        const float y[4] = {__fdiv_rn(r.acc.x, r.sum), __fdiv_rn(r.acc.y, r.sum), __fdiv_rn(r.acc.z, r.sum), __fdiv_rn(r.acc.w, r.sum)};
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[i] = y[i];
            finite = finite && fabsf(y[i]) < INFINITY;
        }
        return finite;
    };
    const bool stores = tid < columns && mine;
    const bool odd = stores && !store();
    if (p.tile_workers == 0) return;
    if (WARPS == 1) {
        if (!__any_sync(MB_FULL, odd)) return;
    } else {
        if (odd) s_again = 1;
        __syncthreads();
        if (s_again == 0) return;
    }
    // Infinities or NaN among the rows: a value kept as planes turns inf into inf - inf, so this
    // head is formed once more from the values themselves, row by row (slowly: 256 lanes behind 4,096 rows,
    // one infinite value in a head of which 1.6 ms).
    const size_t prefix = (size_t)w.prefix * p.prefix_stride + head * p.head_width + d;
    const size_t slot = w.slot * p.slot_stride + head * p.head_width + d;
    r = slice == 0 && x != -INFINITY ? own : none;
    for (unsigned i0 = 0; i0 < w.prefix_rows + w.own_rows; i0 += slices) {
        const unsigned i = i0 + slice;
        const bool in = i < w.prefix_rows + w.own_rows;
        float kx[4] = {0, 0, 0, 0}, vx[4] = {0, 0, 0, 0}, y = 0.0f;
        if (in && mine) {
            const bool shared = i < w.prefix_rows;
            const size_t at = shared ? prefix + (size_t)(i < w.prefix_head ? i : i + w.prefix_jump) * p.prefix_row_stride
                                     : slot + (size_t)own_row(p, w, i - w.prefix_rows) * p.row_stride;
            const T *k = reinterpret_cast<const T *>(shared ? p.prefix_k : p.k) + at;
            const T *v = reinterpret_cast<const T *>(shared ? p.prefix_v : p.v) + at;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                kx[j] = (float)k[j];
                vx[j] = (float)v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) y = fmaf(q[j], kx[j], y);
        for (int o = columns >> 1; o > 0; o >>= 1) y += __shfl_xor_sync(MB_FULL, y, o);
        if (!in) y = -INFINITY;
        const float m = fmaxf(r.top, y), ref = m == -INFINITY ? 0.0f : m, keep = pow2(r.top - ref), e = pow2(y - ref);
        r.top = m;
        r.sum = fmaf(r.sum, keep, e);
        scale4(r.acc, keep);
        if (in) add4(r.acc, make_float4(vx[0], vx[1], vx[2], vx[3]), e);
    }
    r = join_slices<WARPS>(r, columns, s_acc, s_stat);
    if (stores) store();
}

struct Shape { int heads_per_cta, groups, phases, workers, lpr, step, row_bytes, row_pitch; };

Shape lane_shape(size_t heads, size_t head_width, size_t size, int sm_count) {
    Shape s;
    s.groups = (int)((heads + WARPS_MAX - 1) / WARPS_MAX);
    s.heads_per_cta = (int)((heads + s.groups - 1) / s.groups);
    s.workers = CTAS_PER_SM * sm_count / s.groups;
    if (s.workers < 1) s.workers = 1;
    s.lpr = head_width > 64 ? 8 : head_width > 32 ? 4 : head_width > 16 ? 2 : 1;
    s.row_bytes = (int)(s.heads_per_cta * head_width * size);
    const int once = 16 * s.lpr, times = (s.row_bytes + once - 1) / once;
    s.row_pitch = s.lpr < 8 ? (times | 1) * once : s.row_bytes;
    const int rows = 32 / s.lpr * (size == 2 ? ROWS_U<__half> : ROWS_U<float>);        // of a warp in a step
    s.phases = WARPS_MAX / s.heads_per_cta;
    while (s.phases > 1 && 2u * (size_t)s.row_pitch * rows * s.phases > ROWS_STAGE) --s.phases;
    s.step = rows * s.phases;
    return s;
}

// Whether the prefixes go through the tensor cores, from what the host knows: every lane's prefix
// full (prefix_capacity: one far above the lengths in use picks tiles too early), the lanes spread over
// the prefixes.  Walked like own rows they come from L2 and are bound by the arithmetic on groups of 16
// columns per thread; as tiles they cost a start, so much for every block that a CTA takes one after
// the other, and so much for every lane (its query, its partials, its own rows, which get fewer CTAs or
// wait).  The figures are chosen to lose least on 958 pairs of times: 8 layouts of 256 to 1,536 columns,
// 8 .. 256 lanes with 100 .. 300 own rows, prefixes of 100 .. 4,000; the rule takes a side more than 4% above
// the other in 52 of them.  Tiles / walking, in us:
//   12 x 64  f16: 32 lanes behind 1,000 rows 19.3 / 23.4, 16 lanes 18.8 / 16.8; 128 behind 217 31.0 / 29.4
//            f32: 64 lanes behind 1,000 rows 35.0 / 43.5, 32 lanes 28.3 / 27.1; 128 behind 217 43.8 / 37.3
//   8 x 96   f16: 32 lanes behind 1,000 rows 25.8 / 36.3, 8 lanes 17.0 / 14.2; f32: 64 lanes 43.7 / 59.9, 16 lanes 26.5 / 23.9
//   6 x 128  f16: 32 lanes behind 1,000 rows 23.4 / 26.0, 16 lanes 17.6 / 15.2; f32: 64 lanes 41.7 / 44.4, 32 lanes 32.4 / 30.4
constexpr size_t TILE_LANES = 8;   // fewer lanes never use them (and have no workspace for them)

struct TileCost { double start_us, turn_us, lane_us, bytes_per_us; };      // lane_us: of 768 columns
constexpr TileCost TILE_COST[2][2] = {{{0.0, 3.5, 0.03, 25e6}, {4.0, 2.5, 0.04, 22e6}},    // f32: heads up to 64, wider
                                      {{0.0, 2.5, 0.02, 18e6}, {1.5, 2.0, 0.02, 22e6}}};   // f16

bool use_tiles(size_t lanes, size_t heads, size_t head_width, size_t size, size_t prefixes, size_t prefix_capacity, size_t window,
               size_t sinks, int lpr, size_t at_once) {
    if (prefixes == 0 || lanes < TILE_LANES) return false;
    const bool f16 = size == 2u;
    const TileCost cost = TILE_COST[f16][head_width > 64];
    const size_t seen = window > 0 && window + sinks < prefix_capacity ? window + sinks : prefix_capacity;
    const size_t full = (lanes + TILE - 1) / TILE, tiles = prefixes > full ? (prefixes < lanes ? prefixes : lanes) : full;
    const size_t keys = f16 ? TileShape<__half, 1>::KEYS : TileShape<float, 1>::KEYS;
    const size_t blocks = tiles * heads * ((prefix_capacity + keys - 1) / keys), turns = (blocks + at_once - 1) / at_once;
    const double columns = (double)(lanes * heads * (size_t)lpr * 16u);
    const double walk_us = 2.0 * (double)seen * columns * (double)size / cost.bytes_per_us;
    return walk_us > cost.start_us + cost.turn_us * (double)turns + cost.lane_us * columns / 768.0;
}

// Places of the workspace, in floats.
struct Places { size_t offset, stat, acc, tile_lane, tile_prefix, tile_run, tile_stat, tile_acc, floats; };

Places lane_places(size_t lanes, size_t heads, size_t head_width, size_t prefixes, int sm_count) {
    const Shape s = lane_shape(heads, head_width, 4u, sm_count);      // workers go by the heads alone
    const size_t parts = (size_t)s.workers + lanes;
    const size_t workers = prefixes > 0 && lanes >= TILE_LANES ? (size_t)(TILE_CTAS_PER_SM * sm_count) : 0u;
    const size_t rows = workers > 0 ? lanes * heads + workers * TILE : 0u;
    Places w;
    size_t at = 0;
    auto take = [&at](size_t floats) {
        const size_t from = at;
        at += (floats + 3u) & ~(size_t)3u;
        return from;
    };
    w.offset = take(lanes + 2u);
    w.stat = take(2u * parts * heads);
    w.acc = take(parts * heads * head_width);
    w.tile_lane = take(workers > 0 ? lanes : 0u);
    w.tile_prefix = take(workers > 0 ? 4u * prefixes : 0u);
    w.tile_run = take(workers > 0 ? 1u : 0u);
    w.tile_stat = take(2u * rows);
    w.tile_acc = take(rows * head_width);
    w.floats = at;
    return w;
}

// f(kernel) for the kernel of a head width.
template <typename T, typename F>
int with_rows_kernel(int lpr, bool full, F f) {
    if (lpr == 8) return full ? f(k_lane_rows<T, 8, true>) : f(k_lane_rows<T, 8, false>);
    if (lpr == 4) return full ? f(k_lane_rows<T, 4, true>) : f(k_lane_rows<T, 4, false>);
    if (lpr == 2) return full ? f(k_lane_rows<T, 2, true>) : f(k_lane_rows<T, 2, false>);
    return full ? f(k_lane_rows<T, 1, true>) : f(k_lane_rows<T, 1, false>);
}
size_t rows_smem(size_t lanes, const Shape &s) {
    return ((lanes + 1u) * 4u + 15u) / 16u * 16u + (size_t)ROWS_DEPTH * 2u * (size_t)s.step * (size_t)s.row_pitch;
}
// How many CTAs of the prefix tiles an SM holds, TILE_CTAS_PER_SM at most, and whether one of the
// rows fits beside them.
struct TileFit { int ctas; bool beside; };

size_t tile_smem(size_t size, size_t head_width, size_t lanes, size_t prefixes) {
    const size_t operands = size == 2u ? (head_width <= 64 ? TileShape<__half, 1>::SMEM : TileShape<__half, 2>::SMEM)
                                       : (head_width <= 64 ? TileShape<float, 1>::SMEM : TileShape<float, 2>::SMEM);
    return operands + 16u * prefixes + 6u * lanes + 16u;
}

TileFit tile_fit(const mb_lane_device &device, const Shape &s, size_t size, size_t head_width, size_t lanes, size_t prefixes) {
    const auto &tile = device.tiles[size == 2u][head_width > 64];
    const size_t reserved = 1024u;                         // shared memory that a CTA takes besides its own
    const size_t smem = tile.smem + tile_smem(size, head_width, lanes, prefixes) + reserved, registers = tile.registers * TILE;
    TileFit fit = {TILE_CTAS_PER_SM, false};
    while (fit.ctas > 1 && (fit.ctas * smem > device.smem || fit.ctas * registers > device.registers)) --fit.ctas;
    const size_t threads = (size_t)(s.heads_per_cta * s.phases + 1) * 32u;
    fit.beside = fit.ctas * smem + device.rows.smem + rows_smem(lanes, s) + reserved <= device.smem &&
                 fit.ctas * registers + device.rows.registers * threads <= device.registers;
    return fit;
}
// Whether the rows are cut for one CTA per SM instead of two.  f32 tiles last longer than what one gains
// beside them meanwhile, also where it fits (8 x 96, 64 lanes behind 1,000 rows: 44.1 us with runs for two, 56.1 for
// one; 12 x 64, 48 lanes 31.7 / 33.9).  Beside f16 tiles one fits where heads are up to 64 (12 x 64, 32
// lanes behind 1,000: 21.6 / 18.5; 16 behind 4,000 27.2 / 25.3; where the own rows go on for as long as
// the tiles, 256 lanes of up to 500 behind 4,096, 73.3 / 74.6).  Wider ones take nearly all registers, so
// that the rows follow them: runs for two where they are of 8 steps or more (8 x 96, 64 lanes of up to 300
// behind 1,000: 33.9 / 35.2, 256 of up to 2,000 behind 4,000 212 / 362; 6 x 128, 64 lanes of up to 2,000 63 / 78, of
// up to 300 30.8 / 28.5), as far as the capacity tells.
bool one_rows_cta(const TileFit &fit, const Shape &s, size_t size, size_t lanes, size_t capacity) {
    return size == 2u && (fit.beside || lanes * capacity < 8u * (size_t)s.step * (size_t)s.workers);
}
template <typename T>
int launch_rows(const LaneP &p, const Shape &s, bool one_per_sm, cudaStream_t stream) {
    const int workers = one_per_sm && s.workers > 1 ? s.workers / CTAS_PER_SM : s.workers;
    const dim3 grid((unsigned)workers, (unsigned)s.groups), block((unsigned)((s.heads_per_cta * s.phases + 1) * 32));
    return with_rows_kernel<T>(s.lpr, p.head_width == s.lpr * 16, [&](auto kernel) {
        return mb_launch(kernel, grid, block, rows_smem((size_t)p.lanes, s), stream, p);
    });
}

template <typename T, int SLABS>
int launch_tiles(const LaneP &p, cudaStream_t stream) {
    return mb_launch(k_lane_prefix<T, SLABS>, dim3((unsigned)p.tile_workers), dim3(TILE),
                     tile_smem(sizeof(T), (size_t)p.head_width, (size_t)p.lanes, p.prefixes), stream, p);
}

template <typename T>
int launch_all(const LaneP &p, const Shape &s, bool one_per_sm, int sm_count, cudaStream_t stream, unsigned *launched) {
    int rc = 0;
    if (p.tile_workers > 0) {
        rc = p.head_width <= 64 ? launch_tiles<T, 1>(p, stream) : launch_tiles<T, 2>(p, stream);
        if (rc != 0) return rc;
    }
    rc = launch_rows<T>(p, s, one_per_sm, stream);
    if (rc != 0) return rc;
    int columns = 1;
    while (columns * 4 < p.head_width) columns *= 2;
    // Sixteen warps for a head while the device has room for them all: with the rows 6.9 us for one
    // lane of 12 heads (one warp 8.6), 9.6 for 8 (10.3), 21.2 for 5 of 3 heads and 120 partials (34.9); one
    // warp beyond: 48 lanes of 12 heads 32.5 us (sixteen 40.3), 256 lanes behind tiles 66.8 (126.6).
    const unsigned lanes = (unsigned)p.lanes, heads = (unsigned)p.heads;
    if ((size_t)lanes * heads <= 2u * (size_t)sm_count)
        rc = mb_launch(k_lane_merge<T, 16>, dim3(lanes, heads), dim3(512), 0, stream, p, columns);
    else
        rc = mb_launch(k_lane_merge<T, 1>, dim3(lanes, (heads + MERGE_HEADS - 1) / MERGE_HEADS), dim3(MERGE_HEADS * 32), 0, stream, p, columns);
    if (rc == 0 && launched != nullptr) *launched += p.tile_workers > 0 ? 3u : 2u;
    return rc;
}

}  // namespace

extern "C" size_t mb_lane_attention_floats(size_t lanes, size_t heads, size_t head_width, size_t prefixes, int sm_count) {
    return lane_places(lanes, heads, head_width, prefixes, sm_count).floats;
}

extern "C" int mb_lane_attention_init(mb_lane_device *device) {
    const auto allow = [](auto kernel, size_t smem) {
        return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    };
    // steps of one phase are within ROWS_STAGE too: 12 heads of 64 f32 columns are 8 rows of 3,136 bytes, of K and
    // of V; 12 of 32 f16 columns, 32 of 800, are the most
    constexpr size_t ROWS_SMEM_MOST = (MB_LANES_MAX + 4u) * 4u + ROWS_DEPTH * ROWS_STAGE;
    int rc = 0;
    for (int lpr = 1; lpr <= 8; lpr *= 2)
        for (int full = 0; full < 2; ++full) {
            if (rc == 0) rc = with_rows_kernel<float>(lpr, full, [&](auto k) { return allow(k, ROWS_SMEM_MOST); });
            if (rc == 0) rc = with_rows_kernel<__half>(lpr, full, [&](auto k) { return allow(k, ROWS_SMEM_MOST); });
        }
    int current = 0, smem = 0, registers = 0;
    if (rc == 0) rc = (int)cudaGetDevice(&current);
    if (rc == 0) rc = (int)cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerMultiprocessor, current);
    if (rc == 0) rc = (int)cudaDeviceGetAttribute(&registers, cudaDevAttrMaxRegistersPerMultiprocessor, current);
    device->smem = (size_t)smem;
    device->registers = (size_t)registers;
    const auto takes = [](auto kernel, auto &what) {
        cudaFuncAttributes at;
        const int error = (int)cudaFuncGetAttributes(&at, kernel);
        what.smem = at.sharedSizeBytes;
        what.registers = ((size_t)at.numRegs + 7u) / 8u * 8u;
        return error;
    };
    if (rc == 0) rc = takes(k_lane_rows<__half, 4, true>, device->rows);      // all variants: __maxnreg__, the same arrays
    const auto tiles = [&](auto kernel, size_t size, size_t head_width) {
        const int error = takes(kernel, device->tiles[size == 2u][head_width > 64u]);
        return error != 0 ? error : allow(kernel, tile_smem(size, head_width, MB_LANES_MAX, MB_LANES_MAX));
    };
    if (rc == 0) rc = tiles(k_lane_prefix<float, 1>, 4u, 64u);
    if (rc == 0) rc = tiles(k_lane_prefix<float, 2>, 4u, 128u);
    if (rc == 0) rc = tiles(k_lane_prefix<__half, 1>, 2u, 64u);
    if (rc == 0) rc = tiles(k_lane_prefix<__half, 2>, 2u, 128u);
    return rc;
}

extern "C" int mb_lane_attention(const mb_lane_attn_args *a, mb_stream stream) {
    const Shape s = lane_shape(a->heads, a->head_width, a->cache.type == MB_F16 ? 2u : 4u, a->sm_count);
    const Places w = lane_places(a->lanes, a->heads, a->head_width, a->prefixes, a->sm_count);
    LaneP p = {};
    p.lanes = (int)a->lanes;
    p.heads = (int)a->heads;
    p.head_width = (int)a->head_width;
    p.width = (int)(a->heads * a->head_width);
    p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
    p.qkv = a->qkv;
    p.qkv_stride = a->qkv_stride;
    p.qkv_vectors = ((uintptr_t)a->qkv & 15u) == 0 && a->qkv_stride % 4u == 0 && a->head_width % 4u == 0;
    p.k = (char *)a->cache.k;
    p.v = (char *)a->cache.v;
    p.slots = (unsigned)a->cache.slots;
    p.capacity = (unsigned)a->cache.capacity;
    p.row_stride = a->cache.row_stride;
    p.slot_stride = a->cache.slot_stride;
    p.slot = a->slot;
    p.length = a->length;
    p.prefix_k = (const char *)a->prefix_k;
    p.prefix_v = (const char *)a->prefix_v;
    p.prefixes = (unsigned)a->prefixes;
    p.prefix_capacity = (unsigned)a->prefix_capacity;
    p.prefix_row_stride = a->prefix_row_stride;
    p.prefix_stride = a->prefix_stride;
    p.prefix_length = a->prefix_length;
    p.lane_prefix = a->lane_prefix;
    p.window = (unsigned)a->window;
    p.sinks = (unsigned)a->sinks;
    p.live = a->live;
    p.out = a->out;
    p.out_stride = a->out_stride;
    p.status = a->status;
    p.polls = a->polls;
    p.offset = reinterpret_cast<unsigned *>(a->workspace + w.offset);
    p.stat = reinterpret_cast<float2 *>(a->workspace + w.stat);
    p.acc = a->workspace + w.acc;
    p.heads_per_cta = s.heads_per_cta;
    p.phases = s.phases;
    p.step = s.step;
    p.row_bytes = s.row_bytes;
    p.row_pitch = s.row_pitch;
    const size_t size = a->cache.type == MB_F16 ? 2u : 4u;
    const TileFit fit = tile_fit(*a->device, s, size, a->head_width, a->lanes, a->prefixes);
    bool tiles = a->tiles > 0 && a->prefixes > 0 && a->lanes >= TILE_LANES;
    if (a->tiles < 0)
        tiles = use_tiles(a->lanes, a->heads, a->head_width, size, a->prefixes, a->prefix_capacity, a->window, a->sinks, s.lpr,
                          (size_t)(fit.ctas * a->sm_count));
    if (tiles) p.tile_workers = fit.ctas * a->sm_count;
    p.tile_lane = reinterpret_cast<unsigned *>(a->workspace + w.tile_lane);
    p.tile_prefix = reinterpret_cast<uint4 *>(a->workspace + w.tile_prefix);
    p.tile_run = reinterpret_cast<unsigned *>(a->workspace + w.tile_run);
    p.tile_stat = reinterpret_cast<float2 *>(a->workspace + w.tile_stat);
    p.tile_acc = a->workspace + w.tile_acc;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool one_per_sm = tiles && one_rows_cta(fit, s, size, a->lanes, a->cache.capacity);
    return a->cache.type == MB_F16 ? launch_all<__half>(p, s, one_per_sm, a->sm_count, st, a->launched)
                                   : launch_all<float>(p, s, one_per_sm, a->sm_count, st, a->launched);
}
