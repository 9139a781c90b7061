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
// joins a lane's partials in row order, adds the new row and appends it.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "launch.h"

namespace {

constexpr int WARPS_MAX = 12;      // warps of a k_lane_rows CTA
constexpr int CTAS_PER_SM = 2;

struct LaneP {
    int lanes, heads, head_width, width;
    float scale_log2;              // scale * log2(e): scores are powers of two
    const float *qkv;
    size_t qkv_stride;
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
    // workspace
    unsigned *offset;              // [lanes + 1] rows of the lanes counted on, then the run length
    float2 *stat;                  // [part][heads] maximum, sum
    float *acc;                    // [part][heads][head_width]
    int heads_per_cta, phases;     // warps of a CTA: heads x row phases
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

__device__ __forceinline__ LaneView lane_view(const LaneP &p, int b) {
    LaneView w;
    const unsigned live = p.live != nullptr ? *p.live : 0xffffffffu;
    w.ok = (unsigned)b < live;
    w.slot = p.slot != nullptr ? p.slot[b] : (unsigned)b;
    const unsigned n = p.length[b];
    w.prefix = p.prefixes == 0 ? 0u : p.lane_prefix != nullptr ? p.lane_prefix[b] : 0u;
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
__device__ __forceinline__ unsigned own_row(const LaneP &p, const LaneView &w, unsigned i) {
    if (i < w.own_head) return i;
    const unsigned r = w.own_base + (i - w.own_head);
    return r < p.capacity ? r : r - (p.capacity - w.keep);
}

template <typename T>
struct Piece;                      // 16 bytes of a row as floats
template <>
struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const float *at, float (&x)[4]) {
        const float4 v = *reinterpret_cast<const float4 *>(at);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
};
template <>
struct Piece<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const __half *at, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(at);
        const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows of the lanes, counted on, and the length of a run: every CTA forms them (lanes <= 1024).
__device__ void lane_schedule(const LaneP &p, unsigned *off, unsigned *run, int workers, int step) {
    __shared__ unsigned warp_sum_s[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = (blockDim.x + 31) >> 5;
    unsigned carry = 0;
    for (int b0 = 0; b0 < p.lanes; b0 += blockDim.x) {
        const int b = b0 + tid;
        unsigned n = 0;
        if (b < p.lanes) {
            const LaneView w = lane_view(p, b);
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
        const unsigned each = (carry + workers - 1) / workers;
        *run = max((each + step - 1) / step * step, 2u * step);
    }
    __syncthreads();
}

// LPR lanes of a warp share a row's head (16 elements each), so a warp takes 32 / LPR rows at
// a time; a row's score is complete in its lanes after log2(LPR) exchanges, and every group of
// LPR lanes keeps its own running maximum and sum, joined once per run.
template <typename T, int LPR>
__global__ void __launch_bounds__(WARPS_MAX * 32, CTAS_PER_SM) k_lane_rows(LaneP p) {
    extern __shared__ unsigned sm_off[];
    __shared__ unsigned s_run;
    constexpr int PER = Piece<T>::N, V = 16 / PER, GROUPS = 32 / LPR;
    mb_pdl_wait();
    mb_pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int step = GROUPS * p.phases;
    lane_schedule(p, sm_off, &s_run, gridDim.x, step);
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int i = threadIdx.x; i <= p.lanes; i += blockDim.x) p.offset[i] = sm_off[i];
        if (threadIdx.x == 0) p.offset[p.lanes + 1] = s_run;
    }
    const int head = blockIdx.y * p.heads_per_cta + warp % p.heads_per_cta, phase = warp / p.heads_per_cta;
    const unsigned total = sm_off[p.lanes], run = s_run;
    unsigned long long begin = (unsigned long long)blockIdx.x * run;
    if (begin >= total || head >= p.heads) return;
    const unsigned end = (unsigned)min((unsigned long long)total, begin + run);
    unsigned at = (unsigned)begin;
    int b = 0;                                   // the lane that row `at` belongs to
    for (int lo = 0, hi = p.lanes; lo < hi;) {
        const int mid = (lo + hi + 1) >> 1;
        if (mid < p.lanes && sm_off[mid] <= at) { lo = mid; b = mid; } else hi = mid - 1;
    }
    while (sm_off[b + 1] <= at) ++b;
    const int group = lane / LPR, part = lane % LPR;
    while (at < end) {
        const LaneView w = lane_view(p, b);
        const unsigned first = at - sm_off[b], last = min(end, sm_off[b + 1]) - sm_off[b];
        float q[16], acc[16], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int d = ((i / PER) * LPR + part) * PER + i % PER;
            q[i] = d < p.head_width ? p.qkv[(size_t)b * p.qkv_stride + head * p.head_width + d] * p.scale_log2 : 0.0f;
            acc[i] = 0.0f;
        }
        const T *pk = reinterpret_cast<const T *>(p.prefix_k) + w.prefix * p.prefix_stride + head * p.head_width;
        const T *pv = reinterpret_cast<const T *>(p.prefix_v) + w.prefix * p.prefix_stride + head * p.head_width;
        const T *ok = reinterpret_cast<const T *>(p.k) + w.slot * p.slot_stride + head * p.head_width;
        const T *ov = reinterpret_cast<const T *>(p.v) + w.slot * p.slot_stride + head * p.head_width;
        for (unsigned r0 = first + phase * GROUPS; r0 < last; r0 += step) {
            const unsigned r = r0 + group;
            const bool in = r < last;
            const T *rk = ok, *rv = ov;
            if (in) {
                if (r < w.prefix_rows) {
                    const size_t o = (size_t)(r < w.prefix_head ? r : r + w.prefix_jump) * p.prefix_row_stride;
                    rk = pk + o;
                    rv = pv + o;
                } else {
                    const size_t o = (size_t)own_row(p, w, r - w.prefix_rows) * p.row_stride;
                    rk = ok + o;
                    rv = ov + o;
                }
            }
            float kx[V][PER], vx[V][PER];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int d = (j * LPR + part) * PER;
                if (in && d < p.head_width) {
                    Piece<T>::get(rk + d, kx[j]);
                    Piece<T>::get(rv + d, vx[j]);
                } else {
#pragma unroll
                    for (int i = 0; i < PER; ++i) kx[j][i] = vx[j][i] = 0.0f;
                }
            }
            float x = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < PER; ++i) x = fmaf(q[j * PER + i], kx[j][i], x);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(MB_FULL, x, o);
            if (!in) x = -INFINITY;
            const float m = fmaxf(top, x);
            const float ref = m == -INFINITY ? 0.0f : m;      // nothing but -inf so far: weights 0, not NaN
            const float keep = pow2(top - ref), e = pow2(x - ref);
            top = m;
            sum = fmaf(sum, keep, e);
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    acc[j * PER + i] = fmaf(acc[j * PER + i], keep, in ? e * vx[j][i] : 0.0f);
        }
        // join the groups of the warp
        float m = top;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(MB_FULL, m, o));
        const float f = pow2(top - (m == -INFINITY ? 0.0f : m));
        sum *= f;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) sum += __shfl_xor_sync(MB_FULL, sum, o);
        const size_t slot = ((size_t)(blockIdx.x + b) * p.phases + phase) * p.heads + head;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float a = acc[i] * f;
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1) a += __shfl_xor_sync(MB_FULL, a, o);
            acc[i] = a;
        }
        if (group == 0) {
            if (part == 0) p.stat[slot] = make_float2(m, sum);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int d = (j * LPR + part) * PER;
                if (d < p.head_width)
#pragma unroll
                    for (int i = 0; i < PER; i += 4)
                        *reinterpret_cast<float4 *>(p.acc + slot * p.head_width + d + i) =
                            make_float4(acc[j * PER + i], acc[j * PER + i + 1], acc[j * PER + i + 2], acc[j * PER + i + 3]);
            }
        }
        at += last - first;
        if (at < end)
            do ++b; while (sm_off[b + 1] <= at);
    }
}

// One warp per head of a lane: the new row's score, the lane's partials in row order, the
// result, and the new row into the cache.  A lane whose cache is full or whose slot does not
// exist is left out and sets the status word.
template <typename T>
__global__ void k_lane_merge(LaneP p) {
    mb_pdl_wait();
    mb_pdl_trigger();
    const int b = blockIdx.x, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (p.live != nullptr && (unsigned)b >= *p.live) return;
    const LaneView w = lane_view(p, b);
    if (!w.ok) {
        if (threadIdx.x == 0) atomicOr(p.status, 32);
        return;
    }
    const unsigned first = p.offset[b], last = p.offset[b + 1], run = p.offset[p.lanes + 1];
    const unsigned part0 = last > first ? first / run : 0u, parts = last > first ? (last - 1) / run - part0 + 1 : 0u;
    const int n = (int)parts * p.phases;
    const size_t base = ((size_t)part0 + b) * p.phases;
    const int d = lane * 4;
    const bool mine = d < p.head_width;
    for (int head = blockIdx.y * warps + (threadIdx.x >> 5); head < p.heads; head += gridDim.y * warps) {
        const float *row = p.qkv + (size_t)b * p.qkv_stride + head * p.head_width + d;
        float q[4] = {0, 0, 0, 0}, k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0}, acc[4];
        if (mine)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[i] = row[i] * p.scale_log2;
                const T kt = (T)row[p.width + i], vt = (T)row[2 * p.width + i];
                k[i] = (float)kt;
                v[i] = (float)vt;
                const size_t o = w.slot * p.slot_stride + (size_t)w.append * p.row_stride + head * p.head_width + d + i;
                reinterpret_cast<T *>(p.k)[o] = kt;
                reinterpret_cast<T *>(p.v)[o] = vt;
            }
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x = fmaf(q[i], k[i], x);
        x = warp_sum(x);
        float top = x;
        for (int i = lane; i < n; i += 32) top = fmaxf(top, p.stat[(base + i) * p.heads + head].x);
        top = warp_max(top);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float e = pow2(x - ref);
        float sum = e;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = e * v[i];
        for (int i = 0; i < n; ++i) {
            const float2 s = p.stat[(base + i) * p.heads + head];
            const float f = pow2(s.x - ref);
            sum = fmaf(s.y, f, sum);
            if (mine) {
                const float4 a = *reinterpret_cast<const float4 *>(p.acc + ((base + i) * p.heads + head) * p.head_width + d);
                acc[0] = fmaf(a.x, f, acc[0]);
                acc[1] = fmaf(a.y, f, acc[1]);
                acc[2] = fmaf(a.z, f, acc[2]);
                acc[3] = fmaf(a.w, f, acc[3]);
            }
        }
        if (mine)
#pragma unroll
            for (int i = 0; i < 4; ++i) p.out[(size_t)b * p.out_stride + head * p.head_width + d + i] = __fdiv_rn(acc[i], sum);
    }
}

struct Shape { int heads_per_cta, groups, phases, workers, lpr; };

Shape lane_shape(size_t heads, size_t head_width, int sm_count) {
    Shape s;
    s.groups = (int)((heads + WARPS_MAX - 1) / WARPS_MAX);
    s.heads_per_cta = (int)((heads + s.groups - 1) / s.groups);
    s.phases = WARPS_MAX / s.heads_per_cta;
    s.workers = CTAS_PER_SM * sm_count / s.groups;
    if (s.workers < 1) s.workers = 1;
    s.lpr = head_width > 64 ? 8 : head_width > 32 ? 4 : head_width > 16 ? 2 : 1;
    return s;
}

template <typename T>
int launch_rows(const LaneP &p, const Shape &s, cudaStream_t stream) {
    const dim3 grid((unsigned)s.workers, (unsigned)s.groups), block((unsigned)(s.heads_per_cta * s.phases * 32));
    const size_t smem = ((size_t)p.lanes + 1u) * sizeof(unsigned);
    if (s.lpr == 8) return mb_launch(k_lane_rows<T, 8>, grid, block, smem, stream, p);
    if (s.lpr == 4) return mb_launch(k_lane_rows<T, 4>, grid, block, smem, stream, p);
    if (s.lpr == 2) return mb_launch(k_lane_rows<T, 2>, grid, block, smem, stream, p);
    return mb_launch(k_lane_rows<T, 1>, grid, block, smem, stream, p);
}

size_t up4(size_t n) { return (n + 3u) & ~(size_t)3u; }

}  // namespace

extern "C" size_t mb_lane_attention_floats(size_t lanes, size_t heads, size_t head_width, size_t prefixes,
                                           size_t prefix_capacity, int sm_count) {
    (void)prefixes;
    (void)prefix_capacity;
    const Shape s = lane_shape(heads, head_width, sm_count);
    const size_t parts = ((size_t)s.workers + lanes) * (size_t)s.phases;
    return up4(lanes + 2u) + up4(2u * parts * heads) + parts * heads * head_width;
}

extern "C" int mb_lane_attention_init(void) { return 0; }

extern "C" int mb_lane_attention(const mb_lane_attn_args *a, mb_stream stream) {
    const Shape s = lane_shape(a->heads, a->head_width, a->sm_count);
    const size_t parts = ((size_t)s.workers + a->lanes) * (size_t)s.phases;
    LaneP p = {};
    p.lanes = (int)a->lanes;
    p.heads = (int)a->heads;
    p.head_width = (int)a->head_width;
    p.width = (int)(a->heads * a->head_width);
    p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
    p.qkv = a->qkv;
    p.qkv_stride = a->qkv_stride;
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
    p.offset = reinterpret_cast<unsigned *>(a->workspace);
    p.stat = reinterpret_cast<float2 *>(a->workspace + up4(a->lanes + 2u));
    p.acc = a->workspace + up4(a->lanes + 2u) + up4(2u * parts * a->heads);
    p.heads_per_cta = s.heads_per_cta;
    p.phases = s.phases;
    const cudaStream_t st = (cudaStream_t)stream;
    int rc = a->cache.type == MB_F16 ? launch_rows<__half>(p, s, st) : launch_rows<float>(p, s, st);
    if (rc != 0) return rc;
    const unsigned warps = a->heads < 12u ? (unsigned)a->heads : 12u;
    const dim3 grid((unsigned)a->lanes, 1u), block(warps * 32u);
    rc = a->cache.type == MB_F16 ? mb_launch(k_lane_merge<__half>, grid, block, 0, st, p)
                                 : mb_launch(k_lane_merge<float>, grid, block, 0, st, p);
    if (rc == 0 && a->launched != nullptr) *a->launched += 2u;
    return rc;
}
