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
// dealt to the CTAs, each keeps the running maximum and sum of its row and finds the row's
// best `beams` tokens, and the cluster's first CTA, into whose shared memory all results
// are stored, ranks at most 256 continuations.
//
// Best tokens of a part without sorting it: every group of eight threads knows the largest
// key (logit, then lower token) it has seen; the K-th largest of these group maxima is a
// lower bound of the K-th largest key, and only a few more than K keys reach it.  The threads
// whose own maximum does are the only ones whose tokens are read again (by their whole warp).
//
// Scores are formed in 64 bits: beams differ by less than a rounding of a 32-bit sum often
// enough to change a pick.  The sums of exponentials are 32-bit per thread (at most a few
// hundred terms, each off by 1e-7 of itself) and 64-bit across threads.

constexpr int SEL_CLUSTER = 8;     // portable cluster size
constexpr int SEL_CAP = 512;       // keys that may reach the bound before the slow path is taken
constexpr int SEL_GROUPS = 64;     // threads / 8, at most

struct SelPart {                   // what one part of a row found
    float top;                     // running maximum, -inf if no token
    float pad;
    double sum;                    // sum of exp(x - top)
    unsigned long long key[MB_BEAM_MAX];
};

struct SelSmem {
    SelPart part[MB_BEAM_MAX];     // first CTA: all parts of the request
    unsigned long long group[SEL_GROUPS];
    unsigned long long reach[SEL_CAP];
    double wsum[16];
    float wtop[16];
    unsigned n_reach;
    unsigned long long wkey[16];
    double lse[MB_BEAM_MAX];
    double score[MB_BEAM_MAX * MB_BEAM_MAX];
};

// Order-preserving key of a logit and its token: larger logit first, then the lower token.
// 0 is no key: NaN and -inf are not candidates.
__device__ __forceinline__ unsigned long long sel_key(float x, unsigned token) {
    const unsigned u = __float_as_uint(x + 0.0f);      // -0 and +0 are equal
    const unsigned o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)o << 32) | (0xffffffffu - token);
}
__device__ __forceinline__ float sel_logit(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned sel_token(unsigned long long key) { return 0xffffffffu - (unsigned)key; }

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

struct SelRange {
    const float *row;              // token 0
    const float4 *base;            // row + first, rounded down to 16 bytes
    int first, last;               // tokens first .. last - 1
    int shift;                     // tokens between base and row + first
    int vecs;                      // 16-byte pieces that hold the range
};

__device__ __forceinline__ SelRange sel_range(const float *row, int first, int last) {
    SelRange r;
    r.row = row;
    r.first = first;
    r.last = last;
    r.shift = (int)((reinterpret_cast<uintptr_t>(row + first) & 15u) >> 2);
    r.base = reinterpret_cast<const float4 *>(row + first - r.shift);
    r.vecs = last > first ? (last - first + r.shift + 3) >> 2 : 0;
    return r;
}
// The four logits of piece v; tokens outside the range read as -inf and are not touched.
__device__ __forceinline__ float4 sel_load(const SelRange &r, int v) {
    const int t = r.first - r.shift + 4 * v;
    float4 x;
    if (t >= r.first && t + 4 <= r.last) {
        x = r.base[v];
    } else {
        x.x = t >= r.first && t < r.last ? r.row[t] : -INFINITY;
        x.y = t + 1 >= r.first && t + 1 < r.last ? r.row[t + 1] : -INFINITY;
        x.z = t + 2 >= r.first && t + 2 < r.last ? r.row[t + 2] : -INFINITY;
        x.w = t + 3 >= r.first && t + 3 < r.last ? r.row[t + 3] : -INFINITY;
    }
    return x;
}
__device__ __forceinline__ float drop_nan(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ float sel_exp(float x, float top) {
    return exp2f(__fmul_rn(__fsub_rn(x, top), 1.4426950408889634f));
}

struct SelP {
    const float *logits;
    size_t logits_stride;
    int requests, beams, parts, codebook, eos, has_eos;
    const int *allow_eos;
    const float *score;
    const unsigned *done, *live;
    float *score_out;
    unsigned *token, *parent, *done_out;
};

__device__ void sel_part(const SelP &p, SelSmem &sm, const float *row, int first, int last, bool with_eos, SelPart *out) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x, nwarps = nthreads >> 5;
    const SelRange r = sel_range(row, first, last);
    float top = -INFINITY, sum = 0.0f, best = -INFINITY;
    unsigned best_token = 0;
    for (int v = tid; v < r.vecs; v += 4 * nthreads) {
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int w = v + u * nthreads;
            x[u] = w < r.vecs ? sel_load(r, w) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        float m = top;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            x[u].x = drop_nan(x[u].x); x[u].y = drop_nan(x[u].y);
            x[u].z = drop_nan(x[u].z); x[u].w = drop_nan(x[u].w);
            const float m4 = fmaxf(fmaxf(x[u].x, x[u].y), fmaxf(x[u].z, x[u].w));
            if (m4 > best) {           // ascending tokens: equal logits keep the lower one
                const unsigned t = (unsigned)(r.first - r.shift + 4 * (v + u * nthreads));
                best = m4;
                best_token = x[u].x == m4 ? t : x[u].y == m4 ? t + 1 : x[u].z == m4 ? t + 2 : t + 3;
            }
            m = fmaxf(m, m4);
        }
        if (m == -INFINITY) continue;
        sum = __fmul_rn(sum, top == m ? 1.0f : sel_exp(top, m));
        top = m;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            sum += (sel_exp(x[u].x, m) + sel_exp(x[u].y, m)) + (sel_exp(x[u].z, m) + sel_exp(x[u].w, m));
    }
    if (with_eos && tid == 0) {        // one token behind the range
        const float x = drop_nan(row[p.eos]);
        if (x > best) { best = x; best_token = (unsigned)p.eos; }
        if (x != -INFINITY) {
            const float m = fmaxf(top, x);
            sum = __fmul_rn(sum, top == m ? 1.0f : sel_exp(top, m)) + sel_exp(x, m);
            top = m;
        }
    }
    const unsigned long long mine = best == -INFINITY ? 0ull : sel_key(best, best_token);

    // the part's maximum and sum, and the maxima of groups of eight threads
    float wtop = warp_max(top);
    double wsum = top == -INFINITY ? 0.0 : (double)sum * (double)(top == wtop ? 1.0f : sel_exp(top, wtop));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wsum += __shfl_xor_sync(MB_FULL, wsum, o);
    unsigned long long g = mine;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) g = max_u64(g, __shfl_xor_sync(MB_FULL, g, o));
    if (lane == 0) { sm.wtop[warp] = wtop; sm.wsum[warp] = wsum; }
    if ((lane & 7) == 0) sm.group[tid >> 3] = g;
    if (tid == 0) sm.n_reach = 0;
    __syncthreads();

    // the bound: the beams-th largest group maximum, 0 when fewer groups have one
    const int groups = nthreads >> 3;
    unsigned long long bound = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int i = lane + 32 * half;
        const unsigned long long k = i < groups ? sm.group[i] : 0ull;
        int above = 0;
        for (int j = 0; j < groups; ++j) above += sm.group[j] > k;
        const unsigned hit = __ballot_sync(MB_FULL, k != 0ull && above == p.beams - 1);
        if (hit) bound = __shfl_sync(MB_FULL, k, __ffs(hit) - 1);
    }
    // tokens that reach it: the whole warp reads again what a thread with one has seen
    unsigned todo = __ballot_sync(MB_FULL, mine != 0ull && mine >= bound);
    while (todo) {
        const int owner = __ffs(todo) - 1;
        todo &= todo - 1;
        for (int v = warp * 32 + owner + lane * nthreads; v < r.vecs; v += 32 * nthreads) {
            const float4 x = sel_load(r, v);
            const unsigned t = (unsigned)(r.first - r.shift + 4 * v);
            const float e[4] = {drop_nan(x.x), drop_nan(x.y), drop_nan(x.z), drop_nan(x.w)};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (e[j] == -INFINITY) continue;
                const unsigned long long k = sel_key(e[j], t + j);
                if (k < bound) continue;
                const unsigned at = atomicAdd(&sm.n_reach, 1u);
                if (at < SEL_CAP) sm.reach[at] = k;
            }
        }
        if (with_eos && warp == 0 && owner == 0 && lane == 0) {
            const float x = drop_nan(row[p.eos]);
            if (x != -INFINITY && sel_key(x, (unsigned)p.eos) >= bound) {
                const unsigned at = atomicAdd(&sm.n_reach, 1u);
                if (at < SEL_CAP) sm.reach[at] = sel_key(x, (unsigned)p.eos);
            }
        }
    }
    if (tid < MB_BEAM_MAX) out->key[tid] = 0ull;       // out may lie in another CTA's shared memory
    __syncthreads();
    const unsigned n = sm.n_reach;
    if (n <= SEL_CAP) {
        // keys are distinct: a key's place is the number of larger ones
        for (unsigned i = tid; i < n; i += nthreads) {
            const unsigned long long k = sm.reach[i];
            int above = 0;
            for (unsigned j = 0; j < n; ++j) above += sm.reach[j] > k;
            if (above < p.beams) out->key[above] = k;
        }
    } else {
        // Many tokens reach the bound (their large logits lie in a few threads' pieces): take
        // the largest key below the last one, once per place, from a fresh pass each.
        unsigned long long last_key = ~0ull;
        for (int place = 0; place < p.beams; ++place) {
            unsigned long long k = 0;
            for (int v = tid; v < r.vecs; v += nthreads) {
                const float4 x = sel_load(r, v);
                const unsigned t = (unsigned)(r.first - r.shift + 4 * v);
                const float e[4] = {drop_nan(x.x), drop_nan(x.y), drop_nan(x.z), drop_nan(x.w)};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (e[j] == -INFINITY) continue;
                    const unsigned long long c = sel_key(e[j], t + j);
                    if (c < last_key) k = max_u64(k, c);
                }
            }
            if (with_eos && tid == 0) {
                const float x = drop_nan(row[p.eos]);
                const unsigned long long c = x == -INFINITY ? 0ull : sel_key(x, (unsigned)p.eos);
                if (c < last_key) k = max_u64(k, c);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) k = max_u64(k, __shfl_xor_sync(MB_FULL, k, o));
            __syncthreads();
            if (lane == 0) sm.wkey[warp] = k;
            __syncthreads();
            k = 0;
            for (int w = 0; w < nwarps; ++w) k = max_u64(k, sm.wkey[w]);
            if (tid == 0) out->key[place] = k;
            last_key = k;
            if (k == 0ull) break;
        }
    }
    if (tid == 0) {
        float m = -INFINITY;
        for (int w = 0; w < nwarps; ++w) m = fmaxf(m, sm.wtop[w]);
        double s = 0.0;
        for (int w = 0; w < nwarps; ++w)
            if (sm.wtop[w] != -INFINITY) s += sm.wsum[w] * exp((double)sm.wtop[w] - (double)m);
        out->top = m;
        out->sum = s;
    }
    __syncthreads();                   // sm is used again by the next part
}

__global__ void __launch_bounds__(512) k_beam_select(SelP p) {
    __shared__ SelSmem sm;
    mb_pdl_wait();
    mb_pdl_trigger();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
    const int request = blockIdx.x / size;
    if (p.live != nullptr && (unsigned)request >= *p.live) return;      // the whole cluster
    const int tid = threadIdx.x, beams = p.beams, parts = p.parts;
    SelSmem *first = cluster.map_shared_rank(&sm, 0);
    cluster.sync();                    // the first CTA's memory may be written from here on
    const bool allow = p.has_eos && (p.allow_eos == nullptr || p.allow_eos[request] != 0);
    for (int i = rank; i < beams * parts; i += size) {
        const int b = i / parts, part = i - b * parts;
        const int row = request * beams + b;
        if (p.done != nullptr && p.done[row] != 0) continue;
        const int per = (p.codebook + parts - 1) / parts;
        const int from = min(part * per, p.codebook), to = min(from + per, p.codebook);
        sel_part(p, sm, p.logits + (size_t)row * p.logits_stride, from, to, allow && part == parts - 1, &first->part[i]);
    }
    cluster.sync();
    if (rank != 0) return;

    if (tid < beams) {
        const bool done = p.done != nullptr && p.done[request * beams + tid] != 0;
        double lse = 0.0;
        if (done) {
            for (int j = 0; j < parts; ++j)
                for (int k = 0; k < beams; ++k) sm.part[tid * parts + j].key[k] = j + k == 0 ? sel_key(0.0f, (unsigned)p.eos) : 0ull;
        } else {
            float m = -INFINITY;
            for (int j = 0; j < parts; ++j) m = fmaxf(m, sm.part[tid * parts + j].top);
            double s = 0.0;
            for (int j = 0; j < parts; ++j)
                if (sm.part[tid * parts + j].top != -INFINITY)
                    s += sm.part[tid * parts + j].sum * exp((double)sm.part[tid * parts + j].top - (double)m);
            lse = (double)m + log(s);
        }
        sm.lse[tid] = lse;
    }
    __syncthreads();
    // ranked continuations: place (part, k) of the list; at most 16 x 16
    const int n = beams * parts * beams;
    for (int i = tid; i < n; i += blockDim.x) {
        const int part = i / beams, b = part / parts;
        const unsigned long long key = sm.part[part].key[i - part * beams];
        const double c = (double)p.score[request * beams + b] + ((double)sel_logit(key) - sm.lse[b]);
        sm.score[i] = key != 0ull && c > -INFINITY ? c : -INFINITY;     // NaN is no candidate
    }
    __syncthreads();
    int taken = 0;
    for (int i = tid; i < n; i += blockDim.x) {
        const int part = i / beams, b = part / parts;
        const unsigned long long key = sm.part[part].key[i - part * beams];
        const double c = sm.score[i];
        if (c == -INFINITY) continue;
        int above = 0;
        for (int j = 0; j < n; ++j) {
            const int q = j / beams, o = q / parts;
            const double d = sm.score[j];
            above += d > c || (d == c && (o < b || (o == b && sm.part[q].key[j - q * beams] > key)));
        }
        if (above >= beams) continue;
        const int at = request * beams + above;
        const unsigned t = sel_token(key);
        p.score_out[at] = (float)c;
        p.token[at] = t;
        p.parent[at] = (unsigned)b;
        if (p.done_out != nullptr) p.done_out[at] = t == (unsigned)p.eos ? 1u : 0u;
        ++taken;
    }
    // places without a continuation: a dead beam that stays where it is
    taken = __syncthreads_count(taken > 0) ;
    if (tid >= taken && tid < beams) {
        const int at = request * beams + tid;
        p.score_out[at] = -INFINITY;
        p.token[at] = 0u;
        p.parent[at] = (unsigned)tid;
        if (p.done_out != nullptr) p.done_out[at] = 0u;
    }
}

// ------------------------------------------------------------------------ reordering
//
// Rows 0 .. length[parent] of every beam become its parent's, in place, for all layers of K
// and V; the copies are bound by memory.  A thread owns one 16-byte column of one row in ALL
// beams of a request: it has loaded what every moved beam needs before it stores the first,
// so neither a cycle of parents nor a beam that several others follow needs a second buffer,
// and a parent's row that several beams take comes from memory once.  Beams that keep their
// own rows move nothing.

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
        const bool moves = mine && parent != (unsigned)lane && rows > 0 && slot < p.slots && from < p.slots && slot != from;
        const unsigned mask = __ballot_sync(MB_FULL, moves);
        if (moves) {
            const int i = __popc(mask & ((1u << lane) - 1u));
            s_src[i] = from * p.slot_bytes;
            s_dst[i] = slot * p.slot_bytes;
            s_rows[i] = rows;
        }
        if (lane == 0) s_moved = __popc(mask);
        if (mine && p.length_out != nullptr && plane == 0 && blockIdx.x == 0) p.length_out[at] = from_length;
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
    p.score_out = a->score_out;
    p.token = a->token;
    p.parent = a->parent;
    p.done_out = a->done_out;
    // few beams: rows are cut so that the cluster's CTAs all have work, while a part still has
    // eight tokens per thread
    p.parts = 1;
    while (p.beams * p.parts * 2 <= SEL_CLUSTER && p.codebook / (2 * p.parts) >= 2048) p.parts *= 2;
    const int pieces = p.beams * p.parts;
    const int rounds = (pieces + SEL_CLUSTER - 1) / SEL_CLUSTER;
    const int size = (pieces + rounds - 1) / rounds;
    const int threads = p.codebook / p.parts >= 8192 ? 512 : 256;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a->requests * (size_t)size));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = mb_pdl_enabled() ? 2u : 1u;
    return (int)cudaLaunchKernelEx(&cfg, k_beam_select, p);
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
    // eight CTAs per SM where there is that much work; a CTA walks its plane's rows
    const size_t want = 8u * (size_t)a->sm_count, have = (size_t)p.planes * a->requests;
    size_t x = (want + have - 1u) / have, most = (a->cache.capacity + 7u) / 8u;
    if (x > most) x = most;
    const dim3 grid((unsigned)x, (unsigned)p.planes, (unsigned)a->requests);
    if (a->beams <= 4) return mb_launch(k_beam_reorder<4, 2>, grid, dim3(256), 0, (cudaStream_t)stream, p);
    if (a->beams <= 8) return mb_launch(k_beam_reorder<8, 1>, grid, dim3(256), 0, (cudaStream_t)stream, p);
    return mb_launch(k_beam_reorder<16, 1>, grid, dim3(256), 0, (cudaStream_t)stream, p);
}
