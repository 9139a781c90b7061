// Shared-prefix part of the lane attention on the tensor cores: included by lane_attention.cu.
//
// The lanes of one prefix are rows of a tile (128 at most): for a head and a block of KEYS
// prefix rows
//     S = Q K^T,   p = 2^(S - max),   O += p V
// with both products by tcgen05.mma, S, p and O in tensor memory.  The prefix is read once per
// 128 lanes, which is the point; without it every lane would stream it.  Operands are 16-bit,
// results are to be 32-bit: an f16 cache is exact as it is, and a query and a weight are two f16
// planes, 22 bits.  Both planes end at f16's smallest value, 2^-24, so both are scaled to the top of
// its range: a query by a power of two that puts its largest element into [2^14, 2^15), a weight by
// 2^15 (what is kept as the maximum is 15 less).  Then what is lost is below 2^-38 of the largest
// element or weight, also where thousands of rows of small weight outweigh a few.  An f32 cache,
// query and weight are three bf16 planes, 24 bits and the exponent range of f32, and six of the nine
// products (the others are below 2^-24 of the result).
//
// The blocks of all (tile, head) pairs, counted on, are cut into equal runs, one per CTA; a run
// that ends inside a pair leaves a partial result, which k_lane_merge joins.  A thread owns a
// row of the tile: its maximum, sum and weighted sum stay in registers, so tensor memory is never
// rescaled.  A block is a chain of copies, products and a softmax by four warps, so an SM takes
// two CTAs (and one of k_lane_rows, which the memory keeps busy meanwhile) rather than wider
// ones.  The loops over scores are kept rolled: most CTAs run through them a few times only, and
// unrolled code was fetched at 200 cycles per score.
//
// 256 lanes behind 4,096 f16 rows, 12 heads of 64 (two tiles, 1,536 blocks, 5.2 per CTA): 40 us
// alone, 30 of which the blocks take; with them walked the call takes 374.  Bound by the chain of a block,
// 5 us: the tensor pipe is busy for a tenth of it, memory for less.
#pragma once

#include <cuda_bf16.h>

#include "tc_common.cuh"

namespace {

constexpr int TILE = 128;          // rows of a tile, threads of a CTA
constexpr int TILE_CTAS_PER_SM = 2;

template <typename T, int SLABS>
struct TileShape {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int KEYS = F16 ? 64 : 32;                 // prefix rows of a block
    static constexpr int QP = F16 ? 2 : 3, KP = F16 ? 1 : 3;   // planes of q and p, of K and V
    static constexpr float WEIGHT_TOP = F16 ? 15.0f : 0.0f;    // the largest weight, a power of two
    static constexpr int ORDERS = F16 ? 1 : 2;                 // products of planes a and b with a + b up to this
    static constexpr int Q_SLAB = TILE * 128, K_SLAB = KEYS * 128;     // bytes of 64 columns
    static constexpr int Q_PLANE = SLABS * Q_SLAB, K_PLANE = SLABS * K_SLAB;
    static constexpr int PIECES = KEYS * SLABS * 8 / TILE;     // 8 elements of K and of V per thread
    // columns of tensor memory: S, then O in its place, below; p from P on
    static constexpr unsigned P = SLABS * 64, TMEM = P + QP * KEYS / 2 <= 128 ? 128 : 256;
    static constexpr size_t SMEM = (size_t)QP * Q_PLANE + 2u * KP * K_PLANE + 1024u;
};

__device__ __forceinline__ void tmem_ld32u(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
// Completes the loads issued so far; the registers pass through it so that no use moves in front.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
          "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
          "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
          "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
        :: "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// A from tensor memory, B from shared memory.
__device__ __forceinline__ void mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// Rows of 128 bytes (64 columns), 128-byte swizzle, read with the columns as the M or N
// dimension: 8-row groups 1024 bytes apart along K, 64-column slabs `slab` bytes apart.
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(unsigned addr, unsigned slab) {
    uint64_t d = smem_desc_sw128(addr) & ~((uint64_t)0x3fff << 16);
    return d | (uint64_t)((slab >> 4) & 0x3fffu) << 16;
}

// Two values into the QP 16-bit planes that sum to them.
template <bool F16, int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&plane)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (F16) {
            const __half2 h = __floats2half2_rn(a, b);
            const float2 f = __half22float2(h);
            plane[i] = *reinterpret_cast<const uint32_t *>(&h);
            a -= f.x;
            b -= f.y;
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            const float2 f = __bfloat1622float2(h);
            plane[i] = *reinterpret_cast<const uint32_t *>(&h);
            a -= f.x;
            b -= f.y;
        }
    }
}

// Byte of 16-byte piece c of row r in a slab of 128-byte rows with 128-byte swizzle.
__device__ __forceinline__ unsigned swizzled(int r, int c) { return (unsigned)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Ranks of the lanes within their prefixes (in lane order; ~0u: no row of it to see) and, per
// prefix, its first unit, its first row of partials, its lanes and its blocks.  A unit is one
// block of one (tile, head) pair.  Worker v leaves its partial rows of a pair v * TILE rows
// behind where the pair's rows begin: pairs and workers only go up along the units, so no two
// partials meet.
template <int KEYS>
__device__ void tile_schedule(const LaneP &p, unsigned short *voice, unsigned *rank, uint4 *prefix, unsigned *units, unsigned *run) {
    const int tid = threadIdx.x, lane = tid & 31;
    for (int g = tid; g < (int)p.prefixes; g += blockDim.x) {
        const unsigned rows = min(p.prefix_length[g], p.prefix_capacity);
        prefix[g] = make_uint4(0u, 0u, 0u, (rows + KEYS - 1) / KEYS);
    }
    for (int b = tid; b < p.lanes; b += blockDim.x) {
        const LaneView w = lane_view(p, b);
        voice[b] = w.prefix_rows > 0 ? (unsigned short)w.prefix : (unsigned short)0xffffu;
    }
    __syncthreads();
    if (p.prefixes == 1) {             // all warps at once
        __shared__ unsigned s_count[MB_LANES_MAX / 32];
        const int warp = tid >> 5, chunks = (p.lanes + 31) / 32;
        for (int c = warp; c < chunks; c += (int)blockDim.x >> 5) {
            const int b = c * 32 + lane;
            const unsigned has = __ballot_sync(MB_FULL, b < p.lanes && voice[b] == 0);
            if (lane == 0) s_count[c] = __popc(has);
            if (b < p.lanes) rank[b] = has >> lane & 1u ? (unsigned)__popc(has & ((1u << lane) - 1u)) : 0xffffffffu;
        }
        __syncthreads();
        for (int c = warp; c < chunks; c += (int)blockDim.x >> 5) {
            const unsigned before = __reduce_add_sync(MB_FULL, lane < c ? s_count[lane] : 0u);
            const int b = c * 32 + lane;
            if (b < p.lanes && rank[b] != 0xffffffffu) rank[b] += before;
            if (c == chunks - 1 && lane == 0) prefix[0].z = before + s_count[c];
        }
        __syncthreads();
    }
    if (tid < 32) {
        for (int b0 = 0; b0 < p.lanes && p.prefixes > 1; b0 += 32) {
            const int b = b0 + lane;
            const unsigned g = b < p.lanes ? voice[b] : 0xffffu;
            const unsigned peers = __match_any_sync(MB_FULL, g);
            const unsigned before = g != 0xffffu ? prefix[g].z : 0u;
            __syncwarp();
            if (b < p.lanes) rank[b] = g != 0xffffu ? before + __popc(peers & ((1u << lane) - 1u)) : 0xffffffffu;
            if (g != 0xffffu && __ffs(peers) - 1 == lane) prefix[g].z = before + __popc(peers);
            __syncwarp();
        }
        unsigned unit = 0, row = 0;
        for (int g0 = 0; g0 < (int)p.prefixes; g0 += 32) {
            const int g = g0 + lane;
            uint4 v = g < (int)p.prefixes ? prefix[g] : make_uint4(0u, 0u, 0u, 0u);
            const unsigned n = (v.z + TILE - 1) / TILE * (unsigned)p.heads * v.w;
            unsigned x = n, y = v.z;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned a = __shfl_up_sync(MB_FULL, x, o), c = __shfl_up_sync(MB_FULL, y, o);
                if (lane >= o) { x += a; y += c; }
            }
            v.x = unit + x - n;
            v.y = row + (y - v.z) * (unsigned)p.heads;
            if (g < (int)p.prefixes) prefix[g] = v;
            unit += __shfl_sync(MB_FULL, x, 31);
            row += __shfl_sync(MB_FULL, y, 31) * (unsigned)p.heads;
        }
        if (lane == 0) {
            *units = unit;
            *run = max((unit + p.tile_workers - 1) / p.tile_workers, 1u);
        }
    }
    __syncthreads();
}

template <typename T, int SLABS>
__global__ void __launch_bounds__(TILE, SLABS == 1 ? 4 : 2) k_lane_prefix(LaneP p) {
    using C = TileShape<T, SLABS>;
    constexpr bool F16 = C::F16;
    constexpr int KEYS = C::KEYS, QP = C::QP, KP = C::KP, PER_ROW = SLABS * 8;
    extern __shared__ unsigned char sm_tile[];
    __shared__ __align__(8) unsigned long long s_bar;
    __shared__ uint32_t s_tmem;
    __shared__ unsigned s_units, s_run;
    __shared__ unsigned short s_row[TILE];                 // lanes of the tile
    __shared__ float s_unscale[TILE];
    unsigned char *base = sm_tile + ((1024u - (saddr(sm_tile) & 1023u)) & 1023u);
    unsigned char *sq = base, *sk = sq + QP * C::Q_PLANE, *sv = sk + KP * C::K_PLANE;
    unsigned char *rest = base + (C::SMEM - 1024u);        // schedule
    uint4 *s_prefix = reinterpret_cast<uint4 *>(rest);
    unsigned *s_rank = reinterpret_cast<unsigned *>(s_prefix + p.prefixes);
    unsigned short *s_voice = reinterpret_cast<unsigned short *>(s_rank + p.lanes);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    mb_pdl_wait();
    mb_pdl_trigger();
    tile_schedule<KEYS>(p, s_voice, s_rank, s_prefix, &s_units, &s_run);
    if (blockIdx.x == 0) {
        for (int b = tid; b < p.lanes; b += TILE) p.tile_lane[b] = s_rank[b];
        for (int g = tid; g < (int)p.prefixes; g += TILE) p.tile_prefix[g] = s_prefix[g];
        if (tid == 0) *p.tile_run = s_run;
    }
    const unsigned units = s_units, run = s_run;
    if ((unsigned long long)blockIdx.x * run >= units) return;
    unsigned unit = blockIdx.x * run;
    const unsigned end = min(units, unit + run);
    if (tid == 0) {
        bar_init(&s_bar, 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&s_tmem)), "r"(C::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem, my_tmem = tmem + ((uint32_t)(warp * 32) << 16);
    const int hw = p.head_width, ksteps = (hw + 15) / 16, ncols = ksteps * 16;
    const uint32_t format = F16 ? 0u : (1u << 7 | 1u << 10);
    const uint32_t idesc_s = instr_desc_f16(TILE, KEYS) | format;
    const uint32_t idesc_o = instr_desc_f16(TILE, ncols) | format | 1u << 16;              // B along N
    unsigned parity = 0;
    bool fine = true;
    int g = 0;

    while (unit < end && fine) {
        while (g + 1 < (int)p.prefixes && s_prefix[g + 1].x <= unit) ++g;
        const uint4 of = s_prefix[g];
        const unsigned pair = (unit - of.x) / of.w, tile = pair / (unsigned)p.heads;
        const int head = (int)(pair - tile * (unsigned)p.heads);
        unsigned block = unit - of.x - pair * of.w;
        const unsigned stop = min(of.w, block + (end - unit));
        const int rows = (int)min((unsigned)TILE, of.z - tile * TILE);
        const unsigned keys = min(p.prefix_length[g], p.prefix_capacity);
        unit += stop - block;

        // f16 rows of a block on their way, zero beyond the prefix and beyond the head (rows that are
        // not seen may hold anything)
        const size_t origin = (size_t)g * p.prefix_stride + (size_t)head * hw;
        const T *pk = reinterpret_cast<const T *>(p.prefix_k) + origin, *pv = reinterpret_cast<const T *>(p.prefix_v) + origin;
        auto bring = [&](const T *from, unsigned char *to, unsigned block) {
#pragma unroll
            for (int i = 0; i < C::PIECES; ++i) {
                const int at = tid + i * TILE, r = at / PER_ROW, c = at % PER_ROW;
                const unsigned j = block * KEYS + r;
                const bool in = j < keys && c * 8 < hw;
                copy_async(saddr(to) + (c >> 3) * C::K_SLAB + swizzled(r, c & 7),
                           in ? from + (size_t)j * p.prefix_row_stride + c * 8 : from, in ? 16 : 0);
            }
        };
        __syncthreads();                                   // s_row and the queries are read no more
        if (F16) {
            bring(pk, sk, block);
            bring(pv, sv, block);
        }
        for (int b = tid; b < p.lanes; b += TILE)
            if (s_voice[b] == g && s_rank[b] / TILE == tile) s_row[s_rank[b] % TILE] = (unsigned short)b;
        __syncthreads();

        // the queries: scaled, cut into planes, rows of 128 bytes per slab
        constexpr int QUERIES = 4, QUERY_TOP = 14;
#pragma unroll 1
        for (int i0 = tid; i0 - lane < rows * PER_ROW; i0 += QUERIES * TILE) {
            float x[QUERIES][8];
#pragma unroll
            for (int u = 0; u < QUERIES; ++u) {
                const int i = i0 + u * TILE, r = i / PER_ROW, c = i % PER_ROW;
                const float *q = p.qkv + (size_t)(r < rows ? s_row[r] : 0) * p.qkv_stride + head * hw + c * 8;
                if (p.qkv_vectors && r < rows && c * 8 + 8 <= hw) {
                    const float4 a = *reinterpret_cast<const float4 *>(q), b = *reinterpret_cast<const float4 *>(q + 4);
                    x[u][0] = a.x; x[u][1] = a.y; x[u][2] = a.z; x[u][3] = a.w;
                    x[u][4] = b.x; x[u][5] = b.y; x[u][6] = b.z; x[u][7] = b.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[u][j] = r < rows && c * 8 + j < hw ? q[j] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < QUERIES; ++u) {
                const int i = i0 + u * TILE, r = i / PER_ROW, c = i % PER_ROW;
                float most = 0.0f, up = 1.0f, down = 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[u][j] *= p.scale_log2;
                if (F16) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[u][j]));
#pragma unroll
                    for (int o = PER_ROW / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(MB_FULL, most, o));
                    // 2^e <= most < 2^(e + 1); what is not finite stays as it is, and so does what is
                    // so small that all its scores are 0
                    const int e = (int)(__float_as_uint(most) >> 23) - 127;
                    if (e > -100 && e < 127) {
                        up = __uint_as_float((unsigned)(127 + QUERY_TOP - e) << 23);
                        down = __uint_as_float((unsigned)(127 - QUERY_TOP + e) << 23);
                    }
                }
                if (r < rows) {
                    uint32_t plane[4][QP];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_pair<F16>(x[u][2 * j] * up, x[u][2 * j + 1] * up, plane[j]);
#pragma unroll
                    for (int j = 0; j < QP; ++j)
                        *reinterpret_cast<uint4 *>(sq + j * C::Q_PLANE + (c >> 3) * C::Q_SLAB + swizzled(r, c & 7)) =
                            make_uint4(plane[0][j], plane[1][j], plane[2][j], plane[3][j]);
                    if (c == 0) s_unscale[r] = down;
                }
            }
        }
        const bool mine = tid < rows;
        const bool work = warp * 32 < rows;                // a warp without a row has nothing to weigh
        unsigned seen_head = 0, seen_from = 0;             // rows of the prefix it sees: below, and from there on
        if (mine) {
            const LaneView w = lane_view(p, s_row[tid]);
            seen_head = w.prefix_head;
            seen_from = w.prefix_head + w.prefix_jump;
        }
        float unscale = 1.0f, top = -INFINITY, sum = 0.0f, o[SLABS * 64];
#pragma unroll
        for (int i = 0; i < SLABS * 64; ++i) o[i] = 0.0f;

#pragma unroll 1
        for (bool begun = false; block < stop; ++block, begun = true) {
            const unsigned first = block * KEYS;
            if (F16) {
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
#pragma unroll 1
                for (int m = 0; m < 2; ++m) {              // K, then V
                    const T *from = m ? pv : pk;
                    uint4 x[C::PIECES][2];
#pragma unroll
                    for (int i = 0; i < C::PIECES; ++i) {
                        const int at = tid + i * TILE, r = at / PER_ROW, d = at % PER_ROW * 8;
#pragma unroll
                        for (int l = 0; l < 2; ++l) {
                            x[i][l] = make_uint4(0, 0, 0, 0);
                            if (first + r < keys && d + 4 * l < hw)
                                x[i][l] = __ldg(reinterpret_cast<const uint4 *>(from + (size_t)(first + r) * p.prefix_row_stride + d + 4 * l));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < C::PIECES; ++i) {
                        const int at = tid + i * TILE, r = at / PER_ROW, c = at % PER_ROW;
                        uint32_t plane[4][KP];
                        split_pair<F16>(__uint_as_float(x[i][0].x), __uint_as_float(x[i][0].y), plane[0]);
                        split_pair<F16>(__uint_as_float(x[i][0].z), __uint_as_float(x[i][0].w), plane[1]);
                        split_pair<F16>(__uint_as_float(x[i][1].x), __uint_as_float(x[i][1].y), plane[2]);
                        split_pair<F16>(__uint_as_float(x[i][1].z), __uint_as_float(x[i][1].w), plane[3]);
#pragma unroll
                        for (int j = 0; j < KP; ++j)
                            *reinterpret_cast<uint4 *>((m ? sv : sk) + j * C::K_PLANE + (c >> 3) * C::K_SLAB + swizzled(r, c & 7)) =
                                make_uint4(plane[0][j], plane[1][j], plane[2][j], plane[3][j]);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t dq = smem_desc_sw128(saddr(sq)), dk = smem_desc_sw128(saddr(sk));
                uint32_t more = 0u;
                // the smallest products first: what they add to is not yet rounded to the size of the result
#pragma unroll
                for (int order = C::ORDERS; order >= 0; --order)
#pragma unroll
                    for (int a = 0; a < QP; ++a) {
                        const int b = order - a;
                        if (b < 0 || b >= KP) continue;
#pragma unroll
                        for (int s = 0; s < SLABS * 4; ++s) {
                            if (s >= ksteps) break;
                            const unsigned off = (unsigned)(s & 3) * 2u;   // 16 columns, in 16-byte units
                            mma_f16(tmem, dq + (a * C::Q_PLANE + (s >> 2) * C::Q_SLAB) / 16 + off,
                                    dk + (b * C::K_PLANE + (s >> 2) * C::K_SLAB) / 16 + off, idesc_s, more);
                            more = 1u;
                        }
                    }
                mma_commit(&s_bar);
            }
            if (!begun) unscale = mine ? s_unscale[tid] : 1.0f;
            bool done = __all_sync(MB_FULL, bar_wait(&s_bar, parity, p.polls));
            parity ^= 1u;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (F16 && done && block + 1 < stop) bring(pk, sk, block + 1);
            // masked: beyond the prefix, or between the first rows and the window
            const bool all = first + KEYS <= keys && (first + KEYS <= seen_head || first >= seen_from);
            float keep = 1.0f;
            if (done && work) {
                uint32_t x[32];
                auto scores = [&](int i) {
                    tmem_ld32u(my_tmem + i * 32, x);
                    tmem_ld_wait(x);
                    if (!__all_sync(MB_FULL, all)) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const unsigned j = first + i * 32 + k;
                            if (!(j < keys && (j < seen_head || j >= seen_from))) x[k] = 0xff800000u;
                        }
                    }
                };
                float m = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < KEYS / 32; ++i) {
                    scores(i);
#pragma unroll
                    for (int k = 0; k < 32; ++k) m = fmaxf(m, __uint_as_float(x[k]));
                }
                m = fmaxf(top, fmaf(m, unscale, -C::WEIGHT_TOP));
                const float ref = m == -INFINITY ? 0.0f : m;
                keep = pow2(top - ref);
                top = m;
                sum *= keep;
#pragma unroll 1
                for (int i = 0; i < KEYS / 32; ++i) {
                    if (KEYS > 32) scores(i);              // one group: still there
                    uint32_t out[QP][16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float a = pow2(fmaf(__uint_as_float(x[2 * k]), unscale, -ref));
                        const float b = pow2(fmaf(__uint_as_float(x[2 * k + 1]), unscale, -ref));
                        sum += a + b;
                        uint32_t plane[QP];
                        split_pair<F16>(a, b, plane);
#pragma unroll
                        for (int l = 0; l < QP; ++l) out[l][k] = plane[l];
                    }
#pragma unroll
                    for (int l = 0; l < QP; ++l) tmem_st16u(my_tmem + C::P + l * (KEYS / 2) + i * 16, out[l]);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            fine = __syncthreads_and(done);
            if (!fine) break;
            if (tid == 0) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t dv = smem_desc_sw128_mn(saddr(sv), C::K_SLAB);
                uint32_t more = 0u;
#pragma unroll
                for (int order = C::ORDERS; order >= 0; --order)
#pragma unroll
                    for (int a = 0; a < QP; ++a) {
                        const int b = order - a;
                        if (b < 0 || b >= KP) continue;
#pragma unroll
                        for (int s = 0; s < KEYS / 16; ++s) {
                            mma_f16_ts(tmem, tmem + C::P + a * (KEYS / 2) + s * 8, dv + (b * C::K_PLANE + s * 2048) / 16, idesc_o, more);
                            more = 1u;
                        }
                    }
                mma_commit(&s_bar);
            }
            done = __all_sync(MB_FULL, bar_wait(&s_bar, parity, p.polls));
            parity ^= 1u;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (F16 && done && block + 1 < stop) bring(pv, sv, block + 1);
            if (done && work) {
#pragma unroll
                for (int i = 0; i < SLABS * 2; ++i) {
                    if (i * 32 >= ncols) break;
                    uint32_t x[32];
                    tmem_ld32u(my_tmem + i * 32, x);
                    tmem_ld_wait(x);
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[i * 32 + j] = fmaf(o[i * 32 + j], keep, __uint_as_float(x[j]));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            fine = __syncthreads_and(done);                // before S and the operands are written again
            if (!fine) break;
        }
        if (fine && mine) {
            const size_t at = of.y + (size_t)tile * TILE * p.heads + (size_t)head * rows + (size_t)blockIdx.x * TILE + tid;
            p.tile_stat[at] = make_float2(top, sum);
#pragma unroll
            for (int i = 0; i < SLABS * 64; i += 4)
                if (i < hw) *reinterpret_cast<float4 *>(p.tile_acc + at * hw + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
    }
    if (!fine) {
        if (tid == 0) {
            atomicOr(p.status, 16);
            bar_wait(&s_bar, parity ^ 1u, TC_SPIN >> 4);   // what may still be in flight, one more bounded chance
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
}

}  // namespace
