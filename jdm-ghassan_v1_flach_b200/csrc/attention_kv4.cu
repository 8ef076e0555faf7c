// Attention of ragged rows over the 4-bit pages (b200serve.h), on mma.sync with the codes themselves as operands.
//
// The mathematics.  A key's element is d code + m (kind 1; kind 0 has m = -8 d) with d, m of its block of 32, so
//   q . K = sum over blocks  d (sum of q code) + m (sum of q)         the last factor is a constant of the query
//   o     = sum over keys    (p d) (code - 8) + p (m + 8 d)           p d goes to the tensor cores, the rest is one number per block
// and the codes need no arithmetic at all: the bits of a code in the low end of an fp16 word are the subnormal code * 2^-24 (or, one nibble
// up, code * 2^-20), exactly, and a product with them is exact too.  One AND makes a pair of operands.
// Queries and p d travel as two fp16 parts in neighbouring columns.  The tensor cores cut what does not fit where they add, sixteen
// times for one product; so the first part is a whole number of at most 2^11 (the power of two comes from the largest element of the
// query, or the largest p d of the tile), whose sums of 32 with codes are whole numbers below 2^20 and never cut, and the second
// the rest, at most 1/2, whose cuts are 2^-12 of those.  (With parts cut by significance instead, scores of +-10 were off by
// 1e-5.)  Together they hold 2^-24 of the largest.  The values' sums start at -8 times the weights, a product with a constant: sums over thousands
// of positive codes would have to lose most of their size again to p m (2e-6 of the output, where it is now below 5e-7).  An accumulator pair added up is one head's sum; what is beyond 32 dims or keys is
// added in fp32 registers, the softmax statistics too.
//   S^T [16 keys, 4 pairs x 2 parts] = K [16 keys, 16 dims] . q^T      keys as rows: a lane has a key's scores and scales together
//   O^T [16 dims, 4 pairs x 2 parts] = V^T [16 dims, 16 keys] . (p d)^T, the weights' fragments turned by movmatrix
// (pair: a query row and one of the heads that share the KV head).
//
// What bounds it: for single tokens the cache, 2 KV (hd/2 + 4 hd/32) bytes a token once (kind 1), with about 730 instructions of a
// warp per 32 keys behind it, which is what the time goes to (57 % of the issue slots; 64 sequences of 256 to 8192 tokens, 32 / 8 heads of
// 128: 55 us, the bytes alone 29); for many rows the instructions more still.
//
// The split.  The lengths are on the device, so the grid is fixed and every warp takes an equal share of all (sequence, KV head, tile of
// 4 or 8 pairs, 32 keys) units laid end to end, with what an item's set-up costs counted in, found from a prefix sum over the batch that
// every block makes by itself.  What a share cuts off an item's ends goes to the workspace and is joined by a second, small kernel.
// (Shares of whole blocks, their warps joined in shared memory: 74 us where this took 64 then, and takes 55 now.  Warps of a block on different pairs of the
// same keys: idle ones where the pairs are no multiple, 149 us on the drafts below.)  Keys come through a ring of each warp's own in
// shared memory that cp.async fills a tile ahead.
#include <algorithm>
#include <type_traits>

#include "serve.cuh"

namespace b200 {

constexpr int A4_WARPS = 4;
constexpr int A4_THREADS = A4_WARPS * 32;
constexpr int A4_KEYS = 32;                      // keys of a warp's step
constexpr int A4_ITEM = 3;                       // what an item's set-up costs, in units
constexpr int A4_LEAST = 2;                      // units of a worker at the least (one sequence of 300 tokens: 9.2 us, of 4: 10.9; 1 and 4097 tokens: more pieces than it saves)
constexpr int A4_STAGES = 2;
// Blocks on an SM, by a warp's tiles of four pairs: 168 registers a thread, or 255.
__host__ __device__ constexpr int a4_resident(int nt) { return nt > 2 ? 2 : 3; }
// A warp's query fragments where they stay in shared memory: 32 registers that two tiles of pairs have more use for.
__host__ __device__ constexpr int a4_query_bytes(int hd, int nt) { return nt > 1 ? nt * (hd / 32) * 32 * 16 : 0; }

struct Kv4AttnArgs {
    const float* q;
    int64_t qs;
    const int32_t* offsets;
    const uint8_t* pages;
    int num_pages;
    const int32_t* table;
    const int32_t* lens;
    float* out;
    int64_t os;
    int batch, max_pages, page, H, KV, group;
    FastDiv by_page, by_group, by_pairs;
    uint32_t page_bytes, k_scale, v_code;        // of a page, and of its parts
    float scale;
    int window;
    int pairs, workers;                          // pairs of a tile; warps of the grid
    float* piece;                                // [2 * workers][pairs][hd + 4]: o, m, l of cut items
    struct A4Item* item;                         // [workers]
};
// What a worker began and left to those behind it: how many of them (0: nothing), the sequence's first row, the tile's first pair
// and its number of pairs, the KV head.
struct __align__(16) A4Item {
    int more, first, pair, live, kv, pad[3];
};

__device__ __forceinline__ void a4_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// from (c0, c1) in both row halves
__device__ __forceinline__ void a4_mma_from(float (&d)[4], float c0, float c1, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t a4_turn(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t a4_pack(float low, float high) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}
__device__ __forceinline__ float a4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int BYTES>
__device__ __forceinline__ void a4_copy(uint32_t dst, const uint8_t* src, bool there) {   // zeros where there is nothing (src is an address all the same)
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}

// A warp's stage: K codes, V codes, K scales, V scales of 32 keys.
template <int HD, int KIND>
struct A4Stage {
    static constexpr int NB = HD / 32;
    static constexpr int ROW = HD / 2;           // bytes of a row's codes
    static constexpr int SROW = NB * (KIND == 1 ? 4 : 2);
    static constexpr int V = A4_KEYS * ROW, KS = 2 * V, VS = KS + A4_KEYS * SROW, BYTES = VS + A4_KEYS * SROW;
};

// d and m of block b among the NB scales of a key held in registers.
template <int KIND, int NB>
struct A4Scales {
    static constexpr int WORDS = KIND == 1 ? NB : NB / 2;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const uint8_t* p) {
        if (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x; w[WORDS > 1 ? 1 : 0] = v.y; w[WORDS > 2 ? 2 : 0] = v.z; w[WORDS > 3 ? 3 : 0] = v.w;
        } else if (WORDS == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[WORDS > 1 ? 1 : 0] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ void get(int b, float& d, float& m) const {
        if (KIND == 1) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[b]));
            d = f.x;
            m = f.y;
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[b / 2]));
            d = b & 1 ? f.y : f.x;
            m = 0.0f;
        }
    }
};

// A sequence's share of the units: rows, length, tiles of pairs, units of an item.
struct A4Seq {
    int first, rows, len, tiles, units;
};
__device__ __forceinline__ A4Seq a4_seq(const Kv4AttnArgs& a, int b) {
    A4Seq s;
    s.first = a.offsets ? a.offsets[b] : b;
    s.rows = a.offsets ? max(a.offsets[b + 1] - s.first, 0) : 1;      // rows * group: q would not fit the device from 2^31 on
    s.len = max(0, min(a.lens[b], a.max_pages * a.page));
    s.tiles = (int)a.by_pairs.div((uint32_t)(s.rows * a.group + a.pairs - 1));
    s.units = max(1, (s.len + A4_KEYS - 1) / A4_KEYS);
    if (a.window > 0) s.units = (int)min((int64_t)s.units, ((int64_t)a.window + a.pairs / a.group + A4_KEYS + 1) / A4_KEYS + 1);
    return s;
}
__device__ __forceinline__ int64_t a4_units(const Kv4AttnArgs& a, const A4Seq& s) { return (int64_t)s.tiles * a.KV * (s.units + A4_ITEM); }

// The keys that the pairs of one tile see, in units: the item's units are first .. first + units - 1, of which those from `end` on
// (keys from key_end on) hold nothing.
struct A4Range {
    int first, key_end;
};
__device__ __forceinline__ A4Range a4_range(const Kv4AttnArgs& a, const A4Seq& s, int tile) {
    const int last = min(s.rows - 1, (int)a.by_group.div((uint32_t)((tile + 1) * a.pairs - 1)));
    A4Range r;
    r.key_end = max(0, s.len - s.rows + last + 1);
    r.first = max(0, (r.key_end + A4_KEYS - 1) / A4_KEYS - s.units);
    return r;
}

template <int HD, int KIND, int NT>
__global__ void __launch_bounds__(A4_THREADS, a4_resident(NT)) attn_kv4_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using ST = A4Stage<HD, KIND>;
    constexpr int NB = ST::NB, PAIRS = 4 * NT, STAGES = A4_STAGES, RING = STAGES * ST::BYTES;
    constexpr uint32_t LOW = 0x000F000Fu, UP = 0x00F000F0u;      // code * 2^-24, code * 2^-20
    constexpr uint32_t LESS_8 = 0x80088008u, LESS_8_UP = 0x80808080u;        // -8 of each
    constexpr float ROUND = 12582912.0f;                         // 1.5 * 2^23
    extern __shared__ __align__(128) uint8_t a4_ring[];
    __shared__ int64_t s_sum[A4_WARPS], s_from[A4_THREADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();

    // ---- this worker's share of the units ----
    const int share = (a.batch + A4_THREADS - 1) / A4_THREADS;
    int64_t mine = 0;
    for (int i = threadIdx.x * share; i < min(a.batch, (int)(threadIdx.x + 1) * share); ++i) mine += a4_units(a, a4_seq(a, i));
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) {
        if (w < warp) upto += s_sum[w];
        all += s_sum[w];
    }
    s_from[threadIdx.x] = upto - mine;
    __syncthreads();
    // the block's workers lie far apart, so that few of them still reach every SM
    const int worker = warp * gridDim.x + blockIdx.x, workers = A4_WARPS * gridDim.x;
    const int64_t per = max((int64_t)A4_LEAST, (all + workers - 1) / workers);
    int64_t u = worker * per;
    const int64_t u_end = min(all, u + per);
    if (lane == 0) a.item[worker].more = 0;
    if (u >= u_end) return;
    int b = -1;                                                  // the last thread whose sequences begin at u or before
#pragma unroll
    for (int i = 0; i < A4_WARPS; ++i) b += __popc(__ballot_sync(0xffffffffu, s_from[32 * i + lane] <= u));
    int64_t rest = u - s_from[b];
    b *= share;
    A4Seq seq = a4_seq(a, b);
    while (rest >= a4_units(a, seq)) {
        rest -= a4_units(a, seq);
        seq = a4_seq(a, ++b);
    }

    const bool halves = a.page % 16 == 0;                        // sixteen keys lie in one page
    constexpr int step = A4_KEYS;
    constexpr bool Q_SHARED = NT > 1;
    uint8_t* ring = a4_ring + warp * RING;
    uint4(*s_q)[32] = reinterpret_cast<uint4(*)[32]>(a4_ring + A4_WARPS * RING + warp * a4_query_bytes(HD, NT));
    const uint32_t ring_at = smem_u32(ring);

    while (true) {
        const int weight = seq.units + A4_ITEM;
        const int64_t item = rest / weight;
        const int w0 = (int)(rest - item * weight), w1 = (int)min((int64_t)weight, w0 + (u_end - u));
        u += w1 - w0;
        rest += w1 - w0;
        const int i0 = max(0, w0 - A4_ITEM), i1 = max(0, w1 - A4_ITEM);
        if (i0 == i1) break;                                     // the share ends before the item's first unit
        const int kv = (int)(item / seq.tiles), tile = (int)(item - (int64_t)kv * seq.tiles);
        const A4Range range = a4_range(a, seq, tile);
        const int kbeg = (range.first + i0) * A4_KEYS, kend = (int)min((int64_t)range.key_end, ((int64_t)range.first + i1) * A4_KEYS);
        const int32_t* table = a.table + (int64_t)b * a.max_pages;
        const int pair0 = tile * PAIRS, npairs = seq.rows * a.group;

        // ---- one tile of 32 keys into stage s ----
        // A lane brings pieces of 16 bytes of its half's keys, PER keys of the half a round.  K rows stand in the order in which the fragments take them,
        // V rows as they come, the pieces of every other pair of rows swapped so that four rows one apart miss each other's banks.
        constexpr int CH = ST::ROW / 16, PER = 16 / CH;
        const int hkey = lane % 16 / CH, lkey = (lane & 16) + hkey, lpiece = lane % CH * 16;
        const uint32_t kdst = ring_at + ((lane & 16) + 2 * (hkey & 3) + (hkey >> 2)) * ST::ROW + lpiece;
        const uint32_t vdst = ring_at + ST::V + lkey * ST::ROW + (HD == 128 ? lpiece ^ ((lkey & 2) * 16) : lpiece);
        const uint32_t sdst = ring_at + ST::KS + lane * ST::SROW;
        auto k_round = [](int i) { return HD == 128 ? (i >> 1) * 8 + (i & 1) : 8 * i; };           // rows on, in K's order
        const int kv_row = kv * a.page;
        // Page and token in it of the tile's keys: a lane has the first key of its half (sixteen keys lie in one page), or, where pages do
        // not allow that, its own key.
        struct Place {
            int id, off;
        };
        auto place = [&](int k) {
            Place pl{-1, 0};
            if (k < kend) {
                const int key = min(k + (halves ? lane & 16 : lane), kend - 1), p = (int)a.by_page.div(key);
                pl.id = table[p];
                pl.off = key - p * a.page;
            }
            return pl;
        };
        auto issue = [&](int s, int k, Place pl) {
            const uint32_t so = s * ST::BYTES;
            const bool there = (uint32_t)pl.id < (uint32_t)a.num_pages;
            const uint8_t* at = a.pages + (uint64_t)(there ? (uint32_t)pl.id : 0u) * a.page_bytes;
            const uint8_t* codes = at + (uint32_t)(kv_row + pl.off) * ST::ROW;
            const uint8_t* scales = at + a.k_scale + (uint32_t)(kv_row + pl.off + (halves ? lane & 15 : 0)) * ST::SROW;
            if (halves) {
                const uint8_t* p = codes + hkey * ST::ROW + lpiece;
                if (k + A4_KEYS <= kend) {
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        a4_copy<16>(kdst + so + k_round(i) * ST::ROW, p + i * PER * ST::ROW, there);
                        a4_copy<16>(vdst + so + i * PER * ST::ROW, p + a.v_code + i * PER * ST::ROW, there);
                    }
                    a4_copy<ST::SROW>(sdst + so, scales, there);
                    a4_copy<ST::SROW>(sdst + so + (ST::VS - ST::KS), scales + a.v_code, there);      // V's parts follow K's in the same order
                    return;
                }
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const bool ok = there && k + lkey + i * PER < kend;
                    const uint8_t* from = ok ? p + i * PER * ST::ROW : a.pages;
                    a4_copy<16>(kdst + so + k_round(i) * ST::ROW, from, ok);
                    a4_copy<16>(vdst + so + i * PER * ST::ROW, from + a.v_code, ok);
                }
            } else {
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int key_of = lkey + i * PER;
                    const uint8_t* p = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(codes), key_of)) + lpiece;
                    const bool ok = __shfl_sync(0xffffffffu, there, key_of) && k + key_of < kend;
                    a4_copy<16>(kdst + so + k_round(i) * ST::ROW, p, ok);
                    a4_copy<16>(vdst + so + i * PER * ST::ROW, p + a.v_code, ok);
                }
            }
            const bool ok = there && k + lane < kend;
            const uint8_t* from = ok ? scales : a.pages;
            a4_copy<ST::SROW>(sdst + so, from, ok);
            a4_copy<ST::SROW>(sdst + so + (ST::VS - ST::KS), from + a.v_code, ok);
        };
        auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

        int k = kbeg;
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            if (k + s * step < kend) issue(s, k + s * step, place(k + s * step));
            commit();
        }
        Place next = place(k + (STAGES - 1) * step);

        // ---- queries: parts of q 2^e as B fragments, sums of each block ----
        uint32_t qf[NT][NB][2][2];                                // NT > 1: kept in shared memory
        float qsum[NT][NB], less[NT][NB][2], unit[NT];            // kind 1: sums of the blocks; kind 0: -8 times those of the parts
        int lim[NT], from[NT];
        int all_see = 0x7fffffff, none_before = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int p = pair0 + 4 * j + (g >> 1);
            const bool live = p < npairs;
            const int row = live ? (int)a.by_group.div(p) : 0;
            const float* q = a.q + (int64_t)(seq.first + row) * a.qs + ((int64_t)kv * a.group + (live ? p - row * a.group : 0)) * HD + 8 * t;
            float x[NB][8], top = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
                if (live) {
                    lo = __ldg(reinterpret_cast<const float4*>(q + 32 * n));
                    hi = __ldg(reinterpret_cast<const float4*>(q + 32 * n + 4));
                }
                x[n][0] = lo.x; x[n][1] = lo.y; x[n][2] = lo.z; x[n][3] = lo.w;
                x[n][4] = hi.x; x[n][5] = hi.y; x[n][6] = hi.z; x[n][7] = hi.w;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[n][i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = max((int)(__float_as_uint(top) >> 23), 14);             // top < 2^(e - 126)
            const float mul = __uint_as_float((uint32_t)(264 - e) << 23);         // 2^(137 - e): top * mul < 2^11
            const float back = __uint_as_float((uint32_t)(e == 255 ? 254 : e) << 23) * 16384.0f;     // 2^24 / mul
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float sum = 0.0f, rest = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // nibble i of two words, elements i and 4 + i; an odd nibble's codes come 16 times too large
                    const float f = i & 1 ? 0.0625f : 1.0f, u0 = x[n][i] * mul, u1 = x[n][4 + i] * mul, h0 = rintf(u0), h1 = rintf(u1);
                    const uint32_t low = a4_pack((u0 - h0) * f, (u1 - h1) * f);
                    qf[j][n][i >> 1][i & 1] = g & 1 ? low : a4_pack(h0 * f, h1 * f);
                    if (KIND == 0) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&low));
                        sum += h0 + h1;
                        rest += (r.x + r.y) * (i & 1 ? 16.0f : 1.0f);
                    } else {
                        sum += u0 + u1;
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (KIND == 1) qsum[j][n] = __shfl_sync(0xffffffffu, sum * 0x1p-24f, 8 * t);
                if (KIND == 0) {
                    rest += __shfl_xor_sync(0xffffffffu, rest, 1);
                    rest += __shfl_xor_sync(0xffffffffu, rest, 2);
                    less[j][n][0] = __shfl_sync(0xffffffffu, sum * -0x1p-21f, 8 * t);
                    less[j][n][1] = __shfl_sync(0xffffffffu, rest * -0x1p-21f, 8 * t);
                }
            }
            if (Q_SHARED) {
#pragma unroll
                for (int n = 0; n < NB; ++n) s_q[j * NB + n][lane] = make_uint4(qf[j][n][0][0], qf[j][n][0][1], qf[j][n][1][0], qf[j][n][1][1]);
            }
            unit[j] = __shfl_sync(0xffffffffu, back, 8 * t) * (a.scale * 1.4426950408889634f);       // to powers of two
            const int pt = pair0 + 4 * j + t;
            const int pos = pt < npairs ? seq.len - seq.rows + (int)a.by_group.div(pt) : 0x7ffffffe;
            lim[j] = pos + 1;
            from[j] = a.window > 0 && pt < npairs ? max(0, pos - a.window + 1) : 0;
            all_see = min(all_see, lim[j]);
            none_before = max(none_before, from[j]);
        }
        all_see = __reduce_min_sync(0xffffffffu, all_see);
        none_before = __reduce_max_sync(0xffffffffu, none_before);

        float o[NT][2 * NB][2], m[NT], l[NT];
        f32x2 bias[NT][NB];                                      // of even and odd keys
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            m[j] = -INFINITY;
            l[j] = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                bias[j][n] = 0;
                o[j][2 * n][0] = o[j][2 * n][1] = o[j][2 * n + 1][0] = o[j][2 * n + 1][1] = 0.0f;
            }
        }
        const int kk = (g >> 1) + 4 * (g & 1);                    // key (of 8) that fragment row g is

        for (int s = 0; k < kend; k += step, s = s + 1 == STAGES ? 0 : s + 1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();                                         // this tile is here, and the one before it is read
            {
                const int ahead = k + (STAGES - 1) * step;
                if (ahead < kend) issue(s == 0 ? STAGES - 1 : s - 1, ahead, next);
                commit();
                next = place(ahead + step);
            }
            const uint8_t* st = ring + s * ST::BYTES;

            // ---- scores ----
            f32x2 x2[NT][2];                                     // of key rows g and g + 8
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[2][NB];                                // of key rows g and g + 8: nibble i of word t's two halves
                A4Scales<KIND, NB> sc[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint8_t* p = st + (16 * h + 8 * r + g) * ST::ROW;
                    if (HD == 128) {
                        const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * t);
                        w[r][0] = __byte_perm(v.x, v.z, 0x5410);
                        w[r][1] = __byte_perm(v.x, v.z, 0x7632);
                        w[r][NB > 2 ? 2 : 0] = __byte_perm(v.y, v.w, 0x5410);
                        w[r][NB > 2 ? 3 : 0] = __byte_perm(v.y, v.w, 0x7632);
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(p + 8 * t);
                        w[r][0] = __byte_perm(v.x, v.y, 0x5410);
                        w[r][1] = __byte_perm(v.x, v.y, 0x7632);
                    }
                    sc[r].load(st + ST::KS + (16 * h + 8 * r + kk) * ST::SROW);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) x2[j][h] = 0;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t s0 = w[0][n] >> 8, s1 = w[1][n] >> 8;
                    float d0, m0, d1, m1;
                    sc[0].get(n, d0, m0);
                    sc[1].get(n, d1, m1);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float c[4];
                        const uint4 f = Q_SHARED ? s_q[j * NB + n][lane] : make_uint4(qf[j][n][0][0], qf[j][n][0][1], qf[j][n][1][0], qf[j][n][1][1]);
                        if (KIND == 0) a4_mma_from(c, less[j][n][0], less[j][n][1], w[0][n] & LOW, w[1][n] & LOW, w[0][n] & UP, w[1][n] & UP, f.x, f.y);
                        else a4_mma0(c, w[0][n] & LOW, w[1][n] & LOW, w[0][n] & UP, w[1][n] & UP, f.x, f.y);
                        a4_mma(c, s0 & LOW, s1 & LOW, s0 & UP, s1 & UP, f.z, f.w);
                        x2[j][h] = fma2(two(d0, d1), two(c[0] + c[1], c[2] + c[3]), x2[j][h]);
                        if (KIND == 1) x2[j][h] = fma2(two(m0, m1), two(qsum[j][n], qsum[j][n]), x2[j][h]);
                    }
                }
            }
            // ---- softmax ----
            const bool cut = k + A4_KEYS > all_see || k < none_before;
            bool grown = false;
            float top[NT], here[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float v = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x2[j][h] = mul2(x2[j][h], two(unit[j], unit[j]));
                    float2 x = each(x2[j][h]);
                    if (cut) {
                        const int key = k + 16 * h + kk;
                        if (key >= lim[j] || key < from[j]) x.x = -INFINITY;
                        if (key + 8 >= lim[j] || key + 8 < from[j]) x.y = -INFINITY;
                        x2[j][h] = two(x.x, x.y);
                    }
                    v = fmaxf(v, fmaxf(x.x, x.y));
                }
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                here[j] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                top[j] = fmaxf(m[j], here[j]);
                grown |= top[j] != m[j];
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float f = m[j] == top[j] ? 1.0f : a4_exp2(m[j] - top[j]);
                    m[j] = top[j];
                    l[j] *= f;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        if (KIND == 1) bias[j][n] = mul2(bias[j][n], two(f, f));
                        o[j][2 * n][0] *= f; o[j][2 * n][1] *= f;
                        o[j][2 * n + 1][0] *= f; o[j][2 * n + 1][1] *= f;
                    }
                }
            }
            // ---- values ----
            A4Scales<KIND, NB> sv[4];
            uint32_t top_d = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sv[i].load(st + ST::VS + (8 * i + kk) * ST::SROW);
#pragma unroll
                for (int n = 0; n < A4Scales<KIND, NB>::WORDS; ++n) top_d = __vmaxu2(top_d, sv[i].w[n]);      // kind 1: m beside it, unused
            }
            if (KIND == 0) top_d = max(top_d & 0xFFFFu, top_d >> 16);
            const float largest = half_bits_to_float((uint16_t)(__reduce_max_sync(0xffffffffu, top_d & 0x7FFFu)));
            f32x2 pg[NT][2], less_pg[NT][2];                     // weights times grow, and their negatives
            float shrink[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float base = m[j] == -INFINITY ? 0.0f : m[j];
                // every p d of the tile < 2^(e - 126) (or a rounding above)
                const uint32_t e = max(__float_as_uint(a4_exp2(here[j] - base) * largest) >> 23, 11u);
                const float grow = __uint_as_float((264u - e) << 23);             // 2^(137 - e): p d grow < 2^11
                shrink[j] = __uint_as_float((14u + e) << 23);                     // 2^24 / grow
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 x = each(add2(x2[j][h], two(-base, -base)));
                    const float p0 = a4_exp2(x.x), p1 = a4_exp2(x.y);
                    l[j] += p0 + p1;
                    x2[j][h] = two(p0, p1);
                    pg[j][h] = mul2(x2[j][h], two(grow, grow));
                    less_pg[j][h] = mul2(x2[j][h], two(-grow, -grow));
                }
            }
            uint32_t vx[8], vy[8];                                // of keys t, t + 4, .. t + 28: the words of dims 4 g .. 4 g + 3
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint8_t* p = st + ST::V + (4 * i + t) * ST::ROW;
                if (HD == 128) {
                    const uint2 v = *reinterpret_cast<const uint2*>(p + (((g >> 1) ^ (t & 2)) * 16 + (g & 1) * 8));
                    vx[i] = v.x;
                    vy[i] = v.y;
                } else {
                    vx[i] = *reinterpret_cast<const uint32_t*>(p + 4 * g);
                    vy[i] = 0;
                }
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                uint32_t pb[NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float d0, m0, d1, m1;
                    sv[2 * h].get(n, d0, m0);
                    sv[2 * h + 1].get(n, d1, m1);
                    const f32x2 d = two(d0, d1), m8 = KIND == 1 ? fma2(two(8.0f, 8.0f), d, two(m0, m1)) : 0;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        // minus the nearest whole number, and what is left: the first column comes out negative
                        const f32x2 less_whole = add2(fma2(less_pg[j][h], d, two(ROUND, ROUND)), two(-ROUND, -ROUND));
                        const float2 hi = each(less_whole), lo = each(fma2(pg[j][h], d, less_whole));
                        pb[j][2 * h] = a4_turn(a4_pack(hi.x, lo.x));
                        pb[j][2 * h + 1] = a4_turn(a4_pack(hi.y, lo.y));
                        if (KIND == 1) bias[j][n] = fma2(x2[j][h], m8, bias[j][n]);
                    }
                }
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = n < 2 ? __byte_perm(vx[2 * i], vx[2 * i + 1], n & 1 ? 0x7632 : 0x5410) : __byte_perm(vy[2 * i], vy[2 * i + 1], n & 1 ? 0x7632 : 0x5410);
                float eights[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    a4_mma0(eights[j], LESS_8, LESS_8_UP, LESS_8, LESS_8_UP, pb[j][0], pb[j][1]);
                    a4_mma(eights[j], LESS_8, LESS_8_UP, LESS_8, LESS_8_UP, pb[j][2], pb[j][3]);
                }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float c[4] = {eights[j][0], eights[j][1], eights[j][2], eights[j][3]};
                        a4_mma(c, w[0] & LOW, w[0] & UP, w[1] & LOW, w[1] & UP, pb[j][0], pb[j][1]);
                        a4_mma(c, w[2] & LOW, w[2] & UP, w[3] & LOW, w[3] & UP, pb[j][2], pb[j][3]);
                        o[j][2 * n + v][0] = fmaf(c[1] - c[0], shrink[j], o[j][2 * n + v][0]);
                        o[j][2 * n + v][1] = fmaf(c[3] - c[2], shrink[j], o[j][2 * n + v][1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] >>= 8;
                }
            }
        }
        // ---- the lanes' sums ----
        const bool whole = i0 == 0 && i1 == seq.units;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float rest_of[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const float2 y = each(bias[j][n]);
                rest_of[n] = y.x + y.y;
            }
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) {
                l[j] += __shfl_xor_sync(0xffffffffu, l[j], sh);
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    if (KIND == 1) rest_of[n] += __shfl_xor_sync(0xffffffffu, rest_of[n], sh);
            }
            const int p = pair0 + 4 * j + t;
            if (p >= npairs) continue;
            const int row = (int)a.by_group.div(p);
            float* piece = a.piece + ((int64_t)(2 * worker + (i0 == 0)) * PAIRS + 4 * j + t) * (HD + 4);
            float* dst = whole ? a.out + (int64_t)(seq.first + row) * a.os + ((int64_t)kv * a.group + (p - row * a.group)) * HD : piece;
            const float mul = !whole ? 1.0f : l[j] == 0.0f ? 0.0f : 1.0f / l[j];
#pragma unroll
            for (int n = 0; n < NB; ++n)
                *reinterpret_cast<float4*>(dst + 32 * n + 4 * g) =
                    make_float4((o[j][2 * n][0] + rest_of[n]) * mul, fmaf(o[j][2 * n][1], 0.0625f, rest_of[n]) * mul,
                                (o[j][2 * n + 1][0] + rest_of[n]) * mul, fmaf(o[j][2 * n + 1][1], 0.0625f, rest_of[n]) * mul);
            if (!whole && g == 0) {
                piece[HD] = m[j];
                piece[HD + 1] = l[j];
            }
        }
        if (i0 == 0 && !whole && lane == 0)         // units of this item with the workers that follow
            a.item[worker] = A4Item{(int)((seq.units - i1 + per - 1) / per), seq.first, pair0, min(PAIRS, npairs - pair0), kv, {0, 0, 0}};
        if (u >= u_end) break;
        if (rest >= a4_units(a, seq)) {
            rest = 0;
            do seq = a4_seq(a, ++b); while (seq.rows == 0);       // there is one: units are left
        }
        __syncwarp();                                             // the ring is read
    }
}

// Items that a worker began and others went on with, a block each: a thread per four dims of a pair and group of pieces, AT_ONCE pieces at
// a time.  Many items have few pieces: a block with a thread per column or two for every worker, which reads the pieces that there would
// be at the same time as how many there are.  Few items, that is few sequences, have many: large blocks for several workers each.
template <int HD, int THREADS, int AT_ONCE>
__global__ void __launch_bounds__(THREADS, 4096 / AT_ONCE / THREADS) attn_kv4_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
    __shared__ float4 s_o[THREADS];
    __shared__ float2 s_ml[THREADS];
    const int columns = a.pairs * (HD / 4), groups = THREADS / columns, lane = threadIdx.x & 31;
    const int group = threadIdx.x / columns, col = threadIdx.x % columns, p = col / (HD / 4), c = col % (HD / 4) * 4;
    pdl_wait();
    unsigned left = 1;                                           // bit k: worker blockIdx.x + k gridDim.x began something
    if (gridDim.x < (unsigned)a.workers) {
        const int mine = blockIdx.x + lane * gridDim.x;
        left = __ballot_sync(0xffffffffu, mine < a.workers && __ldcg(&a.item[min(mine, a.workers - 1)].more) > 0);
    }
    for (; left; left &= left - 1) {
        const int worker = blockIdx.x + (__ffs(left) - 1) * gridDim.x;
        // piece i: the worker's own second slot, then the first slots of those behind it
        const float* pieces = a.piece + ((int64_t)(2 * worker) * a.pairs + p) * (HD + 4);
        float2 ml[AT_ONCE];
        float4 v[AT_ONCE];
        auto load = [&](int i0, int most) {
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int i = i0 + k * groups;
                if (i <= most) {
                    const float* s = pieces + (int64_t)(2 * i + (i == 0)) * a.pairs * (HD + 4);
                    ml[k] = __ldcg(reinterpret_cast<const float2*>(s + HD));
                    v[k] = __ldcg(reinterpret_cast<const float4*>(s + c));
                }
            }
        };
        load(group, a.workers - 1 - worker);
        const A4Item it = a.item[worker];
        if (it.more == 0) continue;
        float mm = -INFINITY, ll = 0.0f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = group; i0 <= it.more; i0 += AT_ONCE * groups) {
            if (i0 != group) load(i0, it.more);
            float top = mm;
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                if (i0 + k * groups > it.more) {                 // not there, whatever was read
                    ml[k] = make_float2(-INFINITY, 0.0f);
                    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                top = fmaxf(top, ml[k].x);
            }
            const float base = top == -INFINITY ? 0.0f : top, old = a4_exp2(mm - base);
            ll *= old;
            acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const float f = a4_exp2(ml[k].x - base);
                ll = fmaf(ml[k].y, f, ll);
                acc.x = fmaf(v[k].x, f, acc.x); acc.y = fmaf(v[k].y, f, acc.y); acc.z = fmaf(v[k].z, f, acc.z); acc.w = fmaf(v[k].w, f, acc.w);
            }
            mm = top;
        }
        if (groups > 1) {
            __syncthreads();                                     // the item before is read
            s_o[threadIdx.x] = acc;
            s_ml[threadIdx.x] = make_float2(mm, ll);
            __syncthreads();
            if (group == 0)
                for (int i = 1; i < groups; ++i) {
                    const float2 other = s_ml[i * columns + threadIdx.x];
                    const float4 w = s_o[i * columns + threadIdx.x];
                    const float top = fmaxf(mm, other.x), base = top == -INFINITY ? 0.0f : top, f0 = a4_exp2(mm - base), f1 = a4_exp2(other.x - base);
                    ll = ll * f0 + other.y * f1;
                    acc.x = acc.x * f0 + w.x * f1; acc.y = acc.y * f0 + w.y * f1; acc.z = acc.z * f0 + w.z * f1; acc.w = acc.w * f0 + w.w * f1;
                    mm = top;
                }
        }
        if (group == 0 && p < it.live) {
            const int row = (int)a.by_group.div(it.pair + p);
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            float* dst = a.out + (int64_t)(it.first + row) * a.os + ((int64_t)it.kv * a.group + (it.pair + p - row * a.group)) * HD + c;
            *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
    }
}

template <int HD>
static int launch_a4_join(const Kv4AttnArgs& a, int items) {
    constexpr int THREADS = 2 * HD, AT_ONCE = 4;
    if (a.pairs > 8)
        return launch_serve("attn_kv4_join_kernel", attn_kv4_join_kernel<HD, 4 * HD, 4>, dim3(a.workers), dim3(4 * HD), 0, 1, true, a);
    if (items > num_sms()) return launch_serve("attn_kv4_join_kernel", attn_kv4_join_kernel<HD, THREADS, AT_ONCE>, dim3(a.workers), dim3(THREADS), 0, 1, true, a);
    return launch_serve("attn_kv4_join_kernel", attn_kv4_join_kernel<HD, 512, 8>, dim3(num_sms()), dim3(512), 0, 1, true, a);
}

// Tiles of four pairs that a warp takes at once, from the most pairs that a sequence has for a KV head.  A tile's keys are unpacked
// once for all of its pairs, but pairs that are not there cost as much as others: 16 sequences, 5 rows of 32/8 heads (20 pairs)
// 69 us in eights, 84 in sixteens; 72 pairs of 12/4 heads 93 and 101; 96 pairs 223 and 212; prompts' pieces of 300 to 900 pairs 84 and 79.
static int a4_tiles(int64_t most) { return most <= 4 ? 1 : most <= 128 ? 2 : 4; }
static int a4_blocks(int nt) { return a4_resident(nt) * num_sms(); }

template <int HD, int KIND, int NT>
static int launch_a4(const Kv4AttnArgs& a, int blocks) {
    auto kern = attn_kv4_kernel<HD, KIND, NT>;
    constexpr int smem = A4_WARPS * (A4_STAGES * A4Stage<HD, KIND>::BYTES + a4_query_bytes(HD, NT));
    if (smem + 2048 > 48 * 1024) B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return launch_serve("attn_kv4_kernel", kern, dim3(blocks), dim3(A4_THREADS), smem, 1, true, a);
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_attention_paged_kv4_workspace(int H, int KV, int hd, int max_rows, size_t* bytes) {
    int rc = kv4_check("attention_paged_kv4_workspace", 1, 1, KV, hd, 0);
    if (rc) return rc;
    B200_REQUIRE(bytes, "attention_paged_kv4_workspace: null pointer");
    B200_REQUIRE(H >= 1 && H % KV == 0 && max_rows >= 1, "attention_paged_kv4_workspace: H must be a positive multiple of KV, max_rows positive");
    const int nt = a4_tiles((int64_t)max_rows * (H / KV));
    *bytes = (size_t)a4_blocks(nt) * A4_WARPS * (sizeof(A4Item) + (size_t)2 * 4 * nt * (hd + 4) * sizeof(float));
    return B200_OK;
}

int b200_attention_paged_kv4(const float* q, int64_t q_stride, const int32_t* row_offsets, const void* pages, int num_pages,
                             const int32_t* page_table, const int32_t* seq_lens, float* out, int64_t out_stride, int batch,
                             int max_rows, int max_pages, int page, int H, int KV, int hd, int kind, float scale, int window,
                             void* workspace, size_t workspace_bytes) {
    if (batch <= 0) return B200_OK;
    const char* who = "attention_paged_kv4";
    int rc = kv4_check(who, num_pages, page, KV, hd, kind);
    if (rc) return rc;
    B200_REQUIRE(H >= 1 && H % KV == 0, "%s: H must be a positive multiple of KV", who);
    B200_REQUIRE(batch <= 1 << 24, "%s: too many sequences", who);
    if (window >= (int64_t)max_pages * page) window = 0;         // wider than any sequence
    B200_REQUIRE(max_rows >= 1 && max_pages >= 1 && (int64_t)max_pages * page <= 0x7fffff00, "%s: bad max_rows or max_pages", who);
    B200_REQUIRE(q && pages && page_table && seq_lens && out && workspace, "%s: null pointer", who);
    B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(pages) && aligned16(workspace) && q_stride % 4 == 0 && out_stride % 4 == 0,
                 "%s: q, out, pages and workspace must be 16-byte aligned, strides multiples of 4", who);
    B200_REQUIRE(q_stride >= (int64_t)H * hd && out_stride >= (int64_t)H * hd, "%s: a stride is shorter than its row", who);
    size_t need = 0;
    rc = b200_attention_paged_kv4_workspace(H, KV, hd, max_rows, &need);
    if (rc) return rc;
    B200_REQUIRE(workspace_bytes >= need, "%s: the workspace has %zu bytes of %zu", who, workspace_bytes, need);
    const int nt = a4_tiles((int64_t)max_rows * (H / KV)), blocks = a4_blocks(nt), workers = blocks * A4_WARPS;
    const Kv4Page part(page, KV, hd, kind);
    Kv4AttnArgs a{q, q_stride, row_offsets, static_cast<const uint8_t*>(pages), num_pages, page_table, seq_lens, out, out_stride, batch,
                  max_pages, page, H, KV, H / KV, FastDiv(page), FastDiv(H / KV), FastDiv(4 * nt), (uint32_t)part.bytes, (uint32_t)part.k_scale, (uint32_t)part.v_code, scale, window, 4 * nt, workers,
                  reinterpret_cast<float*>(static_cast<A4Item*>(workspace) + workers), static_cast<A4Item*>(workspace)};
    auto go = [&](auto tiles) {
        constexpr int NT = decltype(tiles)::value;
        return hd == 64 ? (kind == 1 ? launch_a4<64, 1, NT>(a, blocks) : launch_a4<64, 0, NT>(a, blocks))
                        : (kind == 1 ? launch_a4<128, 1, NT>(a, blocks) : launch_a4<128, 0, NT>(a, blocks));
    };
    rc = nt == 1 ? go(std::integral_constant<int, 1>()) : nt == 2 ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 4>());
    if (rc) return rc;
    const int64_t items = (int64_t)batch * KV * (((int64_t)max_rows * (H / KV) + a.pairs - 1) / a.pairs);       // at the most
    return hd == 64 ? launch_a4_join<64>(a, (int)std::min<int64_t>(items, 1 << 30)) : launch_a4_join<128>(a, (int)std::min<int64_t>(items, 1 << 30));
}

}  // extern "C"
