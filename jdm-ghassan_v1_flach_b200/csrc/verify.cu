// Drafted tokens against the target's probabilities, from given uniforms.
//
// Two kernels.  The first reads every row of logits once, a chunk per block, and leaves its largest value, where that stands,
// and the sum of 2^(l c - R), c = log2(e) / T.  The second has a cluster of eight blocks per sequence: each joins the chunks of the
// sequence's rows by itself (a few hundred words), decides how many drafts are kept, and then sums its eighth of the one row that the
// next token is drawn from, a segment per warp; the 64 segments' masses are exchanged through the cluster's shared memory, and
// the block that holds the draw walks its segment again.  Mass i is e_i - q_i Z with e_i the weight: nothing is divided by Z.
//
// A check misses by rounding when u falls within its error of p(x) / q(x), 1e-6 of it: fp32 weights do, and the first kernel waits for the logits (4 V
// bytes a row).  A draw misses when u falls within the sums' error of any of 100 000 borders: with weights off by 2^-25 of themselves at
// random, one draw in 10 000 (counted on rows of variance 6).  So the second kernel makes its weights to 2^-29: the argument as two fp32
// numbers, a whole number R taken from it instead of the largest logit (exact, and chunks are joined by powers of
// two), 2^y = 2^(n/16) 2^f with the sixteen powers kept in two parts and 2^f - 1, at most 1/32, from its series; its sums run in
// fp64; and where a drafter's q is taken off it sums Z once more in the same way.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "serve.cuh"

namespace b200 {

namespace cg = cooperative_groups;

constexpr int VD_THREADS = 256;
constexpr int VD_WARPS = VD_THREADS / 32;
constexpr int VD_CHUNK = VD_THREADS * 8;          // logits of a chunk at the least, which sizes the workspace
constexpr int VD_RESIDENT = 4;                    // blocks on an SM (the second kernel's 64 x 8 all at once)
constexpr int VD_CLUSTER = 8;
constexpr int VD_MAX_DRAFTS = 255;
constexpr int VD_ROUND = 64;                      // steps of 128 logits that a block walks at a time

struct __align__(16) VdPart {                     // of one chunk of one row
    double sum;
    float top;
    int at;                                       // -1: no logit above -inf
};

struct VerifyArgs {
    const float* logits;
    int64_t ls;
    const float* draft;
    int64_t ds;
    const int32_t *ids, *offsets;
    int batch, rows, V, chunks;
    float c_hi, c_lo;                             // log2(e) / temperature
    double c, inv_c;
    int chunk;                                    // logits of a chunk, whole steps of 1024
    const float* uniforms;
    int max_drafts;
    int32_t *accepted, *tokens;
    VdPart* part;
};

// What a row's (or chunk's) weights are taken relative to: weight = 2^((l - s) c - r).  r is whole, and s 0 but for logits so large that l c is
// no number to work with; there l - s is exact for every l whose weight counts.
struct VdRef {
    float s;
    int r;
};
__device__ __forceinline__ VdRef vd_ref(const VerifyArgs& a, float top) {
    const float y = top * a.c_hi;
    return fabsf(y) < 30000.0f ? VdRef{0.0f, (int)rintf(y)} : VdRef{top, 0};
}
// 2^(from's exponent - to's): sums taken relative to `from` times this are relative to `to`; from <= to.
__device__ __forceinline__ double vd_rescale(const VerifyArgs& a, float from_top, float to_top) {
    if (from_top == to_top) return 1.0;
    if (isinf(to_top) || isinf(from_top)) return 0.0;
    const VdRef f = vd_ref(a, from_top), t = vd_ref(a, to_top);
    if (f.s == 0.0f && t.s == 0.0f) {
        const int d = f.r - t.r;                  // at most 0
        return d < -1022 ? 0.0 : __hiloint2double((1023 + d) << 20, 0);
    }
    return exp2(((double)f.s - (double)t.s) * a.c + (double)(f.r - t.r));
}

// 2^(k/16), made by every block for itself: the bits of its fp32 value less k << 19, so that adding n << 19 gives 2^(n/16); and
// what the rounding left, relative to it.
__device__ __forceinline__ void vd_table(int2* s_pow) {
    if (threadIdx.x < 16) {
        const double p = exp2(threadIdx.x / 16.0);
        s_pow[threadIdx.x] = make_int2(__float_as_int((float)p) - (int)(threadIdx.x << 19), __float_as_int((float)((p - (double)(float)p) / p)));
    }
}
// What the weights of one row or chunk have in common.
struct VdWeights {
    const int2* s_pow;
    float c_hi, c_lo, s, least;                   // below `least` the weight is under 2^-120 of the largest, and 0
    int shift;                                    // -r, where an exponent stands
    // The weights of two logits as hi + lo, hi the sum's fp32 value.  NaN and -inf have none.
    __device__ __forceinline__ void operator()(float l0, float l1, float2& hi, float2& lo) const {
        const f32x2 round = two(12582912.0f, 12582912.0f), less_round = two(-12582912.0f, -12582912.0f);      // 1.5 * 2^23
        const f32x2 c = two(c_hi, c_hi), x = add2(two(fmaxf(l0, least), fmaxf(l1, least)), two(-s, -s));
        const f32x2 t = mul2(x, c), low = fma2(x, two(c_lo, c_lo), fma2(x, c, mul2(x, two(-c_hi, -c_hi))));
        const f32x2 z = fma2(t, two(16.0f, 16.0f), round), n = add2(z, less_round);      // the low bits of z are those of n
        const f32x2 f = add2(fma2(n, two(-0.0625f, -0.0625f), t), low);
        const float2 zz = each(z);
        const int i0 = __float_as_int(zz.x), i1 = __float_as_int(zz.y);
        const int2 p0 = s_pow[i0 & 15], p1 = s_pow[i1 & 15];
        f32x2 g = fma2(f, two(9.6181291e-3f, 9.6181291e-3f), two(5.5504109e-2f, 5.5504109e-2f));              // ln(2)^k / k!
        g = fma2(f, g, two(0.24022651f, 0.24022651f));
        g = fma2(f, g, two(0.69314718f, 0.69314718f));
        g = fma2(f, g, two(__int_as_float(p0.y), __int_as_float(p1.y)));
        const f32x2 p = two(l0 >= least ? __int_as_float(p0.x + (i0 << 19) + shift) : 0.0f, l1 >= least ? __int_as_float(p1.x + (i1 << 19) + shift) : 0.0f);
        const f32x2 less = two(-1.0f, -1.0f), pg = mul2(p, g), sum = add2(p, pg);        // pg is at most p / 32
        hi = each(sum);
        lo = each(fma2(fma2(p, less, sum), less, pg));                                   // what rounding the sum cut off
    }
};
__device__ __forceinline__ VdWeights vd_weights(const VerifyArgs& a, const int2* s_pow, float top) {
    const VdRef ref = vd_ref(a, top);
    const float least = ref.s + (float)((double)(ref.r - 120) * a.inv_c);
    return VdWeights{s_pow, a.c_hi, a.c_lo, ref.s, fmaxf(least, -3.402823466e38f), (int)((unsigned)-ref.r << 23)};
}

struct VdBest {
    float v;
    int i;
};
__device__ __forceinline__ VdBest vd_better(VdBest a, VdBest b) {    // larger value, then lower index; -1: none
    if (b.i < 0) return a;
    if (a.i < 0) return b;
    return a.v > b.v || (a.v == b.v && a.i < b.i) ? a : b;
}
__device__ __forceinline__ VdBest vd_warp_best(VdBest a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = vd_better(a, VdBest{__shfl_xor_sync(0xffffffffu, a.v, o), __shfl_xor_sync(0xffffffffu, a.i, o)});
    return a;
}

// grid (chunks, rows).  A thread takes sixteen logits of every 4096, the next ones under way, and adds them up relative to the largest of its
// first; the threads' sums meet at the end.  (`top` of a part is then what its sum is relative to, no more than 60 / c below the largest.)
template <bool WIDE, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS, VD_RESIDENT) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int HALF = 4 * VD_THREADS, EACH = 16, STEP = VD_THREADS * EACH;
    __shared__ VdPart s_part[VD_WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int live = min(a.offsets[a.batch], a.rows), c0 = blockIdx.x * a.chunk, c1 = min(a.V, c0 + a.chunk);
    for (int row = blockIdx.y; row < live; row += gridDim.y) {
        const float* l = a.logits + row * a.ls;
        auto load = [&](int at, float (&x)[EACH]) {
#pragma unroll
            for (int i = 0; i < EACH / 4; ++i) {
                const int p = at + i * HALF;
                if (WIDE) {
                    const float4 f = p < c1 ? *reinterpret_cast<const float4*>(l + p) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[4 * i + k] = p + k < c1 ? l[p + k] : -INFINITY;
                }
            }
        };
        VdBest best{-INFINITY, -1};
        float sum = 0.0f, s = 0.0f, less_r = 0.0f, least = 0.0f;
        float limit = -INFINITY;                   // a weight of 2^60 is as good as one of 1: what sums are relative to changes once, as a rule
        auto take = [&](int at, const float (&x)[EACH]) {
            if (GREEDY) {
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                    if (x[i] > best.v) best = VdBest{x[i], at + (i >> 2) * HALF + (i & 3)};
                return;
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < EACH; ++i) top = fmaxf(top, x[i]);
            if (top > limit) {
                sum *= (float)vd_rescale(a, best.v, top);
                best = VdBest{top, 0};             // where it stands is not asked
                const VdRef ref = vd_ref(a, top);
                s = ref.s;
                less_r = (float)-ref.r;
                least = fmaxf(ref.s + (float)((double)(ref.r - 126) * a.inv_c), -3.402823466e38f);
                limit = fminf(top + (float)(60.0 * a.inv_c), 3.402823466e38f);
            }
            if (best.v == INFINITY) {              // infinite logits share the mass
#pragma unroll
                for (int i = 0; i < EACH; ++i) sum += x[i] == INFINITY ? 1.0f : 0.0f;
            } else if (best.i >= 0) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < EACH; ++i) {   // NaN and -inf count 2^-126
                    float e;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(fmaxf(x[i], least) - s, a.c_hi, less_r)));
                    part[i & 3] += e;
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
            }
        };
        float x[EACH], y[EACH];
        int at = c0 + 4 * threadIdx.x;
        load(at, x);
        for (; at < c1; at += 2 * STEP) {
            load(at + STEP, y);
            take(at, x);
            load(at + 2 * STEP, x);
            take(at + STEP, y);
        }
        const VdBest top = vd_warp_best(best);
        double all = 0.0;
        if (!GREEDY) all = warp_sum_d(best.i >= 0 ? (double)sum * vd_rescale(a, best.v, top.v) : 0.0);
        if (lane == 0) s_part[warp] = VdPart{all, top.v, top.i};
        __syncthreads();
        if (warp == 0) {
            const VdPart p = s_part[lane % VD_WARPS];
            best = vd_warp_best(VdBest{p.top, p.at});
            if (!GREEDY) all = warp_sum_d(lane < VD_WARPS && p.at >= 0 ? p.sum * vd_rescale(a, p.top, best.v) : 0.0);
            if (lane == 0) a.part[(int64_t)row * a.chunks + blockIdx.x] = VdPart{all, best.v, best.i};
        }
        __syncthreads();                           // s_part is read
    }
}

// One warp: a row's arg-max and Z relative to it.
template <bool GREEDY>
__device__ __forceinline__ void vd_join(const VerifyArgs& a, int row, int lane, VdBest& best, double& z) {
    const float4* p = reinterpret_cast<const float4*>(a.part + (int64_t)row * a.chunks);       // sum (two words), top, at
    const float4 none = make_float4(0.0f, 0.0f, -INFINITY, __int_as_float(-1)), own = lane < a.chunks ? __ldcg(p + lane) : none;
    best = VdBest{own.z, __float_as_int(own.w)};
    for (int c = lane + 32; c < a.chunks; c += 32) {
        const float4 f = __ldcg(p + c);
        best = vd_better(best, VdBest{f.z, __float_as_int(f.w)});
    }
    best = vd_warp_best(best);
    z = 0.0;
    if (!GREEDY) {
        for (int c = lane; c < a.chunks; c += 32) {
            const float4 f = c == lane ? own : __ldcg(p + c);
            if (__float_as_int(f.w) >= 0) z += __hiloint2double(__float_as_int(f.y), __float_as_int(f.x)) * vd_rescale(a, f.z, best.v);
        }
        z = warp_sum_d(z);
    }
}

// grid (8 per sequence); a cluster has a sequence
template <bool WIDE, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS, VD_RESIDENT) verify_pick_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ bool s_keep[VD_MAX_DRAFTS + 1];
    __shared__ float s_top[VD_MAX_DRAFTS + 1];
    __shared__ int s_at[VD_MAX_DRAFTS + 1];
    __shared__ double s_z[VD_MAX_DRAFTS + 1], s_mass[3][3][VD_WARPS];      // by pass: masses, and with a drafter's q what they lose with Z, all of p
    __shared__ int2 s_pow[16];
    __shared__ double s_step[VD_ROUND];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), b = blockIdx.x / VD_CLUSTER, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    vd_table(s_pow);
    __syncthreads();
    pdl_wait();
    const int first = max(a.offsets[b], 0), count = min(a.offsets[b + 1], a.rows) - first, drafts = min(count - 1, a.max_drafts);
    int32_t* tokens = a.tokens + (int64_t)b * (a.max_drafts + 1);
    if (count <= 0) {                              // no rows: the whole cluster leaves
        if (rank == 0) {
            for (int j = threadIdx.x; j <= a.max_drafts; j += VD_THREADS) tokens[j] = -1;
            if (threadIdx.x == 0) a.accepted[b] = 0;
        }
        return;
    }
    for (int j = warp; j <= drafts; j += VD_WARPS) {
        VdBest best;
        double z;
        const int x = j < drafts ? a.ids[first + j + 1] : -1;
        const bool there = (uint32_t)x < (uint32_t)a.V;
        const float l = !GREEDY && there ? a.logits[(first + j) * a.ls + x] : 0.0f, q = !GREEDY && there && a.draft ? a.draft[(first + j) * a.ds + x] : 1.0f;
        const float u = !GREEDY && there ? a.uniforms[first + j] : 0.0f;
        vd_join<GREEDY>(a, first + j, lane, best, z);
        if (lane == 0) {
            bool keep = false;
            if (GREEDY) {
                keep = there && best.i == x;
            } else if (there && best.i >= 0) {
                float2 hi = make_float2(l == INFINITY ? 1.0f : 0.0f, 0.0f), lo = make_float2(0.0f, 0.0f);
                if (best.v < INFINITY) vd_weights(a, s_pow, best.v)(l, l, hi, lo);
                keep = (double)u * (double)q * z < (double)hi.x + (double)lo.x;
            }
            s_keep[j] = keep;
            s_top[j] = best.v;
            s_at[j] = best.i;
            s_z[j] = z;
        }
    }
    __syncthreads();
    int n = 0;
    while (n < drafts && s_keep[n]) ++n;
    const int next = s_at[n];
    if (!GREEDY && next >= 0) {
        const int row = first + n;
        const bool refused = n < drafts;
        const float* l = a.logits + row * a.ls;
        const float* q = refused && a.draft ? a.draft + row * a.ds : nullptr;
        const int without = refused && !a.draft ? a.ids[row + 1] : -1;
        const float top = s_top[n];
        double z = s_z[n];
        const VdWeights weigh = vd_weights(a, s_pow, top);
        // segment of a warp: whole steps of 128 logits
        const int steps = ((a.V + 127) / 128 + VD_CLUSTER * VD_WARPS - 1) / (VD_CLUSTER * VD_WARPS), seg = steps * 128;
        struct Four {
            float4 l, q;
        };
        auto load = [&](int at, bool with_q) {
            Four f{make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY), make_float4(0.f, 0.f, 0.f, 0.f)};
            if (WIDE) {
                if (at < a.V) {
                    f.l = __ldg(reinterpret_cast<const float4*>(l + at));
                    if (with_q) f.q = __ldg(reinterpret_cast<const float4*>(q + at));
                }
            } else {
                float *x = &f.l.x, *y = &f.q.x;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (at + k < a.V) {
                        x[k] = l[at + k];
                        if (with_q) y[k] = q[at + k];
                    }
            }
            return f;
        };
        auto weights = [&](const Four& f, float (&hi)[4], float (&lo)[4]) {
            if (top < INFINITY) {
                float2 h0, h1, r0, r1;
                weigh(f.l.x, f.l.y, h0, r0);
                weigh(f.l.z, f.l.w, h1, r1);
                hi[0] = h0.x; hi[1] = h0.y; hi[2] = h1.x; hi[3] = h1.y;
                lo[0] = r0.x; lo[1] = r0.y; lo[2] = r1.x; lo[3] = r1.y;
            } else {                               // infinite logits share the mass
                hi[0] = f.l.x == INFINITY; hi[1] = f.l.y == INFINITY; hi[2] = f.l.z == INFINITY; hi[3] = f.l.w == INFINITY;
                lo[0] = lo[1] = lo[2] = lo[3] = 0.0f;
            }
        };
        auto masses = [&](int at, const Four& f, bool from_p, double (&r)[4]) {
            float hi[4], lo[4];
            weights(f, hi, lo);
            const float y[4] = {f.q.x, f.q.y, f.q.z, f.q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                r[k] = !from_p && q ? fma(-(double)y[k], z, (double)hi[k]) : (double)hi[k];
                r[k] = r[k] > 0.0 && (from_p || at + k != without) ? fmax(r[k] + (double)lo[k], 0.0) : 0.0;
            }
        };
        const int own = (rank * VD_WARPS + warp) * seg;
        // With a drafter's q: the masses for the first kernel's Z, which is off by up to 1e-7, how they change with Z, and all of p, which is
        // the Z they are then corrected to.  What of p is left where p and q nearly agree is summed again for the right Z.
        bool from_p = !refused;
        double lane_from = 0.0, lane_mid = 0.0, lane_to = 0.0, total = 0.0;
        for (int pass = 0; pass < 3; ++pass) {
            double sum = 0.0, whole = 0.0;
            float rest = 0.0f, whole_rest = 0.0f, loses = 0.0f;       // rests: what the weights' second parts come to, 2^-24 of the sum
            const bool with_q = !from_p && q;
            auto add = [&](int at, const Four& f) {
                float hi[4], lo[4];
                weights(f, hi, lo);
                if (!from_p && (unsigned)(without - at) < 4u) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (at + k == without) hi[k] = lo[k] = 0.0f;
                }
                const double h[4] = {(double)hi[0], (double)hi[1], (double)hi[2], (double)hi[3]};
                const double all = (h[0] + h[1]) + (h[2] + h[3]);
                const float low = (lo[0] + lo[1]) + (lo[2] + lo[3]);
                if (!with_q) {
                    sum += all;
                    rest += low;
                    return;
                }
                whole += all;
                whole_rest += low;
                const float y[4] = {f.q.x, f.q.y, f.q.z, f.q.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const double r = fma(-(double)y[k], z, h[k]);
                    if (r > 0.0) {
                        sum += r;
                        rest += lo[k];
                        loses += y[k];
                    }
                }
            };
            // two steps at a time, the next two under way
            auto fetch = [&](int s, Four (&f)[2]) {
                f[0] = load(s < steps ? own + s * 128 + 4 * lane : a.V, with_q);
                f[1] = load(s + 1 < steps ? own + (s + 1) * 128 + 4 * lane : a.V, with_q);
            };
            auto take = [&](int s, const Four (&f)[2]) {
                if (s < steps) add(own + s * 128 + 4 * lane, f[0]);
                if (s + 1 < steps) add(own + (s + 1) * 128 + 4 * lane, f[1]);
            };
            Four u[2], v[2];
            fetch(0, u);
            for (int s = 0; s < steps; s += 4) {
                fetch(s + 2, v);
                take(s, u);
                fetch(s + 4, u);
                take(s + 2, v);
            }
            sum = warp_sum_d(sum + (double)rest);
            if (with_q) {
                whole = warp_sum_d(whole + (double)whole_rest);
                loses = warp_sum(loses);
            }
            if (lane == 0) {
                s_mass[pass][0][warp] = sum;
                s_mass[pass][1][warp] = (double)loses;
                s_mass[pass][2][warp] = whole;
            }
            cluster.sync();
            // where the segments begin and end on the line of masses, the same numbers in every warp: lane k has segments 2 k and
            // 2 k + 1, [prev, mid) and [mid, upto), made to ascend whatever the sums' rounding
            const double* of = cluster.map_shared_rank(&s_mass[pass][0][0], lane / 4) + 2 * (lane % 4);
            double m0 = of[0], m1 = of[1];
            if (with_q) {
                const double e0 = of[2 * VD_WARPS], e1 = of[2 * VD_WARPS + 1], right = warp_sum_d(e0 + e1), more = right - z;
                m0 = fmax(m0 - more * of[VD_WARPS], 0.0);
                m1 = fmax(m1 - more * of[VD_WARPS + 1], 0.0);
                z = right;
            }
            double upto = m0 + m1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto = fmax(upto, v);
            }
            total = __shfl_sync(0xffffffffu, upto, 31);
            const double up = __shfl_up_sync(0xffffffffu, upto, 1), prev = lane == 0 ? 0.0 : up, mid = fmin(prev + m0, upto);
            lane_from = prev;
            lane_mid = mid;
            lane_to = upto;
            if (with_q && pass == 0 && total < 1e-3 * z) continue;
            if (total > 0.0 || from_p) break;
            from_p = true;                         // max(p - q, 0) has no mass
        }
        const float u = a.uniforms[first + count - 1];
        const double mark = (u > 0.0f ? fmin((double)u, 1.0 - 1.0 / 16777216.0) : 0.0) * total;
        const unsigned even = __ballot_sync(0xffffffffu, lane_from <= mark && mark < lane_mid), odd = __ballot_sync(0xffffffffu, lane_mid <= mark && mark < lane_to);
        const int holder = max(0, even ? __ffs(even) - 1 : __ffs(odd) - 1);          // lane whose segments hold the draw: there is one
        const int which = 2 * holder + (even == 0);
        if (which / VD_WARPS == rank) {            // this block walks the segment again, its warps a step each
            double run = __shfl_sync(0xffffffffu, even ? lane_from : lane_mid, holder);
            const int from = which * seg;
            int found = -1;                        // the step that holds the draw, or so far the last one that has mass
            double found_run = 0.0;
            bool sure = false;
            for (int s0 = 0; s0 < steps && !sure; s0 += VD_ROUND) {
                const int here = min(VD_ROUND, steps - s0);
                for (int s = warp; s < here; s += VD_WARPS) {
                    const int at = from + (s0 + s) * 128 + 4 * lane;
                    double r[4];
                    masses(at, load(at, !from_p && q), from_p, r);
                    const double sum = warp_sum_d((r[0] + r[1]) + (r[2] + r[3]));
                    if (lane == 0) s_step[s] = sum;
                }
                __syncthreads();
                for (int s = 0; s < here && !sure; ++s) {       // every thread alike
                    const double m = s_step[s];
                    if (m > 0.0) {
                        found = s0 + s;
                        found_run = run;
                        sure = run + m > mark;
                    }
                    run += m;
                }
                __syncthreads();
            }
            if (warp == 0) {
                const int at = from + max(found, 0) * 128 + 4 * lane;
                double r[4];
                masses(at, load(at, !from_p && q), from_p, r);
                const double sum = (r[0] + r[1]) + (r[2] + r[3]);
                double incl = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                double c = found_run + (incl - sum);
                int hit = 0x7fffffff, last = -1;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    c += r[k];
                    if (r[k] > 0.0) {
                        last = at + k;
                        if (c > mark) hit = min(hit, at + k);
                    }
                }
                hit = __reduce_min_sync(0xffffffffu, hit);
                last = __reduce_max_sync(0xffffffffu, last);
                // sums in another order may end a rounding short of the mark: the last one that has mass
                if (lane == 0) tokens[n] = hit != 0x7fffffff ? hit : last >= 0 ? last : min(from, a.V - 1);
            }
        }
        cluster.sync();                            // nobody leaves while its masses are read
    } else if (rank == 0 && threadIdx.x == 0) {
        tokens[n] = next;
    }
    if (rank == 0) {
        for (int j = threadIdx.x; j <= a.max_drafts; j += VD_THREADS)
            if (j != n) tokens[j] = j < n ? a.ids[first + j + 1] : -1;
        if (threadIdx.x == 0) a.accepted[b] = n;
    }
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_verify_drafts_workspace(int rows, int V, size_t* bytes) {
    B200_REQUIRE(bytes, "verify_drafts_workspace: null pointer");
    B200_REQUIRE(rows >= 0 && V >= 1 && V <= 1 << 30, "verify_drafts_workspace: bad sizes");
    *bytes = std::max<size_t>(16, (size_t)rows * ceil_div(V, VD_CHUNK) * sizeof(VdPart));
    return B200_OK;
}

int b200_verify_drafts(const float* logits, int64_t logits_stride, const float* draft_probs, int64_t draft_stride,
                       const int32_t* ids, const int32_t* row_offsets, int batch, int rows, int V, float temperature,
                       const float* uniforms, int max_drafts, int32_t* accepted, int32_t* tokens, void* workspace,
                       size_t workspace_bytes) {
    if (batch <= 0) return B200_OK;
    const char* who = "verify_drafts";
    size_t need = 0;
    int rc = b200_verify_drafts_workspace(rows, V, &need);
    if (rc) return rc;
    B200_REQUIRE(batch <= 1 << 20 && max_drafts >= 0 && max_drafts <= VD_MAX_DRAFTS, "%s: max_drafts must be in [0, %d]", who, VD_MAX_DRAFTS);
    B200_REQUIRE(rows == 0 || (logits && ids && uniforms), "%s: null pointer", who);
    B200_REQUIRE(row_offsets && accepted && tokens && workspace, "%s: null pointer", who);
    B200_REQUIRE(logits_stride >= V && (!draft_probs || draft_stride >= V), "%s: a stride is shorter than its row", who);
    B200_REQUIRE(temperature <= 1e30f, "%s: the temperature must be a number of at most 1e30", who);
    B200_REQUIRE(aligned16(workspace) && workspace_bytes >= need, "%s: the workspace must be 16-byte aligned and have %zu bytes", who, need);
    const bool greedy = temperature <= 0.0f;
    const double c = greedy ? 0.0 : 1.4426950408889634 / (double)temperature;
    const float hi = (float)c;
    B200_REQUIRE(hi < INFINITY, "%s: the temperature is too small", who);
    VerifyArgs a{logits, logits_stride, draft_probs, draft_stride, ids, row_offsets, batch, rows, V, 0,
                 hi, (float)(c - (double)hi), c, greedy ? 0.0 : 1.0 / c, 0, uniforms, max_drafts, accepted, tokens, static_cast<VdPart*>(workspace)};
    const bool wide = aligned16(logits) && V % 4 == 0 && logits_stride % 4 == 0 &&
                      (!draft_probs || (aligned16(draft_probs) && draft_stride % 4 == 0));
    const dim3 block(VD_THREADS);
    if (rows > 0) {
        // Chunks so that the rounds of blocks over the device, each as long as a chunk and what a block costs besides (about 3000 logits'
        // worth), take the least; none of less than 2048 logits.
        const int slots = VD_RESIDENT * num_sms(), most = ceil_div(V, VD_CHUNK);
        int64_t least = INT64_MAX;
        for (int n = 1; n <= std::min(most, 64); ++n) {
            const int chunk = ceil_div(ceil_div(V, n), 1024) * 1024;
            const int64_t cost = ceil_div64((int64_t)rows * ceil_div(V, chunk), slots) * (chunk + 3000);
            if (cost < least) {
                least = cost;
                a.chunk = chunk;
            }
        }
        a.chunks = ceil_div(V, a.chunk);
        const dim3 grid(a.chunks, std::min(rows, 65535));
        auto kern = wide ? (greedy ? verify_stats_kernel<true, true> : verify_stats_kernel<true, false>)
                         : (greedy ? verify_stats_kernel<false, true> : verify_stats_kernel<false, false>);
        rc = launch_serve("verify_stats_kernel", kern, grid, block, 0, 1, short_grid(grid), a);
        if (rc) return rc;
    }
    auto kern = wide ? (greedy ? verify_pick_kernel<true, true> : verify_pick_kernel<true, false>)
                     : (greedy ? verify_pick_kernel<false, true> : verify_pick_kernel<false, false>);
    // Where the clusters fill more than half of the device they start after the first kernel and not while its last blocks run: the
    // slots that these leave free seldom make eight in one place, and clusters that found none waited for another cluster's end (3 of
    // 64 sequences' did: 56.1 -> 52.7 us; 40: 42.3 -> 39.4; 56: 50.9 -> 52.5).  Fewer clusters find room, early or not.
    const bool early = batch * VD_CLUSTER <= VD_RESIDENT / 2 * num_sms();
    return launch_serve("verify_pick_kernel", kern, dim3(batch * VD_CLUSTER), block, 0, VD_CLUSTER, early, a);
}

}  // extern "C"
