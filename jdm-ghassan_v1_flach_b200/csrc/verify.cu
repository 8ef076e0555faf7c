// Drafted tokens against the target's probabilities, from given uniforms.
//
// Two kernels.  The first reads every row of logits once, a chunk of 8192 per block, and leaves its largest value, where that
// stands, and the sum of exp((l - largest) / T).  The second has a cluster of eight blocks per sequence: each joins the chunks
// of the sequence's rows by itself (a few hundred words), decides how many drafts are kept, and then sums its eighth of the one row
// that the next token is drawn from, a segment per warp; the 64 segments' masses are exchanged through the cluster's shared memory,
// and the warp that holds the draw walks its segment again.  Mass i is e_i - q_i Z with e_i = exp((l_i - max) / T): nothing
// is divided by Z.
//
// A draw falls on another index than the exact one where u * mass lies within the sums' error of a border, and a flat row has
// 100 000 borders.  So the argument of exp is kept in two fp32 parts (l - max and its rounding error, 1 / T in two parts), Z
// in two for e - q Z, and sums run in fp64: what is left is the rounding of single weights, 2^-23 of each with either
// sign, which moves a border of a flat row by about 1e-10 of the mass.
//
// What bounds it: the logits, once (4 V bytes a row).
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "serve.cuh"

namespace b200 {

namespace cg = cooperative_groups;

constexpr int VD_THREADS = 256;
constexpr int VD_WARPS = VD_THREADS / 32;
constexpr int VD_EACH = 32;                       // logits of a thread
constexpr int VD_CHUNK = VD_THREADS * VD_EACH;
constexpr int VD_CLUSTER = 8;
constexpr int VD_MAX_DRAFTS = 255;

struct VdPart {                                   // of one chunk of one row
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
    float inv_hi, inv_lo;                         // 1 / temperature
    const float* uniforms;
    int max_drafts;
    int32_t *accepted, *tokens;
    VdPart* part;
};

// exp((l - top) / T), 0 for NaN and -inf; l <= top.
__device__ __forceinline__ float vd_weight(float l, float top, float inv_hi, float inv_lo) {
    if (l == top) return 1.0f;                    // an infinite top too
    const float d = __fsub_rn(l, top);
    // what rounding left of l - top
    const float b = __fadd_rn(d, top), err = __fsub_rn(__fsub_rn(l, b), __fsub_rn(top, __fsub_rn(b, d)));
    const float t = __fmul_rn(d, inv_hi);
    if (!(t > -104.0f)) return 0.0f;              // also NaN, -inf
    const float low = fmaf(d, inv_hi, -t) + fmaf(d, inv_lo, err * inv_hi);
    const float e = expf(t);
    return fmaf(e, low, e);
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

// grid (chunks, rows)
template <bool WIDE, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS) verify_stats_kernel(VerifyArgs a) {
    __shared__ VdBest s_best[VD_WARPS];
    __shared__ double s_sum[VD_WARPS];
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int row = blockIdx.y; row < a.rows; row += gridDim.y) {
        if (row >= a.offsets[a.batch]) return;
        const float* l = a.logits + row * a.ls;
        const int c0 = blockIdx.x * VD_CHUNK;
        float x[VD_EACH];
        VdBest best{-INFINITY, -1};
#pragma unroll
        for (int i = 0; i < VD_EACH; i += 4) {
            const int at = c0 + i * VD_THREADS + 4 * threadIdx.x;
            if (WIDE) {
                const float4 f = at < a.V ? __ldcs(reinterpret_cast<const float4*>(l + at)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i + k] = at + k < a.V ? l[at + k] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < VD_EACH; ++i)
            if (x[i] > best.v) best = VdBest{x[i], c0 + (i & ~3) * VD_THREADS + 4 * (int)threadIdx.x + (i & 3)};
        best = vd_warp_best(best);
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < VD_WARPS; ++w) best = vd_better(best, s_best[w]);
        double sum = 0.0;
        if (!GREEDY && best.i >= 0) {
#pragma unroll
            for (int i = 0; i < VD_EACH; i += 4) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) s += vd_weight(x[i + k], best.v, a.inv_hi, a.inv_lo);
                sum += (double)s;
            }
            sum = warp_sum_d(sum);
            if (lane == 0) s_sum[warp] = sum;
            __syncthreads();
            sum = 0.0;
            for (int w = 0; w < VD_WARPS; ++w) sum += s_sum[w];
        }
        if (threadIdx.x == 0) a.part[(int64_t)row * a.chunks + blockIdx.x] = VdPart{sum, best.v, best.i};
        __syncthreads();
    }
}

// One warp: a row's arg-max and, for the largest value, Z.
template <bool GREEDY>
__device__ __forceinline__ void vd_join(const VerifyArgs& a, int row, int lane, VdBest& best, double& z) {
    const VdPart* p = a.part + (int64_t)row * a.chunks;
    best = VdBest{-INFINITY, -1};
    for (int c = lane; c < a.chunks; c += 32) best = vd_better(best, VdBest{__ldcg(&p[c].top), __ldcg(&p[c].at)});
    best = vd_warp_best(best);
    z = 0.0;
    if (!GREEDY) {
        for (int c = lane; c < a.chunks; c += 32) {
            const float top = __ldcg(&p[c].top);
            if (__ldcg(&p[c].at) < 0) continue;
            const double t = top == best.v ? 0.0 : ((double)top - (double)best.v) * ((double)a.inv_hi + (double)a.inv_lo);
            z += __ldcg(&p[c].sum) * exp(t);
        }
        z = warp_sum_d(z);
    }
}

// grid (8 per sequence); a cluster has a sequence
template <bool WIDE, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS) verify_pick_kernel(VerifyArgs a) {
    __shared__ bool s_keep[VD_MAX_DRAFTS + 1];
    __shared__ float s_top[VD_MAX_DRAFTS + 1];
    __shared__ int s_at[VD_MAX_DRAFTS + 1];
    __shared__ double s_z[VD_MAX_DRAFTS + 1], s_mass[2][VD_WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), b = blockIdx.x / VD_CLUSTER, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
        vd_join<GREEDY>(a, first + j, lane, best, z);
        if (lane == 0) {
            bool keep = false;
            if (j < drafts) {
                const int x = a.ids[first + j + 1];
                if (GREEDY) {
                    keep = best.i >= 0 && best.i == x;
                } else if ((uint32_t)x < (uint32_t)a.V && best.i >= 0) {
                    const float l = a.logits[(first + j) * a.ls + x];
                    const double e = (double)vd_weight(l, best.v, a.inv_hi, a.inv_lo), u = (double)a.uniforms[first + j];
                    const double q = a.draft ? (double)a.draft[(first + j) * a.ds + x] : 1.0;
                    keep = u * q * z < e;
                }
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
    int next = s_at[n];
    if (!GREEDY && next >= 0) {
        const int row = first + n;
        const bool refused = n < drafts;
        const float* l = a.logits + row * a.ls;
        const float* q = refused && a.draft ? a.draft + row * a.ds : nullptr;
        const int without = refused && !a.draft ? a.ids[row + 1] : -1;
        const float top = s_top[n], zh = (float)s_z[n], zl = (float)(s_z[n] - (double)zh);
        // segment of a warp: whole steps of 128 logits
        const int steps = ((a.V + 127) / 128 + VD_CLUSTER * VD_WARPS - 1) / (VD_CLUSTER * VD_WARPS), seg = steps * 128;
        auto masses = [&](int at, bool from_p, float (&r)[4]) {
            float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
            if (WIDE) {
                const float4 f = at < a.V ? __ldg(reinterpret_cast<const float4*>(l + at)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
                if (q && at < a.V) {
                    const float4 g = __ldg(reinterpret_cast<const float4*>(q + at));
                    y[0] = g.x; y[1] = g.y; y[2] = g.z; y[3] = g.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = at + k < a.V ? l[at + k] : -INFINITY;
                    if (q && at + k < a.V) y[k] = q[at + k];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float e = vd_weight(x[k], top, a.inv_hi, a.inv_lo);
                r[k] = from_p ? e : at + k == without ? 0.0f : fmaxf(fmaf(-y[k], zl, fmaf(-y[k], zh, e)), 0.0f);
            }
        };
        const int own = (rank * VD_WARPS + warp) * seg;
        bool from_p = !refused;
        double before = 0.0, total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {                // the second only where max(p - q, 0) has no mass
            double sum = 0.0;
            for (int s = 0; s < steps; ++s) {
                float r[4];
                masses(own + s * 128 + 4 * lane, from_p, r);
                sum += ((double)r[0] + (double)r[1]) + ((double)r[2] + (double)r[3]);
            }
            sum = warp_sum_d(sum);
            if (lane == 0) s_mass[pass][warp] = sum;
            cluster.sync();
            total = 0.0;
            for (int i = 0; i < VD_CLUSTER * VD_WARPS; ++i) {
                if (i == rank * VD_WARPS + warp) before = total;
                total += cluster.map_shared_rank(&s_mass[pass][0], i / VD_WARPS)[i % VD_WARPS];
            }
            if (total > 0.0 || from_p) break;
            from_p = true;
        }
        const float u = a.uniforms[first + count - 1];
        const double mark = (u > 0.0f ? fmin((double)u, 1.0 - 1.0 / 16777216.0) : 0.0) * total;
        const double mine = s_mass[from_p && refused ? 1 : 0][warp];
        if (before <= mark && mark < before + mine) {
            // this warp's segment holds the draw
            double run = before;
            int found = -1, last = -1;
            for (int s = 0; s < steps && found < 0; ++s) {
                float r[4];
                const int at = own + s * 128 + 4 * lane;
                masses(at, from_p, r);
                const double sum = ((double)r[0] + (double)r[1]) + ((double)r[2] + (double)r[3]);
                double incl = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += u;
                }
                double c = run + (incl - sum);
                int hit = 0x7fffffff, any = -1;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    c += (double)r[k];
                    if (r[k] > 0.0f) {
                        any = at + k;
                        if (c > mark) hit = min(hit, at + k);
                    }
                }
                hit = __reduce_min_sync(0xffffffffu, hit);
                any = __reduce_max_sync(0xffffffffu, any);
                if (hit != 0x7fffffff) found = hit;
                last = max(last, any);
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) tokens[n] = found >= 0 ? found : last;     // sums in another order: the segment's last one
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
    B200_REQUIRE(temperature == temperature && temperature < INFINITY, "%s: the temperature must be a finite number", who);
    B200_REQUIRE(aligned16(workspace) && workspace_bytes >= need, "%s: the workspace must be 16-byte aligned and have %zu bytes", who, need);
    const bool greedy = temperature <= 0.0f;
    const double inv = greedy ? 0.0 : 1.0 / (double)temperature;
    const float hi = (float)inv;
    B200_REQUIRE(hi < INFINITY, "%s: the temperature is too small", who);
    VerifyArgs a{logits, logits_stride, draft_probs, draft_stride, ids, row_offsets, batch, rows, V, ceil_div(V, VD_CHUNK),
                 hi, (float)(inv - (double)hi), uniforms, max_drafts, accepted, tokens, static_cast<VdPart*>(workspace)};
    const bool wide = aligned16(logits) && V % 4 == 0 && logits_stride % 4 == 0 &&
                      (!draft_probs || (aligned16(draft_probs) && draft_stride % 4 == 0));
    const dim3 block(VD_THREADS);
    if (rows > 0) {
        const dim3 grid(a.chunks, std::min(rows, 65535));
        auto kern = wide ? (greedy ? verify_stats_kernel<true, true> : verify_stats_kernel<true, false>)
                         : (greedy ? verify_stats_kernel<false, true> : verify_stats_kernel<false, false>);
        rc = launch_serve("verify_stats_kernel", kern, grid, block, 0, 1, false, a);
        if (rc) return rc;
    }
    auto kern = wide ? (greedy ? verify_pick_kernel<true, true> : verify_pick_kernel<true, false>)
                     : (greedy ? verify_pick_kernel<false, true> : verify_pick_kernel<false, false>);
    return launch_serve("verify_pick_kernel", kern, dim3(batch * VD_CLUSTER), block, 0, VD_CLUSTER, rows > 0, a);
}

}  // extern "C"
