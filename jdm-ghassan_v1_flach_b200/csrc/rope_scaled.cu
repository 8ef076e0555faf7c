// Rotary positions: both pair layouts, a leading part of every head, frequencies scaled for long contexts.
//
// (a, b) -> (a c - b s, a s + b c) with c, s = factor * cos, sin(pos * f).  A position of a million times f = 1 leaves an fp32
// product an error of 0.03 rad, so the angle is formed in 64 bits in turns, its whole turns dropped there, and the rest goes to
// sincospif as fp32 with what that rounding cut off added to first order.
//
// What bounds it: q and k read and written once (8 bytes per element).  A block takes one token (or a share of its heads where the
// tokens are few): its rot/2 angles first, into shared memory, then 16 bytes per thread and step.
#include <algorithm>
#include <cmath>

#include "serve.cuh"

namespace b200 {

constexpr int RS_THREADS = 256;
constexpr int RS_MAX_PAIRS = 512;

struct RopeArgs {
    const float *q, *k;
    float *q_out, *k_out;
    const int32_t* pos;
    const double* freq;
    int64_t qs, ks, qos, kos;
    int heads, kv, hd, rot, items;               // items: steps of one head
    FastDiv by_items;
    float factor;
};

template <int W>
struct RsVec { float v[W]; };
template <int W>
__device__ __forceinline__ RsVec<W> rs_load(const float* p) {
    RsVec<W> r;
    if (W == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        r.v[0] = f.x; r.v[W > 1 ? 1 : 0] = f.y; r.v[W > 2 ? 2 : 0] = f.z; r.v[W > 3 ? 3 : 0] = f.w;
    } else if (W == 2) {
        r.v[0] = p[0]; r.v[W > 1 ? 1 : 0] = p[1];
    } else {
        r.v[0] = p[0];
    }
    return r;
}
template <int W>
__device__ __forceinline__ void rs_store(float* p, const RsVec<W>& r) {
    if (W == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[W > 1 ? 1 : 0], r.v[W > 2 ? 2 : 0], r.v[W > 3 ? 3 : 0]);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) p[i] = r.v[i];
    }
}

// HALVES: pairs (i, i + rot/2), a step is W pairs; else pairs (2i, 2i+1), a step is W elements (W even).
// Behind the turned part a step copies W elements.  grid (tokens, shares of the heads).  A thread's first steps are loaded before the
// angles are made, which take as long as the loads do.
template <bool HALVES, int W>
__global__ void __launch_bounds__(RS_THREADS) rope_scaled_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int AT_ONCE = 4;
    __shared__ float2 s_cs[RS_MAX_PAIRS];
    short_begin();
    const int64_t t = blockIdx.x;
    const int half = a.rot / 2;
    const int turned = HALVES ? half / W : a.rot / W;       // steps of a head that turn, the others copy
    const int all = (a.heads + a.kv) * a.items, stride = gridDim.y * RS_THREADS;
    const float *q = a.q + t * a.qs, *k = a.k + t * a.ks;
    float *q_out = a.q_out + t * a.qos, *k_out = a.k_out + t * a.kos;
    const int pos = a.pos[t];
    bool first = true;
    for (int n0 = blockIdx.y * RS_THREADS + threadIdx.x; first || n0 < all; n0 += AT_ONCE * stride) {
        RsVec<W> x[AT_ONCE], y[AT_ONCE];
        float* to[AT_ONCE];
        int at[AT_ONCE];                                    // of the pairs' first one; -1: copied, -2: nothing
#pragma unroll
        for (int s = 0; s < AT_ONCE; ++s) {
            const int n = n0 + s * stride;
            at[s] = -2;
            if (n >= all) continue;
            const int h = (int)a.by_items.div(n), j = n - h * a.items;
            const bool is_q = h < a.heads;
            const float* src = (is_q ? q : k) + (int64_t)(is_q ? h : h - a.heads) * a.hd;
            const int e = j < turned ? j * W : a.rot + (j - turned) * W;
            to[s] = (is_q ? q_out : k_out) + (int64_t)(is_q ? h : h - a.heads) * a.hd + e;
            x[s] = rs_load<W>(src + e);
            if (HALVES && j < turned) y[s] = rs_load<W>(src + e + half);
            at[s] = j >= turned ? (src + e == to[s] ? -2 : -1) : HALVES ? e : e / 2;
        }
        if (first) {
            first = false;
            if (pos < 0) return;
            for (int i = threadIdx.x; i < half; i += RS_THREADS) {
                const double turns = (double)pos * (a.freq[i] * 0.15915494309189533577);
                const double rest = turns - rint(turns);
                const float r = (float)rest;
                float s, c;
                sincospif(2.0f * r, &s, &c);
                const float d = 6.2831853071795865f * (float)(rest - (double)r);
                s_cs[i] = make_float2(a.factor * fmaf(-s, d, c), a.factor * fmaf(c, d, s));
            }
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < AT_ONCE; ++s) {
            if (at[s] == -2) continue;
            if (at[s] >= 0) {
                if (HALVES) {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float2 cs = s_cs[at[s] + i];
                        const float u = x[s].v[i], v = y[s].v[i];
                        x[s].v[i] = u * cs.x - v * cs.y;
                        y[s].v[i] = u * cs.y + v * cs.x;
                    }
                    rs_store<W>(to[s] + half, y[s]);
                } else {
#pragma unroll
                    for (int i = 0; i + 1 < W; i += 2) {
                        const float2 cs = s_cs[at[s] + i / 2];
                        const float u = x[s].v[i], v = x[s].v[i + 1];
                        x[s].v[i] = u * cs.x - v * cs.y;
                        x[s].v[i + 1] = u * cs.y + v * cs.x;
                    }
                }
            }
            rs_store<W>(to[s], x[s]);
        }
    }
}

__global__ void rope_frequencies_kernel(double* out, int rot, double theta, int scaling, double factor, double ctx, double low, double high) {
    const double two_pi = 6.28318530717958647693, base = scaling == 2 && rot > 2 ? theta * pow(factor, rot / (rot - 2.0)) : theta;
    for (int i = threadIdx.x; i < rot / 2; i += blockDim.x) {
        const double f = pow(base, -2.0 * i / rot);
        double r = f;
        if (scaling == 1) r = f / factor;
        if (scaling == 2 && rot == 2) r = f;                 // one pair of frequency 1: nothing for a base to change
        if (scaling == 3) {
            // the dimensions that turn `high` and `low` times over the original context
            const double a = rot * log(ctx / (high * two_pi)) / (2.0 * log(theta)), b = rot * log(ctx / (low * two_pi)) / (2.0 * log(theta));
            const double from = fmax(floor(a), 0.0), to = fmin(ceil(b), rot - 1.0);
            const double ramp = fmin(fmax((i - from) / fmax(to - from, 1e-3), 0.0), 1.0);
            r = f / factor * ramp + f * (1.0 - ramp);
        }
        if (scaling == 4) {
            const double smooth = fmin(fmax((ctx * f / two_pi - low) / (high - low), 0.0), 1.0);
            r = (1.0 - smooth) * f / factor + smooth * f;
        }
        out[i] = r;
    }
}

template <bool HALVES, int W>
static int launch_rope(RopeArgs a, int64_t ntok) {
    a.items = (HALVES ? a.rot / 2 : a.rot) / W + (a.hd - a.rot) / W;
    a.by_items = FastDiv(a.items);
    const int steps = ceil_div((a.heads + a.kv) * a.items, RS_THREADS);
    // one token per block where that fills the device; fewer tokens: their heads are dealt out
    const int shares = ntok >= 2 * num_sms() ? 1 : std::min<int>(steps, ceil_div(2 * num_sms(), (int)ntok));
    const dim3 grid((unsigned)ntok, shares);
    return launch_serve("rope_scaled_kernel", rope_scaled_kernel<HALVES, W>, grid, dim3(RS_THREADS), 0, 1, short_grid(grid), a);
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_rope_frequencies(double* inv_freq, int rot_dim, double theta, int scaling, double factor, int orig_ctx, double low,
                          double high, double* attn_factor_host) {
    B200_REQUIRE(inv_freq, "rope_frequencies: null pointer");
    B200_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= 2 * RS_MAX_PAIRS, "rope_frequencies: rot_dim must be even and in [2, %d]", 2 * RS_MAX_PAIRS);
    B200_REQUIRE(std::isfinite(theta) && theta > 1.0, "rope_frequencies: theta must be above 1");
    B200_REQUIRE(scaling >= 0 && scaling <= 4, "rope_frequencies: unknown scaling %d", scaling);
    B200_REQUIRE(scaling == 0 || (std::isfinite(factor) && factor >= 1.0), "rope_frequencies: factor must be at least 1");
    B200_REQUIRE(scaling < 3 || (orig_ctx >= 1 && low > 0.0 && high > low && std::isfinite(high)),
                 "rope_frequencies: this scaling needs the original context and 0 < low < high");
    rope_frequencies_kernel<<<1, 128, 0, stream()>>>(inv_freq, rot_dim, theta, scaling, factor, (double)orig_ctx, low, high);
    B200_LAUNCH_CHECK("rope_frequencies_kernel");
    if (attn_factor_host) *attn_factor_host = scaling == 3 ? 1.0 + 0.1 * std::log(factor) : 1.0;
    return B200_OK;
}

int b200_rope_forward_scaled(const float* q, const float* k, float* q_out, float* k_out, const int32_t* pos,
                             const double* inv_freq, int64_t ntok, int n_heads, int n_kv, int head_dim, int rot_dim,
                             int rope_type, int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                             float attn_factor) {
    if (ntok <= 0) return B200_OK;
    const char* who = "rope_forward_scaled";
    B200_REQUIRE(ntok <= 0x7fffffff, "%s: too many tokens", who);
    B200_REQUIRE(pos && inv_freq, "%s: null pointer", who);
    B200_REQUIRE(!q == !q_out && !k == !k_out && (q || k), "%s: q and q_out, k and k_out go together, one pair at least", who);
    B200_REQUIRE(head_dim >= 2 && head_dim <= 2 * RS_MAX_PAIRS && rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim,
                 "%s: rot_dim must be even, at least 2 and at most head_dim (which may be %d)", who, 2 * RS_MAX_PAIRS);
    B200_REQUIRE(rope_type == 0 || rope_type == 1, "%s: rope_type must be 0 or 1", who);
    B200_REQUIRE((!q || n_heads >= 1) && (!k || n_kv >= 1) && n_heads <= 65536 && n_kv <= 65536, "%s: bad head counts", who);
    const int64_t qn = q ? (int64_t)n_heads * head_dim : 0, kn = k ? (int64_t)n_kv * head_dim : 0;
    B200_REQUIRE((!q || (q_stride >= qn && q_out_stride >= qn)) && (!k || (k_stride >= kn && k_out_stride >= kn)),
                 "%s: a stride is shorter than its row", who);
    auto apart = [&](const float* x, int64_t xs, const float* y, int64_t ys, int64_t n) {
        if (x + (ntok - 1) * xs + n <= y || y + (ntok - 1) * ys + n <= x) return true;
        if (xs != ys) return false;
        // the same rows: the same columns, or others of each row
        const int64_t off = ((int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x)) / (int64_t)sizeof(float) % xs + xs) % xs;
        return x == y || (off >= n && xs - off >= n);
    };
    B200_REQUIRE((!q || apart(q, q_stride, q_out, q_out_stride, qn)) && (!k || apart(k, k_stride, k_out, k_out_stride, kn)),
                 "%s: an output overlaps its input without being it", who);
    RopeArgs a{q, k, q_out, k_out, pos, inv_freq, q_stride, k_stride, q_out_stride, k_out_stride, q ? n_heads : 0, k ? n_kv : 0,
               head_dim, rot_dim, 0, FastDiv(), attn_factor};
    auto by4 = [](const float* p, int64_t s) { return !p || (aligned16(p) && s % 4 == 0); };
    const bool wide = by4(q, q_stride) && by4(k, k_stride) && by4(q_out, q_out_stride) && by4(k_out, k_out_stride) && head_dim % 4 == 0 && rot_dim % 4 == 0;
    if (rope_type == 1) {
        if (wide && rot_dim % 8 == 0) return launch_rope<true, 4>(a, ntok);
        return launch_rope<true, 1>(a, ntok);
    }
    // pairs of neighbours: two elements a step, unless an odd head width leaves one behind
    if (wide) return launch_rope<false, 4>(a, ntok);
    B200_REQUIRE(head_dim % 2 == 0, "%s: head_dim must be even", who);
    return launch_rope<false, 2>(a, ntok);
}

}  // extern "C"
