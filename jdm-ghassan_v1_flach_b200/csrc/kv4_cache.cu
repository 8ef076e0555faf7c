// Rows of keys and values into the 4-bit pages and back (layout: b200serve.h).
//
// The rule is b200_quantize's for kinds 0 and 1, one correctly rounded fp32 operation at a time, but for two things.  The step of
// kind 1 is (max - min) times fp32(1/15) where that divides by 15: every new token pays for it, and the quotient's last bit
// decides only for a value on the border of two codes.  And a scale or minimum beyond the range of fp16 is kept at its largest
// value, because an infinite one would make a NaN of every code 0, and of every masked probability in the attention over these
// pages.
//
// What bounds both: the fp32 rows (8 KV hd bytes a token), a sixth of that again for the pages.  16 384 rows of 8 x 128, kind 0: store 27 us,
// 5.7 TB/s, with 64 instructions a lane per 16 bytes of row behind it; fetch 26, 134 MB to write, with 48.
// Eight lanes share a token's row of one head: lane g has the four elements 4 g .. 4 g + 3 of each block
// of 32, which is one 16-bit word per block, and those words lie side by side.  So a warp reads and writes whole lines of the row
// and eight bytes a lane of the codes, and the statistics of four blocks take four shuffles.
#include <type_traits>

#include "serve.cuh"

namespace b200 {

constexpr int KC_THREADS = 128;
constexpr int KC_ITEMS = KC_THREADS / 8;         // rows of a head at a time

struct Kv4Rows {
    const float *k_in = nullptr, *v_in = nullptr;
    float *k_out = nullptr, *v_out = nullptr;
    int64_t ks = 0, vs = 0;
    const int32_t* slots = nullptr;
    uint8_t* pages = nullptr;
    int64_t n = 0;
    int num_slots = 0, page = 1, KV = 0;
    FastDiv by_page, by_KV;
    Kv4Page part;
};

int kv4_check(const char* who, int num_pages, int page, int KV, int hd, int kind) {
    B200_REQUIRE(hd == 64 || hd == 128, "%s: hd must be 64 or 128", who);
    B200_REQUIRE(kind == 0 || kind == 1, "%s: kind must be 0 (Q4_0) or 1 (Q4_1)", who);
    B200_REQUIRE(KV >= 1 && KV <= 65536 && page >= 1 && num_pages >= 1, "%s: bad cache geometry", who);
    B200_REQUIRE((int64_t)num_pages * page <= 0x7fffffff, "%s: num_pages * page must fit in 31 bits", who);
    B200_REQUIRE((int64_t)KV * page <= 1 << 23, "%s: a page may have %d rows (tokens times heads)", who, 1 << 23);      // under 2^31 bytes
    return B200_OK;
}

__device__ __forceinline__ uint32_t kc_half(float x) {      // to fp16, the largest value instead of an infinity
    return float_to_half_bits(fminf(fmaxf(x, -65504.0f), 65504.0f));
}
// Largest and smallest, NaN if one is.
__device__ __forceinline__ float kc_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float kc_min(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Two sums, rounded down.
__device__ __forceinline__ f32x2 kc_add_down(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// floor(y + shift), 0 .. 15, of four numbers as nibbles, lowest first, with anything above the low 24 bits: both steps are rounded down,
// which never passes a whole number that the exact sum has not reached, and leave the floor in the low bits of a number of
// exponent 23, the rest of which only reaches bits 24 and up.
__device__ __forceinline__ uint32_t kc_codes(const float2 (&y)[2], float shift) {
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = each(kc_add_down(kc_add_down(two(y[i].x, y[i].y), two(shift, shift)), two(8388608.0f, 8388608.0f)));
        code += ((uint32_t)__float_as_int(f.x) << (8 * i)) + ((uint32_t)__float_as_int(f.y) << (8 * i + 4));
    }
    return code;
}
// One of NB values that eight lanes have each, joined over them: lane g has the one of block g % NB.  Half of the values go
// to a neighbour at each of the first steps, and half as many are left.
template <int NB, typename Join>
__device__ __forceinline__ float kc_join(const float (&x)[NB], int g, Join join) {
    float r;
    if (NB == 4) {
        const bool far = g & 2, odd = g & 1;
        const float a = join(far ? x[2 % NB] : x[0], __shfl_xor_sync(0xffffffffu, far ? x[0] : x[2 % NB], 2));
        const float b = join(far ? x[3 % NB] : x[1], __shfl_xor_sync(0xffffffffu, far ? x[1] : x[3 % NB], 2));
        r = join(odd ? b : a, __shfl_xor_sync(0xffffffffu, odd ? a : b, 1));
    } else {
        const bool odd = g & 1;
        r = join(odd ? x[1] : x[0], __shfl_xor_sync(0xffffffffu, odd ? x[0] : x[1], 1));
        r = join(r, __shfl_xor_sync(0xffffffffu, r, 2));
    }
    return join(r, __shfl_xor_sync(0xffffffffu, r, 4));
}

// A row of a head: its token, its head, and where its codes and scales stand in the pages (K's or V's); slot < 0: in none.
template <int HD, int KIND>
struct KcItem {
    int64_t row;
    int head, slot;
    int64_t codes, scales;
    __device__ __forceinline__ KcItem(const Kv4Rows& a, int64_t item, bool v) {
        row = item < a.n * a.KV ? (int64_t)a.by_KV.div((uint32_t)item) : -1;
        head = (int)(item - row * a.KV);
        slot = row >= 0 ? a.slots[row] : -1;
        if ((uint32_t)slot >= (uint32_t)a.num_slots) slot = -1;
        const int s = max(slot, 0), pg = (int)a.by_page.div(s), off = s - pg * a.page;
        const int64_t at = (int64_t)pg * a.part.bytes + (v ? a.part.v_code : 0), token = (int64_t)head * a.page + off;
        codes = at + token * (HD / 2);
        scales = at + a.part.k_scale + token * (HD / 32 * (KIND == 1 ? 4 : 2));          // V's parts follow as K's do
    }
};

// SIDES 1: K's rows or V's, by blockIdx.y; 2: a thread has its part of both, with both rows' loads under way.
template <int HD, int KIND, bool WIDE, int SIDES>
__global__ void __launch_bounds__(KC_THREADS) kv4_store_kernel(const __grid_constant__ Kv4Rows a) {
    constexpr int NB = HD / 32;
    const int g = threadIdx.x & 7;
    short_begin();
    const KcItem<HD, KIND> it(a, (int64_t)blockIdx.x * KC_ITEMS + (threadIdx.x >> 3), false);
    float rows[SIDES][NB][4];
#pragma unroll
    for (int side = 0; side < SIDES; ++side) {
        const bool v = SIDES == 2 ? side == 1 : blockIdx.y != 0;
        const float* src = (v ? a.v_in + it.row * a.vs : a.k_in + it.row * a.ks) + (int64_t)it.head * HD + 4 * g;
        float(&x)[NB][4] = rows[side];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            x[b][0] = x[b][1] = x[b][2] = x[b][3] = 0.0f;
            if (it.row < 0) continue;
            if (WIDE) {
                const float4 f = *reinterpret_cast<const float4*>(src + 32 * b);
                x[b][0] = f.x; x[b][1] = f.y; x[b][2] = f.z; x[b][3] = f.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[b][i] = src[32 * b + i];
            }
        }
    }
#pragma unroll
    for (int side = 0; side < SIDES; ++side) {
        const bool v = SIDES == 2 ? side == 1 : blockIdx.y != 0;
        float(&x)[NB][4] = rows[side];
        float lo[NB], hi[NB];                                    // kind 0: hi of the magnitudes
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (KIND == 1) {
                lo[b] = kc_min(kc_min(x[b][0], x[b][1]), kc_min(x[b][2], x[b][3]));
                hi[b] = kc_max(kc_max(x[b][0], x[b][1]), kc_max(x[b][2], x[b][3]));
            } else {
                hi[b] = kc_max(kc_max(fabsf(x[b][0]), fabsf(x[b][1])), kc_max(fabsf(x[b][2]), fabsf(x[b][3])));
            }
        }
        // each lane makes one block's scale and inverse, and has the others' from its neighbours
        const float my_hi = kc_join(hi, g, [](float u, float w) { return kc_max(u, w); });
        const float my_lo = KIND == 1 ? kc_join(lo, g, [](float u, float w) { return kc_min(u, w); }) : 0.0f;
        const float d = KIND == 1 ? __fmul_rn(__fsub_rn(my_hi, my_lo), 1.0f / 15.0f) : __fmul_rn(my_hi, 0.125f);
        const bool sound = my_hi < INFINITY && my_lo > -INFINITY;
        const float my_inv = !sound ? -1.0f : d > 0.0f ? __frcp_rn(d) : 0.0f;      // -1: the block is to be zero
        uint32_t word[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float inv = __shfl_sync(0xffffffffu, my_inv, b, 8);
            const float least = KIND == 1 ? __shfl_sync(0xffffffffu, my_lo, b, 8) : 0.0f;
            uint32_t code = KIND == 0 ? 0x8888u : 0u;            // of zeros, of equal ones, of a range that is no fp32 number, and unsound
            if (inv > 0.0f && inv < INFINITY) {
                const f32x2 by = two(inv, inv);
                float2 y[2];
                if (KIND == 1) {                                 // at most 15 of them
                    y[0] = each(mul2(add2(two(x[b][0], x[b][1]), two(-least, -least)), by));
                    y[1] = each(mul2(add2(two(x[b][2], x[b][3]), two(-least, -least)), by));
                    code = kc_codes(y, 0.5f);
                } else {
                    // 8 and the nearest, halves away from zero, 16 as 15: floor(y + 8.5) but for a half below zero, which one bit further from
                    // zero is none
                    y[0] = each(mul2(two(x[b][0], x[b][1]), by));
                    y[1] = each(mul2(two(x[b][2], x[b][3]), by));
                    auto further = [](float v) { return fminf(__int_as_float(__float_as_int(v) + (int)((uint32_t)__float_as_int(v) >> 31)), 7.0f); };
                    y[0] = make_float2(further(y[0].x), further(y[0].y));
                    y[1] = make_float2(further(y[1].x), further(y[1].y));
                    code = kc_codes(y, 8.5f);
                }
            }
            if (inv == INFINITY) {                               // a block of denormals: all that is not its zero (or minimum) is as far as codes go
                code = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) code |= (KIND == 1 ? (x[b][i] > least ? 15u : 0u) : x[b][i] > 0.0f ? 15u : x[b][i] < 0.0f ? 0u : 8u) << (4 * i);
            }
            word[b] = code & 0xFFFFu;
        }
        if (it.slot < 0) continue;
        const int64_t side_at = v ? a.part.v_code : 0;      // V's parts follow as K's do
        uint8_t* codes = a.pages + side_at + it.codes + g * (2 * NB);
        if (NB == 4) *reinterpret_cast<uint2*>(codes) = make_uint2(word[0] | (word[1] << 16), word[NB > 2 ? 2 : 0] | (word[NB > 2 ? 3 : 0] << 16));
        else *reinterpret_cast<uint32_t*>(codes) = word[0] | (word[1] << 16);
        if (g < NB) {
            uint8_t* scale = a.pages + side_at + it.scales + g * (KIND == 1 ? 4 : 2);
            const float m = sound ? my_lo : 0.0f;
            if (KIND == 1) *reinterpret_cast<uint32_t*>(scale) = sound ? kc_half(d) | (kc_half(m) << 16) : 0u;
            else *reinterpret_cast<uint16_t*>(scale) = sound ? (uint16_t)kc_half(d) : (uint16_t)0;
        }
    }
}

template <int HD, int KIND, bool WIDE>
__global__ void __launch_bounds__(KC_THREADS) kv4_fetch_kernel(const __grid_constant__ Kv4Rows a) {
    constexpr int NB = HD / 32;
    const bool v = a.k_out ? blockIdx.y != 0 : true;
    const int g = threadIdx.x & 7;
    short_begin();
    const KcItem<HD, KIND> it(a, (int64_t)blockIdx.x * KC_ITEMS + (threadIdx.x >> 3), v);
    if (it.slot < 0) return;
    uint32_t word[NB / 2], scale[KIND == 1 ? NB : NB / 2];
    auto fill = [](uint32_t* w, int n, const uint8_t* p) {
        if (n == 4) {
            const uint4 f = *reinterpret_cast<const uint4*>(p);
            w[0] = f.x; w[1] = f.y; w[2] = f.z; w[3] = f.w;
        } else if (n == 2) {
            const uint2 f = *reinterpret_cast<const uint2*>(p);
            w[0] = f.x; w[1] = f.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    };
    fill(word, NB / 2, a.pages + it.codes + g * (2 * NB));
    fill(scale, KIND == 1 ? NB : NB / 2, a.pages + it.scales);
    float* dst = (v ? a.v_out + it.row * a.vs : a.k_out + it.row * a.ks) + (int64_t)it.head * HD + 4 * g;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t code = word[b / 2] >> (b & 1 ? 16 : 0);
        const uint32_t s = KIND == 1 ? scale[b < NB && KIND == 1 ? b : 0] : scale[b / 2] >> (b & 1 ? 16 : 0);
        const float d = half_bits_to_float((uint16_t)s), m = KIND == 1 ? half_bits_to_float((uint16_t)(s >> 16)) : 0.0f;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {                       // a code under the exponent of 2^23 is 2^23 and itself
            const float f = __int_as_float(((code >> (4 * i)) & 15) | 0x4B000000);
            x[i] = KIND == 1 ? fmaf(d, f - 8388608.0f, m) : d * (f - 8388616.0f);       // d * code is exact: one rounding
        }
        if (WIDE) {
            *reinterpret_cast<float4*>(dst + 32 * b) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[32 * b + i] = x[i];
        }
    }
}

static void kc_geometry(Kv4Rows& a, void* pages, int num_pages, int page, int KV, int hd, int kind) {
    a.pages = static_cast<uint8_t*>(pages);
    a.num_slots = num_pages * page;
    a.page = page;
    a.KV = KV;
    a.by_page = FastDiv(page);
    a.by_KV = FastDiv(KV);
    a.part = Kv4Page(page, KV, hd, kind);
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_kv4_page_bytes(int page, int KV, int hd, int kind, size_t* bytes) {
    int rc = kv4_check("kv4_page_bytes", 1, page, KV, hd, kind);
    if (rc) return rc;
    B200_REQUIRE(bytes, "kv4_page_bytes: null pointer");
    *bytes = (size_t)Kv4Page(page, KV, hd, kind).bytes;
    return B200_OK;
}

int b200_kv4_store(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* slots, int64_t n,
                   void* pages, int num_pages, int page, int KV, int hd, int kind) {
    if (n <= 0) return B200_OK;
    int rc = kv4_check("kv4_store", num_pages, page, KV, hd, kind);
    if (rc) return rc;
    B200_REQUIRE(n <= 0x7fffffff / KV, "kv4_store: too many rows");
    B200_REQUIRE(k && v && slots && pages, "kv4_store: null pointer");
    B200_REQUIRE(aligned16(pages), "kv4_store: pages must be 16-byte aligned");
    B200_REQUIRE(k_stride >= (int64_t)KV * hd && v_stride >= (int64_t)KV * hd, "kv4_store: a stride is shorter than its row");
    Kv4Rows a;
    kc_geometry(a, pages, num_pages, page, KV, hd, kind);
    a.k_in = k; a.v_in = v; a.ks = k_stride; a.vs = v_stride; a.slots = slots; a.n = n;
    const bool wide = aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0;
    // A thread with both sides finds one address for them and has twice the loads under way, in half as many blocks: better as soon as
    // these are one an SM (8 x 128, kind 0: 512 rows 4.2 -> 3.2 us, 4096 10.4 -> 8.3, 16 384 30.3 -> 26.8; kind 1 of 4 x 64: 1024 rows 4.2 -> 2.3;
    // one case the other way, 1024 rows of 8 x 128, kind 1, 4.6 -> 5.2).  Below, the longer thread is what is waited for (256 rows 2.4 -> 2.5).
    const dim3 block(KC_THREADS);
    const unsigned blocks = (unsigned)ceil_div64(n * KV, KC_ITEMS);
    const bool both = blocks > (unsigned)num_sms();
    const dim3 grid(blocks, both ? 1 : 2);
    auto pick = [&](auto hd_, auto kind_) {
        constexpr int HD = decltype(hd_)::value, KIND = decltype(kind_)::value;
        return wide ? (both ? kv4_store_kernel<HD, KIND, true, 2> : kv4_store_kernel<HD, KIND, true, 1>)
                    : (both ? kv4_store_kernel<HD, KIND, false, 2> : kv4_store_kernel<HD, KIND, false, 1>);
    };
    using std::integral_constant;
    auto kern = hd == 64 ? (kind == 1 ? pick(integral_constant<int, 64>(), integral_constant<int, 1>()) : pick(integral_constant<int, 64>(), integral_constant<int, 0>()))
                         : (kind == 1 ? pick(integral_constant<int, 128>(), integral_constant<int, 1>()) : pick(integral_constant<int, 128>(), integral_constant<int, 0>()));
    return launch_serve("kv4_store_kernel", kern, grid, block, 0, 1, short_grid(grid), a);
}

int b200_kv4_fetch(const void* pages, int num_pages, int page, const int32_t* slots, int64_t n, float* k, float* v,
                   int64_t k_stride, int64_t v_stride, int KV, int hd, int kind) {
    if (n <= 0) return B200_OK;
    int rc = kv4_check("kv4_fetch", num_pages, page, KV, hd, kind);
    if (rc) return rc;
    B200_REQUIRE(n <= 0x7fffffff / KV, "kv4_fetch: too many rows");
    B200_REQUIRE((k || v) && slots && pages, "kv4_fetch: null pointer");
    B200_REQUIRE(aligned16(pages), "kv4_fetch: pages must be 16-byte aligned");
    B200_REQUIRE((!k || k_stride >= (int64_t)KV * hd) && (!v || v_stride >= (int64_t)KV * hd), "kv4_fetch: a stride is shorter than its row");
    Kv4Rows a;
    kc_geometry(a, const_cast<void*>(pages), num_pages, page, KV, hd, kind);
    a.k_out = k; a.v_out = v; a.ks = k_stride; a.vs = v_stride; a.slots = slots; a.n = n;
    const bool wide = (!k || (aligned16(k) && k_stride % 4 == 0)) && (!v || (aligned16(v) && v_stride % 4 == 0));
    const dim3 grid((unsigned)ceil_div64(n * KV, KC_ITEMS), k && v ? 2 : 1), block(KC_THREADS);
    auto kern = hd == 64 ? (kind == 1 ? (wide ? kv4_fetch_kernel<64, 1, true> : kv4_fetch_kernel<64, 1, false>)
                                      : (wide ? kv4_fetch_kernel<64, 0, true> : kv4_fetch_kernel<64, 0, false>))
                         : (kind == 1 ? (wide ? kv4_fetch_kernel<128, 1, true> : kv4_fetch_kernel<128, 1, false>)
                                      : (wide ? kv4_fetch_kernel<128, 0, true> : kv4_fetch_kernel<128, 0, false>));
    return launch_serve("kv4_fetch_kernel", kern, grid, block, 0, 1, short_grid(grid), a);
}

}  // extern "C"
