// Rows of keys and values into the 4-bit pages and back (layout: b200serve.h).
//
// The rule is b200_quantize's for kinds 0 and 1, one correctly rounded fp32 operation at a time, but for two things.  The step of
// kind 1 is (max - min) times fp32(1/15) where that divides by 15: every new token pays for it, and the quotient's last bit
// decides only for a value on the border of two codes.  And a scale or minimum beyond the range of fp16 is kept at its largest
// value, because an infinite one would make a NaN of every code 0, and of every masked probability in the attention over these
// pages.
//
// What bounds both: the fp32 rows (8 KV hd bytes a token), a quarter of that again for the pages' lines.  Eight lanes share a block of 32, each
// with the four elements of one 16-bit word, so a warp reads 512 consecutive bytes and the block's statistics take three
// shuffles.
#include <type_traits>

#include "serve.cuh"

namespace b200 {

constexpr int KC_THREADS = 256;

struct Kv4Rows {
    const float *k_in = nullptr, *v_in = nullptr;
    float *k_out = nullptr, *v_out = nullptr;
    int64_t ks = 0, vs = 0;
    const int32_t* slots = nullptr;
    uint8_t* pages = nullptr;
    int64_t n = 0;
    int num_slots = 0, page = 1, KV = 0, nb = 0;
    FastDiv by_page, by_nb;
    Kv4Page part;
};

int kv4_check(const char* who, int num_pages, int page, int KV, int hd, int kind) {
    B200_REQUIRE(hd == 64 || hd == 128, "%s: hd must be 64 or 128", who);
    B200_REQUIRE(kind == 0 || kind == 1, "%s: kind must be 0 (Q4_0) or 1 (Q4_1)", who);
    B200_REQUIRE(KV >= 1 && KV <= 65536 && page >= 1 && num_pages >= 1, "%s: bad cache geometry", who);
    B200_REQUIRE((int64_t)num_pages * page <= 0x7fffffff, "%s: num_pages * page must fit in 31 bits", who);
    return B200_OK;
}

// Where block `blk` (head * nb + b) of `slot` stands: its codes' 16-bit words (stride nb) and its scale.
struct KcPlace {
    uint16_t* word;
    uint8_t* scale;
};
template <int KIND>
__device__ __forceinline__ KcPlace kc_place(const Kv4Rows& a, int slot, int blk, bool v) {
    const int pg = (int)a.by_page.div(slot), off = slot - pg * a.page;
    const int h = (int)a.by_nb.div(blk), b = blk - h * a.nb;
    uint8_t* base = a.pages + (int64_t)pg * a.part.bytes;
    const int64_t row = (int64_t)h * a.page + off;
    return {reinterpret_cast<uint16_t*>(base + (v ? a.part.v_code : 0) + row * (a.nb * 16)) + b,
            base + (v ? a.part.v_scale : a.part.k_scale) + (row * a.nb + b) * (KIND == 1 ? 4 : 2)};
}

__device__ __forceinline__ uint32_t kc_half(float x) {      // to fp16, the largest value instead of an infinity
    return float_to_half_bits(fminf(fmaxf(x, -65504.0f), 65504.0f));
}

// Rows of a thread: its loads are all under way before the first is used.  Few rows: one, so that they spread over the device.
constexpr int KC_ROWS = 4;

// blockIdx.y: 0 K, 1 V.  Eight lanes per block of 32 elements, ROWS rows one after another.
template <int KIND, bool WIDE, int ROWS>
__global__ void __launch_bounds__(KC_THREADS) kv4_store_kernel(const __grid_constant__ Kv4Rows a) {
    const bool v = blockIdx.y != 0;
    const float* src = v ? a.v_in : a.k_in;
    const int64_t stride = v ? a.vs : a.ks, row0 = (int64_t)blockIdx.x * ROWS;
    const int blocks = a.KV * a.nb, g = threadIdx.x & 7;
    int slot[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) slot[r] = row0 + r < a.n ? a.slots[row0 + r] : -1;
    for (int blk = threadIdx.x >> 3; blk < (blocks + 3) / 4 * 4; blk += KC_THREADS / 8) {       // whole warps: four blocks each
        float x[ROWS][4];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            x[r][0] = x[r][1] = x[r][2] = x[r][3] = 0.0f;
            if (row0 + r >= a.n || blk >= blocks) continue;
            const float* p = src + (row0 + r) * stride + (int64_t)blk * 32 + 4 * g;
            if (WIDE) {
                const float4 f = *reinterpret_cast<const float4*>(p);
                x[r][0] = f.x; x[r][1] = f.y; x[r][2] = f.z; x[r][3] = f.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[r][i] = p[i];
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            bool bad = !(isfinite(x[r][0]) && isfinite(x[r][1]) && isfinite(x[r][2]) && isfinite(x[r][3]));
            bad = (__ballot_sync(0xffffffffu, bad) & (0xFFu << (threadIdx.x & 24))) != 0;
            uint32_t code = 0, scale;
            if (KIND == 0) {
                float top = fmaxf(fmaxf(fabsf(x[r][0]), fabsf(x[r][1])), fmaxf(fabsf(x[r][2]), fabsf(x[r][3])));
#pragma unroll
                for (int s = 1; s < 8; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                const float d = __fdiv_rn(top, 8.0f), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) code |= (uint32_t)(min(max((int)roundf(__fmul_rn(x[r][i], inv)), -8), 7) + 8) << (4 * i);
                scale = kc_half(d);
                if (bad) { code = 0x8888u; scale = 0; }
            } else {
                float lo = fminf(fminf(x[r][0], x[r][1]), fminf(x[r][2], x[r][3])), hi = fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3]));
#pragma unroll
                for (int s = 1; s < 8; s <<= 1) {
                    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
                    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
                }
                const float d = __fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) code |= (uint32_t)min(max((int)roundf(__fmul_rn(__fsub_rn(x[r][i], lo), inv)), 0), 15) << (4 * i);
                scale = kc_half(d) | (kc_half(lo) << 16);
                if (bad) { code = 0; scale = 0; }
            }
            if (blk < blocks && (uint32_t)slot[r] < (uint32_t)a.num_slots) {
                const KcPlace at = kc_place<KIND>(a, slot[r], blk, v);
                at.word[g * a.nb] = (uint16_t)code;
                if (g == 0) {
                    if (KIND == 1) *reinterpret_cast<uint32_t*>(at.scale) = scale;
                    else *reinterpret_cast<uint16_t*>(at.scale) = (uint16_t)scale;
                }
            }
        }
    }
}

template <int KIND, bool WIDE, int ROWS>
__global__ void __launch_bounds__(KC_THREADS) kv4_fetch_kernel(const __grid_constant__ Kv4Rows a) {
    const bool v = a.k_out ? blockIdx.y != 0 : true;
    float* dst = v ? a.v_out : a.k_out;
    const int64_t stride = v ? a.vs : a.ks, row0 = (int64_t)blockIdx.x * ROWS;
    const int words = a.KV * a.nb * 8;
    int slot[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) slot[r] = row0 + r < a.n ? a.slots[row0 + r] : -1;
    for (int w = threadIdx.x; w < words; w += KC_THREADS) {
        uint32_t code[ROWS], scale[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            code[r] = scale[r] = 0;
            if ((uint32_t)slot[r] >= (uint32_t)a.num_slots) continue;
            const KcPlace at = kc_place<KIND>(a, slot[r], w >> 3, v);
            code[r] = at.word[(w & 7) * a.nb];
            scale[r] = KIND == 1 ? *reinterpret_cast<const uint32_t*>(at.scale) : *reinterpret_cast<const uint16_t*>(at.scale);
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if ((uint32_t)slot[r] >= (uint32_t)a.num_slots) continue;
            const float d = half_bits_to_float((uint16_t)scale[r]), m = half_bits_to_float((uint16_t)(scale[r] >> 16));
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = (code[r] >> (4 * i)) & 15;
                x[i] = KIND == 1 ? __fadd_rn(__fmul_rn(d, (float)c), m) : __fmul_rn(d, (float)(c - 8));
            }
            float* p = dst + (row0 + r) * stride + (int64_t)w * 4;
            if (WIDE) {
                *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = x[i];
            }
        }
    }
}

static void kc_geometry(Kv4Rows& a, void* pages, int num_pages, int page, int KV, int hd, int kind) {
    a.pages = static_cast<uint8_t*>(pages);
    a.num_slots = num_pages * page;
    a.page = page;
    a.KV = KV;
    a.nb = hd / 32;
    a.by_page = FastDiv(page);
    a.by_nb = FastDiv(a.nb);
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
    B200_REQUIRE(n <= 0x7fffffff, "kv4_store: too many rows");
    B200_REQUIRE(k && v && slots && pages, "kv4_store: null pointer");
    B200_REQUIRE(aligned16(pages), "kv4_store: pages must be 16-byte aligned");
    B200_REQUIRE(k_stride >= (int64_t)KV * hd && v_stride >= (int64_t)KV * hd, "kv4_store: a stride is shorter than its row");
    Kv4Rows a;
    kc_geometry(a, pages, num_pages, page, KV, hd, kind);
    a.k_in = k; a.v_in = v; a.ks = k_stride; a.vs = v_stride; a.slots = slots; a.n = n;
    const bool wide = aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0;
    const bool many = n >= KC_ROWS * num_sms();
    const dim3 grid((unsigned)(many ? ceil_div64(n, KC_ROWS) : n), 2), block(KC_THREADS);
    auto pick = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        return kind == 1 ? (wide ? kv4_store_kernel<1, true, R> : kv4_store_kernel<1, false, R>)
                         : (wide ? kv4_store_kernel<0, true, R> : kv4_store_kernel<0, false, R>);
    };
    auto kern = many ? pick(std::integral_constant<int, KC_ROWS>()) : pick(std::integral_constant<int, 1>());
    return launch_serve("kv4_store_kernel", kern, grid, block, 0, 1, false, a);
}

int b200_kv4_fetch(const void* pages, int num_pages, int page, const int32_t* slots, int64_t n, float* k, float* v,
                   int64_t k_stride, int64_t v_stride, int KV, int hd, int kind) {
    if (n <= 0) return B200_OK;
    int rc = kv4_check("kv4_fetch", num_pages, page, KV, hd, kind);
    if (rc) return rc;
    B200_REQUIRE(n <= 0x7fffffff, "kv4_fetch: too many rows");
    B200_REQUIRE((k || v) && slots && pages, "kv4_fetch: null pointer");
    B200_REQUIRE(aligned16(pages), "kv4_fetch: pages must be 16-byte aligned");
    B200_REQUIRE((!k || k_stride >= (int64_t)KV * hd) && (!v || v_stride >= (int64_t)KV * hd), "kv4_fetch: a stride is shorter than its row");
    Kv4Rows a;
    kc_geometry(a, const_cast<void*>(pages), num_pages, page, KV, hd, kind);
    a.k_out = k; a.v_out = v; a.ks = k_stride; a.vs = v_stride; a.slots = slots; a.n = n;
    const bool wide = (!k || (aligned16(k) && k_stride % 4 == 0)) && (!v || (aligned16(v) && v_stride % 4 == 0));
    const bool many = n >= KC_ROWS * num_sms();
    const dim3 grid((unsigned)(many ? ceil_div64(n, KC_ROWS) : n), k && v ? 2 : 1), block(KC_THREADS);
    auto pick = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        return kind == 1 ? (wide ? kv4_fetch_kernel<1, true, R> : kv4_fetch_kernel<1, false, R>)
                         : (wide ? kv4_fetch_kernel<0, true, R> : kv4_fetch_kernel<0, false, R>);
    };
    auto kern = many ? pick(std::integral_constant<int, KC_ROWS>()) : pick(std::integral_constant<int, 1>());
    return launch_serve("kv4_fetch_kernel", kern, grid, block, 0, 1, false, a);
}

}  // extern "C"
