// Attention of ragged rows over the 4-bit pages: the plain kernel, one block per row and head.
#include <algorithm>

#include "serve.cuh"

namespace b200 {

constexpr int A4_WARPS = 4;

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
    FastDiv by_page;
    Kv4Page part;
    float scale;
    int window;
};

template <int HD, int KIND>
__global__ void __launch_bounds__(A4_WARPS * 32) attn_kv4_plain_kernel(Kv4AttnArgs a) {
    constexpr int NB = HD / 32, E = HD / 32;                 // elements per lane: element 32 e + lane
    __shared__ float s_ml[A4_WARPS][2], s_o[A4_WARPS][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
        const int first = a.offsets ? a.offsets[b] : b, rows = a.offsets ? a.offsets[b + 1] - first : 1;
        const int len = min(a.lens[b], a.max_pages * a.page);
        for (int i = blockIdx.z; i < rows; i += gridDim.z) {
            const int h = blockIdx.x, kv = h / a.group, pos = len - rows + i;
            const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) { q[e] = a.q[(first + i) * a.qs + (int64_t)h * HD + 32 * e + lane] * a.scale; o[e] = 0.0f; }
            for (int j = lo + warp; j <= pos; j += A4_WARPS) {
                const int p = (int)a.by_page.div(j), off = j - p * a.page, id = a.table[(int64_t)b * a.max_pages + p];
                const bool there = (uint32_t)id < (uint32_t)a.num_pages;
                const uint8_t* base = a.pages + (int64_t)(there ? id : 0) * a.part.bytes;
                const int64_t row = (int64_t)kv * a.page + off;
                auto value = [&](int64_t codes, int64_t scales, int e) {
                    if (!there) return 0.0f;
                    const int g = lane >> 2;
                    const int c = (reinterpret_cast<const uint16_t*>(base + codes + row * (HD / 2))[g * NB + e] >> (4 * (lane & 3))) & 15;
                    const uint16_t* s = reinterpret_cast<const uint16_t*>(base + scales) + (row * NB + e) * (KIND == 1 ? 2 : 1);
                    return KIND == 1 ? half_bits_to_float(s[0]) * (float)c + half_bits_to_float(s[KIND]) : half_bits_to_float(s[0]) * (float)(c - 8);
                };
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) x += q[e] * value(0, a.part.k_scale, e);
                x = warp_sum(x);
                const float mn = fmaxf(m, x), f = expf(m - mn), w = expf(x - mn);
                l = l * f + w;
                m = mn;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * value(a.part.v_code, a.part.v_scale, e);
            }
            if (lane == 0) { s_ml[warp][0] = m; s_ml[warp][1] = l; }
#pragma unroll
            for (int e = 0; e < E; ++e) s_o[warp][32 * e + lane] = o[e];
            __syncthreads();
            if (warp == 0) {
                float mm = -INFINITY, ll = 0.0f;
                for (int w = 0; w < A4_WARPS; ++w) mm = fmaxf(mm, s_ml[w][0]);
                for (int w = 0; w < A4_WARPS; ++w) ll += s_ml[w][1] == 0.0f ? 0.0f : s_ml[w][1] * expf(s_ml[w][0] - mm);
                for (int e = 0; e < E; ++e) {
                    float v = 0.0f;
                    for (int w = 0; w < A4_WARPS; ++w) v += s_ml[w][1] == 0.0f ? 0.0f : s_o[w][32 * e + lane] * expf(s_ml[w][0] - mm);
                    a.out[(first + i) * a.os + (int64_t)h * HD + 32 * e + lane] = ll == 0.0f ? 0.0f : v / ll;
                }
            }
            __syncthreads();
        }
    }
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_attention_paged_kv4_workspace(int H, int KV, int hd, int max_rows, size_t* bytes) {
    int rc = kv4_check("attention_paged_kv4_workspace", 1, 1, KV, hd, 0);
    if (rc) return rc;
    B200_REQUIRE(bytes, "attention_paged_kv4_workspace: null pointer");
    B200_REQUIRE(H >= 1 && H % KV == 0 && max_rows >= 1, "attention_paged_kv4_workspace: H must be a positive multiple of KV, max_rows positive");
    *bytes = 16;
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
    B200_REQUIRE(max_rows >= 1 && max_pages >= 1 && (int64_t)max_pages * page <= 0x7fffffff, "%s: bad max_rows or max_pages", who);
    B200_REQUIRE(q && pages && page_table && seq_lens && out && workspace, "%s: null pointer", who);
    B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(pages) && aligned16(workspace) && q_stride % 4 == 0 && out_stride % 4 == 0,
                 "%s: q, out, pages and workspace must be 16-byte aligned, strides multiples of 4", who);
    B200_REQUIRE(q_stride >= (int64_t)H * hd && out_stride >= (int64_t)H * hd, "%s: a stride is shorter than its row", who);
    size_t need = 0;
    rc = b200_attention_paged_kv4_workspace(H, KV, hd, max_rows, &need);
    if (rc) return rc;
    B200_REQUIRE(workspace_bytes >= need, "%s: the workspace has %zu bytes of %zu", who, workspace_bytes, need);
    Kv4AttnArgs a{q, q_stride, row_offsets, static_cast<const uint8_t*>(pages), num_pages, page_table, seq_lens, out, out_stride, batch,
                  max_pages, page, H, KV, H / KV, FastDiv(page), Kv4Page(page, KV, hd, kind), scale, window};
    const dim3 grid(H, std::min(batch, 65535), std::min(max_rows, 65535)), block(A4_WARPS * 32);
    auto kern = hd == 64 ? (kind == 1 ? attn_kv4_plain_kernel<64, 1> : attn_kv4_plain_kernel<64, 0>)
                         : (kind == 1 ? attn_kv4_plain_kernel<128, 1> : attn_kv4_plain_kernel<128, 0>);
    return launch_serve("attn_kv4_plain_kernel", kern, grid, block, 0, 1, false, a);
}

}  // extern "C"
