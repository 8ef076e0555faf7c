// Block tables, row offsets, positions and slots of a serving step from the requests' lengths.
//
// Three prefix sums over the requests in order - rows, pages taken, pages given back - say everything: a request is admitted
// while its inclusive sums fit the rows and the free pages, both of which only grow, so the refused requests with rows are a
// tail and the offsets are the sums cut off at the last admitted one.  Row r then belongs to the last request whose offset is
// at most r, found by bisection in shared memory; the same for the pages.
//
// What bounds it: latency (a few kilobytes in, 8 bytes per row out).  So every block reads the requests and sums them by itself,
// and writes its share of the rows and pages; the first also what belongs to the requests.  Where those outputs are the inputs and one
// block is not enough, a second launch of one block writes them when nobody reads any more.
// 5 requests 4.0 us, 700 with 88 000 rows 6.3 (a cluster of eight blocks that waits before it writes: 24.6).
#include <algorithm>

#include "serve.cuh"

namespace b200 {

constexpr int PP_THREADS = 512;
constexpr int PP_EACH = 4;                       // requests of a thread
constexpr int PP_BATCH = PP_THREADS * PP_EACH;

struct PlanArgs {
    const int32_t *ctx, *fresh, *held;
    int batch;
    int32_t* table;
    int max_pages, page, num_pages;
    FastDiv by_page;
    int32_t* ring;
    uint32_t ring_size;
    const int64_t* at;
    int64_t* at_out;
    int32_t *seq_lens, *held_out, *offsets, *positions, *slots;
    int max_rows;
    int32_t* counts;
    bool expand, report;                         // rows and pages; what belongs to the requests
};

// Last index in [0, n) whose entry is at most x (s[0] = 0 <= x, s ascending).
__device__ __forceinline__ int pp_find(const int* s, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PP_THREADS) paged_plan_kernel(const __grid_constant__ PlanArgs a) {
    __shared__ int s_row[PP_BATCH + 1], s_take[PP_BATCH + 1], s_back[PP_BATCH], s_ctx[PP_BATCH], s_held[PP_BATCH];
    __shared__ long long s_part[PP_THREADS / 32][3];
    __shared__ int s_most[2], s_refused;
    __shared__ uint32_t s_ring[2];                 // where the ring starts and ends
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    short_begin();
    const long long head = a.at[0], tail = a.at[1];
    const bool sound = head >= 0 && tail >= head && tail - head <= (long long)a.ring_size;
    const long long avail = sound ? tail - head : 0;
    const int warps = (a.batch + 32 * PP_EACH - 1) / (32 * PP_EACH);        // that have requests
    if (warp == PP_THREADS / 32 - 1) {             // the one that has them last; a quotient of 64 bits is a hundred instructions
        if (lane < 2) {
            s_ring[lane] = sound ? (uint32_t)((lane ? tail : head) % a.ring_size) : 0;
            s_most[lane] = 0;
        }
        if (lane == 2) s_refused = 0;
    }
    int ctx[PP_EACH], fresh[PP_EACH], held[PP_EACH];
    long long rows[PP_EACH], take[PP_EACH], back[PP_EACH], sum[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < PP_EACH; ++i) {
        const int b = tid * PP_EACH + i;
        const bool there = b < a.batch;
        ctx[i] = there ? a.ctx[b] : 0;
        fresh[i] = there ? a.fresh[b] : 0;
        held[i] = there ? a.held[b] : 0;
    }
#pragma unroll
    for (int i = 0; i < PP_EACH; ++i) {
        const uint32_t want = (uint32_t)ctx[i] + (uint32_t)fresh[i];        // of two numbers below 2^31
        const bool fits = fresh[i] > 0 && ctx[i] >= 0 && held[i] >= 0 && held[i] <= a.max_pages && want <= (uint32_t)(a.max_pages * a.page);
        rows[i] = fits ? fresh[i] : 0;
        const uint32_t full = a.by_page.div(fits ? want : 0u), pages = full + (want > full * a.page);
        take[i] = fits ? max(0, (int)pages - held[i]) : 0;
        back[i] = fresh[i] < 0 ? min(max(held[i], 0), a.max_pages) : 0;
        sum[0] += rows[i];
        sum[1] += take[i];
        sum[2] += back[i];
    }
    long long before[3] = {0, 0, 0};
    if (warp < warps) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            long long v = sum[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            before[k] = v - sum[k];
            if (lane == 31) s_part[warp][k] = v;
        }
    }
    __syncthreads();
    long long all_back = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp)
#pragma unroll
            for (int k = 0; k < 3; ++k) before[k] += s_part[w][k];
        all_back += s_part[w][2];
    }
    // admission; the largest sums among the admitted are the step's totals
    bool ok[PP_EACH];
    int refused = 0, most_rows = 0, most_take = 0;
    long long first_row[PP_EACH], first_take[PP_EACH], first_back[PP_EACH];
#pragma unroll
    for (int i = 0; i < PP_EACH; ++i) {
        first_row[i] = before[0];
        first_take[i] = before[1];
        first_back[i] = before[2];
        before[0] += rows[i];
        before[1] += take[i];
        before[2] += back[i];
        ok[i] = rows[i] > 0 && before[0] <= a.max_rows && before[1] <= avail;
        if (ok[i]) {
            most_rows = (int)before[0];
            most_take = (int)before[1];
        }
        refused += fresh[i] > 0 && !ok[i];
    }
    if (warp < warps) {
        most_rows = __reduce_max_sync(0xffffffffu, most_rows);
        most_take = __reduce_max_sync(0xffffffffu, most_take);
        refused = __reduce_add_sync(0xffffffffu, refused);
        if (lane == 0) {
            atomicMax(&s_most[0], most_rows);
            atomicMax(&s_most[1], most_take);
            if (refused) atomicAdd(&s_refused, refused);
        }
    }
    __syncthreads();
    const int all_rows = s_most[0], all_take = s_most[1];
    // more pages than the ring has room for: a page held twice; none is put in
    const int given = sound && all_back <= (long long)a.ring_size - avail ? (int)all_back : 0;
#pragma unroll
    for (int i = 0; i < PP_EACH; ++i) {
        const int b = tid * PP_EACH + i;
        if (b < a.batch) {
            s_row[b] = (int)min(first_row[i], (long long)all_rows);
            s_take[b] = (int)min(first_take[i], (long long)all_take);
            s_back[b] = (int)first_back[i];
            s_ctx[b] = ctx[i];
            s_held[b] = held[i];
        }
    }
    if (tid == 0) {
        s_row[a.batch] = all_rows;
        s_take[a.batch] = all_take;
    }
    __syncthreads();                             // everything is read that a single block's outputs may overwrite
    const uint32_t nthreads = gridDim.x * PP_THREADS, id = blockIdx.x * PP_THREADS + tid;
    if (a.report && blockIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < PP_EACH; ++i) {
            const int b = tid * PP_EACH + i;
            if (b >= a.batch) continue;
            a.seq_lens[b] = fresh[i] < 0 ? 0 : ok[i] ? ctx[i] + fresh[i] : ctx[i];
            a.held_out[b] = fresh[i] < 0 ? 0 : ok[i] ? held[i] + (int)take[i] : held[i];
            a.offsets[b] = s_row[b];
        }
        if (tid == 0) {
            a.offsets[a.batch] = all_rows;
            a.at_out[0] = head + all_take;
            a.at_out[1] = tail + given;
            a.counts[0] = all_rows;
            a.counts[1] = all_take;
            a.counts[2] = given;
            a.counts[3] = s_refused;
        }
    }
    if (!a.expand) return;
    const uint32_t ring_head = s_ring[0], ring_tail = s_ring[1];
    auto ring_index = [&](uint32_t from, uint32_t j) {      // both below the ring's size
        const uint32_t i = from + j;
        return i >= a.ring_size ? i - a.ring_size : i;
    };
    for (uint32_t j = id; j < (uint32_t)all_take; j += nthreads) {
        const int b = pp_find(s_take, a.batch, (int)j);
        a.table[(int64_t)b * a.max_pages + s_held[b] + ((int)j - s_take[b])] = a.ring[ring_index(ring_head, j)];
    }
    // the pages of the finished: behind the ring's end, never over entries that are being taken
    for (uint32_t j = id; j < (uint32_t)given; j += nthreads) {
        const int b = pp_find(s_back, a.batch, (int)j);
        a.ring[ring_index(ring_tail, j)] = a.table[(int64_t)b * a.max_pages + ((int)j - s_back[b])];
    }
    // two rows at a time, both looked up before either is written (a store might be what the next load reads, for all the compiler knows)
    for (uint32_t r0 = id; r0 < (uint32_t)a.max_rows; r0 += 2 * nthreads) {
        int pos[2], off[2], id_of[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t r = r0 + s * nthreads;
            pos[s] = id_of[s] = -1;
            off[s] = 0;
            if (r >= (uint32_t)all_rows) continue;
            const int b = pp_find(s_row, a.batch, (int)r);
            pos[s] = s_ctx[b] + ((int)r - s_row[b]);
            const int p = (int)a.by_page.div(pos[s]), more = p - s_held[b];
            off[s] = pos[s] - p * a.page;
            id_of[s] = more < 0 ? a.table[(int64_t)b * a.max_pages + p] : a.ring[ring_index(ring_head, s_take[b] + more)];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t r = r0 + s * nthreads;
            if (r >= (uint32_t)a.max_rows) continue;
            a.positions[r] = pos[s];
            a.slots[r] = (uint32_t)id_of[s] < (uint32_t)a.num_pages ? id_of[s] * a.page + off[s] : -1;
        }
    }
}

}  // namespace b200

using namespace b200;

extern "C" int b200_paged_plan(const int32_t* ctx_lens, const int32_t* new_lens, const int32_t* held, int batch, int32_t* page_table,
                               int max_pages, int page, int num_pages, int32_t* free_ring, int ring_size, const int64_t* ring_at,
                               int64_t* ring_at_out, int32_t* seq_lens, int32_t* held_out, int32_t* row_offsets,
                               int32_t* positions, int32_t* slots, int max_rows, int32_t* counts) {
    B200_REQUIRE(batch >= 0 && batch <= PP_BATCH, "paged_plan: batch must be in [0, %d]", PP_BATCH);
    B200_REQUIRE(page >= 1 && max_pages >= 1 && num_pages >= 1, "paged_plan: bad page geometry");
    B200_REQUIRE((int64_t)num_pages * page <= 0x7fffffff && (int64_t)max_pages * page <= 0x7fffffff,
                 "paged_plan: num_pages * page and max_pages * page must fit in 31 bits");
    B200_REQUIRE(ring_size >= num_pages, "paged_plan: the ring must have room for every page");
    B200_REQUIRE(max_rows >= 0, "paged_plan: negative max_rows");
    B200_REQUIRE(ring_at && ring_at_out && free_ring && row_offsets && counts, "paged_plan: null pointer");
    B200_REQUIRE(batch == 0 || (ctx_lens && new_lens && held && page_table && seq_lens && held_out), "paged_plan: null pointer");
    B200_REQUIRE(max_rows == 0 || (positions && slots), "paged_plan: null pointer");
    PlanArgs a{ctx_lens, new_lens, held, batch, page_table, max_pages, page, num_pages, FastDiv(page), free_ring, (uint32_t)ring_size,
               ring_at, ring_at_out, seq_lens, held_out, row_offsets, positions, slots, max_rows, counts, true, true};
    // A row a thread where that takes no second launch (700 requests with 88 000 rows 6.3 us, with two 6.8), else two.
    const bool in_place = seq_lens == ctx_lens || held_out == held || ring_at_out == ring_at;
    const int blocks = std::min(num_sms(), std::max(ceil_div(std::min(max_rows, 1 << 30), in_place ? 2 * PP_THREADS : PP_THREADS), ceil_div(batch, 128)));
    a.report = blocks <= 1 || !in_place;
    int rc = launch_serve("paged_plan_kernel", paged_plan_kernel, dim3(std::max(blocks, 1)), dim3(PP_THREADS), 0, 1, true, a);
    if (rc || a.report) return rc;
    a.expand = false;
    a.report = true;
    return launch_serve("paged_plan_kernel", paged_plan_kernel, dim3(1), dim3(PP_THREADS), 0, 1, true, a);
}
