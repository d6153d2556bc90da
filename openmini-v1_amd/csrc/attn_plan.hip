// Pages and slots of a step's tokens (openmini_kv_plan): one launch, whole numbers.
//
// With c cached and n new tokens a request needs ceil((c + n) / P) - ceil(c / P) pages;
// prefix sums of the needs and of the new tokens over the requests place every page and
// every token.  Each workgroup makes both sums for itself (at most 4096 requests: two
// words each from L2, and LDS for the sums), so no workgroup waits for another and one
// launch does; then pages and tokens are spread over all threads, each finding its
// request by bisection in LDS.
//
// Bound by latency: a launch, two dependent loads, the sums, and one more load for a
// token's page.
#include "attn_internal.hpp"

namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMost = 0x7FFFFFFFu;

// Sums stop at 2^31 - 1 (which a step's counts then report) instead of wrapping.
__device__ __forceinline__ uint32_t add_most(uint32_t a, uint32_t b) { return min(a + b, kMost); }

struct Request {
    uint32_t cached, fresh, held, need;  // tokens, tokens, pages, pages
    bool too_long;
};

__device__ __forceinline__ uint32_t pages_of(const FastDiv& page, uint32_t tokens) {
    return tokens ? page.div(tokens - 1) + 1 : 0;
}

__device__ __forceinline__ Request request(const PlanArgs& a, uint32_t r) {
    Request q;
    q.cached = (uint32_t)max(a.cached[r], 0);
    q.fresh = (uint32_t)max(a.fresh[r], 0);
    q.too_long = q.cached + q.fresh > a.max_held;  // both below 2^31
    q.held = q.too_long ? 0 : pages_of(a.page, q.cached);
    q.need = q.too_long ? 0 : pages_of(a.page, q.cached + q.fresh) - q.held;
    return q;
}

// The last r with sums[r] <= v (sums ascend from sums[0] = 0).
__device__ __forceinline__ uint32_t owner(const uint32_t* sums, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;  // sums[lo] <= v; hi is past it or past the end
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sums[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    extern __shared__ uint32_t sums[];  // [requests] first tokens, [requests] pages before
    __shared__ uint32_t wave_tokens[kThreads / 64], wave_pages[kThreads / 64];
    __shared__ uint32_t taken, refused;
    uint32_t* first = sums;
    uint32_t* before = sums + a.requests;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t each = (a.requests + kThreads - 1) / kThreads;
    const uint32_t r0 = min(tid * each, a.requests), r1 = min(r0 + each, a.requests);
    const uint32_t head = a.head ? (uint32_t)max(*a.head, 0) : 0;
    const uint32_t avail = head < a.n_free ? a.n_free - head : 0;
    if (tid == 0) taken = refused = 0;

    uint32_t tokens = 0, pages = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const Request q = request(a, r);
        tokens = add_most(tokens, q.fresh);
        pages = add_most(pages, q.need);
    }
    uint32_t t_upto = tokens, p_upto = pages;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t t = __shfl_up(t_upto, d), p = __shfl_up(p_upto, d);
        if (lane >= (uint32_t)d) {
            t_upto = add_most(t_upto, t);
            p_upto = add_most(p_upto, p);
        }
    }
    if (lane == 63) {
        wave_tokens[wave] = t_upto;
        wave_pages[wave] = p_upto;
    }
    uint32_t t_at = __shfl_up(t_upto, 1), p_at = __shfl_up(p_upto, 1);
    if (lane == 0) t_at = p_at = 0;
    __syncthreads();
    uint32_t total = 0, total_pages = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) {
        if (w == wave) {
            t_at = add_most(t_at, total);
            p_at = add_most(p_at, total_pages);
        }
        total = add_most(total, wave_tokens[w]);
        total_pages = add_most(total_pages, wave_pages[w]);
    }
    for (uint32_t r = r0; r < r1; ++r) {
        const Request q = request(a, r);
        first[r] = t_at;
        before[r] = p_at;
        const bool no = q.too_long || (q.need && p_at + q.need > avail);
        if (blockIdx.x == 0) {
            // requests that need pages are refused from some point on, so the largest sum
            // of one that is not is the number of pages taken
            if (no)
                atomicAdd(&refused, 1u);
            else if (q.need)
                atomicMax(&taken, p_at + q.need);
        }
        t_at = add_most(t_at, q.fresh);
        p_at = add_most(p_at, q.need);
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.counts[0] = (int32_t)total;
        a.counts[1] = (int32_t)taken;
        a.counts[2] = (int32_t)refused;
        a.counts[3] = (int32_t)min(head + taken, kMost);
    }

    const uint32_t most = max(max(a.max_tokens, a.requests + 1), total_pages);
    for (uint64_t at = (uint64_t)blockIdx.x * kThreads + tid; at < most; at += (uint64_t)gridDim.x * kThreads) {
        const uint32_t i = (uint32_t)at;
        if (i < a.requests) {
            const Request q = request(a, i);
            const bool no = q.too_long || (q.need && before[i] + q.need > avail);
            a.starts[i] = (int32_t)first[i];
            a.lens[i] = (int32_t)(no ? q.cached : q.cached + q.fresh);
        } else if (i == a.requests) {
            a.starts[i] = (int32_t)total;
        }
        if (i < total_pages) {
            const uint32_t r = owner(before, a.requests, i);
            const Request q = request(a, r);
            if (before[r] + q.need <= avail)
                a.tables[(int64_t)r * a.table_stride + q.held + (i - before[r])] = a.free[head + i];
        }
        if (i >= a.max_tokens) continue;
        int32_t row = -1, pos = -1, slot = -1, len = 0;
        if (i < total) {
            const uint32_t r = owner(first, a.requests, i);
            const Request q = request(a, r);
            row = (int32_t)r;
            const uint32_t p = q.cached + (i - first[r]);
            pos = (int32_t)min(p, kMost);
            if (!q.too_long && !(q.need && before[r] + q.need > avail)) {
                const uint32_t col = a.page.div(p);
                // the request's own last page, or one taken above (from the list: another
                // workgroup may be writing the table)
                const int32_t page = col < q.held ? a.tables[(int64_t)r * a.table_stride + col]
                                                  : a.free[head + before[r] + (col - q.held)];
                const int64_t s = (int64_t)page * a.page.d + (p - col * a.page.d);
                if (page >= 0 && s <= (int64_t)kMost) slot = (int32_t)s;
                len = (int32_t)(p + 1);
            }
        }
        a.rows[i] = row;
        a.positions[i] = pos;
        a.slots[i] = slot;
        a.row_lens[i] = len;
    }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, hipStream_t s) {
    const uint64_t most = a.max_tokens > a.requests + 1 ? a.max_tokens : a.requests + 1;
    const uint64_t wgs = (most + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(plan_kernel, dim3((unsigned)(wgs < 1024 ? wgs : 1024)), dim3(kThreads), 2 * 4 * (size_t)a.requests,
                       s, a);
    return hipGetLastError();
}

}  // namespace attn
