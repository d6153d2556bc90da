// Pages and slots of a step's tokens (openmini_kv_plan): one launch, whole numbers.
//
// With c cached and n new tokens a request needs ceil((c + n) / P) - ceil(c / P) pages;
// prefix sums of the needs and of the new tokens over the requests place every page and
// every token.  Each workgroup makes both sums for itself (at most 4096 requests: two words
// each from L2, three in LDS), so no workgroup waits for another and one launch does; then
// pages and tokens are spread over all threads, each finding its request by bisection in
// LDS, which also holds what it needs of the request.
//
// Bound by latency: a launch, one load, the sums, the bisection, one more load for a
// token's page.  Measured (MI355X): one request and token 2.3 us, 256 requests with 33000
// tokens 4.5 us (554 KB; with the call from Python 4.7 us either way).
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

__device__ __forceinline__ Request request(const FastDiv& page, uint32_t max_held, int32_t cached, int32_t fresh) {
    Request q;
    q.cached = (uint32_t)max(cached, 0);
    q.fresh = (uint32_t)max(fresh, 0);
    q.too_long = q.cached + q.fresh > max_held;  // both below 2^31
    q.held = q.too_long ? 0 : pages_of(page, q.cached);
    q.need = q.too_long ? 0 : pages_of(page, q.cached + q.fresh) - q.held;
    return q;
}

// Inclusive prefix over the wave.
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false));  // row_shr 1, 2, 4, 8
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false));
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false));
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false));
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));  // row_bcast 15 into rows 1 and 3
    v = add_most(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));  // row_bcast 31 into rows 2 and 3
    return v;
}

// The last r with sums[r] <= v (sums ascend from sums[0] = 0; the refusal bit apart).
__device__ __forceinline__ uint32_t owner(const uint32_t* sums, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;  // sums[lo] <= v; hi is past it or past the end
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((sums[mid] & kMost) <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

constexpr uint32_t kRefused = 0x80000000u;  // in `before`, whose sums stay below it

__global__ __launch_bounds__(kThreads) void plan_kernel(const int32_t* __restrict__ cached, const int32_t* __restrict__ fresh,
                                                        const int32_t* __restrict__ free, uint32_t requests, uint32_t max_held,
                                                        uint32_t max_tokens, uint32_t page_d, uint32_t page_m,
                                                        uint32_t page_shift, uint32_t threads, PlanArgs a) {
    extern __shared__ uint32_t lds[];  // [requests] first tokens, [requests] pages before, [requests] cached tokens
    __shared__ uint32_t wave_tokens[kThreads / 64], wave_pages[kThreads / 64];
    __shared__ uint32_t taken, refused;
    uint32_t *first = lds, *before = lds + requests, *had = before + requests;
    FastDiv page;
    page.d = page_d;
    page.m = page_m;
    page.shift = page_shift;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t each = (requests + kThreads - 1) / kThreads;
    const uint32_t r0 = min(tid * each, requests), r1 = min(r0 + each, requests);
    if (tid == 0) taken = refused = 0;

    // the thread's requests, in LDS what pass two needs of them, and their sums
    uint32_t tokens = 0, pages = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const Request q = request(page, max_held, cached[r], fresh[r]);
        first[r] = q.fresh;
        before[r] = q.need | (q.too_long ? kRefused : 0);
        had[r] = q.cached;
        tokens = add_most(tokens, q.fresh);
        pages = add_most(pages, q.need);
    }
    const uint32_t head = a.head ? (uint32_t)max(*a.head, 0) : 0;
    const uint32_t avail = head < a.n_free ? a.n_free - head : 0;
    const uint32_t t_upto = wave_upto(tokens), p_upto = wave_upto(pages);
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
        const uint32_t fresh_r = first[r], need = before[r] & ~kRefused;
        const bool no = (before[r] & kRefused) || (need && p_at + need > avail);
        first[r] = t_at;
        before[r] = p_at | (no ? kRefused : 0);
        if (blockIdx.x == 0) {
            // requests that need pages are refused from some point on, so the largest sum of
            // one that is not is the number of pages taken
            if (no)
                atomicAdd(&refused, 1u);
            else if (need)
                atomicMax(&taken, p_at + need);
        }
        t_at = add_most(t_at, fresh_r);
        p_at = add_most(p_at, need);
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.counts[0] = (int32_t)total;
        a.counts[1] = (int32_t)taken;
        a.counts[2] = (int32_t)refused;
        a.counts[3] = (int32_t)min(head + taken, kMost);
    }

    const uint32_t most = max(max(max_tokens, requests + 1), total_pages);
    for (uint64_t at = (uint64_t)blockIdx.x * kThreads + tid; at < most; at += threads) {
        const uint32_t i = (uint32_t)at;
        if (i < requests) {
            a.starts[i] = (int32_t)first[i];
            a.lens[i] = (int32_t)(had[i] + (before[i] & kRefused ? 0 : (uint32_t)max(fresh[i], 0)));
        } else if (i == requests) {
            a.starts[i] = (int32_t)total;
        }
        if (i < total_pages) {
            const uint32_t r = owner(before, requests, i);
            if (!(before[r] & kRefused))
                a.tables[(int64_t)r * a.table_stride + pages_of(page, had[r]) + (i - before[r])] = free[head + i];
        }
        if (i >= max_tokens) continue;
        int32_t row = -1, pos = -1, slot = -1, len = 0;
        if (i < total) {
            const uint32_t r = owner(first, requests, i);
            row = (int32_t)r;
            const uint32_t p = had[r] + (i - first[r]);
            pos = (int32_t)min(p, kMost);
            if (!(before[r] & kRefused)) {
                const uint32_t col = page.div(p), held = pages_of(page, had[r]);
                // the request's own last page, or one taken above (from the list: another
                // workgroup may be writing the table)
                const int32_t id = col < held ? a.tables[(int64_t)r * a.table_stride + col] : free[head + before[r] + (col - held)];
                const int64_t s = (int64_t)id * page_d + (p - col * page_d);
                if (id >= 0 && s <= (int64_t)kMost) slot = (int32_t)s;
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
    const uint64_t all = (most + kThreads - 1) / kThreads;
    const unsigned wgs = (unsigned)(all < 1024 ? all : 1024);
    hipLaunchKernelGGL(plan_kernel, dim3(wgs), dim3(kThreads), 3 * 4 * (size_t)a.requests,
                       s, a.cached, a.fresh, a.free, a.requests, a.max_held, a.max_tokens, a.page.d, a.page.m, a.page.shift, wgs * kThreads, a);
    return hipGetLastError();
}

}  // namespace attn
