// pages.cu -- one serving step's page plan from the requests' lengths
// (attn_page_plan_ex): block-table entries, slot map, positions, free list.
//
// All of it follows from three running sums over the requests: the new tokens
// (which token rows a request has), the pages the ended ones return, and the
// pages the others need.  The list that pages are taken from is
//   L = free_pages[0 .. free_count) ++ pages of ended requests,
// taken from its end, so request s's i-th new page is
//   L[|L| - 1 - (need of the requests before s) - i],
// and no page depends on another CTA's writes: the kernel is one launch
// without atomics, and what it writes is the same on every run.
//
// Every CTA forms the three sums of all requests in shared memory (12 bytes a
// request) and then writes its share of the outputs; token rows and new pages
// find their request by bisection in the sums.  What bounds a step of a few
// thousand requests is latency: the loads of the lengths, two block scans and
// the dependent loads behind a token's bisection.
#include <algorithm>

#include "common.cuh"

namespace attn {
namespace pages {

constexpr int kThreads = 1024;
constexpr int kMaxSeq = 16384;            // 12 bytes each of shared memory

struct Params {
    const int *lens, *new_lens, *pos_base;
    int *free_pages;
    const int *free_count;
    int *table, *lens_out, *cu_new;
    long long *slot_map;
    int *positions, *token_seq, *counts;
    long long table_stride;
    int n_seq, log_page, max_pages, max_tokens, n_pages;
};

// sums of non-negative ints that stay at 2^31 - 1 once they pass it
__device__ __forceinline__ int sat_add(int a, int b) {
    const unsigned s = (unsigned)a + (unsigned)b;
    return (int)min(s, 0x7fffffffu);
}

// Inclusive sums of `v` over the block's threads, on top of `carry` (the sum
// so far, which becomes the sum with this block's).  Two barriers.
__device__ __forceinline__ int block_scan(int v, int &carry, int *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s = sat_add(s, u);
    }
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int w = lane < kThreads / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w = sat_add(w, u);
    }
    const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    const int total = __shfl_sync(0xffffffffu, w, 31);
    const int r = sat_add(carry, sat_add(before, s));
    carry = sat_add(carry, total);
    __syncthreads();                       // warp_sums may be written again
    return r;
}

// the smallest i with sums[i] > x (sums ascending, n entries; n if none)
__device__ __forceinline__ int first_above(const int *sums, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads)
page_plan_kernel(const Params p)
{
    extern __shared__ int sums[];
    int *cu = sums;                        // new tokens up to and with request s
    int *need_sum = sums + p.n_seq;        // pages needed
    int *back_sum = need_sum + p.n_seq;    // pages returned
    __shared__ int warp_sums[kThreads / 32];
    __shared__ int s_used, s_refused;
    pdl_begin();                           // launched by launch_pdl

    const int page = 1 << p.log_page;
    const int cap = p.max_pages << p.log_page;
    auto length = [&](int s) { return min(max(__ldg(p.lens + s), 0), cap); };
    auto pages_of = [&](long long tokens) { return (int)((tokens + page - 1) >> p.log_page); };

    if (threadIdx.x == 0) { s_used = 0; s_refused = 0; }
    int tokens = 0, returned = 0, needed = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) {
        const int s = s0 + threadIdx.x;
        int len = 0, nw = 0;
        bool in = s < p.n_seq, ended = false;
        if (in) { len = length(s); nw = __ldg(p.new_lens + s); ended = nw < 0; nw = max(nw, 0); }
        const int c = block_scan(nw, tokens, warp_sums);
        const int b = block_scan(ended ? pages_of(len) : 0, returned, warp_sums);
        const long long end = (long long)len + nw;
        const bool fits = in && !ended && (nw == 0 || (end <= cap && c <= p.max_tokens));
        const int n = block_scan(fits ? pages_of(end) - pages_of(len) : 0, needed, warp_sums);
        if (in) { cu[s] = c; back_sum[s] = b; need_sum[s] = n; }
    }
    __syncthreads();

    const int have_free = min(max(__ldg(p.free_count), 0), p.n_pages);
    const int avail = sat_add(have_free, returned);
    // a page of an ended request by its place among the returned ones
    auto returned_page = [&](int i) {
        const int s = first_above(back_sum, p.n_seq, i);
        return __ldg(p.table + (long long)s * p.table_stride + (i - (s ? back_sum[s - 1] : 0)));
    };
    auto list_page = [&](int i) { return i < have_free ? __ldg(p.free_pages + i) : returned_page(i - have_free); };
    auto need_before = [&](int s) { return s ? need_sum[s - 1] : 0; };
    // served: nothing asked of the list, or the list reaches
    auto served = [&](int s, int len, int nw) {
        if (nw <= 0) return nw == 0;
        const long long end = (long long)len + nw;
        if (end > cap || cu[s] > p.max_tokens) return false;
        return need_sum[s] == need_before(s) || need_sum[s] <= avail;
    };

    // requests
    const int tid = (int)(blockIdx.x * kThreads + threadIdx.x), total = (int)(gridDim.x * kThreads);
    for (int s = tid; s < p.n_seq; s += total) {
        const int len = length(s), nw = __ldg(p.new_lens + s);
        p.lens_out[s] = nw < 0 ? 0 : served(s, len, nw) ? len + nw : len;
        p.cu_new[s + 1] = cu[s];
    }
    // Pages taken: the need of the requests up to the last one that the list
    // reaches (every later need sum is larger, so the served ones come first).
    {
        const int k = first_above(need_sum, p.n_seq, avail);       // the first that the list does not reach
        if (threadIdx.x == 0) s_used = k ? need_sum[k - 1] : 0;
    }
    if (blockIdx.x == 0) {
        int refused = 0;
        for (int s = threadIdx.x; s < p.n_seq; s += kThreads) {
            const int nw = __ldg(p.new_lens + s);
            refused += nw > 0 && !served(s, length(s), nw);
        }
        if (refused) atomicAdd(&s_refused, refused);
    }
    __syncthreads();
    const int used = s_used;
    for (int i = tid; i < used; i += total) {
        const int s = first_above(need_sum, p.n_seq, i);
        p.table[(long long)s * p.table_stride + pages_of(length(s)) + (i - need_before(s))] = list_page(avail - 1 - i);
    }
    for (int i = have_free + tid; i < min(avail - used, p.n_pages); i += total) p.free_pages[i] = returned_page(i - have_free);
    if (tid == 0) {
        p.cu_new[0] = 0;
        p.counts[0] = min(avail - used, p.n_pages);
        p.counts[1] = tokens;
        p.counts[2] = s_refused;
        p.counts[3] = used;
    }

    // token rows
    for (int t = tid; t < p.max_tokens; t += total) {
        long long slot = -1;
        int pos = 0, s = -1;
        if (t < tokens) {
            s = first_above(cu, p.n_seq, t);
            const int len = length(s), first = s ? cu[s - 1] : 0;
            const long long at = (long long)len + (t - first);
            pos = (int)((p.pos_base ? __ldg(p.pos_base + s) : 0) + at);
            if (served(s, len, __ldg(p.new_lens + s))) {
                const int i = (int)(at >> p.log_page) - pages_of(len);       // >= 0: the i-th new page
                const int id = i < 0 ? __ldg(p.table + (long long)s * p.table_stride + (at >> p.log_page))
                                     : list_page(avail - 1 - (need_before(s) + i));
                if (id >= 0) slot = ((long long)id << p.log_page) + (at & (page - 1));
            }
        }
        p.slot_map[t] = slot;
        p.positions[t] = pos;
        if (p.token_seq) p.token_seq[t] = s;
    }
}

}  // namespace pages
}  // namespace attn

namespace attn_host {

bool ensure_smem_attr(const void *func, size_t bytes);
int sm_count_here();

int launch_page_plan(const attn_page_shape *s, const int *lens, const int *new_lens, const int *pos_base,
                     int *free_pages, const int *free_count, int *block_table, int *lens_out, int *cu_new,
                     long long *slot_map, int *positions, int *token_seq, int *counts, cudaStream_t stream) {
    using namespace attn::pages;
    Params p;
    p.lens = lens; p.new_lens = new_lens; p.pos_base = pos_base;
    p.free_pages = free_pages; p.free_count = free_count; p.table = block_table;
    p.lens_out = lens_out; p.cu_new = cu_new; p.slot_map = slot_map; p.positions = positions;
    p.token_seq = token_seq; p.counts = counts;
    p.table_stride = s->table_stride ? s->table_stride : s->max_pages;
    p.n_seq = s->n_seq; p.max_pages = s->max_pages; p.max_tokens = s->max_tokens; p.n_pages = s->n_pages;
    p.log_page = __builtin_ctz((unsigned)s->page_size);
    // A CTA for every 1024 token rows, or for as many pages as come back when an
    // eighth of the tables does, up to one per SM (2048 requests of up to 8192
    // tokens, 5 % ending: 20 us with the 2 CTAs of their 2048 rows, %STEP% us).
    const long long back = std::min<long long>(s->n_pages, (long long)s->n_seq * s->max_pages) / 8;
    const int grid = (int)std::max<long long>(1, std::min<long long>((std::max<long long>(s->max_tokens, back) + kThreads - 1) / kThreads,
                                                                     sm_count_here()));
    const size_t smem = (size_t)s->n_seq * 12;
    if (!ensure_smem_attr((const void *)page_plan_kernel, (size_t)kMaxSeq * 12))
        return set_error(ATTN_ERR_CUDA, "page plan: cannot set shared-memory size");
    return check_pdl(launch_pdl(page_plan_kernel, dim3(grid), dim3(kThreads), smem, stream, p), "page_plan_kernel");
}

}  // namespace attn_host
