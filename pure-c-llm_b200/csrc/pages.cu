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

constexpr int kThreads = 512;             // (256: 10.5 us, 1024: 9.8 us on the 2048-request step below)
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

// Sums of `a` and of `b` over the threads before this one; the block's totals
// in total_a and total_b.  `warp_sums` holds two ints per warp.
__device__ __forceinline__ void block_scan(int &a, int &b, int &total_a, int &total_b, int2 *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) { x = sat_add(x, u); y = sat_add(y, v); }
    }
    __syncthreads();                       // warp_sums may be written
    if (lane == 31) warp_sums[warp] = make_int2(x, y);
    __syncthreads();
    int2 w = lane < (int)blockDim.x / 32 ? warp_sums[lane] : make_int2(0, 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, w.x, o), v = __shfl_up_sync(0xffffffffu, w.y, o);
        if (lane >= o) { w.x = sat_add(w.x, u); w.y = sat_add(w.y, v); }
    }
    total_a = __shfl_sync(0xffffffffu, w.x, 31);
    total_b = __shfl_sync(0xffffffffu, w.y, 31);
    // warps before, lanes before
    const int wa = __shfl_sync(0xffffffffu, w.x, max(warp - 1, 0)), wb = __shfl_sync(0xffffffffu, w.y, max(warp - 1, 0));
    const int la = __shfl_up_sync(0xffffffffu, x, 1), lb = __shfl_up_sync(0xffffffffu, y, 1);
    a = sat_add(warp ? wa : 0, lane ? la : 0);
    b = sat_add(warp ? wb : 0, lane ? lb : 0);
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
page_plan_kernel(const __grid_constant__ Params p)
{
    extern __shared__ int sums[];
    int *cu = sums;                        // new tokens up to and with request s
    int *need_sum = sums + p.n_seq;        // pages needed
    int *back_sum = need_sum + p.n_seq;    // pages returned
    __shared__ int2 warp_sums[kThreads / 32];
    __shared__ int s_used, s_refused;
    pdl_begin();                           // launched by launch_pdl

    const int page = 1 << p.log_page;
    const int cap = p.max_pages << p.log_page;
    auto length = [&](int s) { return min(max(__ldg(p.lens + s), 0), cap); };
    auto pages_of = [&](long long tokens) { return (int)((tokens + page - 1) >> p.log_page); };
    const int have_free = min(max(__ldg(p.free_count), 0), p.n_pages);
    if (threadIdx.x == 0) s_refused = 0;

    // The lengths, side by side, and then: a thread sums up n_seq / threads
    // requests that follow one another, the block the threads' sums.  What a
    // request needs depends on the first of the sums.
    for (int s = threadIdx.x; s < p.n_seq; s += blockDim.x) {
        cu[s] = __ldg(p.new_lens + s);
        need_sum[s] = length(s);
    }
    __syncthreads();
    const int per = (p.n_seq + (int)blockDim.x - 1) / (int)blockDim.x;
    const int s0 = min((int)threadIdx.x * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    int c = 0, b = 0, n = 0, none = 0, tokens, returned, needed, ignored;
    for (int s = s0; s < s1; s++) {
        c = sat_add(c, max(cu[s], 0));
        if (cu[s] < 0) b = sat_add(b, pages_of(need_sum[s]));
    }
    block_scan(c, b, tokens, returned, warp_sums);
    for (int s = s0; s < s1; s++) {
        const int len = need_sum[s], nw = cu[s];
        const long long end = (long long)len + nw;
        cu[s] = c = sat_add(c, max(nw, 0));
        back_sum[s] = b = sat_add(b, nw < 0 ? pages_of(len) : 0);
        const int need = nw > 0 && end <= cap && c <= p.max_tokens ? pages_of(end) - pages_of(len) : 0;
        need_sum[s] = need;
        n = sat_add(n, need);
    }
    block_scan(n, none, needed, ignored, warp_sums);
    for (int s = s0; s < s1; s++) need_sum[s] = n = sat_add(n, need_sum[s]);
    __syncthreads();

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
    // (consecutive warps of the grid on different SMs: most outputs are short)
    const int tid = (int)(((threadIdx.x >> 5) * gridDim.x + blockIdx.x) * 32 + (threadIdx.x & 31));
    const int total = (int)(gridDim.x * blockDim.x);
    for (int s = tid; s < p.n_seq; s += total) {
        const int len = length(s), nw = __ldg(p.new_lens + s);
        p.lens_out[s] = nw < 0 ? 0 : served(s, len, nw) ? len + nw : len;
        p.cu_new[s + 1] = cu[s];
    }
    // Pages taken: the need of the requests up to the last one that the list
    // reaches (every later need sum is larger, so the served ones come first).
    if (threadIdx.x == 0) {
        const int reached = first_above(need_sum, p.n_seq, avail); // the first that the list does not reach
        s_used = reached ? need_sum[reached - 1] : 0;
    }
    __syncthreads();
    const int used = s_used;
    for (int i = tid; i < used; i += total) {
        const int s = first_above(need_sum, p.n_seq, i);
        p.table[(long long)s * p.table_stride + pages_of(length(s)) + (i - need_before(s))] = list_page(avail - 1 - i);
    }
    for (int i = have_free + tid; i < min(avail - used, p.n_pages); i += total) p.free_pages[i] = returned_page(i - have_free);
    if (blockIdx.x == gridDim.x - 1) {
        int refused = 0;
        for (int s = threadIdx.x; s < p.n_seq; s += blockDim.x) {
            const int nw = __ldg(p.new_lens + s);
            refused += nw > 0 && !served(s, length(s), nw);
        }
        if (refused) atomicAdd(&s_refused, refused);
        __syncthreads();
        if (threadIdx.x == 0) {
            p.cu_new[0] = 0;
            p.counts[0] = min(avail - used, p.n_pages);
            p.counts[1] = tokens;
            p.counts[2] = s_refused;
            p.counts[3] = used;
        }
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
    // A thread for every token row and request, and for as many pages as come
    // back when an eighth of the tables does, up to one CTA per SM (2048
    // requests of up to 8192 tokens, 5 % ending: 20 us with CTAs for their
    // 2048 rows alone, 8.6 us).
    const long long back = std::min<long long>(s->n_pages, (long long)s->n_seq * s->max_pages) / 8;
    const long long work = std::max<long long>(std::max(s->max_tokens, s->n_seq), back);
    const int threads = work <= 256 ? 256 : kThreads;
    const int grid = (int)std::max<long long>(1, std::min<long long>((work + threads - 1) / threads, sm_count_here()));
    const size_t smem = (size_t)s->n_seq * 12;
    if (!ensure_smem_attr((const void *)page_plan_kernel, (size_t)kMaxSeq * 12))
        return set_error(ATTN_ERR_CUDA, "page plan: cannot set shared-memory size");
    return check_pdl(launch_pdl(page_plan_kernel, dim3(grid), dim3(threads), smem, stream, p), "page_plan_kernel");
}

}  // namespace attn_host
