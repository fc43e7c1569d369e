// prefix.cuh -- what the kernels of attn_prefix_decode_ex share: the call's
// arguments on the device, and the walk through a page table.
#pragma once
#include "common.cuh"

namespace attn {
namespace prefix {

struct Params {
    const void *q;
    const void *k, *v;
    const float *kscale, *vscale;
    const int *group_begin, *prefix_table, *prefix_lens, *block_table, *lens;
    void *out;
    float *lse;
    int *err;
    long long q_stride, out_stride, row_stride;
    int n_seq, n_groups, heads, kv_heads, ratio;      // ratio: query heads per key head
    int log_page, n_pages;
    int max_prefix_pages, max_pages, max_prefix_len, max_len;
    float scale_log2;                                 // scale * log2(e)
};

__device__ __forceinline__ int checked_len(const Params &p, int len, int most) {
    if (len < 0 || len > most) {
        atomicExch(p.err, 0x703);
        return len < 0 ? 0 : most;
    }
    return len;
}
__device__ __forceinline__ int own_len(const Params &p, int s) { return checked_len(p, __ldg(p.lens + s), p.max_len); }
__device__ __forceinline__ int prefix_len(const Params &p, int g) {
    return checked_len(p, __ldg(p.prefix_lens + g), p.max_prefix_len);
}
// first request of group g, within [0, n_seq]
__device__ __forceinline__ int group_first(const Params &p, int g) {
    return min(max(__ldg(p.group_begin + g), 0), p.n_seq);
}

// Cache row of token t of a table line, or -1 where the page lies outside the cache.
__device__ __forceinline__ long long cache_row(const Params &p, const int *line, int t) {
    const int page = __ldg(line + (t >> p.log_page));
    if ((unsigned)page >= (unsigned)p.n_pages) {
        atomicExch(p.err, 0x702);
        return -1;
    }
    return ((long long)page << p.log_page) + (t & ((1 << p.log_page) - 1));
}

}  // namespace prefix
}  // namespace attn
