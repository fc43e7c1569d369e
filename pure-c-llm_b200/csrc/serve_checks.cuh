// serve_checks.cuh -- argument checks that the serving entry points share
// (abi_serve.cu, abi_tree.cu).
#pragma once
#include "common.cuh"

namespace attn_host {

inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }
inline bool head_dim_ok(int d) { return d == 32 || d == 64 || d == 96 || d == 128; }
inline bool page_size_ok(int n) { return n >= 1 && n <= 1024 && (n & (n - 1)) == 0; }
inline bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

// Checks of a paged cache for kv_heads heads of d; the row stride in elements.
inline int check_cache(const attn_paged_kv *c, int kv_heads, int d, long long *row_stride, const char *who) {
    if (!c) return set_error(ATTN_ERR_INVALID, "%s: cache is NULL", who);
    if (c->kv_dtype != ATTN_F32 && c->kv_dtype != ATTN_BF16 && c->kv_dtype != ATTN_I8)
        return set_error(ATTN_ERR_UNSUPPORTED, "%s: kv_dtype %d not supported", who, c->kv_dtype);
    const long long hd = (long long)kv_heads * d;
    const int unit = c->kv_dtype == ATTN_F32 ? 4 : c->kv_dtype == ATTN_BF16 ? 8 : 16;
    *row_stride = c->row_stride ? c->row_stride : hd;
    if (*row_stride < hd || *row_stride % unit)
        return set_error(ATTN_ERR_INVALID, "%s: cache row_stride %lld must be >= kv_heads*d=%lld and a multiple of %d",
                         who, *row_stride, hd, unit);
    if (c->rows < 0) return set_error(ATTN_ERR_INVALID, "%s: cache of %lld rows", who, c->rows);
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16))
        return set_error(ATTN_ERR_INVALID, "%s: cache k and v must be 16-byte aligned and not NULL", who);
    if (c->kv_dtype == ATTN_I8 && (!c->kscale || !c->vscale || !aligned(c->kscale, 4) || !aligned(c->vscale, 4)))
        return set_error(ATTN_ERR_INVALID, "%s: an INT8 cache needs kscale and vscale", who);
    return ATTN_OK;
}

}  // namespace attn_host
