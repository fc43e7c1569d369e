// abi_tree.cu -- the C ABI of drafted token trees over a paged cache
// (include/attn_b200.h): argument checks of the tree plan, the tree decode and
// the commit.
#include <algorithm>

#include "common.cuh"
#include "prefix.cuh"
#include "serve_checks.cuh"

namespace attn_host {
int launch_tree_plan(int n_seq, int n_rows, int words, const int *cu_rows, const int *parents, const int *positions, int *positions_out,
                     uint32_t *masks, int *err, cudaStream_t s);
int launch_tree_decode(const attn::prefix::Params &p, int d, int kv_dtype, void *ws, size_t *need, cudaStream_t s);
int launch_tree_commit(const attn_page_shape *s, int n_layers, const attn_paged_kv *caches, int kv_heads, int head_dim, const int *cu_rows,
                       const int *ctx_lens, const int *lens, const int *leaf, const uint32_t *masks, int words, const int *table,
                       int *free_pages, const int *free_count, int *lens_out, int *counts, int *err, cudaStream_t stream);
int *device_error_ptr();
}  // namespace attn_host

using namespace attn_host;

extern "C" {

// ---------------------------------------------------------------------------
// tree plan
// ---------------------------------------------------------------------------
int attn_tree_plan_ex(int n_seq, int n_rows, int mask_words, const int *cu_rows, const int *parents, const int *positions,
                      int *positions_out, uint32_t *masks, attn_stream_t stream) {
    if (n_seq < 0 || n_seq > 65535 || n_rows < 0 || n_rows > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "tree plan: bad shape n_seq=%d n_rows=%d", n_seq, n_rows);
    if (mask_words < 1 || mask_words > 32)
        return set_error(ATTN_ERR_UNSUPPORTED, "tree plan: %d mask words, not 1 to 32", mask_words);
    if (n_seq == 0) return ATTN_OK;
    if (!cu_rows || (n_rows && (!parents || !positions || !positions_out || !masks)))
        return set_error(ATTN_ERR_INVALID, "tree plan: NULL pointer");
    const void *const words[] = {cu_rows, parents, positions, positions_out, masks};
    for (const void *w : words)
        if (!aligned(w, 4)) return set_error(ATTN_ERR_INVALID, "tree plan: arrays must be 4-byte aligned");
    if (positions != positions_out && overlap(positions, (size_t)n_rows * 4, positions_out, (size_t)n_rows * 4))
        return set_error(ATTN_ERR_INVALID, "tree plan: positions and positions_out overlap and are not the same");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "tree plan: no device error word");
    return launch_tree_plan(n_seq, n_rows, mask_words, cu_rows, parents, positions, positions_out, masks, err,
                            reinterpret_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// tree decode
// ---------------------------------------------------------------------------
static int check_tree(const attn_tree_shape *s, const attn_paged_kv *c, long long *rs) {
    if (!s) return set_error(ATTN_ERR_INVALID, "tree decode: shape is NULL");
    if (s->n_seq < 0 || s->n_seq > 65535 || s->n_rows < 0 || s->n_groups < 0 || s->n_groups > 65535 || s->heads < 1 || s->kv_heads < 1 ||
        s->heads > 65535 || s->heads % s->kv_heads || (long long)s->n_rows * s->heads > (1 << 24))
        return set_error(ATTN_ERR_INVALID, "tree decode: bad shape n_seq=%d n_rows=%d n_groups=%d heads=%d kv_heads=%d", s->n_seq,
                         s->n_rows, s->n_groups, s->heads, s->kv_heads);
    if (!head_dim_ok(s->head_dim))
        return set_error(ATTN_ERR_UNSUPPORTED, "tree decode: head_dim %d not in {32,64,96,128}", s->head_dim);
    if (!page_size_ok(s->page_size))
        return set_error(ATTN_ERR_UNSUPPORTED, "tree decode: page_size %d is not a power of two in [1, 1024]", s->page_size);
    if (s->max_len < 0 || s->max_prefix_len < 0 || s->max_pages < 0 || s->max_prefix_pages < 0 ||
        s->max_len > (long long)s->max_pages * s->page_size ||
        (s->n_groups && s->max_prefix_len > (long long)s->max_prefix_pages * s->page_size) ||
        s->max_len > (1 << 30) || s->max_prefix_len > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "tree decode: max_len %d in %d pages, max_prefix_len %d in %d pages of %d",
                         s->max_len, s->max_pages, s->max_prefix_len, s->max_prefix_pages, s->page_size);
    if (s->max_nodes < 0 || s->max_nodes > 1024)
        return set_error(ATTN_ERR_UNSUPPORTED, "tree decode: max_nodes %d, at most 1024", s->max_nodes);
    if (s->mask_words < 0 || s->mask_words > 32 || (s->mask_words && s->max_nodes > 32 * s->mask_words))
        return set_error(ATTN_ERR_INVALID, "tree decode: %d mask words for %d nodes", s->mask_words, s->max_nodes);
    const int st = check_cache(c, s->kv_heads, s->head_dim, rs, "tree decode");
    if (st) return st;
    if (c->rows > 0x7fffffffLL)
        return set_error(ATTN_ERR_UNSUPPORTED, "tree decode: a cache of %lld rows, at most 2^31 - 1", c->rows);
    if (c->rows < s->page_size && (s->max_len || (s->n_groups && s->max_prefix_len)))
        return set_error(ATTN_ERR_INVALID, "tree decode: a cache of %lld rows holds no page of %d", c->rows, s->page_size);
    if (s->dtype != (c->kv_dtype == ATTN_BF16 ? ATTN_BF16 : ATTN_F32))
        return set_error(ATTN_ERR_UNSUPPORTED, "tree decode: dtype %d with a cache of dtype %d", s->dtype, c->kv_dtype);
    const long long hd = (long long)s->heads * s->head_dim;
    const int unit = s->dtype == ATTN_F32 ? 4 : 8;
    if ((s->q_row_stride && (s->q_row_stride < hd || s->q_row_stride % unit)) ||
        (s->out_row_stride && (s->out_row_stride < hd || s->out_row_stride % unit)))
        return set_error(ATTN_ERR_INVALID, "tree decode: q and out row strides must be >= heads*d=%lld and multiples of %d", hd, unit);
    if (!(s->scale >= 0.f) || s->scale > 1e30f) return set_error(ATTN_ERR_INVALID, "tree decode: scale %g", (double)s->scale);
    return ATTN_OK;
}

static attn::prefix::Params tree_params(const attn_tree_shape *s, const attn_paged_kv *cache, long long rs) {
    attn::prefix::Params p = {};
    p.k = cache->k; p.v = cache->v; p.kscale = cache->kscale; p.vscale = cache->vscale;
    const long long hd = (long long)s->heads * s->head_dim;
    p.q_stride = s->q_row_stride ? s->q_row_stride : hd;
    p.out_stride = s->out_row_stride ? s->out_row_stride : hd;
    p.row_stride = rs;
    p.n_seq = s->n_rows; p.n_req = s->n_seq; p.n_groups = s->n_groups; p.heads = s->heads; p.kv_heads = s->kv_heads;
    p.ratio = s->heads / s->kv_heads;
    p.log_page = __builtin_ctz((unsigned)s->page_size);
    p.n_pages = (int)(cache->rows / s->page_size);
    p.max_prefix_pages = s->max_prefix_pages; p.max_pages = s->max_pages;
    p.max_prefix_len = s->max_prefix_len; p.max_len = s->max_len;
    p.max_nodes = s->max_nodes; p.mask_words = s->mask_words;
    p.scale_log2 = attn::kLog2e * (s->scale > 0.f ? s->scale : 1.f / sqrtf((float)s->head_dim));
    return p;
}

size_t attn_tree_decode_workspace_bytes(const attn_tree_shape *s, const attn_paged_kv *cache) {
    long long rs;
    if (check_tree(s, cache, &rs) || s->n_seq == 0 || s->n_rows == 0) return 0;
    size_t need = 0;
    launch_tree_decode(tree_params(s, cache, rs), s->head_dim, cache->kv_dtype, nullptr, &need, nullptr);
    return need;
}

int attn_tree_decode_ex(const attn_tree_shape *s, const attn_paged_kv *cache, const void *q, const int *cu_rows, const int *ctx_lens,
                        const int *lens, const uint32_t *masks, const int *group_begin, const int *prefix_table, const int *prefix_lens,
                        const int *block_table, void *out, float *lse, void *workspace, size_t workspace_bytes, attn_stream_t stream) {
    long long rs;
    const int st = check_tree(s, cache, &rs);
    if (st) return st;
    if (s->n_seq == 0 || s->n_rows == 0) return ATTN_OK;
    if (!q || !out || !cu_rows || !ctx_lens || !lens || (s->max_pages && !block_table) ||
        (s->n_groups && (!group_begin || !prefix_lens || (s->max_prefix_pages && !prefix_table))))
        return set_error(ATTN_ERR_INVALID, "tree decode: NULL pointer");
    if (masks && !s->mask_words && s->max_nodes) return set_error(ATTN_ERR_INVALID, "tree decode: masks of 0 words");
    if (!aligned(q, 16) || !aligned(out, 16)) return set_error(ATTN_ERR_INVALID, "tree decode: q and out must be 16-byte aligned");
    const void *const words[] = {cu_rows, ctx_lens, lens, masks, group_begin, prefix_table, prefix_lens, block_table, lse};
    for (const void *w : words)
        if (!aligned(w, 4)) return set_error(ATTN_ERR_INVALID, "tree decode: int arrays and lse must be 4-byte aligned");
    attn::prefix::Params p = tree_params(s, cache, rs);
    size_t need = 0;
    launch_tree_decode(p, s->head_dim, cache->kv_dtype, nullptr, &need, nullptr);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
        return set_error(ATTN_ERR_WORKSPACE, "tree decode: needs a workspace of %zu bytes (256-byte aligned), got %zu", need,
                         workspace ? workspace_bytes : 0);
    p.q = q; p.out = out; p.lse = lse;
    p.row_begin = cu_rows; p.ctx_lens = ctx_lens; p.lens = lens; p.masks = masks;
    p.group_begin = group_begin; p.prefix_table = prefix_table; p.prefix_lens = prefix_lens; p.block_table = block_table;
    p.err = device_error_ptr();
    if (!p.err) return set_error(ATTN_ERR_CUDA, "tree decode: no device error word");
    return launch_tree_decode(p, s->head_dim, cache->kv_dtype, workspace, nullptr, reinterpret_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// commit
// ---------------------------------------------------------------------------
int attn_tree_commit_ex(const attn_page_shape *s, int n_layers, const attn_paged_kv *caches, int kv_heads, int head_dim,
                        const int *cu_rows, const int *ctx_lens, const int *lens, const int *leaf, const uint32_t *masks, int mask_words,
                        const int *block_table, int *free_pages, const int *free_count, int *lens_out, int *counts, attn_stream_t stream) {
    if (!s) return set_error(ATTN_ERR_INVALID, "tree commit: shape is NULL");
    if (s->n_seq < 0 || s->max_pages < 0 || s->max_tokens < 0 || s->n_pages < 0 || s->max_tokens > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "tree commit: bad shape n_seq=%d max_pages=%d max_tokens=%d n_pages=%d",
                         s->n_seq, s->max_pages, s->max_tokens, s->n_pages);
    if (s->n_seq > 16384) return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: %d requests, at most 16384", s->n_seq);
    if (!page_size_ok(s->page_size))
        return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: page_size %d is not a power of two in [1, 1024]", s->page_size);
    if ((long long)s->max_pages * s->page_size > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "tree commit: max_pages*page_size %lld past 2^30", (long long)s->max_pages * s->page_size);
    if (s->table_stride && s->table_stride < s->max_pages)
        return set_error(ATTN_ERR_INVALID, "tree commit: table_stride %d < max_pages %d", s->table_stride, s->max_pages);
    if (mask_words < 1 || mask_words > 32)
        return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: %d mask words, not 1 to 32", mask_words);
    if (n_layers < 0 || n_layers > ATTN_MAX_LAYERS || (n_layers && !caches))
        return set_error(ATTN_ERR_INVALID, "tree commit: %d layers, at most %d", n_layers, ATTN_MAX_LAYERS);
    if (n_layers) {
        if (kv_heads < 1 || kv_heads > 65535) return set_error(ATTN_ERR_INVALID, "tree commit: kv_heads %d", kv_heads);
        if (!head_dim_ok(head_dim)) return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: head_dim %d not in {32,64,96,128}", head_dim);
    }
    for (int i = 0; i < n_layers; i++) {
        long long rs;
        const int st = check_cache(caches + i, kv_heads, head_dim, &rs, "tree commit");
        if (st) return st;
        if (caches[i].kv_dtype != caches[0].kv_dtype)
            return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: caches of types %d and %d", caches[0].kv_dtype, caches[i].kv_dtype);
        if (caches[i].rows > 0x7fffffffLL)
            return set_error(ATTN_ERR_UNSUPPORTED, "tree commit: a cache of %lld rows, at most 2^31 - 1", caches[i].rows);
    }
    if (!free_count || !counts || (s->n_pages && !free_pages) ||
        (s->n_seq && (!cu_rows || !ctx_lens || !lens || !leaf || !lens_out || (s->max_pages && !block_table))))
        return set_error(ATTN_ERR_INVALID, "tree commit: NULL pointer");
    const void *const words[] = {cu_rows, ctx_lens, lens, leaf, masks, block_table, free_pages, free_count, lens_out, counts};
    for (const void *w : words)
        if (!aligned(w, 4)) return set_error(ATTN_ERR_INVALID, "tree commit: int arrays must be 4-byte aligned");
    const size_t n = (size_t)s->n_seq * 4;
    const struct { const void *at; size_t bytes; } inputs[] = {{ctx_lens, n}, {lens, n}, {leaf, n}, {free_count, 4}};
    for (const auto &in : inputs)
        if (overlap(lens_out, n, in.at, in.bytes) || overlap(counts, 16, in.at, in.bytes))
            return set_error(ATTN_ERR_INVALID, "tree commit: lens_out and counts must not overlap lens, ctx_lens, leaf and free_count");
    // Rows and scales are moved by a CTA for each layer, K and V side by side, so none may be there twice, in whatever
    // part.  (Buffers that meet otherwise are left to the caller: layers may be interleaved in one.)
    const int arrays = n_layers && caches[0].kv_dtype == ATTN_I8 ? 4 : 2;
    const void *held[4 * ATTN_MAX_LAYERS];
    for (int i = 0; i < n_layers; i++) {
        const void *const mine[4] = {caches[i].k, caches[i].v, caches[i].kscale, caches[i].vscale};
        for (int a = 0; a < arrays; a++) {
            const void **end = held + arrays * i + a;
            if (std::find((const void **)held, end, mine[a]) != end)
                return set_error(ATTN_ERR_INVALID, "tree commit: the %s of layer %d is there twice",
                                 a < 2 ? "K or V" : "scale of K or V", i);
            *end = mine[a];
        }
    }
    if (overlap(lens_out, n, counts, 16)) return set_error(ATTN_ERR_INVALID, "tree commit: lens_out and counts overlap");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "tree commit: no device error word");
    return launch_tree_commit(s, n_layers, caches, kv_heads, head_dim, cu_rows, ctx_lens, lens, leaf, masks, mask_words, block_table,
                              free_pages, free_count, lens_out, counts, err, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
