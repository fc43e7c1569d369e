// abi_serve.cu -- the C ABI of serving over a paged cache
// (include/attn_b200.h): argument checks and workspaces of the page plan, the
// rotary embedding, plain and with normed heads, and the shared-prefix decode.
#include <algorithm>

#include "common.cuh"
#include "prefix.cuh"
#include "serve_checks.cuh"

namespace attn_host {
int launch_page_plan(const attn_page_shape *s, const int *lens, const int *new_lens, const int *pos_base,
                     int *free_pages, const int *free_count, int *block_table, int *lens_out, int *cu_new,
                     long long *slot_map, int *positions, int *token_seq, int *counts, cudaStream_t stream);
int launch_rope_table(const attn_rope_config *c, float *table, cudaStream_t s);
int launch_rope(const attn_rope_shape *s, int dtype, const float *table, const int *positions, const void *q,
                const void *k, void *q_out, void *k_out, int transpose, int *err, cudaStream_t stream);
int launch_rope_append(const attn_rope_shape *s, const attn_paged_kv *c, int dtype, const float *table,
                       const int *positions, const long long *slots, const void *q, const void *k, const void *v,
                       void *q_out, int *err, cudaStream_t stream);
int launch_norm_rope(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions, const void *q,
                     const void *k, void *q_out, void *k_out, int *err, cudaStream_t stream);
size_t norm_rope_bwd_workspace(const attn_rope_shape *s);
int launch_norm_rope_bwd(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions, const void *q,
                         const void *k, const void *dq_out, const void *dk_out, void *dq, void *dk, float *dq_weight, float *dk_weight,
                         int accumulate, void *ws, int *err, cudaStream_t stream);
int launch_norm_rope_append(const attn_rope_shape *s, const attn_head_norm *n, const attn_paged_kv *c, int dtype, const float *table,
                            const int *positions, const long long *slots, const void *q, const void *k, const void *v, void *q_out, int *err,
                            cudaStream_t stream);
size_t prefix_decode_workspace(const attn_prefix_shape *s, int kv_dtype);
int launch_prefix_decode(const attn::prefix::Params &p, int d, int kv_dtype, void *ws, cudaStream_t s);
void *library_workspace(int which, size_t bytes, cudaStream_t s);      // slot 4: the prefix decode's pieces
int *device_error_ptr();
}  // namespace attn_host

using namespace attn_host;

extern "C" {

// ---------------------------------------------------------------------------
// page plan
// ---------------------------------------------------------------------------
int attn_page_plan_ex(const attn_page_shape *s, const int *lens, const int *new_lens, const int *pos_base,
                      int *free_pages, const int *free_count, int *block_table, int *lens_out, int *cu_new,
                      long long *slot_map, int *positions, int *token_seq, int *counts, attn_stream_t stream) {
    if (!s) return set_error(ATTN_ERR_INVALID, "page plan: shape is NULL");
    if (s->n_seq < 0 || s->max_pages < 0 || s->max_tokens < 0 || s->n_pages < 0 || s->max_tokens > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "page plan: bad shape n_seq=%d max_pages=%d max_tokens=%d n_pages=%d",
                         s->n_seq, s->max_pages, s->max_tokens, s->n_pages);
    if (s->n_seq > 16384) return set_error(ATTN_ERR_UNSUPPORTED, "page plan: %d requests, at most 16384", s->n_seq);
    if (!page_size_ok(s->page_size))
        return set_error(ATTN_ERR_UNSUPPORTED, "page plan: page_size %d is not a power of two in [1, 1024]", s->page_size);
    if ((long long)s->max_pages * s->page_size > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "page plan: max_pages*page_size %lld past 2^30",
                         (long long)s->max_pages * s->page_size);
    if (s->table_stride && s->table_stride < s->max_pages)
        return set_error(ATTN_ERR_INVALID, "page plan: table_stride %d < max_pages %d", s->table_stride, s->max_pages);
    if (!free_count || !cu_new || !counts || (s->n_pages && !free_pages) ||
        (s->n_seq && (!lens || !new_lens || !lens_out || (s->max_pages && !block_table))) ||
        (s->max_tokens && (!slot_map || !positions)))
        return set_error(ATTN_ERR_INVALID, "page plan: NULL pointer");
    const void *const words[] = {lens, new_lens, pos_base, free_pages, free_count, block_table,
                                 lens_out, cu_new, positions, token_seq, counts};
    for (const void *w : words)
        if (!aligned(w, 4)) return set_error(ATTN_ERR_INVALID, "page plan: int arrays must be 4-byte aligned");
    if (!aligned(slot_map, 8)) return set_error(ATTN_ERR_INVALID, "page plan: slot_map must be 8-byte aligned");
    if (overlap(lens_out, (size_t)s->n_seq * 4, lens, (size_t)s->n_seq * 4) || overlap(counts, 16, free_count, 4))
        return set_error(ATTN_ERR_INVALID, "page plan: lens_out and counts must not overlap lens and free_count");
    return launch_page_plan(s, lens, new_lens, pos_base, free_pages, free_count, block_table, lens_out, cu_new,
                            slot_map, positions, token_seq, counts, reinterpret_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
int attn_rope_table_ex(const attn_rope_config *c, float *table, attn_stream_t stream) {
    if (!c) return set_error(ATTN_ERR_INVALID, "rope table: config is NULL");
    if (c->rot_dim < 2 || c->rot_dim > 128 || c->rot_dim % 2 || c->max_pos < 0 || !(c->base > 1.0))
        return set_error(ATTN_ERR_INVALID, "rope table: bad rot_dim=%d max_pos=%d base=%g", c->rot_dim, c->max_pos, c->base);
    if (c->scaling < ATTN_ROPE_PLAIN || c->scaling > ATTN_ROPE_RAMP)
        return set_error(ATTN_ERR_UNSUPPORTED, "rope table: scaling %d", c->scaling);
    if (c->scaling != ATTN_ROPE_PLAIN && !(c->factor >= 1.0))
        return set_error(ATTN_ERR_INVALID, "rope table: factor %g < 1", c->factor);
    if (c->scaling == ATTN_ROPE_BASE && c->rot_dim <= 2)
        return set_error(ATTN_ERR_INVALID, "rope table: ATTN_ROPE_BASE needs rot_dim > 2");
    if (c->scaling == ATTN_ROPE_RAMP && (c->trained_len < 1 || !(c->slow > 0.0) || !(c->fast > c->slow)))
        return set_error(ATTN_ERR_INVALID, "rope table: ATTN_ROPE_RAMP needs trained_len >= 1 and fast > slow > 0");
    if (c->max_pos == 0) return ATTN_OK;
    if (!table || !aligned(table, 8)) return set_error(ATTN_ERR_INVALID, "rope table: table must be 8-byte aligned and not NULL");
    return launch_rope_table(c, table, reinterpret_cast<cudaStream_t>(stream));
}

static int check_rope(const attn_rope_shape *s, int dtype, const float *table, const int *positions) {
    if (!s) return set_error(ATTN_ERR_INVALID, "rope: shape is NULL");
    if (s->tokens < 0 || s->tokens > (1 << 30) || s->heads < 1 || s->kv_heads < 1 || s->heads > 65535 || s->kv_heads > 65535)
        return set_error(ATTN_ERR_INVALID, "rope: bad shape tokens=%d heads=%d kv_heads=%d", s->tokens, s->heads, s->kv_heads);
    if (!head_dim_ok(s->head_dim))
        return set_error(ATTN_ERR_UNSUPPORTED, "rope: head_dim %d not in {32,64,96,128}", s->head_dim);
    if (s->rot_dim < 0 || s->rot_dim > s->head_dim || s->rot_dim % 2)
        return set_error(ATTN_ERR_INVALID, "rope: rot_dim %d must be even and within head_dim %d", s->rot_dim, s->head_dim);
    if (dtype != ATTN_F32 && dtype != ATTN_BF16) return set_error(ATTN_ERR_UNSUPPORTED, "rope: dtype %d not supported", dtype);
    if (s->rot_dim && (s->max_pos < 1 || !table || !aligned(table, 8)))
        return set_error(ATTN_ERR_INVALID, "rope: a table of %d rows; it must be 8-byte aligned and not NULL", s->max_pos);
    if (s->rot_dim && !positions && s->seq_len < 1)
        return set_error(ATTN_ERR_INVALID, "rope: positions is NULL and seq_len is %d", s->seq_len);
    if (positions && !aligned(positions, 4)) return set_error(ATTN_ERR_INVALID, "rope: misaligned positions");
    const long long qw = (long long)s->heads * s->head_dim, kw = (long long)s->kv_heads * s->head_dim;
    if ((s->q_row_stride && s->q_row_stride < qw) || (s->q_out_row_stride && s->q_out_row_stride < qw) ||
        (s->k_row_stride && s->k_row_stride < kw) || (s->k_out_row_stride && s->k_out_row_stride < kw) ||
        (s->v_row_stride && s->v_row_stride < kw))
        return set_error(ATTN_ERR_INVALID, "rope: a row stride is shorter than its rows");
    return ATTN_OK;
}

int attn_rope_ex(const attn_rope_shape *s, int dtype, const float *table, const int *positions, const void *q,
                 const void *k, void *q_out, void *k_out, int transpose, attn_stream_t stream) {
    const int st = check_rope(s, dtype, table, positions);
    if (st) return st;
    if (s->tokens == 0) return ATTN_OK;
    const size_t e = dtype == ATTN_F32 ? 4 : 2;
    if (!q || !q_out || !k != !k_out) return set_error(ATTN_ERR_INVALID, "rope: NULL tensor pointer");
    if (!aligned(q, e) || !aligned(k, e) || !aligned(q_out, e) || !aligned(k_out, e))
        return set_error(ATTN_ERR_INVALID, "rope: tensors must be %zu-byte aligned", e);
    const long long qw = (long long)s->heads * s->head_dim, kw = (long long)s->kv_heads * s->head_dim;
    if ((q == q_out && (s->q_row_stride ? s->q_row_stride : qw) != (s->q_out_row_stride ? s->q_out_row_stride : qw)) ||
        (k && k == k_out && (s->k_row_stride ? s->k_row_stride : kw) != (s->k_out_row_stride ? s->k_out_row_stride : kw)))
        return set_error(ATTN_ERR_INVALID, "rope: in place, the strides of input and output must be the same");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "rope: no device error word");
    return launch_rope(s, dtype, table, positions, q, k, q_out, k_out, transpose ? 1 : 0, err,
                       reinterpret_cast<cudaStream_t>(stream));
}

int attn_rope_append_ex(const attn_rope_shape *s, const attn_paged_kv *cache, int dtype, const float *table,
                        const int *positions, const long long *slot_map, const void *q, const void *k, const void *v,
                        void *q_out, attn_stream_t stream) {
    int st = check_rope(s, dtype, table, positions);
    if (st) return st;
    long long rs;
    if ((st = check_cache(cache, s->kv_heads, s->head_dim, &rs, "rope append"))) return st;
    if ((dtype == ATTN_BF16) != (cache->kv_dtype == ATTN_BF16))
        return set_error(ATTN_ERR_UNSUPPORTED, "rope append: dtype %d into a cache of dtype %d", dtype, cache->kv_dtype);
    if (s->tokens == 0) return ATTN_OK;
    const size_t e = dtype == ATTN_F32 ? 4 : 2;
    if (!q || !k || !v || !q_out || !slot_map) return set_error(ATTN_ERR_INVALID, "rope append: NULL pointer");
    if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(q_out, e) || !aligned(slot_map, 8))
        return set_error(ATTN_ERR_INVALID, "rope append: tensors must be %zu-byte aligned, slot_map 8-byte", e);
    const long long qw = (long long)s->heads * s->head_dim;
    if (q == q_out && (s->q_row_stride ? s->q_row_stride : qw) != (s->q_out_row_stride ? s->q_out_row_stride : qw))
        return set_error(ATTN_ERR_INVALID, "rope append: in place, the strides of q and q_out must be the same");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "rope append: no device error word");
    return launch_rope_append(s, cache, dtype, table, positions, slot_map, q, k, v, q_out, err,
                              reinterpret_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// normed heads, turned
// ---------------------------------------------------------------------------
static int check_norm(const attn_head_norm *n) {
    if (!n) return set_error(ATTN_ERR_INVALID, "norm rope: norm is NULL");
    if (!(n->eps >= 0.f) || n->eps > 1e30f) return set_error(ATTN_ERR_INVALID, "norm rope: eps %g", (double)n->eps);
    if (!aligned(n->q_weight, 4) || !aligned(n->k_weight, 4)) return set_error(ATTN_ERR_INVALID, "norm rope: misaligned weights");
    return ATTN_OK;
}

// Row strides of q and k, and of their outputs (or gradients): the same where two tensors are one.
static bool strides_differ(const attn_rope_shape *s, bool of_q) {
    const long long w = (long long)(of_q ? s->heads : s->kv_heads) * s->head_dim;
    const long long in = of_q ? s->q_row_stride : s->k_row_stride, out = of_q ? s->q_out_row_stride : s->k_out_row_stride;
    return (in ? in : w) != (out ? out : w);
}

int attn_norm_rope_ex(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions,
                      const void *q, const void *k, void *q_out, void *k_out, attn_stream_t stream) {
    int st = check_rope(s, dtype, table, positions);
    if (st || (st = check_norm(n))) return st;
    if (s->tokens == 0) return ATTN_OK;
    const size_t e = dtype == ATTN_F32 ? 4 : 2;
    if (!q || !q_out || !k != !k_out) return set_error(ATTN_ERR_INVALID, "norm rope: NULL tensor pointer");
    if (!aligned(q, e) || !aligned(k, e) || !aligned(q_out, e) || !aligned(k_out, e))
        return set_error(ATTN_ERR_INVALID, "norm rope: tensors must be %zu-byte aligned", e);
    if ((q == q_out && strides_differ(s, true)) || (k && k == k_out && strides_differ(s, false)))
        return set_error(ATTN_ERR_INVALID, "norm rope: in place, the strides of input and output must be the same");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "norm rope: no device error word");
    return launch_norm_rope(s, n, dtype, table, positions, q, k, q_out, k_out, err, reinterpret_cast<cudaStream_t>(stream));
}

size_t attn_norm_rope_bwd_workspace_bytes(const attn_rope_shape *s) {
    if (!s || s->tokens < 0 || s->tokens > (1 << 30) || s->heads < 1 || s->heads > 65535 || s->kv_heads < 1 || s->kv_heads > 65535 ||
        !head_dim_ok(s->head_dim))
        return 0;
    return norm_rope_bwd_workspace(s);
}

int attn_norm_rope_bwd_ex(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions,
                          const void *q, const void *k, const void *dq_out, const void *dk_out, void *dq, void *dk, float *dq_weight,
                          float *dk_weight, int accumulate, void *workspace, size_t workspace_bytes, attn_stream_t stream) {
    int st = check_rope(s, dtype, table, positions);
    if (st || (st = check_norm(n))) return st;
    const size_t e = dtype == ATTN_F32 ? 4 : 2;
    if (s->tokens && (!q || !dq_out || !dq || !k != !dk_out || !k != !dk))
        return set_error(ATTN_ERR_INVALID, "norm rope backward: NULL tensor pointer");
    const void *const tensors[] = {q, k, dq_out, dk_out, dq, dk};
    for (const void *t : tensors)
        if (!aligned(t, e)) return set_error(ATTN_ERR_INVALID, "norm rope backward: tensors must be %zu-byte aligned", e);
    if (!aligned(dq_weight, 4) || !aligned(dk_weight, 4))
        return set_error(ATTN_ERR_INVALID, "norm rope backward: misaligned weight gradients");
    if ((dq && dq == dq_out && strides_differ(s, true)) || (dk && dk == dk_out && strides_differ(s, false)))
        return set_error(ATTN_ERR_INVALID, "norm rope backward: in place, the strides of input and output must be the same");
    if (dq_weight || dk_weight) {
        const size_t need = norm_rope_bwd_workspace(s);
        if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
            return set_error(ATTN_ERR_WORKSPACE, "norm rope backward: weight gradients need a workspace of %zu bytes (256-byte aligned), got %zu",
                             need, workspace ? workspace_bytes : 0);
        const size_t w = (size_t)s->head_dim * 4;
        if (dq_weight && dk_weight && overlap(dq_weight, w, dk_weight, w))
            return set_error(ATTN_ERR_INVALID, "norm rope backward: dq_weight and dk_weight overlap");
    }
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "norm rope backward: no device error word");
    return launch_norm_rope_bwd(s, n, dtype, table, positions, q, k, dq_out, dk_out, dq, dk, dq_weight, dk_weight, accumulate ? 1 : 0,
                                workspace, err, reinterpret_cast<cudaStream_t>(stream));
}

int attn_norm_rope_append_ex(const attn_rope_shape *s, const attn_head_norm *n, const attn_paged_kv *cache, int dtype, const float *table,
                             const int *positions, const long long *slot_map, const void *q, const void *k, const void *v, void *q_out,
                             attn_stream_t stream) {
    int st = check_rope(s, dtype, table, positions);
    if (st || (st = check_norm(n))) return st;
    long long rs;
    if ((st = check_cache(cache, s->kv_heads, s->head_dim, &rs, "norm rope append"))) return st;
    if ((dtype == ATTN_BF16) != (cache->kv_dtype == ATTN_BF16))
        return set_error(ATTN_ERR_UNSUPPORTED, "norm rope append: dtype %d into a cache of dtype %d", dtype, cache->kv_dtype);
    if (s->tokens == 0) return ATTN_OK;
    const size_t e = dtype == ATTN_F32 ? 4 : 2;
    if (!q || !k || !v || !q_out || !slot_map) return set_error(ATTN_ERR_INVALID, "norm rope append: NULL pointer");
    if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(q_out, e) || !aligned(slot_map, 8))
        return set_error(ATTN_ERR_INVALID, "norm rope append: tensors must be %zu-byte aligned, slot_map 8-byte", e);
    if (q == q_out && strides_differ(s, true))
        return set_error(ATTN_ERR_INVALID, "norm rope append: in place, the strides of q and q_out must be the same");
    int *err = device_error_ptr();
    if (!err) return set_error(ATTN_ERR_CUDA, "norm rope append: no device error word");
    return launch_norm_rope_append(s, n, cache, dtype, table, positions, slot_map, q, k, v, q_out, err,
                                   reinterpret_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// shared-prefix decode
// ---------------------------------------------------------------------------
static int check_prefix(const attn_prefix_shape *s, const attn_paged_kv *c, long long *rs) {
    if (!s) return set_error(ATTN_ERR_INVALID, "prefix decode: shape is NULL");
    if (s->n_seq < 0 || s->n_seq > 65535 || s->n_groups < 0 || s->n_groups > 65535 || s->heads < 1 || s->kv_heads < 1 ||
        s->heads > 65535 || s->heads % s->kv_heads || (long long)s->n_seq * s->heads > (1 << 24))
        return set_error(ATTN_ERR_INVALID, "prefix decode: bad shape n_seq=%d n_groups=%d heads=%d kv_heads=%d",
                         s->n_seq, s->n_groups, s->heads, s->kv_heads);
    if (!head_dim_ok(s->head_dim))
        return set_error(ATTN_ERR_UNSUPPORTED, "prefix decode: head_dim %d not in {32,64,96,128}", s->head_dim);
    if (!page_size_ok(s->page_size))
        return set_error(ATTN_ERR_UNSUPPORTED, "prefix decode: page_size %d is not a power of two in [1, 1024]", s->page_size);
    if (s->max_len < 0 || s->max_prefix_len < 0 || s->max_pages < 0 || s->max_prefix_pages < 0 ||
        s->max_len > (long long)s->max_pages * s->page_size ||
        (s->n_groups && s->max_prefix_len > (long long)s->max_prefix_pages * s->page_size) ||
        s->max_len > (1 << 30) || s->max_prefix_len > (1 << 30))
        return set_error(ATTN_ERR_INVALID, "prefix decode: max_len %d in %d pages, max_prefix_len %d in %d pages of %d",
                         s->max_len, s->max_pages, s->max_prefix_len, s->max_prefix_pages, s->page_size);
    const int st = check_cache(c, s->kv_heads, s->head_dim, rs, "prefix decode");
    if (st) return st;
    if (c->rows > 0x7fffffffLL)
        return set_error(ATTN_ERR_UNSUPPORTED, "prefix decode: a cache of %lld rows, at most 2^31 - 1", c->rows);
    if (c->rows < s->page_size && (s->max_len || (s->n_groups && s->max_prefix_len)))
        return set_error(ATTN_ERR_INVALID, "prefix decode: a cache of %lld rows holds no page of %d", c->rows, s->page_size);
    if (s->dtype != (c->kv_dtype == ATTN_BF16 ? ATTN_BF16 : ATTN_F32))
        return set_error(ATTN_ERR_UNSUPPORTED, "prefix decode: dtype %d with a cache of dtype %d", s->dtype, c->kv_dtype);
    const long long hd = (long long)s->heads * s->head_dim;
    const int unit = s->dtype == ATTN_F32 ? 4 : 8;
    if ((s->q_row_stride && (s->q_row_stride < hd || s->q_row_stride % unit)) ||
        (s->out_row_stride && (s->out_row_stride < hd || s->out_row_stride % unit)))
        return set_error(ATTN_ERR_INVALID, "prefix decode: q and out row strides must be >= heads*d=%lld and multiples of %d",
                         hd, unit);
    if (!(s->scale >= 0.f) || s->scale > 1e30f)
        return set_error(ATTN_ERR_INVALID, "prefix decode: scale %g", (double)s->scale);
    return ATTN_OK;
}

size_t attn_prefix_decode_workspace_bytes(const attn_prefix_shape *s, const attn_paged_kv *cache) {
    long long rs;
    if (check_prefix(s, cache, &rs) || s->n_seq == 0) return 0;
    return prefix_decode_workspace(s, cache->kv_dtype);
}

int attn_prefix_decode_ex(const attn_prefix_shape *s, const attn_paged_kv *cache, const void *q, const int *group_begin,
                          const int *prefix_table, const int *prefix_lens, const int *block_table, const int *lens,
                          void *out, float *lse, void *workspace, size_t workspace_bytes, attn_stream_t stream) {
    long long rs;
    const int st = check_prefix(s, cache, &rs);
    if (st) return st;
    if (s->n_seq == 0) return ATTN_OK;
    if (!q || !out || !lens || (s->max_pages && !block_table) ||
        (s->n_groups && (!group_begin || !prefix_lens || (s->max_prefix_pages && !prefix_table))))
        return set_error(ATTN_ERR_INVALID, "prefix decode: NULL pointer");
    if (!aligned(q, 16) || !aligned(out, 16))
        return set_error(ATTN_ERR_INVALID, "prefix decode: q and out must be 16-byte aligned");
    const void *const words[] = {group_begin, prefix_table, prefix_lens, block_table, lens, lse};
    for (const void *w : words)
        if (!aligned(w, 4)) return set_error(ATTN_ERR_INVALID, "prefix decode: int arrays and lse must be 4-byte aligned");
    const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
    const size_t need = prefix_decode_workspace(s, cache->kv_dtype);
    if (workspace) {
        if (workspace_bytes < need || !aligned(workspace, 256))
            return set_error(ATTN_ERR_WORKSPACE, "prefix decode: workspace needs %zu bytes (256-byte aligned), got %zu",
                             need, workspace_bytes);
    } else {
        // A graph would keep the address of a buffer that a later, larger call replaces.
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        const cudaError_t e = cudaStreamIsCapturing(cs, &capture);
        if (e != cudaSuccess) (void)cudaGetLastError();
        if (capture != cudaStreamCaptureStatusNone || e == cudaErrorStreamCaptureImplicit)
            return set_error(ATTN_ERR_WORKSPACE, "prefix decode: a graph needs a workspace of the caller's (%zu bytes)", need);
        if (!(workspace = library_workspace(4, need, cs)))
            return set_error(ATTN_ERR_NOMEM, "prefix decode: cannot allocate %zu-byte workspace", need);
    }
    attn::prefix::Params p = {};
    p.q = q; p.k = cache->k; p.v = cache->v; p.kscale = cache->kscale; p.vscale = cache->vscale;
    p.group_begin = group_begin; p.prefix_table = prefix_table; p.prefix_lens = prefix_lens;
    p.block_table = block_table; p.lens = lens; p.out = out; p.lse = lse;
    p.err = device_error_ptr();
    if (!p.err) return set_error(ATTN_ERR_CUDA, "prefix decode: no device error word");
    const long long hd = (long long)s->heads * s->head_dim;
    p.q_stride = s->q_row_stride ? s->q_row_stride : hd;
    p.out_stride = s->out_row_stride ? s->out_row_stride : hd;
    p.row_stride = rs;
    p.n_seq = s->n_seq; p.n_groups = s->n_groups; p.heads = s->heads; p.kv_heads = s->kv_heads;
    p.ratio = s->heads / s->kv_heads;
    p.log_page = __builtin_ctz((unsigned)s->page_size);
    p.n_pages = (int)(cache->rows / s->page_size);
    p.max_prefix_pages = s->max_prefix_pages; p.max_pages = s->max_pages;
    p.max_prefix_len = s->max_prefix_len; p.max_len = s->max_len;
    p.scale_log2 = attn::kLog2e * (s->scale > 0.f ? s->scale : 1.f / sqrtf((float)s->head_dim));
    return launch_prefix_decode(p, s->head_dim, cache->kv_dtype, workspace, cs);
}

}  // extern "C"
