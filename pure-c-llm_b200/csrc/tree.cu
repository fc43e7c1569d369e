// tree.cu -- what surrounds the attention of drafted token trees:
// attn_tree_plan_ex (positions and visibility from the drafts' parents) and
// attn_tree_commit_ex (an accepted path's cache rows moved together in every
// layer, the lengths after it, the pages behind it handed back).
#include <algorithm>

#include "common.cuh"

namespace attn {
namespace tree {

constexpr int kMaxNodes = 1024;

struct PlanParams {
    const int *cu_rows, *parents, *positions;
    int *positions_out;
    uint32_t *masks;
    int *err;
    int n_seq, n_rows, words;
};

// A CTA per request.  A node's mask is its own bit and those of its ancestors,
// whose indexes descend, so a thread walks up from its node through the parents
// in shared memory and writes the words from the last to the first; the number
// of steps is the depth.  Bound by latency: two dependent loads and a walk of a
// few nodes (a chain of 1024 takes that many steps).
__global__ void __launch_bounds__(256)
tree_plan_kernel(const __grid_constant__ PlanParams p)
{
    extern __shared__ int parent[];
    pdl_begin();                          // launched by launch_pdl
    const int s = blockIdx.x;
    const int first = min(max(__ldg(p.cu_rows + s), 0), p.n_rows), end = min(max(__ldg(p.cu_rows + s + 1), first), p.n_rows);
    const int rows = end - first, n = min(rows, 32 * p.words);
    if (rows == 0) return;
    const int base = p.positions[first];  // (positions_out may be positions)
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        int up = __ldg(p.parents + first + i);
        if (up < -1 || up >= i) {
            atomicExch(p.err, 0x704);
            up = -1;
        }
        parent[i] = up;
    }
    if (rows > n && threadIdx.x == 0) atomicExch(p.err, 0x705);
    __syncthreads();
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
        int at = i < n ? i : -1, depth = -1;
        uint32_t *mask = p.masks + (long long)(first + i) * p.words;
        for (int w = p.words - 1; w >= 0; w--) {
            uint32_t bits = 0;
            while (at >= 32 * w) {
                bits |= 1u << (at & 31);
                at = parent[at];
                depth++;
            }
            mask[w] = bits;
        }
        p.positions_out[first + i] = base + max(depth, 0);
    }
}

struct Layer { char *k, *v; float *kscale, *vscale; long long pitch, pages; };   // bytes between rows
struct CommitParams {
    const int *cu_rows, *ctx_lens, *lens, *leaf;
    const uint32_t *masks;
    const int *table;
    int *free_pages;
    const int *free_count;
    int *lens_out, *counts, *err;
    long long table_stride;
    int n_seq, n_rows, words, log_page, max_pages, n_pages, row_bytes, kv_heads;
    Layer layers[ATTN_MAX_LAYERS];
};
constexpr int kThreads = 256, kRows = 8;

// What request s holds and accepts: its rows before the drafts, its rows in
// all, and the words of its path (the leaf's mask up to the leaf).
struct Accepted {
    int ctx, len, drafts, leaf;
    const uint32_t *mask;                 // NULL: all up to the leaf
    __device__ __forceinline__ uint32_t word(int w) const {
        const int last = leaf - 32 * w;
        if (last < 0) return 0;
        const uint32_t upto = last >= 31 ? 0xffffffffu : (2u << last) - 1;
        return mask ? __ldg(mask + w) & upto : upto;
    }
};
__device__ __forceinline__ Accepted accepted(const CommitParams &p, int s, bool report) {
    Accepted a;
    const int cap = p.max_pages << p.log_page;
    // (clamped to the rows of masks, as the plan and the decode clamp to theirs; chains have none)
    const int most = p.masks ? p.n_rows : 0x7fffffff;
    const int first = min(max(__ldg(p.cu_rows + s), 0), most), end = min(max(__ldg(p.cu_rows + s + 1), first), most);
    int leaf = __ldg(p.leaf + s);
    a.len = min(max(__ldg(p.lens + s), 0), cap);
    a.ctx = min(max(__ldg(p.ctx_lens + s), 0), a.len);
    a.drafts = min(a.len - a.ctx, 32 * p.words);
    // a leaf that is no draft accepts nothing; one of a request without drafted rows (refused ones) is not reported
    if (leaf < -1 || leaf >= a.drafts || leaf >= end - first) {
        if (report && a.drafts > 0) atomicExch(p.err, 0x706);
        leaf = -1;
    }
    a.leaf = leaf;
    a.mask = p.masks && leaf >= 0 ? p.masks + (long long)(first + leaf) * p.words : nullptr;
    return a;
}

// CTA (s, l): the rows of request s in layer l.  The path's i-th draft goes to
// row ctx + i; as drafts of a path ascend, that is at or before its own row, so
// a thread that takes its 16 bytes of kRows rows at a time, reading all before
// writing any, overwrites nothing that is still to be read.  The drafts at the
// path's beginning that are in place already are not touched.  CTA (n_seq, 0):
// lengths, pages and counts of all requests.
__global__ void __launch_bounds__(kThreads)
tree_commit_kernel(const __grid_constant__ CommitParams p)
{
    __shared__ int from[kMaxNodes], to[kMaxNodes];     // cache rows
    __shared__ int s_moves, s_sum[kThreads / 32][2], s_none;
    pdl_begin();                          // launched by launch_pdl
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int page = 1 << p.log_page;
    auto pages_of = [&](int tokens) { return (tokens + page - 1) >> p.log_page; };

    if ((int)blockIdx.x == p.n_seq) {
        if (blockIdx.y) return;
        const int have = min(max(__ldg(p.free_count), 0), p.n_pages);
        if (tid == 0) s_none = 0;
        int tokens = 0, back = 0;         // of the requests before this round's
        for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) {
            const int s = s0 + tid;
            int n = 0, ret = 0, keep = 0;
            if (s < p.n_seq) {
                const Accepted a = accepted(p, s, true);
                for (int w = 0; 32 * w <= a.leaf; w++) n += __popc(a.word(w));
                keep = pages_of(a.ctx + n);
                ret = pages_of(a.len) - keep;
                p.lens_out[s] = a.ctx + n;
            }
            int x = n, y = ret;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) { x += u; y += v; }
            }
            __syncthreads();              // the round before is done with the sums
            if (lane == 31) { s_sum[warp][0] = x; s_sum[warp][1] = y; }
            const int none = __popc(__ballot_sync(0xffffffffu, s < p.n_seq && n == 0));
            if (lane == 0 && none) atomicAdd(&s_none, none);
            __syncthreads();
            int at = back + y - ret;
            for (int w = 0; w < kThreads / 32; w++) {
                if (w < warp) at += s_sum[w][1];
                tokens += s_sum[w][0];
                back += s_sum[w][1];
            }
            for (int i = 0; i < ret; i++)
                if (have + at + i < p.n_pages) p.free_pages[have + at + i] = __ldg(p.table + s * p.table_stride + keep + i);
        }
        __syncthreads();
        if (tid == 0) {
            p.counts[0] = min(have + back, p.n_pages);
            p.counts[1] = tokens;
            p.counts[2] = s_none;
            p.counts[3] = back;
        }
        return;
    }

    const int s = blockIdx.x;
    const Layer &layer = p.layers[blockIdx.y];
    if (!layer.k) return;                 // a call without caches
    const Accepted a = accepted(p, s, false);
    if (warp == 0) {
        // the drafts at the beginning that are in place, then the others' rows in the path's order
        auto row_of = [&](int t) {
            const int id = __ldg(p.table + s * p.table_stride + (t >> p.log_page));
            if ((unsigned long long)id < (unsigned long long)layer.pages) return (id << p.log_page) + (t & (page - 1));
            atomicExch(p.err, 0x702);
            return -1;
        };
        int before = 0, moves = 0;
        for (int w = 0; 32 * w <= a.leaf; w++) {
            const uint32_t bits = a.word(w);
            const int i = before + __popc(bits & ((1u << lane) - 1)), j = 32 * w + lane;
            const bool moves_here = (bits >> lane & 1) && i != j;
            const unsigned all = __ballot_sync(0xffffffffu, moves_here);
            if (moves_here) {
                const int k = moves + __popc(all & ((1u << lane) - 1));
                from[k] = row_of(a.ctx + j);
                to[k] = row_of(a.ctx + i);
            }
            moves += __popc(all);
            before += __popc(bits);
        }
        if (lane == 0) s_moves = moves;
    }
    __syncthreads();
    const int moves = s_moves;
    const int columns = p.row_bytes / 16;
    for (int c = tid; c < 2 * columns; c += kThreads) {
        char *base = (c < columns ? layer.k : layer.v) + (c < columns ? c : c - columns) * 16;
        for (int i0 = 0; i0 < moves; i0 += kRows) {
            uint4 x[kRows];
#pragma unroll
            for (int i = 0; i < kRows; i++)
                if (i0 + i < moves && from[i0 + i] >= 0) x[i] = *reinterpret_cast<const uint4 *>(base + from[i0 + i] * layer.pitch);
#pragma unroll
            for (int i = 0; i < kRows; i++)
                if (i0 + i < moves && from[i0 + i] >= 0 && to[i0 + i] >= 0) *reinterpret_cast<uint4 *>(base + to[i0 + i] * layer.pitch) = x[i];
        }
    }
    if (!layer.kscale) return;
    for (int c = tid; c < 2 * p.kv_heads; c += kThreads) {
        float *base = c < p.kv_heads ? layer.kscale + c : layer.vscale + c - p.kv_heads;
        for (int i = 0; i < moves; i++)
            if (from[i] >= 0 && to[i] >= 0) base[(long long)to[i] * p.kv_heads] = base[(long long)from[i] * p.kv_heads];
    }
}

}  // namespace tree
}  // namespace attn

namespace attn_host {

int launch_tree_plan(int n_seq, int n_rows, int words, const int *cu_rows, const int *parents, const int *positions, int *positions_out,
                     uint32_t *masks, int *err, cudaStream_t s) {
    using namespace attn::tree;
    const PlanParams p = {cu_rows, parents, positions, positions_out, masks, err, n_seq, n_rows, words};
    const int threads = std::min(256, 32 * words);
    return check_pdl(launch_pdl(tree_plan_kernel, dim3(n_seq), dim3(threads), (size_t)words * 128, s, p), "tree_plan_kernel");
}

int launch_tree_commit(const attn_page_shape *s, int n_layers, const attn_paged_kv *caches, int kv_heads, int head_dim, const int *cu_rows,
                       const int *ctx_lens, const int *lens, const int *leaf, const uint32_t *masks, int words, const int *table,
                       int *free_pages, const int *free_count, int *lens_out, int *counts, int *err, cudaStream_t stream) {
    using namespace attn::tree;
    CommitParams p = {};
    p.cu_rows = cu_rows; p.ctx_lens = ctx_lens; p.lens = lens; p.leaf = leaf; p.masks = masks; p.table = table;
    p.free_pages = free_pages; p.free_count = free_count; p.lens_out = lens_out; p.counts = counts; p.err = err;
    p.table_stride = s->table_stride ? s->table_stride : s->max_pages;
    p.n_seq = s->n_seq; p.n_rows = s->max_tokens; p.words = words; p.log_page = __builtin_ctz((unsigned)s->page_size);
    p.max_pages = s->max_pages; p.n_pages = s->n_pages; p.kv_heads = kv_heads;
    for (int i = 0; i < n_layers; i++) {
        const attn_paged_kv &c = caches[i];
        const int e = c.kv_dtype == ATTN_F32 ? 4 : c.kv_dtype == ATTN_BF16 ? 2 : 1;
        const long long stride = c.row_stride ? c.row_stride : (long long)kv_heads * head_dim;
        p.row_bytes = kv_heads * head_dim * e;
        const bool i8 = c.kv_dtype == ATTN_I8;
        p.layers[i] = {(char *)c.k, (char *)c.v, i8 ? c.kscale : nullptr, i8 ? c.vscale : nullptr, stride * e, c.rows >> p.log_page};
    }
    return check_pdl(launch_pdl(tree_commit_kernel, dim3(s->n_seq + 1, std::max(n_layers, 1)), dim3(kThreads), 0, stream, p),
                     "tree_commit_kernel");
}

}  // namespace attn_host
