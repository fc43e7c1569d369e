// tree_decode.cu -- attn_tree_decode_ex: several query tokens per request (the
// drafts of a token tree), each over the rows that its request's group shares,
// its request's context, and the drafted rows that it may see.
//
// One softmax over three sets of keys, joined from triples (m, l, o) as
// prefix_decode.cu describes.  Prefixes and contexts are seen by every query
// token of their group or request, so they are that file's prefix lines with
// more of them: one launch walks both (prefix.cuh, TREES), a line's rows read
// once for each block of its query rows.  What is left is small and masked: a
// token sees as many drafted rows as it is deep in the tree, out of up to 1024.
// The joining kernel goes through just those by the bits of its mask, so a
// drafted row that a token does not see is not read for it, whatever it holds.
#include "prefix.cuh"
#include "prefix_rows.cuh"

namespace attn {
namespace prefix {

constexpr int kJoinWarps = 4, kMany = 8, kKeys = 4;

// The request of query token r (the last whose tokens begin at or before r),
// or -1 where it has none.  By a warp, 32 probes at a time.
__device__ __forceinline__ int request_of(const Params &p, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = p.n_req;
    while (true) {
        const int step = (n + 31) / 32, i = lane * step;
        const unsigned at = __ballot_sync(0xffffffffu, i < n && __ldg(p.row_begin + lo + i) <= r);
        if (!at) return -1;
        const int k = (__popc(at) - 1) * step;
        lo += k;
        n = min(step, n - k);
        if (step == 1) break;
    }
    return r >= row_first(p, lo) && r < row_first(p, lo + 1) ? lo : -1;
}

// The pieces of a query row in one line, from teams t0 .. t1; with `twice` each team left two.
struct Pieces {
    const float *o;
    const float2 *ml;
    long long step;
    int apart, n;
    bool twice;
    __device__ __forceinline__ long long at(int j) const { return twice ? (j >> 1) * step + (j & 1) * apart : j * step; }
};
template <int D>
__device__ __forceinline__ Pieces pieces_of(const Params &p, const Part &w, const Line &l, int row, int hk, int t0, int t1) {
    Pieces r = {};
    if (l.steps == 0) return r;
    const int rb = row >> w.log_rows, hb = w.n_blocks == 1 ? 0 : hk / w.head_block, hw = hk - hb * w.head_block;
    const Place x = place_of<TREES>(p, w, l, rb, hb);
    const long long at = x.first + t0 * x.step + (w.half ? 0 : (long long)hw * x.apart) + row - (rb << w.log_rows);
    r.o = w.o + at * D;
    r.ml = w.ml + at;
    r.step = x.step;
    r.apart = x.apart;
    r.twice = w.half && l.rows - (rb << w.log_rows) <= w.half;
    r.n = (t1 - t0 + 1) * (r.twice ? 2 : 1);
    return r;
}

// Output type of a cache's calls.
template <typename KV> struct Out { using Type = float; };
template <> struct Out<__nv_bfloat16> { using Type = __nv_bfloat16; };

// One query row (token x head) per warp; SHARED: per CTA, whose warps share its
// pieces and drafted rows.
template <typename KV, int D, bool SHARED>
__global__ void __launch_bounds__(kJoinWarps * 32)
tree_join_kernel(const __grid_constant__ Params p, const __grid_constant__ Part w)
{
    pdl_begin();                          // launched by launch_pdl
    using T = typename Out<KV>::Type;
    constexpr int E = D / 32;
    constexpr bool I8 = sizeof(KV) == 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x, h = (int)blockIdx.y * (SHARED ? 1 : kJoinWarps) + (SHARED ? 0 : warp);
    if (h >= p.heads) return;
    const int req = request_of(p, r);
    if (req < 0) return;
    const int hk = p.ratio == 1 ? h : h / p.ratio, hr = h - hk * p.ratio;

    const Line ctx = line_of<TREES>(p, w, p.n_groups + req);
    Line pre = {};
    long long ctx_begin = 0, pre_begin = 0, team = 1;
    if (w.lines) {
        ctx_begin = __ldcg(w.line_first + p.n_groups + req);
        team = __ldcg(w.line_first + w.lines + 1);
    }
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const bool in = g < p.n_groups && r >= group_first<TREES>(p, g) && r < group_first<TREES>(p, g + 1);
        const unsigned found = __ballot_sync(0xffffffffu, in);
        if (found) {
            const int mine = g0 + __ffs(found) - 1;
            if (w.lines) pre_begin = __ldcg(w.line_first + mine);
            pre = line_of<TREES>(p, w, mine);
            break;
        }
    }
    const int ctx_row = (r - ctx.first_req) * p.ratio + hr, pre_row = (r - pre.first_req) * p.ratio + hr;
    // teams of the first and last step of both segments: four divisions, one in each of four lanes
    const long long x = segment_begin(w, ctx, ctx_row, hk, ctx_begin), y = segment_begin(w, pre, pre_row, hk, pre_begin);
    const int k = lane & 3;
    const int mine = (int)quotient(max((k < 2 ? x : y) + (k & 1 ? (k < 2 ? ctx.steps : pre.steps) - 1 : 0), 0LL), team);
    const Pieces a = pieces_of<D>(p, w, ctx, ctx_row, hk, __shfl_sync(0xffffffffu, mine, 0), __shfl_sync(0xffffffffu, mine, 1));
    const Pieces b = pieces_of<D>(p, w, pre, pre_row, hk, __shfl_sync(0xffffffffu, mine, 2), __shfl_sync(0xffffffffu, mine, 3));

    float m = -INFINITY, l = 0.f, o[E];
    bool bad = false;                     // a score or a sum that is no number
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = 0.f;

    // the drafted rows that the token sees, kKeys at a time
    const int drafts = checked_len(p, checked_len(p, __ldg(p.lens + req), p.max_len) - ctx.keys, p.max_nodes);
    float q[E];
    const T *query = static_cast<const T *>(p.q) + r * p.q_stride + (long long)h * D + lane;
#pragma unroll
    for (int i = 0; i < E; i++) q[i] = to_f32(query[32 * i]);
    const int *table = p.block_table + (long long)req * p.max_pages;
    int seen = 0;
    for (int j0 = 0; j0 < drafts; j0 += 32) {
        const int last = r - ctx.first_req - j0;              // without masks a token sees itself and those before it
        unsigned bits = p.masks ? __ldg(p.masks + (long long)r * p.mask_words + j0 / 32)
                                : last >= 31 ? 0xffffffffu : last < 0 ? 0u : (2u << last) - 1;
        if (drafts - j0 < 32) bits &= (1u << (drafts - j0)) - 1;
        while (bits) {
            long long row[kKeys];
#pragma unroll
            for (int i = 0; i < kKeys; i++) {
                row[i] = -1;
                while (bits) {
                    const int j = __ffs(bits) - 1;
                    bits &= bits - 1;
                    if (SHARED && (seen++ % kJoinWarps) != warp) continue;
                    row[i] = cache_row(p, table, ctx.keys + j0 + j);
                    break;
                }
            }
            float s[kKeys], v[kKeys][E], mx = m;
#pragma unroll
            for (int i = 0; i < kKeys; i++) {
                const long long at = max(row[i], 0LL) * p.row_stride + (long long)hk * D + lane;
                s[i] = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if constexpr (I8) {
                        s[i] = fmaf(q[e], (float)static_cast<const int8_t *>(p.k)[at + 32 * e], s[i]);
                        v[i][e] = (float)static_cast<const int8_t *>(p.v)[at + 32 * e];
                    } else {
                        s[i] = fmaf(q[e], to_f32(static_cast<const KV *>(p.k)[at + 32 * e]), s[i]);
                        v[i][e] = to_f32(static_cast<const KV *>(p.v)[at + 32 * e]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kKeys; i++) {
                s[i] = warp_sum(s[i]) * p.scale_log2;
                if constexpr (I8) s[i] *= p.kscale[max(row[i], 0LL) * p.kv_heads + hk];
                if (row[i] < 0) s[i] = -INFINITY;
                bad |= s[i] != s[i];
                mx = fmaxf(mx, s[i]);
            }
            if (mx == -INFINITY) continue;
            const float old = exp2f(m - mx);
            l *= old;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] *= old;
            m = mx;
#pragma unroll
            for (int i = 0; i < kKeys; i++) {
                if (row[i] < 0) continue;
                float c = exp2f(s[i] - m);
                l += c;
                if constexpr (I8) c *= p.vscale[row[i] * p.kv_heads + hk];
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = fmaf(c, v[i][e], o[e]);
            }
        }
    }

    // the pieces
    const int n = a.n + b.n;
    auto which = [&](int j) { return SHARED ? j * kJoinWarps + warp : j; };
    for (int j0 = 0; which(j0) < n; j0 += 32) {
        const int j = which(j0 + lane);
        const float2 ml = j < a.n ? __ldcg(a.ml + a.at(j)) : j < n ? __ldcg(b.ml + b.at(j - a.n)) : make_float2(-INFINITY, 0.f);
        const float mx = fmaxf(m, warp_max(ml.x));
        bad |= ml.y != ml.y;
        if (mx == -INFINITY) continue;    // no valid row in these pieces
        const bool rows = ml.x != -INFINITY;
        const float old = exp2f(m - mx), c = rows ? exp2f(ml.x - mx) : 0.f;
        l = l * old + warp_sum(ml.y * c);
#pragma unroll
        for (int i = 0; i < E; i++) o[i] *= old;
        m = mx;
        for (int k0 = 0; k0 < 32 && which(j0 + k0) < n; k0 += kMany) {
            float z[kMany][E];
#pragma unroll
            for (int k = 0; k < kMany; k++) {
                const int q = which(j0 + k0 + k);
                const float *from = (q < a.n ? a.o + a.at(q) * D : b.o + b.at(q - a.n) * D) + lane;
#pragma unroll
                for (int i = 0; i < E; i++) z[k][i] = q < n ? __ldcg(from + 32 * i) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kMany; k++) {
                // A piece without a valid row has an o that may not have been written; one whose weight is 0
                // because its scores are low still hands on a value that is no number.
                const float f = __shfl_sync(0xffffffffu, rows ? c : -1.f, k0 + k);
#pragma unroll
                for (int i = 0; i < E; i++) o[i] = f >= 0.f ? fmaf(z[k][i], f, o[i]) : o[i];
            }
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    if constexpr (SHARED) {
        __shared__ bool s_bad[kJoinWarps];
        __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_o[kJoinWarps][D];
        if (lane == 0) { s_m[warp] = m; s_l[warp] = l; s_bad[warp] = bad; }
#pragma unroll
        for (int i = 0; i < E; i++) s_o[warp][lane + 32 * i] = o[i];
        __syncthreads();
        if (warp) return;
        m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        l = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = 0.f;
#pragma unroll
        for (int k = 0; k < kJoinWarps; k++) {
            const float c = s_m[k] == -INFINITY ? 0.f : exp2f(s_m[k] - m);
            l += s_l[k] * c;
            bad |= s_bad[k];
#pragma unroll
            for (int i = 0; i < E; i++) o[i] += s_o[k][lane + 32 * i] * c;
        }
    }
    T *out = static_cast<T *>(p.out) + r * p.out_stride + (long long)h * D + lane;
    if (bad) m = l = NAN;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < E; i++) out[32 * i] = from_f32<T>(o[i] * inv);
    if (p.lse && lane == 0) p.lse[(long long)r * p.heads + h] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace prefix
}  // namespace attn

namespace attn_host {

int launch_tree_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s);

namespace {

using attn::prefix::Params;
using attn::prefix::Part;

// The part on the workspace `base` (NULL to learn its size), in pieces of up to
// seg_rows query rows.
size_t lay_out(Part &w, const Params &p, int d, int seg_rows, int keys, int grid, bool tile, char *base) {
    using namespace attn::prefix;
    w = {};
    if (!p.max_len && !(p.n_groups && p.max_prefix_len)) return 256;
    divide_part(w, p, p.n_groups + p.n_req, seg_rows, keys, grid, tile);
    const long long rows = (long long)p.n_seq * p.ratio, heads = (long long)w.n_blocks * w.head_block;
    w.rows = tile ? seg_rows : (int)std::min<long long>(rows, seg_rows);
    w.after = p.n_groups ? (rows + (long long)w.half * p.n_groups) * heads : 0;
    const size_t all = (size_t)(w.after + rows * (w.half ? 2 : 1) * heads + (long long)w.teams * w.head_block * w.rows);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *at = base ? base + off : nullptr;
        off += (bytes + 255) / 256 * 256;
        return at;
    };
    w.line_first = reinterpret_cast<long long *>(take(((size_t)w.lines + 2) * 8));
    w.ml = reinterpret_cast<float2 *>(take(all * 8));
    w.o = reinterpret_cast<float *>(take(all * d * 4));
    return off;
}

template <typename KV, int D>
int join(const Params &p, const Part &w, cudaStream_t s) {
    using namespace attn::prefix;
    const bool shared = p.n_seq * p.heads < sm_count_here() * 16;
    return check_pdl(launch_pdl(shared ? tree_join_kernel<KV, D, true> : tree_join_kernel<KV, D, false>,
                                dim3(p.n_seq, shared ? p.heads : (p.heads + kJoinWarps - 1) / kJoinWarps), dim3(kJoinWarps * 32), 0, s, p, w),
                     "tree_join_kernel");
}

template <typename KV, class Path, int D>
int run(const Params &p, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    constexpr int CTAS = Path::LEAN ? 2 : 1;
    Part w;
    const size_t bytes = lay_out(w, p, D, Path::ROWS, Path::KEYS, sm_count_here() * CTAS, false, static_cast<char *>(ws));
    if (need) { *need = bytes; return ATTN_OK; }
    const int st = w.lines ? run_part<Path, TREES, D, CTAS>(p, w, 0, s) : ATTN_OK;
    return st ? st : join<KV, D>(p, w, s);
}
template <int D>
int run_tile(const Params &p, void *ws, size_t *need, cudaStream_t s) {
    Part w;
    const size_t bytes = lay_out(w, p, D, 256, 128, sm_count_here(), true, static_cast<char *>(ws));
    if (need) { *need = bytes; return ATTN_OK; }
    const int st = w.lines ? launch_tree_tile(p, w, D, s) : ATTN_OK;
    return st ? st : join<__nv_bfloat16, D>(p, w, s);
}

// Paths by the query rows that a line has on average (counted from the shape:
// their numbers are on the device), as for prefixes (prefix_decode.cu).
template <int D>
int run_d(const Params &p, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    const long long all = (long long)p.n_seq * p.ratio, rows = (all + p.n_req - 1) / p.n_req;
    if (kv_dtype == ATTN_BF16) {
        if constexpr (D == 64 || D == 128) {
            if (rows >= 32 || (p.n_groups && p.max_prefix_len && all >= 32LL * p.n_groups)) return run_tile<D>(p, ws, need, s);
        }
        if (rows <= 8) return run<__nv_bfloat16, Bf16Path<D, 1>, D>(p, ws, need, s);
        return run<__nv_bfloat16, Bf16Path<D, D == 32 ? 8 : D == 64 ? 4 : 2>, D>(p, ws, need, s);
    }
    if (kv_dtype == ATTN_I8) {
        if (rows <= 4) return run<int8_t, I8Path<D, 1>, D>(p, ws, need, s);
        return run<int8_t, I8Path<D, D <= 64 ? 4 : 2>, D>(p, ws, need, s);
    }
    if (rows <= 4) return run<float, F32Path<D, 4>, D>(p, ws, need, s);
    return run<float, F32Path<D, 8>, D>(p, ws, need, s);
}

}  // namespace

// need: the size of the workspace alone.
int launch_tree_decode(const Params &p, int d, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    switch (d) {
        case 32: return run_d<32>(p, kv_dtype, ws, need, s);
        case 64: return run_d<64>(p, kv_dtype, ws, need, s);
        case 96: return run_d<96>(p, kv_dtype, ws, need, s);
        default: return run_d<128>(p, kv_dtype, ws, need, s);
    }
}

}  // namespace attn_host
