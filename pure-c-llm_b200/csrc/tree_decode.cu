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

constexpr int kJoinWarps = 8;

// Line i as the first kernel has told it.
__device__ __forceinline__ Line told_line(const Params &p, const Part &w, int i, int4 info) {
    Line l;
    l.prefix = i < p.n_groups;
    l.first_req = info.x;
    l.rows = info.y;
    l.keys = info.z;
    l.blocks = ceil_shift(l.rows, w.log_rows);
    l.base = (l.first_req * p.ratio >> w.log_rows) + (l.prefix ? i : i - p.n_groups);
    line_steps<TREES>(w, l);
    return l;
}

// The pieces of a query row in one line, from teams t0 .. t1, by their rows on
// the workspace; where each team left two (Part::half), `apart` is not 0.
struct Pieces {
    long long first;
    int step, apart, n;
    __device__ __forceinline__ long long at(int j) const { return first + (apart ? (long long)(j >> 1) * step + (j & 1) * apart : (long long)j * step); }
};
template <int D>
__device__ __forceinline__ Pieces pieces_of(const Params &p, const Part &w, const Line &l, int row, int hk, int t0, int t1) {
    const int rb = row >> w.log_rows, hb = w.n_blocks == 1 ? 0 : hk / w.head_block, hw = hk - hb * w.head_block;
    const Place x = place_of<TREES>(p, w, l, rb, hb);
    const bool twice = w.half && l.rows - (rb << w.log_rows) <= w.half;
    return {x.first + t0 * x.step + (w.half ? 0 : (long long)hw * x.apart) + row - (rb << w.log_rows), (int)x.step, twice ? x.apart : 0,
            (t1 - t0 + 1) * (twice ? 2 : 1)};
}

// Output type of a cache's calls.
template <typename KV> struct Out { using Type = float; };
template <> struct Out<__nv_bfloat16> { using Type = __nv_bfloat16; };

using sm100::mul2;
// Four consecutive elements as two packed pairs of floats.
struct Quad { uint64_t a, b; };
__device__ __forceinline__ Quad quad(float4 x) { return {f2(x.x, x.y), f2(x.z, x.w)}; }
__device__ __forceinline__ Quad four(const float *p) { return quad(*reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ Quad four(const __nv_bfloat16 *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return {f2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u)), f2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u))};
}
__device__ __forceinline__ Quad four(const int8_t *p) {
    const char4 c = *reinterpret_cast<const char4 *>(p);
    return {f2(c.x, c.y), f2(c.z, c.w)};
}
__device__ __forceinline__ float4 floats(const Quad &q) {
    float4 x;
    f2_split(q.a, x.x, x.y);
    f2_split(q.b, x.z, x.w);
    return x;
}

// A warp takes one query token and four adjacent query heads, eight lanes a
// head: lane i has elements 4 i .. 4 i + 3 of every 32.  A score is then three
// exchanges for all four heads, and each lane keeps its head's maximum and sum,
// so weights need none.  SHARED: the warps of a CTA share that, each taking some
// of the drafted rows and pieces.
// 3 CTAs an SM: at d 96 and 128 that spills up to 96 bytes, which costs
// nothing: with 2 at d 128, without spills, the case of two documents took 1143,
// 1140 and 1157 us in turn with 1149, 1136 and 1156.
template <typename KV, int D, bool SHARED>
__global__ void __launch_bounds__(kJoinWarps * 32, 3)
tree_join_kernel(const __grid_constant__ Params p, const __grid_constant__ Part w)
{
    pdl_begin();                          // launched by launch_pdl
    using T = typename Out<KV>::Type;
    constexpr int C = D / 32, KB = 2;     // elements of a lane, in fours; drafted rows, and pieces, at once
    constexpr bool I8 = sizeof(KV) == 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x;
    const int unit = (int)blockIdx.y * (SHARED ? 1 : kJoinWarps) + (SHARED ? 0 : warp);
    if (4 * unit >= p.heads) return;
    // What counts here is the chain of dependent loads, so each link's go out together: the token's request, its mask and
    // the number of tokens; then the lines; then the pieces' maxima and the page table; then the rows.
    const int2 of = __ldcg(w.row_of + r);                     // (not written for rows of no request)
    const int req = of.x, total = row_first(p, p.n_req);
    unsigned bits = p.masks && p.max_nodes ? __ldg(p.masks + (long long)r * p.mask_words) : 0u;
    if (r >= total || (unsigned)req >= (unsigned)p.n_req || r < row_first(p, req) || r >= row_first(p, req + 1)) return;
    const int h = min(4 * unit + lane / 8, p.heads - 1), mine = lane % 8 * 4;      // (idle lanes repeat the last head)
    const int hk = p.ratio == 1 ? h : h / p.ratio, hr = h - hk * p.ratio;

    const int own = p.n_groups + req, group = (unsigned)of.y < (unsigned)p.n_groups ? of.y : -1;
    const long long team = __ldcg(w.line_first + w.lines + 1), ctx_begin = __ldcg(w.line_first + own);
    const long long pre_begin = group >= 0 ? __ldcg(w.line_first + group) : 0;
    const int len = __ldg(p.lens + req);
    const Line ctx = told_line(p, w, own, __ldcg(w.line_info + own));
    Line pre = {};
    if (group >= 0) {
        pre = told_line(p, w, group, __ldcg(w.line_info + group));
        if ((r - pre.first_req) * p.ratio < 0 || (r - pre.first_req) * p.ratio >= pre.rows) pre.steps = 0;
    }
    const int drafts = checked_len(p, checked_len(p, len, p.max_len) - ctx.keys, p.max_nodes);
    // the pieces of the two lines, and the maxima and sums of the first ones
    auto line_pieces = [&](const Line &line, long long begin) {
        if (line.steps == 0) return Pieces{};
        const int row = (r - line.first_req) * p.ratio + hr;
        const long long first = segment_begin(w, line, row, hk, begin);
        const int t0 = (int)quotient(max(first, 0LL), team), t1 = (int)quotient(max(first + (long long)(line.steps - 1) * line.weight, 0LL), team);
        return pieces_of<D>(p, w, line, row, hk, t0, t1);
    };
    auto bring_ml = [&](const Pieces &a, int j0, float2 (&ml)[KB]) {
#pragma unroll
        for (int i = 0; i < KB; i++) ml[i] = j0 + i < a.n ? __ldcg(w.ml + a.at(j0 + i)) : make_float2(-INFINITY, 0.f);
    };
    const Pieces ctx_pieces = line_pieces(ctx, ctx_begin), pre_pieces = line_pieces(pre, pre_begin);
    const int j_first = SHARED ? warp * KB : 0;
    float2 ctx_ml[KB], pre_ml[KB];
    bring_ml(ctx_pieces, j_first, ctx_ml);
    bring_ml(pre_pieces, j_first, pre_ml);

    Quad q[C], o[C];
    float m = -INFINITY, l = 0.f;
    const T *query = static_cast<const T *>(p.q) + r * p.q_stride + (long long)h * D + mine;
#pragma unroll
    for (int c = 0; c < C; c++) {
        q[c] = four(query + 32 * c);
        o[c] = {0, 0};
    }
    auto add = [&](float f, const Quad (&v)[C]) {
        const uint64_t ff = f2(f, f);
#pragma unroll
        for (int c = 0; c < C; c++) o[c] = {fma2(ff, v[c].a, o[c].a), fma2(ff, v[c].b, o[c].b)};
    };
    // Takes in maxima x (-inf: none) with sums s; x becomes the weights.
    auto fold = [&](float (&x)[KB], const float (&s)[KB]) {
        float mx = m;
#pragma unroll
        for (int i = 0; i < KB; i++) mx = fmaxf(mx, x[i]);
        const float old = mx == m ? 1.f : exp2f(m - mx);
        if (__any_sync(0xffffffffu, old != 1.f)) {
            const uint64_t ff = f2(old, old);
            l *= old;
#pragma unroll
            for (int c = 0; c < C; c++) o[c] = {mul2(o[c].a, ff), mul2(o[c].b, ff)};
        }
        m = mx;
#pragma unroll
        for (int i = 0; i < KB; i++) {
            x[i] = x[i] == -INFINITY ? 0.f : exp2f(x[i] - mx);
            l = fmaf(x[i], s[i], l);
        }
    };

    // the drafted rows that the token sees
    const int *table = p.block_table + (long long)req * p.max_pages;
    int seen = 0;
    for (int j0 = 0; j0 < drafts; j0 += 32) {
        const int last = r - ctx.first_req - j0;              // without masks a token sees itself and those before it
        if (!p.masks) bits = last >= 31 ? 0xffffffffu : last < 0 ? 0u : (2u << last) - 1;
        else if (j0) bits = __ldg(p.masks + (long long)r * p.mask_words + j0 / 32);
        if (drafts - j0 < 32) bits &= (1u << (drafts - j0)) - 1;
        while (bits) {
            int row[KB];
            bool any = false;
#pragma unroll
            for (int i = 0; i < KB; i++) {
                row[i] = -1;
                while (bits) {
                    const int j = __ffs(bits) - 1;
                    bits &= bits - 1;
                    if (SHARED && (seen++ % kJoinWarps) != warp) continue;
                    row[i] = (int)cache_row(p, table, ctx.keys + j0 + j);
                    any = true;
                    break;
                }
            }
            if (!any) continue;
            Quad v[KB][C];
            float x[KB], one[KB];
#pragma unroll
            for (int i = 0; i < KB; i++) {
                x[i] = 0.f;
                one[i] = 1.f;
                if (row[i] < 0) continue;
                const long long at = row[i] * p.row_stride + (long long)hk * D + mine;
                uint64_t dot = 0;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const Quad k = four(static_cast<const KV *>(p.k) + at + 32 * c);
                    v[i][c] = four(static_cast<const KV *>(p.v) + at + 32 * c);
                    dot = fma2(q[c].b, k.b, fma2(q[c].a, k.a, dot));
                }
                float even, odd;
                f2_split(dot, even, odd);
                x[i] = even + odd;
            }
#pragma unroll
            for (int k = 1; k < 8; k *= 2)
#pragma unroll
                for (int i = 0; i < KB; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], k);
            float vscale[KB];
#pragma unroll
            for (int i = 0; i < KB; i++) {
                x[i] *= p.scale_log2;
                if constexpr (I8) {
                    const long long at = (long long)max(row[i], 0) * p.kv_heads + hk;
                    x[i] *= __ldg(p.kscale + at);
                    vscale[i] = __ldg(p.vscale + at);
                }
                if (row[i] < 0) x[i] = -INFINITY;
            }
            fold(x, one);
#pragma unroll
            for (int i = 0; i < KB; i++) {
                if (row[i] < 0) continue;
                if constexpr (I8) x[i] *= vscale[i];
                add(x[i], v[i]);
            }
        }
    }

    auto join = [&](const Pieces &a, float2 (&ml)[KB]) {
        int most = a.n;                   // of the four heads
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
        for (int j0 = j_first; j0 < most; j0 += KB * (SHARED ? kJoinWarps : 1)) {
            if (j0 != j_first) bring_ml(a, j0, ml);
            float x[KB], s[KB];
            Quad v[KB][C];
#pragma unroll
            for (int i = 0; i < KB; i++) {
                x[i] = ml[i].x;
                s[i] = ml[i].y;
                const long long at = j0 + i < a.n ? a.at(j0 + i) : 0;
#pragma unroll
                for (int c = 0; c < C; c++)
                    v[i][c] = quad(j0 + i < a.n ? __ldcg(reinterpret_cast<const float4 *>(w.o + at * D + mine + 32 * c)) : make_float4(0.f, 0.f, 0.f, 0.f));
            }
            bool there[KB];
#pragma unroll
            for (int i = 0; i < KB; i++) there[i] = x[i] != -INFINITY;
            fold(x, s);
            // A piece without a valid row has an o that may not have been written; one whose weight is 0 because its
            // scores are low still hands on a value that is no number.
#pragma unroll
            for (int i = 0; i < KB; i++)
                if (there[i]) add(x[i], v[i]);
        }
    };
    join(ctx_pieces, ctx_ml);
    join(pre_pieces, pre_ml);

    if constexpr (SHARED) {
        __shared__ float2 s_ml[kJoinWarps][4];
        __shared__ float4 s_o[kJoinWarps][C][32];
        if (lane % 8 == 0) s_ml[warp][lane / 8] = make_float2(m, l);
#pragma unroll
        for (int c = 0; c < C; c++) s_o[warp][c][lane] = floats(o[c]);
        __syncthreads();
        if (warp) return;
        for (int k0 = 1; k0 < kJoinWarps; k0 += KB) {
            float x[KB], s[KB];
#pragma unroll
            for (int i = 0; i < KB; i++) {
                const float2 ml = k0 + i < kJoinWarps ? s_ml[k0 + i][lane / 8] : make_float2(-INFINITY, 0.f);
                x[i] = ml.x;
                s[i] = ml.y;
            }
            fold(x, s);
#pragma unroll
            for (int i = 0; i < KB; i++) {
                if (k0 + i >= kJoinWarps) continue;
                Quad v[C];
#pragma unroll
                for (int c = 0; c < C; c++) v[c] = quad(s_o[k0 + i][c][lane]);
                add(x[i], v);
            }
        }
    }
    if (4 * unit + lane / 8 >= p.heads) return;
    T *out = static_cast<T *>(p.out) + r * p.out_stride + (long long)h * D + mine;
    const float inv = l != l ? NAN : m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const float4 x = floats(o[c]);
        store4(out + 32 * c, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    }
    if (p.lse && lane % 8 == 0) p.lse[(long long)r * p.heads + h] = l != l ? NAN : m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
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
size_t lay_out(Part &w, const Params &p, int d, int seg_rows, int keys, int grid, bool tile, int warps, char *base) {
    using namespace attn::prefix;
    w = {};
    divide_part(w, p, p.n_groups + p.n_req, seg_rows, keys, grid, tile, warps);
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
    w.row_of = reinterpret_cast<int2 *>(take((size_t)p.n_seq * 8));
    w.line_info = reinterpret_cast<int4 *>(take((size_t)w.lines * 16));
    w.ml = reinterpret_cast<float2 *>(take(all * 8));
    w.o = reinterpret_cast<float *>(take(all * d * 4));
    return off;
}

template <typename KV, int D>
int join(const Params &p, const Part &w, cudaStream_t s) {
    using namespace attn::prefix;
    // SHARED while the tokens' units leave most warps without one (fp32, 16 heads of
    // 32, contexts of up to 500: 32 tokens 15.8 us, 17.4 unshared, 128 tokens 17.6 to
    // 18.5, 256 tokens 25.6 to 22.4, 512 41.2 to 34.2)
    const int units = (p.heads + 3) / 4;
    const bool shared = (long long)p.n_seq * units < 4LL * sm_count_here();
    return check_pdl(launch_pdl(shared ? tree_join_kernel<KV, D, true> : tree_join_kernel<KV, D, false>,
                                dim3(p.n_seq, shared ? units : (units + kJoinWarps - 1) / kJoinWarps), dim3(kJoinWarps * 32), 0, s, p, w),
                     "tree_join_kernel");
}

template <typename KV, class Path, int D, int WARPS = attn::prefix::kWarps>
int run(const Params &p, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    constexpr int CTAS = Path::LEAN ? 2 : 1;
    Part w;
    const size_t bytes = lay_out(w, p, D, Path::ROWS, Path::KEYS, sm_count_here() * CTAS, false, WARPS, static_cast<char *>(ws));
    if (need) { *need = bytes; return ATTN_OK; }
    const int st = run_part<Path, TREES, D, CTAS, WARPS>(p, w, 0, s);
    return st ? st : join<KV, D>(p, w, s);
}
template <int D>
int run_tile(const Params &p, void *ws, size_t *need, cudaStream_t s) {
    Part w;
    const size_t bytes = lay_out(w, p, D, 256, 128, sm_count_here(), true, 0, static_cast<char *>(ws));
    if (need) { *need = bytes; return ATTN_OK; }
    const int st = launch_tree_tile(p, w, D, s);
    return st ? st : join<__nv_bfloat16, D>(p, w, s);
}

// The path with the least time, by bounds: rows of keys (the shape's bounds of
// the lengths, as the lengths are on the device) times the blocks of query rows
// that pass over them (the rows that a line has on average) times what such a
// pass costs.  Costs are us of full blocks, one to each of 64 contexts of 500 to
// 4500 rows (bf16, 500 to 8200 for INT8, 250 to 4000 for fp32; 0.25 to 0.6 GB), and
// both sides of each choice follow from them and hold as measured:
//   bf16, d 64, 32 heads, tiles, blocks of 32, 16, 8: 16 rows 202, 143, 114, 180, 32 rows
//     235, 171, 204, 341, 64 rows 300, 338, -, 686; 8 groups sharing 8192 rows, 32 rows
//     of a group 261, 154, -, 264, 128 rows 271, 333, -, 616.
//   bf16, d 128, 8 key heads, tiles, blocks of 16, 8: 16 rows 73, 68, 92, 32 rows 83, 105, 157.
//   bf16, d 32, blocks of 64, 16, 8: 8 rows 157, 72, 63, 32 rows 191, 148, 184, 64 rows 246, 298, 367.
//   INT8, d 64, blocks of 16, 8, 4: 4 rows 229, 156, 127, 8 rows 240, 165, 234, 16 rows 252, 306, -.
//   fp32, blocks of 8, 4: d 32, 4 rows 132, 104, 8 rows 139, 177; d 96, 12 heads, 2 rows 270, 206, 4 rows 277, 231;
//     d 128, 4 rows 210, 231, 8 rows 215, 404, with 12 heads, 2 rows 304, 309, 4 rows 315, 325: blocks of 8 alone.
// Lines of fewer rows than the shape leaves room for would want smaller blocks:
// INT8 with room for 16 rows and 8 on average takes 245 in blocks of 16, 234 in 8.
template <int N>
int least(const Params &p, const int (&blocks)[N], const int (&costs)[N]) {
    const long long all = (long long)p.n_seq * p.ratio, own = (all + p.n_req - 1) / p.n_req, group = p.n_groups ? (all + p.n_groups - 1) / p.n_groups : 0;
    int best = 0;
    double time = 0.;
    for (int i = 0; i < N; i++) {
        const double passes = (double)p.n_req * p.max_len * (double)((own + blocks[i] - 1) / blocks[i]) +
                              (double)p.n_groups * p.max_prefix_len * (double)((group + blocks[i] - 1) / blocks[i]);
        if (i && passes * costs[i] >= time) continue;
        best = i;
        time = passes * costs[i];
    }
    return best;
}
// Blocks of 8 INT8 or 16 bf16 rows at d 32 and 64 leave the registers for 12
// warps an SM (INT8, d 64: 160 us, 183 with 8 warps; bf16 104 and 109).
constexpr int kMoreWarps = 12;

template <int D>
int run_d(const Params &p, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    using B = __nv_bfloat16;
    if (kv_dtype == ATTN_BF16) {
        if constexpr (D == 32) {
            switch (least<3>(p, {8, 16, 64}, {63, 82, 220})) {
                case 0: return run<B, Bf16Path<D, 1>, D>(p, ws, need, s);
                case 1: return run<B, Bf16Path<D, 2>, D, kMoreWarps>(p, ws, need, s);
                default: return run<B, Bf16Path<D, 8>, D>(p, ws, need, s);
            }
        } else if constexpr (D == 64) {
            switch (least<4>(p, {8, 16, 32, 128}, {103, 114, 171, 250})) {
                case 0: return run<B, Bf16Path<D, 1>, D>(p, ws, need, s);
                case 1: return run<B, Bf16Path<D, 2>, D, kMoreWarps>(p, ws, need, s);
                case 2: return run<B, Bf16Path<D, 4>, D>(p, ws, need, s);
                default: return run_tile<D>(p, ws, need, s);
            }
        } else if constexpr (D == 96) {
            return least<2>(p, {8, 16}, {50, 55}) ? run<B, Bf16Path<D, 2>, D>(p, ws, need, s) : run<B, Bf16Path<D, 1>, D>(p, ws, need, s);
        } else {
            switch (least<3>(p, {8, 16, 128}, {64, 68, 90})) {
                case 0: return run<B, Bf16Path<D, 1>, D>(p, ws, need, s);
                case 1: return run<B, Bf16Path<D, 2>, D>(p, ws, need, s);
                default: return run_tile<D>(p, ws, need, s);
            }
        }
    }
    if (kv_dtype == ATTN_I8) {
        if constexpr (D <= 64) {
            switch (D == 32 ? least<3>(p, {4, 8, 16}, {200, 253, 365}) : least<3>(p, {4, 8, 16}, {127, 163, 245})) {
                case 0: return run<int8_t, I8Path<D, 1>, D>(p, ws, need, s);
                case 1: return run<int8_t, I8Path<D, 2>, D, kMoreWarps>(p, ws, need, s);
                default: return run<int8_t, I8Path<D, 4>, D>(p, ws, need, s);
            }
        } else {
            return (D == 96 ? least<2>(p, {4, 8}, {103, 133}) : least<2>(p, {4, 8}, {130, 146})) ? run<int8_t, I8Path<D, 2>, D>(p, ws, need, s)
                                                                                               : run<int8_t, I8Path<D, 1>, D>(p, ws, need, s);
        }
    }
    if constexpr (D < 128) {
        const bool eight = D == 32   ? least<2>(p, {4, 8}, {104, 137})
                           : D == 64 ? least<2>(p, {4, 8}, {193, 226})
                                     : least<2>(p, {4, 8}, {231, 277});
        if (!eight) return run<float, F32Path<D, 4>, D>(p, ws, need, s);
    }
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
