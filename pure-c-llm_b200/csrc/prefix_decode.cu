// prefix_decode.cu -- attn_prefix_decode_ex: one query token per request over
// the rows that its group shares and its own, both in a paged cache.
//
// With keys j over prefix and own rows, out = sum_j p_j v_j / sum_j p_j and
// p_j = 2^(x_j - m), x_j = scale log2(e) q.k_j, m = max_j x_j.  Any split of
// the keys gives triples (m, l, o) that join exactly: with M = max m_i,
// l = sum l_i 2^(m_i - M) and o likewise.
//
// Work.  There are two parts with a launch each: the groups' prefixes, with the
// query rows of all their requests, and the requests' own rows, with
// heads/kv_heads query rows per key head.  A "line" is one page-table line of
// a part; a segment is a line x a block of query rows x a block of key heads,
// its keys counted in steps of KEYS.  All steps of a part, in order, are cut
// into equal ranges, one per team of warps, so no length decides how busy an
// SM is; a team's warps take one key head each and read adjacent parts of the
// same cache rows.  What a warp leaves of a segment (its piece) goes to the
// workspace, at slot segment + team, and prefix_merge_kernel joins the pieces
// of each query row.
//
// Bound: HBM (the cache rows, once).  Little else may cost: each warp
// copies its rows through a ring of its own in shared memory, from which the
// lanes read them in the layout that the arithmetic takes (prefix_paths.cuh),
// and meets no other warp until the merge.
#include "prefix.cuh"
#include "prefix_rows.cuh"

namespace attn {
namespace prefix {

// Joins the pieces of the query rows, a lane D/32 elements.  What counts is the
// chain of dependent loads (lengths and first steps, then the pieces' m and l,
// then their o), so each link's loads go out together: lane i takes piece i's
// m and l, and the o's of kMany pieces are on their way at once.  With few rows
// the four warps of a CTA share a row's pieces; with many, each takes a row
// (8192 rows of 128: 35 us with four warps a row, 21 with one; 64 rows of 32
// with some 20 pieces: 8 and 15 us).
//
// A slot of the tile kernel (w.half rows twice) holds, for a block of up to
// w.half query rows, the pieces of its two warpgroups, which share the keys.
struct Pieces {
    const float *o;
    const float2 *ml;
    long long step;                       // rows between pieces
    int n;
};
constexpr int kMergeWarps = 4, kMany = 8;

// The pieces of a row, from teams t0 .. t1.
template <int LINES, int D>
__device__ __forceinline__ Pieces pieces_of(const Params &p, const Part &w, const Line &l, int row, int hk, int t0, int t1) {
    Pieces r = {};
    if (l.steps == 0) return r;
    const int rb = row >> w.log_rows, hb = w.n_blocks == 1 ? 0 : hk / w.head_block, hw = hk - hb * w.head_block;
    const Place x = place_of<LINES>(p, w, l, rb, hb);
    const long long at = x.first + t0 * x.step + (w.half ? 0 : (long long)hw * x.apart) + row - (rb << w.log_rows);
    r.o = w.o + at * D;
    r.ml = w.ml + at;
    r.step = x.step;
    r.n = t1 - t0 + 1;
    if (w.half && l.rows - (rb << w.log_rows) <= w.half) {      // two pieces of a team's, one behind the other
        r.step = w.half;
        r.n *= 2;
    }
    return r;
}

template <typename T, int D, bool SHARED>   // SHARED: a row per CTA
__global__ void __launch_bounds__(kMergeWarps * 32)
prefix_merge_kernel(const __grid_constant__ Params p, const __grid_constant__ Part own, const __grid_constant__ Part pre)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = (int)blockIdx.x * (SHARED ? 1 : kMergeWarps) + (SHARED ? 0 : warp), s = blockIdx.y;
    if (h >= p.heads) return;
    const int hk = p.ratio == 1 ? h : h / p.ratio, hr = h - hk * p.ratio;

    // The request's lines: its own and, by the lanes, 32 groups at a time.  A
    // part whose bound is 0 has no launch of its own; its lengths are checked here.
    long long own_begin = 0, own_team = 1, pre_begin = 0, pre_team = 1;
    const Line own_line = line_of<OWN>(p, own, s);
    Line pre_line = {};
    if (own.lines) {
        own_begin = __ldcg(own.line_first + s);
        own_team = __ldcg(own.line_first + own.lines + 1);
    }
    if (pre.lines) pre_team = __ldcg(pre.line_first + pre.lines + 1);
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const bool in = g < p.n_groups && s >= group_first<PREFIX>(p, g) && s < group_first<PREFIX>(p, g + 1);
        const unsigned found = __ballot_sync(0xffffffffu, in);
        if (found) {
            const int mine = g0 + __ffs(found) - 1;
            if (pre.lines) pre_begin = __ldcg(pre.line_first + mine);
            pre_line = line_of<PREFIX>(p, pre, mine);
            break;
        }
    }
    // teams of the first and last step of both segments: four divisions, one in each of four lanes
    const int pre_row = (s - pre_line.first_req) * p.ratio + hr;
    const long long x = segment_begin(own, own_line, hr, hk, own_begin), y = segment_begin(pre, pre_line, pre_row, hk, pre_begin);
    const int k = lane & 3;
    const int team = (int)quotient(max((k < 2 ? x : y) + (k & 1 ? (k < 2 ? own_line.steps : pre_line.steps) - 1 : 0), 0LL),
                                   k < 2 ? own_team : pre_team);
    const Pieces a = pieces_of<OWN, D>(p, own, own_line, hr, hk, __shfl_sync(0xffffffffu, team, 0), __shfl_sync(0xffffffffu, team, 1));
    const Pieces b = pieces_of<PREFIX, D>(p, pre, pre_line, pre_row, hk, __shfl_sync(0xffffffffu, team, 2), __shfl_sync(0xffffffffu, team, 3));

    const int n = a.n + b.n;
    float m = -INFINITY, l = 0.f, o[E];
    bool bad = false;                     // a sum that is no number, also of a piece without a maximum (all its scores are none)
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = 0.f;
    // piece j of the row; with SHARED, this warp's j-th
    auto which = [&](int j) { return SHARED ? j * kMergeWarps + warp : j; };
    for (int j0 = 0; which(j0) < n; j0 += 32) {
        const int j = which(j0 + lane);
        const float2 ml = j < a.n ? __ldcg(a.ml + j * a.step) : j < n ? __ldcg(b.ml + (j - a.n) * b.step) : make_float2(-INFINITY, 0.f);
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
            float x[kMany][E];
#pragma unroll
            for (int k = 0; k < kMany; k++) {
                const int q = which(j0 + k0 + k);
                const float *from = (q < a.n ? a.o + q * a.step * D : b.o + (q - a.n) * b.step * D) + lane;
#pragma unroll
                for (int i = 0; i < E; i++) x[k][i] = q < n ? __ldcg(from + 32 * i) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kMany; k++) {
                // A piece without a valid row has an o that may not have been written; one whose weight is 0
                // because its scores are low still hands on a value that is no number.
                const float w = __shfl_sync(0xffffffffu, rows ? c : -1.f, k0 + k);
#pragma unroll
                for (int i = 0; i < E; i++) o[i] = w >= 0.f ? fmaf(x[k][i], w, o[i]) : o[i];
            }
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    if constexpr (SHARED) {
        __shared__ bool s_bad[kMergeWarps];
        __shared__ float s_m[kMergeWarps], s_l[kMergeWarps], s_o[kMergeWarps][D];
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
        for (int k = 0; k < kMergeWarps; k++) {
            const float c = s_m[k] == -INFINITY ? 0.f : exp2f(s_m[k] - m);
            l += s_l[k] * c;
            bad |= s_bad[k];
#pragma unroll
            for (int i = 0; i < E; i++) o[i] += s_o[k][lane + 32 * i] * c;
        }
    }
    T *out = static_cast<T *>(p.out) + s * p.out_stride + (long long)h * D + lane;
    if (bad) m = l = NAN;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < E; i++) out[32 * i] = from_f32<T>(o[i] * inv);
    if (p.lse && lane == 0) p.lse[(long long)s * p.heads + h] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace prefix
}  // namespace attn

namespace attn_host {

int launch_prefix_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s);

namespace {

// The parts of a call on the workspace `base` (NULL to learn its size).
struct Layout {
    attn::prefix::Part own, pre;
    size_t bytes;
};

Layout lay_out(const attn::prefix::Params &p, int d, int own_rows, int own_keys, int own_grid, int pre_rows, int pre_keys,
               int pre_grid, bool tile, char *base) {
    using namespace attn::prefix;
    Layout r = {};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *at = base ? base + off : nullptr;
        off += (bytes + 255) / 256 * 256;
        return at;
    };
    auto part = [&](Part &w, int lines, int seg_rows, int keys, int grid, bool pre) {
        if (!lines) return;
        divide_part(w, p, lines, seg_rows, keys, grid, pre && tile);
        w.blocks = (p.ratio + seg_rows - 1) / seg_rows;
        const long long all_rows = (long long)p.n_seq * p.ratio;
        w.rows = pre && tile ? seg_rows : (int)std::min<long long>(pre ? all_rows : p.ratio, seg_rows);
        const long long blocks = pre ? all_rows / seg_rows + lines : (long long)lines * w.blocks;
        const size_t slots = (size_t)(blocks * w.n_blocks + w.teams) * w.head_block * w.rows;
        w.line_first = reinterpret_cast<long long *>(take(((size_t)lines + 2) * 8));
        w.ml = reinterpret_cast<float2 *>(take(slots * 8));
        w.o = reinterpret_cast<float *>(take(slots * d * 4));
    };
    part(r.own, p.max_len ? p.n_seq : 0, own_rows, own_keys, own_grid, false);
    part(r.pre, p.max_prefix_len ? p.n_groups : 0, tile ? 256 : pre_rows, tile ? 128 : pre_keys, pre_grid, true);
    r.bytes = std::max<size_t>(off, 256);
    return r;
}

template <class Own, class Pre, int D>
int run(const attn::prefix::Params &p, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    using T = typename Own::Type;
    constexpr int OWN_CTAS = Own::LEAN ? 2 : 1, PRE_CTAS = Pre::LEAN ? 2 : 1;
    // The tensor-core tiles take prefixes of bf16 caches from 32 query rows a
    // group on (counted on average: the groups' sizes are on the device).  A call
    // on an 8192-row prefix in us, warps and tiles, 8 x 128: 24 rows 30.4 and 28.5, 32 rows
    // 32.2 and 29.0, 64 rows 40.2 and 32.0; 16 x 64: 31.9 and 32.1, 33.1 and 32.7, 39.6 and 35.0.
    const bool tile = sizeof(T) == 2 && (D == 64 || D == 128) && p.n_groups &&
                      (long long)p.n_seq * p.ratio >= 32LL * p.n_groups;
    const Layout L = lay_out(p, D, Own::ROWS, Own::KEYS, sm_count_here() * OWN_CTAS, Pre::ROWS, Pre::KEYS,
                             sm_count_here() * (tile ? 1 : PRE_CTAS), tile, static_cast<char *>(ws));
    if (need) { *need = L.bytes; return ATTN_OK; }
    int st;
    if (L.pre.lines && (st = tile ? launch_prefix_tile(p, L.pre, D, s) : run_part<Pre, PREFIX, D, PRE_CTAS>(p, L.pre, 0, s)))
        return st;
    if (L.own.lines && (st = run_part<Own, OWN, D, OWN_CTAS>(p, L.own, L.pre.lines != 0, s))) return st;
    const int rows = p.n_seq * p.heads;
    const bool shared = rows < sm_count_here() * 16;
    return check_pdl(launch_pdl(shared ? prefix_merge_kernel<T, D, true> : prefix_merge_kernel<T, D, false>,
                                dim3(shared ? p.heads : (p.heads + kMergeWarps - 1) / kMergeWarps, p.n_seq), dim3(kMergeWarps * 32), 0, s, p,
                                L.own, L.pre),
                     "prefix_merge_kernel");
}

// Paths by the rows a part has: own rows have ratio of them (more than a path
// holds make more blocks, which read the cache again); a prefix has those of
// its group, counted on average, since the groups' sizes are on the device.
template <class Own, int D>
int run_pre(const attn::prefix::Params &p, void *ws, size_t *need, cudaStream_t s, long long rows) {
    using namespace attn::prefix;
    // As many rows as the registers hold (o takes D NT / 4 of them), where there are more than one tile's.
    // A call on an 8192-row prefix in us, one tile and several: bf16 8 x 128: 8 rows 27.9 and 24.9, 16 rows
    // 27.5 and 26.1, 48 rows 39.0 and 36.4; 16 x 64: 23.3 and 25.0, 25.6 and 29.9, 38.1 and 38.1.  INT8 8 x 128:
    // 4 rows 25.1 and 23.4, 8 rows 24.5 and 24.6, 16 rows 28.4 and 27.2; 16 x 64: 20.3 and 24.9, 22.4 and 26.4,
    // 31.8 and 30.7.  (One tile a piece reads the rows again for each 8, or 4, query rows, from L2 mostly.)
    constexpr bool BF16 = sizeof(typename Own::Type) == 2;
    if constexpr (BF16) {
        if (rows <= 8) return run<Own, Bf16Path<D, 1>, D>(p, ws, need, s);
        return run<Own, Bf16Path<D, D == 32 ? 8 : D == 64 ? 4 : 2>, D>(p, ws, need, s);
    } else {
        if (rows <= 4) return run<Own, I8Path<D, 1>, D>(p, ws, need, s);
        return run<Own, I8Path<D, D <= 64 ? 4 : 2>, D>(p, ws, need, s);
    }
}
template <class Own, int D>
int run_pre_f32(const attn::prefix::Params &p, void *ws, size_t *need, cudaStream_t s, long long rows) {
    using namespace attn::prefix;
    // 4 rows a piece and 8, in us on an 8192-row prefix: 12 x 128: 4 rows 43.6 and 36.4, 5 rows 55.2 and 36.7;
    // 16 x 64: 31.1 and 33.0, 37.2 and 33.0
    if (rows <= 4) return run<Own, F32Path<D, 4>, D>(p, ws, need, s);
    return run<Own, F32Path<D, 8>, D>(p, ws, need, s);
}

template <int D>
int run_d(const attn::prefix::Params &p, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    const long long rows = p.n_groups ? ((long long)p.n_seq * p.ratio + p.n_groups - 1) / p.n_groups : 0;
    if (kv_dtype == ATTN_BF16)
        return p.ratio <= 8 ? run_pre<Bf16Path<D, 1>, D>(p, ws, need, s, rows) : run_pre<Bf16Path<D, 2>, D>(p, ws, need, s, rows);
    // INT8: two rows fill a tile of digits (8192 own rows of 8 x 128: 110 us a call, 116 in f16 parts; 32 x 32: 173 and 188)
    if (kv_dtype == ATTN_I8)
        return p.ratio <= 2   ? run_pre<I8Digits<D>, D>(p, ws, need, s, rows)
               : p.ratio <= 4 ? run_pre<I8Path<D, 1>, D>(p, ws, need, s, rows)
                              : run_pre<I8Path<D, 2>, D>(p, ws, need, s, rows);
    // fp32: FMAs grow with the rows, so own rows take the request's
    if (p.ratio == 1) return run_pre_f32<F32Path<D, 1>, D>(p, ws, need, s, rows);
    if (p.ratio == 2) return run_pre_f32<F32Path<D, 2>, D>(p, ws, need, s, rows);
    if (p.ratio <= 4) return run_pre_f32<F32Path<D, 4>, D>(p, ws, need, s, rows);
    return run_pre_f32<F32Path<D, 8>, D>(p, ws, need, s, rows);
}

int run_any(const attn::prefix::Params &p, int d, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    switch (d) {
        case 32: return run_d<32>(p, kv_dtype, ws, need, s);
        case 64: return run_d<64>(p, kv_dtype, ws, need, s);
        case 96: return run_d<96>(p, kv_dtype, ws, need, s);
        default: return run_d<128>(p, kv_dtype, ws, need, s);
    }
}

}  // namespace

size_t prefix_decode_workspace(const attn_prefix_shape *s, int kv_dtype) {
    attn::prefix::Params p = {};
    p.n_seq = s->n_seq; p.n_groups = s->n_groups; p.heads = s->heads; p.kv_heads = s->kv_heads;
    p.ratio = s->heads / s->kv_heads;
    p.max_len = s->max_len; p.max_prefix_len = s->max_prefix_len;
    size_t need = 0;
    run_any(p, s->head_dim, kv_dtype, nullptr, &need, nullptr);
    return need;
}

int launch_prefix_decode(const attn::prefix::Params &p, int d, int kv_dtype, void *ws, cudaStream_t s) {
    return run_any(p, d, kv_dtype, ws, nullptr, s);
}

}  // namespace attn_host
