// prefix_decode.cu -- attn_prefix_decode_ex: one query token per request over
// the rows that its group shares and its own, both in a paged cache.
//
// With keys j over prefix and own rows, out = sum_j p_j v_j / sum_j p_j and
// p_j = 2^(x_j - m), x_j = scale log2(e) q.k_j, m = max_j x_j.  Any split of
// the keys gives triples (m, l, o) that join exactly: with M = max m_i,
// l = sum l_i 2^(m_i - M) and o likewise.
//
// Work.  A "line" is one page-table line: a group's prefix, with the query
// rows of all its requests, or a request's own rows, with its heads/kv_heads
// query rows per key head.  A segment is a line x a block of query rows x a
// block of key heads; its keys are counted in steps of KEYS.  All steps of all
// segments, in order, are cut into equal ranges, one per team of warps, so no
// length decides how busy an SM is; a team's warps take one key head each and
// read adjacent parts of the same cache rows.  What a warp leaves of a segment
// (its piece) goes to the workspace, at slot segment + team, and
// prefix_merge_kernel joins the pieces of each query row.
//
// Bound: HBM (the cache rows, once).  Little else may cost: each warp
// copies its rows through a ring of its own in shared memory, from which the
// lanes read them in the layout that the arithmetic takes (prefix_paths.cuh),
// and meets no other warp until the merge.
#include <algorithm>

#include "prefix.cuh"
#include "prefix_paths.cuh"

namespace attn {
namespace prefix {

constexpr int kEntries = 2048;            // running sums of steps kept per CTA
constexpr int kWarps = 8;

struct Work {
    float *own_o, *pre_o;                 // pieces: [slot][heads of the block][rows][D]
    float2 *own_ml, *pre_ml;              //         [slot][heads of the block][rows] (m in base 2, l)
    long long *line_first;                // first step of each line, and the total
    int lines, per_entry;                 // lines, lines per entry of the running sums
    int pre_lines;                        // prefix lines this kernel takes (0 or n_groups)
    int head_block, n_blocks;             // key heads per team, teams' blocks
    int splits;                           // teams per CTA
    int own_blocks;                       // blocks of query rows of an own line
    int own_rows, pre_rows;               // rows of a slot
    int own_seg_rows, pre_seg_rows;       // rows of a block
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Blocks of query rows of a group, and the index of its first one: an
// ascending numbering without a sum over the groups before.
__device__ __forceinline__ void group_blocks(const Params &p, const Work &w, int g, int &first_req, int &rows,
                                             int &blocks, int &base) {
    first_req = group_first(p, g);
    rows = max(group_first(p, g + 1) - first_req, 0) * p.ratio;
    blocks = ceil_div(rows, w.pre_seg_rows);
    base = first_req * p.ratio / w.pre_seg_rows + g;
}

struct Line {
    int keys, steps, blocks;              // blocks of query rows
    __device__ long long total(const Work &w) const { return (long long)steps * blocks * w.n_blocks; }
};
template <int OWN_KEYS, int PRE_KEYS>
__device__ __forceinline__ Line line_of(const Params &p, const Work &w, int i) {
    Line l;
    if (i < w.pre_lines) {
        int first, rows, base;
        group_blocks(p, w, i, first, rows, l.blocks, base);
        l.keys = rows ? prefix_len(p, i) : 0;
        l.steps = ceil_div(l.keys, PRE_KEYS);
    } else {
        l.keys = own_len(p, i - w.pre_lines);
        l.blocks = w.own_blocks;
        l.steps = ceil_div(l.keys, OWN_KEYS);
    }
    return l;
}

// One warp's piece: steps [a, b) of a line for the query rows of one block and
// one key head.
template <class Path, int STAGES>
__device__ __forceinline__ void run_piece(const Params &p, uint32_t ring, const int *table, int keys, int a, int b,
                                          int first_req, int row0, int rows, int hk, float *o, float2 *ml) {
    const int lane = threadIdx.x & 31;
    Path path;
    // Cache row of this lane's key of a step: bad pages and keys past the line
    // have no valid row.  In pages of 16 rows or more, a run of 16 keys is
    // copied from its first key's row, which keys past the line do not decide.
    auto row_of = [&](int step, bool &valid) {
        const int t = step * Path::KEYS + lane;
        valid = lane < Path::KEYS && t < keys && step < b;
        int row = 0;
        if (valid) {
            const long long r = cache_row(p, table, t);
            valid = r >= 0;
            row = max((int)r, 0);
        }
        return row;
    };
    unsigned masks[STAGES];               // keys with a row, of the steps in flight
    bool next_valid;
    int next_row = row_of(a, next_valid);
    path.begin(p, first_req, row0, rows, hk);
    auto issue = [&](int step, int stage) {
        masks[stage] = __ballot_sync(0xffffffffu, next_valid);
        if (step < b) {
            if (p.log_page >= 4) path.template issue<true>(p, ring + stage * Path::STAGE, next_row);
            else path.template issue<false>(p, ring + stage * Path::STAGE, next_row);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next_row = row_of(step + 1, next_valid);
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) issue(a + i, i);
    constexpr unsigned all = Path::KEYS == 32 ? 0xffffffffu : (1u << (Path::KEYS & 31)) - 1;
    for (int step = a; step < b; step += STAGES) {
#pragma unroll
        for (int u = 0; u < STAGES; u++) {
            if (step + u < b) {
                issue(step + u + STAGES - 1, (u + STAGES - 1) % STAGES);
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
                __syncwarp();             // every lane's copies of the stage are there
                const uint32_t st = ring + u * Path::STAGE;
                if (masks[u] == all) path.template compute<false>(p, st, all);
                else path.template compute<true>(p, st, masks[u]);
                __syncwarp();             // the stage may be copied over
            }
        }
    }
    path.finish(o, ml, rows);
}

// Stages of a warp's ring: as many as fit a CTA's shared memory, up to 6.
template <class Own, class Pre> struct Ring {
    static constexpr int STAGE = Own::STAGE > Pre::STAGE ? Own::STAGE : Pre::STAGE;
    static constexpr int FIT = (208 * 1024 / kWarps) / STAGE;
    static constexpr int STAGES = FIT > 4 ? 4 : FIT;
    static constexpr int BYTES = STAGES * STAGE;
    static_assert(STAGES >= 2 && Own::STAGE % 128 == 0 && Pre::STAGE % 128 == 0, "ring");
};

template <class Own, class Pre, int D>
__global__ void __launch_bounds__(kWarps * 32, 1)
prefix_rows_kernel(const __grid_constant__ Params p, const __grid_constant__ Work w)
{
    using R = Ring<Own, Pre>;
    extern __shared__ __align__(128) uint8_t ring_bytes[];
    __shared__ long long sums[kEntries + 1];
    __shared__ long long warp_sums[kWarps];
    pdl_begin();                          // launched by launch_pdl

    // running sums of the steps, per entry of w.per_entry lines
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int entries = ceil_div(w.lines, w.per_entry);
    long long carry = 0;
    for (int e0 = 0; e0 < entries; e0 += (int)blockDim.x) {
        const int e = e0 + threadIdx.x;
        long long v = 0;
        if (e < entries)
            for (int i = e * w.per_entry; i < min((e + 1) * w.per_entry, w.lines); i++)
                v += line_of<Own::KEYS, Pre::KEYS>(p, w, i).total(w);
        long long s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        if (lane == 31) warp_sums[warp] = s;
        __syncthreads();
        long long before = carry;
        for (int i = 0; i < (int)blockDim.x / 32; i++) {
            if (i < warp) before += warp_sums[i];
            carry += warp_sums[i];
        }
        if (e < entries) sums[e + 1] = before + s;
        __syncthreads();
    }
    if (threadIdx.x == 0) sums[0] = 0;
    __syncthreads();
    const long long total = entries ? sums[entries] : 0;
    if (blockIdx.x == 0) {                // for the merge
        for (int e = threadIdx.x; e < entries; e += blockDim.x) {
            long long at = sums[e];
            for (int i = e * w.per_entry; i < min((e + 1) * w.per_entry, w.lines); i++) {
                w.line_first[i] = at;
                at += line_of<Own::KEYS, Pre::KEYS>(p, w, i).total(w);
            }
        }
        if (threadIdx.x == 0) w.line_first[w.lines] = total;
    }

    // this team's range
    const uint32_t ring = sm100::smem_u32(ring_bytes) + warp * R::BYTES;
    const int team_warp = warp % w.head_block, split = warp / w.head_block;
    // no more teams than steps, so that none between a segment's first and last is without a piece
    const int teams = (int)min((long long)gridDim.x * w.splits, total), team = split * (int)gridDim.x + (int)blockIdx.x;
    if (split >= w.splits || team >= teams) return;
    const long long first = total * team / teams, last = total * (team + 1) / teams;
    int e;
    {
        int lo = 0, hi = entries;         // the last entry that begins at or before `first`
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sums[mid] <= first) lo = mid;
            else hi = mid;
        }
        e = lo;
    }
    long long at = sums[e];
    for (int i = e * w.per_entry; i < w.lines && at < last; i++) {
        const Line l = line_of<Own::KEYS, Pre::KEYS>(p, w, i);
        const long long n = l.total(w);
        if (at + n > first && n > 0) {
            // segments of the line that the range meets
            const int s0 = (int)((max(first, at) - at) / l.steps), s1 = (int)((min(last, at + n) - 1 - at) / l.steps);
            for (int s = s0; s <= s1; s++) {
                const long long begin = at + (long long)s * l.steps;
                const int a = (int)(max(first, begin) - begin), b = (int)(min(last, begin + l.steps) - begin);
                const int rb = s / w.n_blocks, hb = s - rb * w.n_blocks;
                const int hk = hb * w.head_block + team_warp;
                if (hk >= p.kv_heads) continue;
                if (i < w.pre_lines) {
                    int req, rows, blocks, base;
                    group_blocks(p, w, i, req, rows, blocks, base);
                    const long long slot =
                        ((long long)(base + rb) * w.n_blocks + hb + team) * w.head_block + team_warp;
                    run_piece<Pre, R::STAGES>(p, ring, p.prefix_table + (long long)i * p.max_prefix_pages, l.keys, a, b, req,
                                   rb * w.pre_seg_rows, min(rows - rb * w.pre_seg_rows, w.pre_seg_rows), hk,
                                   w.pre_o + slot * w.pre_rows * D, w.pre_ml + slot * w.pre_rows);
                } else {
                    const int req = i - w.pre_lines;
                    const long long slot =
                        (((long long)req * w.own_blocks + rb) * w.n_blocks + hb + team) * w.head_block + team_warp;
                    run_piece<Own, R::STAGES>(p, ring, p.block_table + (long long)req * p.max_pages, l.keys, a, b, req,
                                   rb * w.own_seg_rows, min(p.ratio - rb * w.own_seg_rows, w.own_seg_rows), hk,
                                   w.own_o + slot * w.own_rows * D, w.own_ml + slot * w.own_rows);
                }
            }
        }
        at += n;
    }
}

// Joins the pieces of one query row: a CTA per (request, query head), its
// warps taking the pieces in turn, a lane D/32 elements.
struct Pieces {
    const float *o;
    const float2 *ml;
    long long step;                       // rows between pieces
    int n;
};
constexpr int kMergeWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32)
prefix_merge_kernel(const __grid_constant__ Params p, const __grid_constant__ Work w, int all_teams, int own_keys, int pre_keys)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int E = D / 32;
    __shared__ float s_m[kMergeWarps], s_l[kMergeWarps], s_o[kMergeWarps][D];
    const int s = blockIdx.y, h = blockIdx.x, hk = h / p.ratio, hr = h - hk * p.ratio;
    const int hb = hk / w.head_block, hw = hk - hb * w.head_block;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long total = w.line_first[w.lines];
    const long long teams = min((long long)all_teams, total);
    // the team whose range [total t / teams, total (t + 1) / teams) holds a step
    auto team_of = [&](long long step) { return (int)(((step + 1) * teams - 1) / total); };
    auto find = [&](int line, int seg_in_line, long long seg, int keys, int keys_per_step, int rows, int row,
                    const float *o, const float2 *ml) {
        Pieces r = {};
        const int steps = ceil_div(keys, keys_per_step);
        if (steps == 0) return r;
        const long long begin = w.line_first[line] + (long long)seg_in_line * steps;
        const int t0 = team_of(begin), t1 = team_of(begin + steps - 1);
        const long long slot = ((seg + t0) * w.head_block + hw) * rows + row;
        r.o = o + slot * D;
        r.ml = ml + slot;
        r.step = (long long)w.head_block * rows;
        r.n = t1 - t0 + 1;
        return r;
    };
    const int rb = hr / w.own_seg_rows;
    Pieces part[2];
    part[0] = find(w.pre_lines + s, rb * w.n_blocks + hb, ((long long)s * w.own_blocks + rb) * w.n_blocks + hb,
                   own_len(p, s), own_keys, w.own_rows, hr - rb * w.own_seg_rows, w.own_o, w.own_ml);
    part[1] = Pieces{};
    for (int g = 0; g < w.pre_lines; g++) {
        int req, rows, blocks, base;
        group_blocks(p, w, g, req, rows, blocks, base);
        if (s < req || (s - req) * p.ratio >= rows) continue;
        const int row = (s - req) * p.ratio + hr, b = row / w.pre_seg_rows;
        part[1] = find(g, b * w.n_blocks + hb, (long long)(base + b) * w.n_blocks + hb, prefix_len(p, g), pre_keys,
                       w.pre_rows, row - b * w.pre_seg_rows, w.pre_o, w.pre_ml);
        break;
    }
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const Pieces &r = part[k];
        for (int j = warp; j < r.n; j += kMergeWarps) {
            const float2 ml = __ldcg(r.ml + j * r.step);
            float x[E];
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = __ldcg(r.o + j * r.step * D + lane + 32 * i);
            if (ml.x == -INFINITY) continue;          // no valid row in this piece
            const float mx = fmaxf(m, ml.x), a = exp2f(m - mx), c = exp2f(ml.x - mx);
            l = l * a + ml.y * c;
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = o[i] * a + x[i] * c;
            m = mx;
        }
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < E; i++) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float M = s_m[0];
#pragma unroll
    for (int i = 1; i < kMergeWarps; i++) M = fmaxf(M, s_m[i]);
    float c[kMergeWarps], L = 0.f;
#pragma unroll
    for (int i = 0; i < kMergeWarps; i++) {
        c[i] = s_m[i] == -INFINITY ? 0.f : exp2f(s_m[i] - M);
        L += s_l[i] * c[i];
    }
    if (threadIdx.x < D) {
        float r = 0.f;
#pragma unroll
        for (int i = 0; i < kMergeWarps; i++) r += s_o[i][threadIdx.x] * c[i];
        static_cast<T *>(p.out)[s * p.out_stride + (long long)h * D + threadIdx.x] =
            from_f32<T>(M == -INFINITY ? 0.f : r / L);
    }
    if (p.lse && threadIdx.x == 0)
        p.lse[(long long)s * p.heads + h] = M == -INFINITY ? -INFINITY : (M + log2f(L)) * kLn2;
}

}  // namespace prefix
}  // namespace attn

namespace attn_host {

int sm_count_here();
bool ensure_smem_attr(const void *func, size_t bytes);

namespace {

struct Layout {
    attn::prefix::Work w;
    int grid_ctas;
    size_t bytes;
};

// The workspace of a call, on `base` (NULL to learn its size).
Layout lay_out(int n_seq, int n_groups, int ratio, int kv_heads, int d, int own_seg_rows, int pre_seg_rows, int ctas,
               char *base) {
    using namespace attn::prefix;
    Layout r = {};
    Work &w = r.w;
    w.pre_lines = n_groups;
    w.lines = n_groups + n_seq;
    w.per_entry = std::max(1, (w.lines + kEntries - 1) / kEntries);
    w.n_blocks = (kv_heads + kWarps - 1) / kWarps;
    w.head_block = (kv_heads + w.n_blocks - 1) / w.n_blocks;
    w.splits = kWarps / w.head_block;
    w.own_seg_rows = own_seg_rows;
    w.pre_seg_rows = pre_seg_rows;
    w.own_blocks = (ratio + own_seg_rows - 1) / own_seg_rows;
    w.own_rows = std::min(ratio, own_seg_rows);
    w.pre_rows = (int)std::min<long long>((long long)n_seq * ratio, pre_seg_rows);
    r.grid_ctas = ctas;
    const long long teams = (long long)ctas * w.splits;
    const long long own_slots = ((long long)n_seq * w.own_blocks * w.n_blocks + teams) * w.head_block * w.own_rows;
    const long long pre_segs = n_groups ? (long long)n_seq * ratio / pre_seg_rows + n_groups : 0;
    const long long pre_slots = n_groups ? (pre_segs * w.n_blocks + teams) * w.head_block * w.pre_rows : 0;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *at = base ? base + off : nullptr;
        off += (bytes + 255) / 256 * 256;
        return at;
    };
    w.line_first = reinterpret_cast<long long *>(take(((size_t)w.lines + 1) * 8));
    w.own_ml = reinterpret_cast<float2 *>(take((size_t)own_slots * 8));
    w.pre_ml = reinterpret_cast<float2 *>(take((size_t)pre_slots * 8));
    w.own_o = reinterpret_cast<float *>(take((size_t)own_slots * d * 4));
    w.pre_o = reinterpret_cast<float *>(take((size_t)pre_slots * d * 4));
    r.bytes = off;
    return r;
}

template <class Own, class Pre, typename T, int D>
int run(const attn::prefix::Params &p, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    const Layout L = lay_out(p.n_seq, p.n_groups, p.ratio, p.kv_heads, D, Own::ROWS, Pre::ROWS,
                             sm_count_here(), static_cast<char *>(ws));
    if (need) { *need = L.bytes; return ATTN_OK; }
    const int warps = L.w.splits * L.w.head_block;
    const size_t smem = (size_t)Ring<Own, Pre>::BYTES * warps;
    if (!ensure_smem_attr((const void *)prefix_rows_kernel<Own, Pre, D>, (size_t)Ring<Own, Pre>::BYTES * kWarps))
        return set_error(ATTN_ERR_CUDA, "prefix decode: cannot set shared-memory size");
    int st = check_pdl(launch_pdl(prefix_rows_kernel<Own, Pre, D>, dim3(L.grid_ctas), dim3(warps * 32), smem, s, p, L.w),
                       "prefix_rows_kernel");
    if (st) return st;
    return check_pdl(launch_pdl(prefix_merge_kernel<T, D>, dim3(p.heads, p.n_seq), dim3(kMergeWarps * 32), 0, s, p, L.w,
                                L.grid_ctas * L.w.splits, (int)Own::KEYS, (int)Pre::KEYS),
                     "prefix_merge_kernel");
}

template <int D>
int run_d(const attn::prefix::Params &p, int kv_dtype, void *ws, size_t *need, cudaStream_t s) {
    using namespace attn::prefix;
    // Tiles of query rows per warp: own rows as the request needs (more rows
    // than two tiles hold make more blocks); for a prefix, K and V are read
    // again for every block, so as many as the registers hold (o takes D NT / 4).
    if (kv_dtype == ATTN_BF16) {
        constexpr int N = D == 32 ? 8 : D == 64 ? 4 : 2;
        return p.ratio <= 8 ? run<Bf16Path<D, 1>, Bf16Path<D, N>, __nv_bfloat16, D>(p, ws, need, s)
                            : run<Bf16Path<D, 2>, Bf16Path<D, N>, __nv_bfloat16, D>(p, ws, need, s);
    }
    if (kv_dtype == ATTN_I8) {
        constexpr int N = D <= 64 ? 4 : 2;
        return p.ratio <= 4 ? run<I8Path<D, 1>, I8Path<D, N>, float, D>(p, ws, need, s)
                            : run<I8Path<D, 2>, I8Path<D, N>, float, D>(p, ws, need, s);
    }
    // own rows with the request's query rows, up to 8 at a time; prefixes with 8
    if (p.ratio == 1) return run<F32Path<D, 1>, F32Path<D, 8>, float, D>(p, ws, need, s);
    if (p.ratio == 2) return run<F32Path<D, 2>, F32Path<D, 8>, float, D>(p, ws, need, s);
    if (p.ratio <= 4) return run<F32Path<D, 4>, F32Path<D, 8>, float, D>(p, ws, need, s);
    return run<F32Path<D, 8>, F32Path<D, 8>, float, D>(p, ws, need, s);
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
    size_t need = 0;
    run_any(p, s->head_dim, kv_dtype, nullptr, &need, nullptr);
    return need;
}

int launch_prefix_decode(const attn::prefix::Params &p, int d, int kv_dtype, void *ws, cudaStream_t s) {
    return run_any(p, d, kv_dtype, ws, nullptr, s);
}

}  // namespace attn_host
