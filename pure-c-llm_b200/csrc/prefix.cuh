// prefix.cuh -- what the kernels of attn_prefix_decode_ex and
// attn_tree_decode_ex share: the call's arguments on the device, and the walk
// through a page table.
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
    // attn_tree_decode_ex (n_seq: query tokens, of n_req requests)
    const int *row_begin, *ctx_lens;                  // first query token of each request; rows before its drafts
    const uint32_t *masks;
    int n_req, max_nodes, mask_words;
};

__device__ __forceinline__ int checked_len(const Params &p, int len, int most) {
    if (len < 0 || len > most) {
        atomicExch(p.err, 0x703);
        return len < 0 ? 0 : most;
    }
    return len;
}
__device__ __forceinline__ int own_len(const Params &p, int s) { return checked_len(p, __ldg(p.lens + s), p.max_len); }
// What the lines of a part are: the requests' own rows, each with one query
// token; the groups' prefixes; or the groups' prefixes and then the requests'
// contexts, of requests with several query tokens (drafts).
enum Lines { OWN, PREFIX, TREES };

// first query token of request r, within [0, n_seq]
__device__ __forceinline__ int row_first(const Params &p, int r) { return min(max(__ldg(p.row_begin + r), 0), p.n_seq); }
// first query token of group g, within [0, n_seq]
template <int LINES>
__device__ __forceinline__ int group_first(const Params &p, int g) {
    if constexpr (LINES == TREES) return row_first(p, min(max(__ldg(p.group_begin + g), 0), p.n_req));
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

// ---------------------------------------------------------------------------
// The division of the work (prefix_decode.cu describes it)
// ---------------------------------------------------------------------------
constexpr int kEntries = 512;             // running sums of steps kept per CTA

// a / b for a >= 0, b > 0: mostly in 32 bits, where a division is a quarter of
// the instructions (the starts of the kernels are chains of them)
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
constexpr int kBegin = 1;                 // steps that the beginning and end of a segment count for
// TREES by tiles: a step of more than 128 query rows costs that many of fewer,
// and so does a segment's beginning and end (256 contexts of 1000 rows behind
// two prefixes of 8192, in one run: 1147 us; with costs of 1.5 and 3 1193, of 2.5
// and 3 1261, of 2 and 5 1154.  Runs and boxes range from 1126 to 1216).
constexpr int kFullStep = 2, kTileBegin = 3;

// One part of the work.
struct Part {
    float *o;                             // pieces: [slot][heads of the block][rows][D]
    float2 *ml;                           //         [slot][heads of the block][rows] (m in base 2, l)
    long long *line_first;                // first step of each line, the total, and the steps of a team
    int lines, per_entry, entries;        // lines, lines per entry of the running sums, entries
    int head_block, n_blocks;             // key heads per team, their blocks
    int splits, teams;                    // teams per CTA, in all
    int blocks;                           // blocks of query rows of an own line
    int log_rows, rows;                   // query rows of a block (2^log_rows), of a slot
    int log_keys;                         // keys of a step (2^log_keys)
    int half;                             // see Pieces (0: one piece per slot)
    // TREES: rows of the prefixes' pieces; for the join, each query token's request and group (-1: none), and each
    // line's first query token, query rows and keys
    long long after;
    int2 *row_of;
    int4 *line_info;
};

__device__ __forceinline__ int ceil_shift(int a, int log_b) { return (a + (1 << log_b) - 1) >> log_b; }

// Query rows of line i, the query tokens [first, next), and their blocks, and
// the index of the first block: an ascending numbering without a sum over the
// lines before.
__device__ __forceinline__ void line_blocks(const Params &p, const Part &w, int i, int first, int next, int &rows,
                                            int &blocks, int &base) {
    rows = max(next - first, 0) * p.ratio;
    blocks = ceil_shift(rows, w.log_rows);
    base = (first * p.ratio >> w.log_rows) + i;
}

struct Line {
    int keys, steps, blocks;              // blocks of query rows
    int first_req, rows, base;            // of the line's query rows (first query token); index of its first block
    bool prefix;                          // TREES
    int weight = 1, begin = kBegin;       // cost of a step, and of a segment's beginning and end
    // cost of a segment, and of the line
    __host__ __device__ int cost() const { return steps * weight + begin; }
    __device__ long long total(const Part &w) const { return steps ? (long long)cost() * blocks * w.n_blocks : 0; }
};
// First step of a query row's segment in the order of all steps (by their
// costs), for a row of the line that begins at line_begin; 0 in a part that the
// call does not have.
__host__ __device__ __forceinline__ long long segment_begin(const Part &w, const Line &l, int row, int hk, long long line_begin) {
    if (!w.lines) return 0;
    const int rb = row >> w.log_rows, hb = w.n_blocks == 1 ? 0 : hk / w.head_block;
    return line_begin + (long long)(rb * w.n_blocks + hb) * l.cost() + l.begin;
}
// Steps and costs of a line with its query tokens' rows and keys.
template <int LINES>
__device__ __forceinline__ void line_steps(const Part &w, Line &l) {
    l.steps = ceil_shift(l.keys, w.log_keys);
    if (LINES == TREES && w.half) {
        l.weight = l.rows > w.half ? kFullStep : 1;
        l.begin = kTileBegin;
    }
}
template <int LINES>
__device__ __forceinline__ Line line_of(const Params &p, const Part &w, int i) {
    Line l;
    l.prefix = LINES == PREFIX || (LINES == TREES && i < p.n_groups);
    if (l.prefix) {
        const int len = __ldg(p.prefix_lens + i);            // on its way with the group's bounds
        l.first_req = group_first<LINES>(p, i);
        line_blocks(p, w, i, l.first_req, group_first<LINES>(p, i + 1), l.rows, l.blocks, l.base);
        l.keys = l.rows ? checked_len(p, len, p.max_prefix_len) : 0;
    } else if (LINES == TREES) {
        const int r = i - p.n_groups, len = __ldg(p.ctx_lens + r);
        l.first_req = row_first(p, r);
        line_blocks(p, w, r, l.first_req, row_first(p, r + 1), l.rows, l.blocks, l.base);
        l.keys = l.rows ? checked_len(p, len, p.max_len) : 0;
    } else {
        l.first_req = i;
        l.rows = p.ratio;
        l.blocks = w.blocks;
        l.base = i * w.blocks;
        l.keys = own_len(p, i);
    }
    line_steps<LINES>(w, l);
    return l;
}
// TREES: request s's query tokens are told the request and its group (ascending: by bisection).
__device__ __forceinline__ void tell_rows(const Params &p, const Part &w, int s) {
    int lo = 0, hi = p.n_groups;          // the last group that begins at or before s
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.group_begin + mid) <= s) lo = mid;
        else hi = mid;
    }
    const bool in = p.n_groups && __ldg(p.group_begin + lo) <= s && s < __ldg(p.group_begin + lo + 1);
    for (int r = row_first(p, s), end = row_first(p, s + 1); r < end; r++) w.row_of[r] = make_int2(s, in ? lo : -1);
}

// Running sums of the lines' costs, one per entry of w.per_entry lines, in
// sums[0 .. entries], by all threads of the CTA; CTA 0 also writes each line's
// own for the merge.  Returns the steps of a team: team t takes steps
// [t n, (t + 1) n), so none between a segment's first and last is without a
// piece, and a step's team is one division.
template <int LINES>
__device__ __forceinline__ long long sum_lines(const Params &p, const Part &w, long long *sums, long long *warp_sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int entries = w.entries;
    if constexpr (LINES == TREES) {
        for (int s = (int)(blockIdx.x + gridDim.x * threadIdx.x); s < p.n_req; s += (int)(gridDim.x * blockDim.x)) tell_rows(p, w, s);
    }
    long long carry = 0;
    for (int e0 = 0; e0 < entries; e0 += (int)blockDim.x) {
        const int e = e0 + threadIdx.x;
        long long v = 0;
        if (e < entries)
            for (int i = e * w.per_entry; i < min((e + 1) * w.per_entry, w.lines); i++)
                v += line_of<LINES>(p, w, i).total(w);
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
    // (no fewer than a step costs: else a team between a segment's first and last would be without one)
    const long long of_team = max(quotient(total + w.teams - 1, w.teams), LINES == TREES ? (long long)kFullStep : 1LL);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < entries; e += blockDim.x) {
            long long at = sums[e];
            for (int i = e * w.per_entry; i < min((e + 1) * w.per_entry, w.lines); i++) {
                const Line l = line_of<LINES>(p, w, i);
                w.line_first[i] = at;
                if constexpr (LINES == TREES) w.line_info[i] = make_int4(l.first_req, l.rows, l.keys, 0);
                at += l.total(w);
            }
        }
        if (threadIdx.x == 0) {
            w.line_first[w.lines] = total;
            w.line_first[w.lines + 1] = of_team;
        }
    }
    return of_team;
}

// Steps [a, b) of a segment: keys of a page-table line against query rows
// [row0, row0 + rows) of the line, for block hb of key heads.
struct Piece {
    const int *table;
    long long at;                         // its first row on the workspace
    int keys, a, b, first_req, row0, rows, hb;
    int apart;                            // rows between its key heads' states, or its two halves (Part::half)
};

// Where the pieces of a segment lie on the workspace: team t's at row
// first + t * step, `apart` rows for each key head of the block (tiles: for
// each of the two halves).  As segments and teams ascend together, no two
// pieces meet.
//   OWN, PREFIX: slots of w.rows rows for each key head.
//   TREES: a request's few rows would leave most of a slot empty, so its
//   pieces take as many rows as they have, behind those of the tokens before.
//   With half, where a block of up to w.half rows has two states, a prefix
//   takes w.half rows more for that, and a request's rows count twice.
struct Place { long long first, step; int apart; };
template <int LINES>
__host__ __device__ __forceinline__ Place place_of(const Params &p, const Part &w, const Line &l, int rb, int hb) {
    Place x;
    x.step = (long long)w.head_block * w.rows;
    if constexpr (LINES != TREES) {
        x.first = ((long long)(l.base + rb) * w.n_blocks + hb) * x.step;
        x.apart = w.half ? w.half : w.rows;
        return x;
    }
    const int left = l.rows - (rb << w.log_rows), rows = left < 1 << w.log_rows ? left : 1 << w.log_rows;
    const long long row = (long long)l.first_req * p.ratio + (rb << w.log_rows);
    const int times = w.half && rows <= w.half ? 2 : 1;
    x.apart = w.half && times == 1 ? w.half : rows;
    const long long before = l.prefix ? row + (long long)w.half * (l.base - (l.first_req * p.ratio >> w.log_rows)) : row * (w.half ? 2 : 1);
    x.first = (l.prefix ? 0 : w.after) + (before * w.n_blocks + (long long)hb * rows * times) * w.head_block;
    return x;
}

// The pieces of team `team`'s range.
template <int LINES>
struct Walk {
    const Params &p;
    const Part &w;
    long long first = 0, last = 0, at = 0;
    int i = 0, s = 0, s1 = -1, team;
    Line l;

    __device__ __forceinline__ Walk(const Params &p_, const Part &w_, const long long *sums, long long of_team, int team_)
        : p(p_), w(w_), team(team_) {
        l.steps = l.blocks = 0;
        const long long total = w.entries ? sums[w.entries] : 0;
        first = of_team * team;
        last = min(first + of_team, total);
        if (first >= last) {
            last = 0;
            return;
        }
        int lo = 0, hi = w.entries;       // the last entry that begins at or before `first`
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sums[mid] <= first) lo = mid;
            else hi = mid;
        }
        i = lo * w.per_entry - 1;
        at = sums[lo];
    }
    __device__ __forceinline__ bool next(Piece &x) {
        while (true) {
            while (s > s1) {              // the next line that the range meets, and its segments in the range
                at += l.total(w);
                if (++i >= w.lines || at >= last) { i = w.lines; at = last; l.steps = 0; return false; }
                l = line_of<LINES>(p, w, i);
                const long long n = l.total(w);
                s = 0;
                s1 = -1;
                if (n > 0 && at + n > first) {
                    s = first > at ? (int)quotient(first - at, l.cost()) : 0;
                    s1 = last < at + n ? (int)quotient(last - 1 - at, l.cost()) : l.blocks * w.n_blocks - 1;
                }
            }
            // a step is the team's that its first unit of cost is
            const long long begin = at + (long long)s * l.cost() + l.begin;
            x.a = (int)(max(first, begin) - begin);
            x.b = (int)(min(last, begin + (long long)l.steps * l.weight) - begin);
            if (LINES == TREES && l.weight > 1) {
                x.a = (x.a + l.weight - 1) / l.weight;
                x.b = (x.b + l.weight - 1) / l.weight;
            }
            const int rb = w.n_blocks == 1 ? s : s / w.n_blocks;
            x.hb = s - rb * w.n_blocks;
            s++;
            if (x.a >= x.b) continue;     // the range holds the segment's beginning alone
            const Place at = place_of<LINES>(p, w, l, rb, x.hb);
            x.at = at.first + team * at.step;
            x.apart = at.apart;
            x.table = l.prefix ? p.prefix_table + (long long)i * p.max_prefix_pages
                               : p.block_table + (long long)(LINES == TREES ? i - p.n_groups : i) * p.max_pages;
            x.keys = l.keys;
            x.first_req = l.first_req;
            x.row0 = rb << w.log_rows;
            x.rows = min(l.rows - x.row0, 1 << w.log_rows);
            return true;
        }
    }
};

}  // namespace prefix
}  // namespace attn
