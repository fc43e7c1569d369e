// prefix_rows.cuh -- the kernel in which each warp takes its pieces of the work
// by itself (the paths of prefix_paths.cuh), and the layout of a part's pieces,
// for attn_prefix_decode_ex and attn_tree_decode_ex.
#pragma once
#include <algorithm>

#include "prefix.cuh"
#include "prefix_paths.cuh"

namespace attn {
namespace prefix {

constexpr int kWarps = 8;

// One warp's piece: steps [a, b) of a line for the query rows of one block and
// one key head.  The ring holds SLOTS halves of steps (K, V, K, ...): AHEAD
// whole steps are in flight beside the half at work.
template <class Path, int SLOTS>
__device__ __forceinline__ void run_piece(const Params &p, uint32_t ring, const int *table, int keys, int a, int b,
                                          int first_req, int row0, int rows, int hk, float *o, float2 *ml) {
    static_assert(SLOTS % 2 == 1 && SLOTS >= 3, "ring");
    constexpr int AHEAD = SLOTS / 2;
    constexpr unsigned all = Path::KEYS == 32 ? 0xffffffffu : (1u << (Path::KEYS & 31)) - 1;
    const int lane = threadIdx.x & 31;
    const bool runs = p.log_page >= 4;
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
    bool next_valid;
    int next_row = row_of(a, next_valid), row = 0;
    path.place(p, hk);
    unsigned masks[AHEAD + 1];            // keys with a row, of this step and the ones in flight
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    auto copy_k = [&](int step, int slot) {
        row = next_row;
        if (step < b) {
            if (runs) path.template copy_k<true>(p, ring + slot * Path::SLOT, row);
            else path.template copy_k<false>(p, ring + slot * Path::SLOT, row);
        }
        commit();
        const unsigned mask = __ballot_sync(0xffffffffu, next_valid);
        next_row = row_of(step + 1, next_valid);
        return mask;
    };
    auto copy_v = [&](int step, int slot) {
        if (step < b) {
            if (runs) path.template copy_v<true>(p, ring + slot * Path::SLOT, row);
            else path.template copy_v<false>(p, ring + slot * Path::SLOT, row);
        }
        commit();
    };
    auto wait = [] {
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
        __syncwarp();                     // every lane's copies of the half are there
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        masks[i] = copy_k(a + i, 2 * i);
        copy_v(a + i, 2 * i + 1);
    }
    path.begin(p, ring + SLOTS * Path::SLOT, first_req, row0, rows, hk);      // the queries, behind the first copies
    int at = 0;                           // slot of this step's K
    for (int step = a; step < b; step++) {
        const int after = at + 1 == SLOTS ? 0 : at + 1, before = at ? at - 1 : SLOTS - 1;
        masks[AHEAD] = copy_k(step + AHEAD, before);
        wait();
        if (masks[0] == all) path.template scores<false>(p, ring + at * Path::SLOT, all);
        else path.template scores<true>(p, ring + at * Path::SLOT, masks[0]);
        __syncwarp();                     // K's slot may be copied over
        copy_v(step + AHEAD, at);
        wait();
        if (masks[0] == all) path.template values<false>(p, ring + after * Path::SLOT, all);
        else path.template values<true>(p, ring + after * Path::SLOT, masks[0]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < AHEAD; i++) masks[i] = masks[i + 1];
        at = after + 1 == SLOTS ? 0 : after + 1;
    }
    path.finish(o, ml, rows);
}

// Slots of a warp's ring: as many (an odd number) as CTAS rings of WARPS fit an SM, up to 7.
template <class Path, int CTAS, int WARPS> struct Ring {
    static constexpr int FIT = ((CTAS == 1 ? 216 : 108) * 1024 / WARPS - Path::SCRATCH) / Path::SLOT;
    static constexpr int SLOTS = FIT > 7 ? 7 : (FIT - 1) / 2 * 2 + 1;
    static constexpr int BYTES = SLOTS * Path::SLOT + Path::SCRATCH;
    static_assert(Path::SLOT % 128 == 0 && Path::SCRATCH % 128 == 0, "swizzled rows begin on 128 bytes");
};

// `second`: the launch before this one is the prefix part's, which has waited
// for the work before it when this one may start; the two run side by side, and
// this one ends after both.
template <class Path, int LINES, int D, int CTAS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
prefix_rows_kernel(const __grid_constant__ Params p, const __grid_constant__ Part w, int second)
{
    using R = Ring<Path, CTAS, WARPS>;
    extern __shared__ __align__(128) uint8_t ring_bytes[];
    __shared__ long long sums[kEntries + 1];
    __shared__ long long warp_sums[32];
    if (!second) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const long long of_team = sum_lines<LINES>(p, w, sums, warp_sums);
    const int warp = threadIdx.x >> 5;
    const uint32_t ring = sm100::smem_u32(ring_bytes) + warp * R::BYTES;
    const int team_warp = warp % w.head_block, team = warp / w.head_block * (int)gridDim.x + (int)blockIdx.x;
    Walk<LINES> walk(p, w, sums, of_team, team);
    for (Piece x; walk.next(x);) {
        const int hk = x.hb * w.head_block + team_warp;
        if (hk >= p.kv_heads) continue;
        const long long at = x.at + (long long)team_warp * x.apart;
        run_piece<Path, R::SLOTS>(p, ring, x.table, x.keys, x.a, x.b, x.first_req, x.row0, x.rows, hk,
                                  w.o + at * D, w.ml + at);
    }
    if (second) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace prefix
}  // namespace attn

namespace attn_host {

int sm_count_here();
bool ensure_smem_attr(const void *func, size_t bytes);

// Divides a part among the teams of `grid` CTAs: key heads per team, query rows of a block, keys of a step.
inline void divide_part(attn::prefix::Part &w, const attn::prefix::Params &p, int lines, int seg_rows, int keys, int grid, bool tile,
                        int warps = attn::prefix::kWarps) {
    using namespace attn::prefix;
    w.lines = lines;
    w.per_entry = (lines + kEntries - 1) / kEntries;
    w.entries = (lines + w.per_entry - 1) / w.per_entry;
    // Key heads per team: adjacent ones, in blocks that leave as few of a CTA's warps idle as may be.
    int best = 0;
    for (int n = tile ? p.kv_heads : (p.kv_heads + warps - 1) / warps; n <= p.kv_heads; n++) {
        const int block = (p.kv_heads + n - 1) / n, splits = tile ? 1 : warps / block;
        const int used = p.kv_heads * splits * 1000 / n;          // warps at work, in thousandths
        if (used <= best) continue;
        best = used;
        w.n_blocks = n;
        w.head_block = block;
        w.splits = splits;
    }
    w.teams = grid * w.splits;
    w.log_rows = __builtin_ctz((unsigned)seg_rows);
    w.log_keys = __builtin_ctz((unsigned)keys);
    w.half = tile ? 128 : 0;
}

template <class Path, int LINES, int D, int CTAS, int WARPS = attn::prefix::kWarps>
int run_part(const attn::prefix::Params &p, const attn::prefix::Part &w, int second, cudaStream_t s) {
    using namespace attn::prefix;
    using R = Ring<Path, CTAS, WARPS>;
    const auto kernel = prefix_rows_kernel<Path, LINES, D, CTAS, WARPS>;
    const int warps = w.splits * w.head_block;
    if (!ensure_smem_attr((const void *)kernel, (size_t)R::BYTES * WARPS))
        return set_error(ATTN_ERR_CUDA, "paged decode: cannot set shared-memory size");
    return check_pdl(launch_pdl(kernel, dim3(w.teams / w.splits), dim3(warps * 32), (size_t)R::BYTES * warps, s, p, w, second),
                     "prefix_rows_kernel");
}

}  // namespace attn_host
