// prefix_tile_sm100.cu -- the prefix part of attn_prefix_decode_ex, and the
// prefixes and contexts of attn_tree_decode_ex, on the Blackwell tensor cores,
// for bf16 caches whose groups (or drafts) have many query rows (query tokens x
// query heads per key head).
//
// With r rows a prefix costs r flops per byte, so past about 250 rows the
// tensor cores bound it and not HBM; mma.sync, at a quarter of their rate,
// already from 64 (two 32768-row prefixes of 512 rows each, 8 x 128, called with
// one own row a request: 174 us, merge included: 742 TFLOP/s; 957 us on mma.sync
// with probabilities in one part).  The times in brackets below were taken with
// one part too, when the same call took 143 us.
//
// One CTA per SM walks its range of steps (prefix.cuh) of 128 keys.  A piece has
// up to 256 query rows: with more than 128, warpgroup w takes rows [128 w, 128 w + 128)
// of every step; with fewer, both take the same rows and every other step, and
// each leaves a state of its own.  12 warps:
//   warp 0      K rows, warp 1 V rows.  With pages of 8 rows or more a step is a
//               TMA box of 64 dims for each page that there is (or 128 rows of
//               one), a lane per box; a page's rows behind the line's last key
//               come with it.  In K's place keys without a row hold those, or what
//               was there before: it is the scores that are masked, by the key
//               masks that the K warp leaves, and they have to be.  In V's place
//               the warp writes zeros over them before it reports the half (K or V
//               of a step), so that a probability of 0 never meets a NaN.
//               With smaller pages the lanes copy 16 bytes each into the same
//               128-byte swizzled layout, zeros for keys without a row, and
//               report a half when their next one is on its way.
//               (All steps by lanes: 299 us, the copying instructions setting the pace.)
//               The K warp walks and tells the others the pieces through a queue.
//   warp 2      S_wu = Q_w K_u^T for the two halves u of a step's keys, M = 128,
//               N = 64, both operands in shared memory
//   warp 3      O_w += P_wu V_u (P in two bf16 parts from TMEM, V as it lies, MN-major)
//   warps 4-7   softmax of warpgroup 0, warps 8-11 of warpgroup 1: a warp
//               brings 32 query rows in, a thread keeps the maximum and sum of its row
//               (a TMEM lane), writes its probabilities to TMEM, and rescales O when the maximum grew by
//               more than 2^8 (a stale one leaves P <= 256, and the piece's
//               (m, l, o) stay consistent).  All exponentials on MUFU: lse is an
//               output.
// A probability goes in as two bf16 parts, its rounding and the rest, which leaves
// no error but that of rounding the output (one part: 1.4 times it).  The second
// product and its packing took that call from 143 to 174 us.
// TMEM: four S of 64 columns, each overwritten by the two parts of its P, and two
// O (512 columns at d 128).  S_w1 is formed while S_w0 is in the softmax, so a warpgroup does
// not wait for its own products.  (With 128 keys in one S per warpgroup the
// chain softmax, PV, next S took 5,300 cycles a step, of which the exponentials
// of both warpgroups are 2,048; with P in halves but S in one product 171 us, the
// warpgroup waiting for its last PV and the S after it.  One warp for both products
// in a fixed order: 217 us, its own instructions and waits take 1,730 cycles a pair;
// four, one per product and warpgroup: no faster than two.)
//
// The instruction cache sets a limit of its own: the roles run different code
// side by side, and what is unrolled only for convenience (a piece's end, the
// lanes' copies, a copy of the products for each warpgroup where one piece
// takes turns) cost 465 us, and 366 with one copy each, on 256 contexts of up to
// 2000 rows with 16 drafts of four heads.  So did a warp that divided the pieces into a stream
// for each warpgroup, with its own 300 instructions a step: slower by a fifth.
//
// Every wait is bounded; a timeout records a code in the device error word and
// raises a CTA-wide flag, on which all roles fall through to the teardown.
#include <algorithm>
#include <cudaTypedefs.h>

#include "prefix.cuh"
#include "sm100.cuh"

namespace attn {
namespace ptile {

using namespace sm100;
using namespace prefix;

constexpr int BM = 128, BN = 128, BH = 64;   // query rows; keys of a step, of an S
constexpr int kThreads = 384;
constexpr int kMasks = 8;                 // steps whose key masks are kept: more than K's ring holds, and the ones at work
// Pieces of which the K warp has told the others: it is as many ahead of them as K's ring has slots, and two.  (Each warp
// walking by itself kept the walk's state in the softmax's registers, which spilled: 8 % on the long prefixes of drafts.)
constexpr int kQueue = 16;
struct __align__(16) Queued { long long at; int a, b, first_req, row0, rows, hb, apart; };       // rows 0: no more

template <int D>
struct Cfg {
    // rings of K and V tiles (V waits longer for its use); one ring for both would be ambiguous to parity
    // waits once one of the two copying warps runs ahead of the other
    static constexpr int KS = D == 64 ? 4 : 2, VS = D == 64 ? 4 : 3, SLOTS = KS + VS;
    static constexpr int TILE = BM * D * 2;                   // Q tile, K or V tile: D / 64 blocks of 128 rows x 128 bytes
    // The places of two query tiles, each also of what both warpgroups turn over of O (16 KB a warpgroup)
    static constexpr int QTILE = TILE > 32768 ? TILE : 32768;
    static constexpr int OFF_KV = 2 * QTILE;
    static constexpr int OFF_BAR = OFF_KV + SLOTS * TILE;
    static constexpr int OFF_MASK = OFF_BAR + 416;           // (barriers, the TMEM address, the abort flag)
    static constexpr int OFF_QUEUE = OFF_MASK + kMasks * 16;
    static constexpr int SMEM = OFF_QUEUE + kQueue * (int)sizeof(Queued) + 1024;
    static_assert(SMEM <= 232448, "shared memory of a CTA");
};
// TMEM columns
__device__ __forceinline__ uint32_t col_s(int wg, int u) { return (uint32_t)(wg * 2 + u) * BH; }
template <int D> __device__ __forceinline__ uint32_t col_o(int wg) { return 4 * BH + (uint32_t)wg * D; }

enum {
    B_QF = 0, B_QE = 1,                   // Q there; its last S finished
    B_OF = 2,                             // per warpgroup: O read out
    B_SF = 4, B_PF = 8, B_OD = 12,        // per warpgroup and half (2 w + u): S ready; P written; PV finished
    B_FULL = 16, B_FREE = 24,             // per slot: copied; used
    B_VE = 32,                            // a step's V rows that come as some boxes are there
    B_TD = 33,                            // a piece's O is out: the query tiles' places are free of it
    B_PQ = 34,                            // per place of the queue: a piece is there
    B_COUNT = B_PQ + kQueue
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Place of 16-byte piece ch of row r in a tile: block of 64 dims, row, piece XOR row % 8.
__device__ __forceinline__ uint32_t tile_at(int r, int ch) {
    return (uint32_t)((ch / 8) * BM * 128 + r * 128 + (((ch % 8) ^ (r & 7)) << 4));
}

template <int D, int LINES>
__global__ void __launch_bounds__(kThreads, 1)
prefix_tile_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ Params p, const __grid_constant__ Part w, int boxes)
{
    using C = Cfg<D>;
    constexpr int CPR = D / 8;            // 16-byte pieces of a row
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sb = smem_raw + (base - raw);
    const uint32_t sQ = base, sKV = base + C::OFF_KV, bar0 = base + C::OFF_BAR;
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
    static_assert(8 * B_COUNT <= 400, "barriers");
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sb + C::OFF_BAR + 400);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sb + C::OFF_BAR + 404);
    volatile uint32_t *masks = reinterpret_cast<volatile uint32_t *>(sb + C::OFF_MASK);   // [step % kMasks][4]: keys with a row

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(BAR(B_QF), 256);
        mbar_init(BAR(B_QE), 1);
        mbar_init(BAR(B_VE), 1);
        mbar_init(BAR(B_TD), 256);
        for (int i = 0; i < kQueue; i++) mbar_init(BAR(B_PQ + i), 1);
        for (int i = 0; i < 2; i++) mbar_init(BAR(B_OF + i), 128);
        for (int i = 0; i < 4; i++) {
            mbar_init(BAR(B_SF + i), 2);
            mbar_init(BAR(B_PF + i), 128);
            mbar_init(BAR(B_OD + i), 1);
        }
        for (int s = 0; s < C::SLOTS; s++) {
            mbar_init(BAR(B_FULL + s), 32);
            mbar_init(BAR(B_FREE + s), 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    // The own rows' launch may start once this one's CTAs have all seen the work before them finished.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // (the sums lie where the query rows come after the next barrier)
    long long *sums = reinterpret_cast<long long *>(sb);
    static_assert((kEntries + 1 + 32) * 8 <= 2 * C::QTILE, "sums in the query tiles");
    const long long of_team = sum_lines<LINES>(p, w, sums, sums + kEntries + 1);
    Walk<LINES> walk(p, w, sums, of_team, (int)blockIdx.x);      // (of the copying warps)
    volatile Queued *queue = reinterpret_cast<volatile Queued *>(sb + C::OFF_QUEUE);
    Queued x;
    // Piece k, for the other warps; false where there is none, or on a timeout.
    auto piece = [&](int k, Queued &y) {
        const bool ok = mbar_wait(BAR(B_PQ + k % kQueue), (k / kQueue) & 1, abort_flag, p.err, 0x805);
        if (!__all_sync(0xffffffffu, ok)) return false;
        const volatile Queued &q = queue[k % kQueue];
        y.at = q.at; y.a = q.a; y.b = q.b; y.first_req = q.first_req; y.row0 = q.row0; y.rows = q.rows; y.hb = q.hb; y.apart = q.apart;
        return y.rows > 0;
    };
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // 384 x 168 registers at launch: 128 x 88 + 256 x 208
    if (warp < 4) regs_dec<88>();
    if (warp < 2) {
        // ------------------------------------------------------------ K, V
        const int kv = warp;
        const CUtensorMap *map = kv ? &tv : &tk;
        if (lane == 0) prefetch_tmap(map);
        int due = -1;                     // slot of a half that is on its way and not reported
        int edges = 0;                    // halves of V that came as some boxes
        bool boxed = false;               // the due half is one of them, without the keys `absent`
        unsigned absent[4];
        bool ok = true;
        auto flush = [&] {
            if (due < 0) return;
            if (boxed) {
                // zeros for the keys without a row, over what a page holds behind its last key: a probability of 0
                // must not meet a NaN
                ok = ok && mbar_wait(BAR(B_VE), edges & 1, abort_flag, p.err, 0x804);
                ok = __all_sync(0xffffffffu, ok);
                edges++;
                if (!ok) return;
                const uint32_t to = sKV + due * C::TILE;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (!absent[i]) continue;
                    for (int r = lane / CPR; r < 32; r += 32 / CPR)
                        if (absent[i] >> r & 1)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to + tile_at(32 * i + r, lane % CPR)), "r"(0) : "memory");
                }
                boxed = false;
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            fence_async_smem();           // this thread's copies, for the tensor cores
            mbar_arrive(BAR(B_FULL + due));
            due = -1;
        };
        constexpr int RPI = 32 / CPR;     // rows per copy instruction
        const int lr = lane / CPR, ch = lane % CPR;
        auto tell = [&](int k, const Piece &x, int rows) {
            if (kv == 0 && lane == 0) {
                volatile Queued &q = queue[k % kQueue];
                q.at = x.at; q.a = x.a; q.b = x.b; q.first_req = x.first_req; q.row0 = x.row0; q.rows = rows; q.hb = x.hb; q.apart = x.apart;
                mbar_arrive(BAR(B_PQ + k % kQueue));
            }
        };
        int g = 0, k = 0;                 // steps, pieces
        Piece x;
        for (; ok && walk.next(x); k++) {
            tell(k, x, x.rows);
            const __nv_bfloat16 *from = static_cast<const __nv_bfloat16 *>(kv ? p.v : p.k) + (long long)x.hb * D + ch * 8;
            // cache rows of a step's 128 keys (-1: none), four per lane, read a step ahead
            int next[4];
            auto look_up = [&](int j) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = j * BN + 32 * i + lane;
                    next[i] = j < x.b && t < x.keys ? (int)cache_row(p, x.table, t) : -1;
                }
            };
            look_up(x.a);
            for (int j = x.a; j < x.b; j++, g++) {
                int row[4];
                unsigned valid[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    row[i] = next[i];
                    valid[i] = __ballot_sync(0xffffffffu, next[i] >= 0);
                }
                look_up(j + 1);
                const bool whole = (valid[0] & valid[1] & valid[2] & valid[3]) == 0xffffffffu;
                const int ring = kv ? C::VS : C::KS, slot = kv ? C::KS + g % C::VS : g % C::KS;
                const uint32_t to = sKV + slot * C::TILE;
                if (g >= ring) {
                    flush();              // nothing may stay due behind the wait
                    if (!ok) break;
                    ok = mbar_wait(BAR(B_FREE + slot), (g / ring + 1) & 1, abort_flag, p.err, 0x801 + kv);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                }
                if (kv == 0 && lane == 0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) masks[g % kMasks * 4 + i] = valid[i];
                }
                __syncwarp();
                if (boxes) {
                    // A box for each page that there is (its first key's row): of K as it comes, since scores of keys
                    // without a row are masked; of V, where some have none, with zeros in their place before it is reported
                    const int rows = BN / boxes, key = lane * rows & 127;     // of lane n's box
                    int r = -1;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int y = __shfl_sync(0xffffffffu, row[i], key & 31);
                        if (key >> 5 == i) r = y;
                    }
                    const bool mine = lane < boxes && r >= 0, edge = kv && !whole;
                    const int bytes = __popc(__ballot_sync(0xffffffffu, mine)) * rows * D * 2;
                    if (edge) flush();
                    if (!ok) break;
                    const uint32_t bar = edge ? BAR(B_VE) : BAR(B_FULL + slot);
                    if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                    else if (!edge) mbar_arrive(bar);
                    __syncwarp();
                    if (mine) {
#pragma unroll
                        for (int d = 0; d < D / 64; d++)
                            tma_load_3d(to + d * BN * 128 + key * 128, map, bar, x.hb * D + 64 * d, r, 0);
                    }
                    __syncwarp();
                    if (edge) {
                        due = slot;
                        boxed = true;
#pragma unroll
                        for (int i = 0; i < 4; i++) absent[i] = ~valid[i];
                    }
                    continue;
                }
                flush();
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll 1
                    for (int r0 = 0; r0 < 32; r0 += RPI) {
                        const int r = __shfl_sync(0xffffffffu, row[i], r0 + lr);
                        copy16(to + tile_at(32 * i + r0 + lr, ch), from + (long long)max(r, 0) * p.row_stride, r >= 0);
                    }
                asm volatile("cp.async.commit_group;" ::: "memory");
                due = slot;
            }
        }
        x = {};
        tell(k, x, 0);
        if (ok) flush();
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 2) {
        // ------------------------------------------------------------ S = Q K^T
        const bool leader = elect_one();
        auto wait = [&](int b, int parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(BAR(b), parity & 1, abort_flag, p.err, code));
        };
        constexpr uint32_t id = idesc_bf16(BM, BH, 0, 0);
        int g = 0, t[2] = {0, 0};         // steps; steps per warpgroup
        bool ok = true;
        int place = 0;                    // of a single query tile (as in the softmax)
        bool single = false;
        for (int k = 0; ok && piece(k, x); k++) {
            const bool two = x.rows > BM;
            place = !two && single ? 1 - place : 0;
            single = !two;
            if (!(ok = wait(B_QF, k, 0x811))) break;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int slot = g % C::KS;
                if (!(ok = wait(B_FULL + slot, g / C::KS, 0x812))) break;
                auto half = [&](int wg, int u) {
                    const int b = 2 * wg + u;
                    // the product that reads this half's last P is done
                    const int mine = wg ? t[1] : t[0];
                    if (mine > 0 && !(ok = wait(B_OD + b, mine - 1, 0x813 + b))) return;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t qd = sw128_desc(sQ + (two ? wg : place) * C::QTILE, 16, 1024);
                        const uint64_t kd = sw128_desc(sKV + slot * C::TILE + u * BH * 128, 16, 1024);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {   // 32 bytes on per step, a block of 16 KB on per 64 dims
                            const uint32_t off = (kk / 4) * (BM * 128 >> 4) + (kk % 4) * 2;
                            mma_bf16_ss(tmem + col_s(wg, u), qd + off, kd + off, id, kk > 0);
                        }
                        mma_commit(BAR(B_SF + b));
                        mbar_arrive(BAR(B_SF + b));               // (hands on the copying warps' masks)
                    }
                    __syncwarp();
                    if (u == 1) {
                        if (wg) t[1]++;
                        else t[0]++;
                    }
                };
                if (two) {
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        if (ok) half(n & 1, n >> 1);
                } else {                  // (one copy of the code: the SM's instruction cache is short of room)
#pragma unroll 1
                    for (int u = 0; ok && u < 2; u++) half((j - x.a) & 1, u);
                }
                if (!ok) break;
                if (leader) {
                    mma_commit(BAR(B_FREE + slot));
                    if (j == x.b - 1) mma_commit(BAR(B_QE));
                }
                __syncwarp();
            }
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ O += P V
        const bool leader = elect_one();
        auto wait = [&](int b, int parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(BAR(b), parity & 1, abort_flag, p.err, code));
        };
        constexpr uint32_t id = idesc_bf16(BM, D, 0, 1);
        int g = 0, t[2] = {0, 0}, done[2] = {0, 0};   // steps; steps and pieces per warpgroup
        bool ok = true;
        for (int k = 0; ok && piece(k, x); k++) {
            const bool two = x.rows > BM;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int slot = C::KS + g % C::VS;
                if (!(ok = wait(B_FULL + slot, g / C::VS, 0x821))) break;
                auto half = [&](int wg, int u) {
                    const int b = 2 * wg + u;
                    const bool first = u == 0 && j - x.a < (two ? 1 : 2);   // of this warpgroup in this piece
                    const int mine = wg ? t[1] : t[0], pieces = wg ? done[1] : done[0];
                    if (first && pieces > 0 && !(ok = wait(B_OF + wg, pieces - 1, 0x822 + wg))) return;
                    if (!(ok = wait(B_PF + b, mine, 0x824 + b))) return;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = sw128_desc(sKV + slot * C::TILE + u * BH * 128, BM * 128, 1024);
#pragma unroll
                        for (int kk = 0; kk < 2 * BH / 16; kk++)  // 16 keys: 8 columns of a part of P, 2 KB of V
                            mma_bf16_ts(tmem + col_o<D>(wg), tmem + col_s(wg, u) + kk * 8, vd + 128 * (kk % (BH / 16)), id, !first || kk > 0);
                        mma_commit(BAR(B_OD + b));
                    }
                    __syncwarp();
                    if (u == 1) {
                        if (wg) t[1]++;
                        else t[0]++;
                    }
                };
                if (two) {
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        if (ok) half(n & 1, n >> 1);
                } else {
#pragma unroll 1
                    for (int u = 0; ok && u < 2; u++) half((j - x.a) & 1, u);
                }
                if (!ok) break;
                if (leader) mma_commit(BAR(B_FREE + slot));
                __syncwarp();
            }
            done[0]++;
            if (two || x.b - x.a > 1) done[1]++;
        }
    } else {
        // ------------------------------------------------------------ softmax
        regs_inc<208>();
        const int wg = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), tO = lanes + col_o<D>(wg);
        int g = 0, t = 0;                 // steps of the CTA; of this warpgroup
        bool ok = true;
        // the warp's 32 query rows of a piece, CPR lanes a row, to the tile at `place`
        // (a lane to a row, 16 bytes of 32 rows an instruction, took 2.5 us instead of 1.1)
        auto copy_queries = [&](const Queued &y, int place) {
            constexpr int RPI = 32 / CPR;
            const int r = y.rows > BM ? wg * BM + row : row, at = y.row0 + min(r, y.rows - 1);
            const int s = y.first_req + at / p.ratio, h = y.hb * p.ratio + at % p.ratio;
            const long long from = s * p.q_stride + (long long)h * D;
#pragma unroll 4
            for (int r0 = 0; r0 < 32; r0 += RPI) {
                const int n = r0 + lane / CPR, to = quad * 32 + n, ch = lane % CPR;
                const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.q) + __shfl_sync(0xffffffffu, from, n) + 8 * ch;
                copy16(sQ + place * C::QTILE + tile_at(to, ch), src, r - row + to < y.rows);
            }
        };
        auto queries_there = [&] {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            mbar_arrive(BAR(B_QF));
        };
        // Query tiles.  A piece of more than 128 rows has both places, warpgroup w place w, for its queries and later its
        // O.  A smaller one has one place, whose queries warpgroup 0 brings in for both; where two such pieces follow one
        // another they take turns, so the second one's queries come while the first one's O goes out.
        int place = 0;
        bool ahead = false;               // x's queries have come with the piece before
        bool more = piece(0, x);
        for (int k = 0; ok && more; k++) {
            const bool two = x.rows > BM;
            if (!ahead) {
                if (two || wg == 0) copy_queries(x, two ? wg : place);
                queries_there();
            }
            const int mine = two ? x.rows - wg * BM : x.rows;     // query rows of this warpgroup
            const bool idle = quad * 32 >= mine;                  // none of them in this warp: it only keeps step
            float m = -INFINITY, l = 0.f;
            bool any = false, ready = false;
            for (int j = x.a; ok && j < x.b; j++) {
                if (!two && ((j - x.a) & 1) != wg) continue;
#pragma unroll 1
                for (int u = 0; u < 2; u++) {
                    const int b = 2 * wg + u;
                    const uint32_t tS = lanes + col_s(wg, u);
                    if (!__all_sync(0xffffffffu, ready)) {
                        ok = mbar_wait(BAR(B_SF + b), t & 1, abort_flag, p.err, 0x831 + u);
                        if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    }
                    tc_fence_after();
                    if (!idle) {
                        uint32_t s[BH];
#pragma unroll
                        for (int q = 0; q < BH / 32; q++) {
                            uint32_t tt[32];
                            tmem_ld32(tS + 32 * q, tt);
#pragma unroll
                            for (int c = 0; c < 32; c++) s[32 * q + c] = tt[c];
                        }
                        uint32_t valid[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) valid[i] = masks[(g + j - x.a) % kMasks * 4 + 2 * u + i];
                        tmem_wait_ld();
                        if ((valid[0] & valid[1]) != 0xffffffffu) {
#pragma unroll
                            for (int c = 0; c < BH; c++)
                                if (!(valid[c >> 5] >> (c & 31) & 1)) s[c] = __float_as_uint(-INFINITY);
                        }
                        float mp[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) mp[i] = -INFINITY;
#pragma unroll
                        for (int c = 0; c < BH; c += 2)
                            mp[(c >> 1) & 3] = max3(mp[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                        const float mx = fmaxf(max3(mp[0], mp[1], mp[2]), mp[3]) * p.scale_log2;
                        float alpha = 1.f;
                        const bool grow = mx > m + 8.f;           // also at the first half with a key
                        if (grow) {
                            alpha = ex2(m - mx);
                            m = mx;
                            l *= alpha;
                        }
                        const float neg = m == -INFINITY ? 0.f : -m;
                        const uint64_t scale2 = f2(p.scale_log2, p.scale_log2), neg2 = f2(neg, neg);
                        uint64_t l2[4] = {0ull, 0ull, 0ull, 0ull};
                        uint32_t hi[32], lo[32];
#pragma unroll
                        for (int c = 0; c < 32; c++) {
                            float e, f;
                            f2_split(fma2(f2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, neg2), e, f);
                            e = ex2(e);
                            f = ex2(f);
                            l2[c & 3] = add2(l2[c & 3], f2(e, f));
                            bf16_parts(e, f, hi[c], lo[c]);
                        }
                        {
                            float e, f;
                            f2_split(add2(add2(l2[0], l2[1]), add2(l2[2], l2[3])), e, f);
                            l += e + f;
                        }
                        tmem_st32(tS, hi);                        // over S, which is in registers
                        tmem_st32(tS + 32, lo);
                        if (__any_sync(0xffffffffu, any && grow)) {
                            // O is the previous half's product's until that is done
                            ok = mbar_wait(BAR(B_OD + 2 * wg + 1 - u), (t - 1 + u) & 1, abort_flag, p.err, 0x833 + u);
                            if (!(ok = __all_sync(0xffffffffu, ok))) break;
                            tc_fence_after();
                            uint32_t o[32];
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                tmem_ld32(tO + c0, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int c = 0; c < 32; c++) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                                tmem_st32(tO + c0, o);
                            }
                        }
                        // the next half's S, looked for while P is on its way to TMEM (P in one part: 143 us so, 146.5 after it)
                        ready = mbar_test_wait(BAR(B_SF + 2 * wg + 1 - u), (t + u) & 1);
                        tmem_wait_st();
                        tc_fence_before();
                    }
                    mbar_arrive(BAR(B_PF + b));
                    any = true;
                }
                t++;
            }
            if (!ok) break;
            g += x.b - x.a;
            Queued y;                     // the next piece
            more = piece(k + 1, y);
            ahead = more && !two && y.rows <= BM;
            if (ahead && wg == 0) {
                // the other place: warpgroup 1 has taken O of the piece before this one out through it
                ok = k == 0 || mbar_wait(BAR(B_TD), (k - 1) & 1, abort_flag, p.err, 0x837);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                copy_queries(y, 1 - place);
            }
            ok = mbar_wait(BAR(B_QE), k & 1, abort_flag, p.err, 0x830);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            if (ahead && wg == 1) mbar_arrive(BAR(B_QF));     // (behind the queries of this piece, which QE followed)
            // The piece: this warpgroup's half of the slot.  A warp turns 32 dims of its 32 rows
            // over in what was the place of their queries and writes them 128 bytes at a time.
            // (Each thread writing its own row, 512 bytes apart: 6.4 us from a piece's last P to the next piece, 3.4 so.)
            const long long at = x.at + wg * x.apart + row;
            if (any) {
                ok = mbar_wait(BAR(B_OD + 2 * wg), (t - 1) & 1, abort_flag, p.err, 0x835) &&
                     mbar_wait(BAR(B_OD + 2 * wg + 1), (t - 1) & 1, abort_flag, p.err, 0x836);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
            }
            if (ahead && wg == 0) queries_there();
            if (any) {
                tc_fence_after();
                if (!idle) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(tO + c0, o);
                        tmem_wait_ld();
                        float4 *turn = reinterpret_cast<float4 *>(sb + (two ? wg * C::QTILE : place * C::QTILE + wg * 16384) + quad * 32 * 128);
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            turn[lane * 8 + (c ^ (lane & 7))] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]),
                                                                            __uint_as_float(o[4 * c + 2]), __uint_as_float(o[4 * c + 3]));
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int r = 4 * i + lane / 8, c = lane % 8;
                            const float4 f = turn[r * 8 + (c ^ (r & 7))];
                            if (quad * 32 + r < mine)
                                *reinterpret_cast<float4 *>(w.o + (at - lane + r) * D + c0 + 4 * c) = f;
                        }
                        __syncwarp();
                    }
                    tc_fence_before();
                }
                mbar_arrive(BAR(B_OF + wg));      // the next piece's first product may overwrite O
            }
            if (row < mine) w.ml[at] = make_float2(m, l);
            mbar_arrive(BAR(B_TD));
            // both places next: the other warpgroup may still be taking its O out through this one's
            if (more && !two && y.rows > BM) {
                ok = mbar_wait(BAR(B_TD), k & 1, abort_flag, p.err, 0x838);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
            }
            place = ahead ? 1 - place : 0;
            x = y;
        }
    }

    // ---------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // let what is in flight finish before the CTA releases its memory
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
#undef BAR
}

}  // namespace ptile
}  // namespace attn

namespace attn_host {

bool ensure_smem_attr(const void *func, size_t bytes);

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
        return nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
}

// {key heads x D, rows} of a bf16 cache in boxes of 64 dims x `box` rows, 128-byte swizzle.
static bool cache_map(CUtensorMap *m, const void *ptr, int cols, long long rows, long long stride, int box) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
    const cuuint64_t strides[2] = {(cuuint64_t)stride * 2, (cuuint64_t)stride * 2 * (cuuint64_t)rows};
    const cuuint32_t extent[3] = {64, (cuuint32_t)box, 1}, steps[3] = {1, 1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, extent, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int LINES>
static int launch_d(const attn::prefix::Params &p, const attn::prefix::Part &w, cudaStream_t s) {
    using namespace attn::ptile;
    if (!ensure_smem_attr((const void *)prefix_tile_kernel<D, LINES>, Cfg<D>::SMEM))
        return set_error(ATTN_ERR_CUDA, "prefix decode: cannot set shared-memory size");
    // A step is BN / box boxes; a box of the swizzled layout begins on 8 rows.
    CUtensorMap tk = {}, tv = {};
    const int box = std::min(1 << p.log_page, BN);
    const long long rows = (long long)p.n_pages << p.log_page;
    const bool maps = box >= 8 && cache_map(&tk, p.k, p.kv_heads * D, rows, p.row_stride, box) &&
                      cache_map(&tv, p.v, p.kv_heads * D, rows, p.row_stride, box);
    return check_pdl(launch_pdl(prefix_tile_kernel<D, LINES>, dim3(w.teams), dim3(kThreads), Cfg<D>::SMEM, s, tk, tv, p, w,
                                maps ? BN / box : 0),
                     "prefix_tile_kernel");
}

int launch_prefix_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s) {
    return d == 64 ? launch_d<64, attn::prefix::PREFIX>(p, w, s) : launch_d<128, attn::prefix::PREFIX>(p, w, s);
}
int launch_tree_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s) {
    return d == 64 ? launch_d<64, attn::prefix::TREES>(p, w, s) : launch_d<128, attn::prefix::TREES>(p, w, s);
}

}  // namespace attn_host
