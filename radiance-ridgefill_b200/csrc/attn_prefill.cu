/* attn_prefill.cu -- ridgefill_attn_prefill: causal attention of packed prompts on B200 (ridgefill_serve.h holds the
 * formula): the exact rows of a prompt (all of them, or the tail) over its keys, grouped heads, head dim 256.
 *
 * Tensor-bound: 4 D flops a (row, key) pair and query head. S = Q K^T and O = P V run on tcgen05 over CTA pairs
 * (cta_group::2): 256 rows x 128 keys x 256 and 256 x 256 x 128 a key tile, 2,048 cycles at the full rate together. The
 * pair halves what each SM's shared memory carries: one CTA alone would read 192 KiB of operands and take in 128 KiB of
 * copies a key tile, 2,500 cycles of its 128 bytes a cycle; a CTA of a pair reads 128 KiB and takes in 64 KiB. The
 * exponentials, 16,384 a CTA and tile at 16 a cycle, take another pipe 1,024 cycles beside them.
 *
 * A CTA's 128 rows are the 128 / group tokens' rows of all `group` query heads of one kv head, the pair's second CTA
 * taking the next tokens: a key tile is read once for the whole group, and the causal edge cuts at 2 x 128 / group rows,
 * not at 256. Persistent pairs take query tiles from the longest to the shortest, in turns that run back and forth, so
 * that their sums are near alike (past 32 sequences in the batch's order: Order); few query tiles over long keys are split
 * along the keys instead (Spans).
 *
 * Tensor memory (512 columns a CTA): two 128-column buffers of scores, and O's 256. P, rounded to bf16, replaces its
 * scores in place (64 columns) and is the second product's A operand from there. Shared memory: Q's 64 KiB and a ring of
 * 16 KiB stages; a CTA's share of a key tile is two stages of K (its 64 keys x 128 elements) and two of V (64 keys x its
 * 128 elements). The issue order S(0), S(1), PV(0), S(2), PV(1), ... gives the softmax of tile j the time of PV(j - 1)
 * and S(j + 1).
 *   warps 0-7   softmax, two threads a row: 64 scores each from tensor memory, the maxima exchanged in shared memory,
 *               exponentials, sums, P. The running maximum is followed only when a tile exceeds it by 2^8: rescaling O,
 *               256 columns of tensor memory a row, is then rare, and the weights of a row stay below 2^8
 *   warps 8-11  the output: O from tensor memory, divided by the row's sum, rounded once to bf16, turned in shared memory
 *               so that eight lanes write 128 bytes of a row, while the next query tile's products run
 *   warp 12     TMA loads     warp 13  the products' issue (the pair's first CTA)     warp 14  the order of the tiles
 *   warp 15     where a sequence's last key tile is not full, the zeroing of its V rows past the end (another sequence's
 *               rows, or anything behind the last one: P is zero there, but a NaN times zero is not). Its release to the
 *               pair's first CTA waits for all that the warp has under way; a warp of its own has nothing (released by the
 *               output's warps, behind their stores, 60 prompts of 37 rows took 27.5 us, 21.9 so; one such prompt alone 10.3 both ways)
 * P as bf16 costs half a bf16 step a weight, of the order of the output's own rounding; f32 elsewhere.
 *
 * Measured, 16 query heads over 2: 16,384 rows 1,364 us (1.61 PFLOP/s; the tensor pipe is active 89 % of the SMs' time),
 * 2,048 rows over 32,768 keys 670 us (1.59 PFLOP/s), 2,048 rows 33.4 us (1.03), six prompts of 256 to 2,048 rows 74.5 us
 * (1.09), 37 rows 10 us, each replayed from a graph for milliseconds. Run on for seconds the card is at its power limit,
 * 1,410 MHz under the long calls: 1,582, 788, 38.8 and 88 us. What the shorter ones lose lies between query tiles: the
 * next one's PV(0) waits for O to be read: 5,100 cycles from one PV to the next there, 2,800 elsewhere.
 */
#include <cuda_bf16.h>

#include "common.cuh"
#include "ridgefill_serve.h"
#include "sm100.cuh"

namespace {

constexpr int D = 256, kTileM = 128, kTileN = 128;           /* rows of a CTA (the pair's tile has 256); keys */
constexpr int kStages = 8, kStageBytes = 16384, kQBytes = kTileM * D * 2;
constexpr int kBoxBytes = 64 * 64 * 2;                       /* one TMA box of K or V: 64 rows x 64 elements */
constexpr int kSoftWarps = 8, kOutWarps = 4, kWarps = kSoftWarps + kOutWarps + 4, kThreads = 32 * kWarps;
constexpr int kTurnBytes = 32 * 128;                         /* an output warp's 32 rows x 64 elements */
constexpr int kRing = 4;                                     /* query tiles announced ahead */
constexpr uint32_t kTmemCols = 512, kColO = 256;
constexpr float kGrow = 8.0f, kNone = -INFINITY;
/* kind::f16 over the pair, D f32 (bit 4), A and B bf16 (bits 7, 10), N >> 3 at 17, M >> 4 at 24; B MN-major bit 16 */
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTileN >> 3) << 17) | ((uint32_t)(2 * kTileM >> 4) << 24);
constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(2 * kTileM >> 4) << 24);

struct Plan {
    RidgeFillAttnPrefill g;
    int group, tokens;      /* query heads a kv head; tokens of a CTA's rows (128 / group) */
    float scale_log2;
    void* partials;         /* split over the keys: [pairs][2 slots][2 CTAs] Partial; null: whole query tiles */
    int pairs;              /* of the split */
};

/* A CTA's part of a query tile's result: O's sums by column, and the rows' maxima (log2 units) and sums of weights. */
struct Partial {
    float o[D][kTileM];
    float2 ml[kTileM];
};

/* One query tile as a CTA sees it: `rows` tokens of its own from row q0 of q, keys from row k0 of k and v, key tiles first
 * .. first + tiles - 1 (the pair's); its token t sees the sequence's keys 0 .. limit + t, of which there are `keys`. slot
 * -1: all of its key tiles, the output is written; 0, 1: a piece, its Partial goes to that slot. rows < 0: no more. */
struct Item {
    int q0, rows, k0, keys, first, tiles, limit, head, slot;
};

/* Whether the item's last key tile is not full: its V rows past the sequence are zeroed before the product reads them. */
__device__ __forceinline__ bool cut_short(const Item& it) { return (it.first + it.tiles) * kTileN > it.keys; }

struct Shared {
    Item item[kRing];
    int64_t at[kTileM];                    /* where row r of the CTA's lies in o, from the first one's place */
    float top[2][2][kTileM];               /* rows' maxima of a tile's two halves, by the tile's parity */
    float top_of[3][kTileM];               /* and the maxima they go by */
    float sum[3][2][kTileM];               /* rows' sums (two halves) of the query tiles under way */
    uint64_t item_full[kRing], item_empty[kRing];
    uint64_t q_full, q_empty, kv_full[kStages], kv_empty[kStages];
    uint64_t s_full[2], p_full[2], pv_done[2], v_land[2], v_clean[2], o_full, o_empty, sum_full[3], drain;
    uint32_t tmem;
    int abort;
};
constexpr int kSmemBytes = 1024 + kQBytes + kStages * kStageBytes + kOutWarps * kTurnBytes + (int)sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t*)&p;
}

/* ------------------------------------------------------------------ the order of the query tiles */

struct Seq {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ Seq sequence(const RidgeFillAttnPrefill& g, int i) {
    Seq s;
    s.q0 = (int)rf::seq_start(g.cu_q, g.T, i);
    s.nq = (int)min(max((int64_t)g.cu_q[i + 1], (int64_t)s.q0), g.T) - s.q0;
    s.k0 = (int)rf::seq_start(g.cu_k, g.Tk, i);
    s.nk = (int)min(max((int64_t)g.cu_k[i + 1], (int64_t)s.k0), g.Tk) - s.k0;
    return s;
}
/* Query tile i of a sequence (2 `tokens` of them), the share of the pair's CTA `rank`. */
__device__ __forceinline__ Item tile_of(const Seq& s, int i, int tokens, int head, int rank) {
    Item t;
    const int from = i * 2 * tokens, both = min(2 * tokens, s.nq - from);
    t.rows = min(max(both - rank * tokens, 0), tokens);
    t.q0 = s.q0 + from + rank * tokens;
    t.k0 = s.k0;
    t.keys = s.nk;
    t.limit = s.nk - s.nq + from + rank * tokens;
    const int last = s.nk - s.nq + from + both - 1;   /* the pair's last row's last key */
    t.first = 0;
    t.tiles = last < 0 ? 0 : last / kTileN + 1;
    t.head = head;
    t.slot = -1;
    return t;
}
/* How many query tiles of a sequence have more than `depth` key tiles: the last ones. depth -1: all. */
__device__ __forceinline__ int deeper(const Seq& s, int depth, int tokens) {
    const int all = (int)((uint32_t)(s.nq + tokens - 1) / (uint32_t)tokens);
    if (depth < 0) return all;
    const int rows = depth * kTileN - s.nk + s.nq + 1;   /* a tile ending at this many rows or more is one; depth <= nk / 128 + 1 */
    if (rows > s.nq) return 0;
    return rows <= 0 ? all : all - ((int)((uint32_t)(rows + tokens - 1) / (uint32_t)tokens) - 1);
}
__device__ __forceinline__ int warp_sum(int x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
/* The first lane whose inclusive running sum of x exceeds `at`, and the sum before it; -1 when none does. */
__device__ __forceinline__ int lane_holding(int x, int at, int lane, int* before, int* total) {
    int sum = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    *total = __shfl_sync(0xffffffffu, sum, 31);
    const unsigned past = __ballot_sync(0xffffffffu, sum > at);
    if (!past) return -1;
    const int k = __ffs(past) - 1;
    *before = __shfl_sync(0xffffffffu, sum - x, k);
    return k;
}

/* ------------------------------------------------------------------ the split over the keys
 * All key tiles of all query tiles in a row -- sequence, query tile, kv head, key -- cut into equal spans, one a pair. A
 * span that holds all key tiles of a query tile writes its output; the at most two that it cuts leave Partials (slot 1 of
 * the pair that has the first of them, slot 0 of the others), which join_kernel adds up. */
struct Spans {
    int n, each, extra;   /* the first `extra` spans one longer; with few tiles fewer spans, of two, or one where that is odd */
    __device__ __forceinline__ Spans(int total, int most) {
        n = max(min((total + 1) / 2, most), 1);
        each = total / n;
        extra = total - each * n;
    }
    __device__ __forceinline__ int first(int i) const { return i * each + min(i, extra); }
    __device__ __forceinline__ int owner(int u) const {
        const int longer = extra * (each + 1);
        return u < longer ? u / (each + 1) : extra + (u - longer) / each;
    }
};

/* Query tile `i` of a sequence has this many key tiles (0 past its last one). */
__device__ __forceinline__ int depth_of(const Seq& q, int i, int tokens) {
    return i * 2 * tokens < q.nq ? tile_of(q, i, tokens, 0, 0).tiles : 0;
}

/* Walks the query tiles in order, 32 at a time; `at`(sequence, first query tile, this lane's key tiles of one head) is asked
 * for each 32 and ends the walk by answering true. The whole warp. */
template <class F>
__device__ __forceinline__ void walk(const Plan& p, int lane, F&& at) {
    for (int q = 0; q < (int)p.g.n_seq; ++q) {
        const Seq s = sequence(p.g, q);
        for (int i = 0; i * 2 * p.tokens < s.nq; i += 32)
            if (at(s, i, depth_of(s, i + lane, p.tokens))) return;
    }
}

/* The order of this pair's query tiles, the whole warp 14 of both CTAs, which reach the same order by themselves. Up to 32
 * sequences (a lane each) the tiles go from the most key tiles to the fewest over all sequences, in turns back and forth;
 * with more, in the batch's order, which costs up to 15 %: 32 prompts of 1 to 500 rows 62 us sorted, 68 in their order, of 100
 * to 2,048 406 and 402, of 256 and a last one of 4,096 134 and 154, of 64 to 2,048 falling 356 and 384. Split over the keys:
 * the pieces of the pair's span. */
struct Order {
    const Plan& p;
    int rank, lane, heads, pairs, pair, tokens;
    bool sorted;
    Seq mine = {};               /* sorted: this lane's sequence */
    int most = 0, total = 0;     /* the most key tiles of any query tile at most; the query tiles of one kv head */
    int block = 0, base = 0;     /* unsorted: the block of 32 sequences reached, and the tiles before it */
    int unit = 0, end = 0;       /* split: the rest of the span */
    Item own = {};               /* this lane's tile, if it is the owner of the one asked for */

    __device__ __forceinline__ Order(const Plan& plan, int rank_, int lane_) : p(plan), rank(rank_), lane(lane_) {
        const int n_seq = (int)p.g.n_seq;
        heads = (int)p.g.n_head_kv;
        pairs = (int)rf::cluster_count_x();
        pair = (int)rf::cluster_id_x();
        tokens = 2 * p.tokens;   /* of a query tile */
        sorted = n_seq <= 32 && !p.partials;
        if (p.partials) {
            int units = 0;
            walk(p, lane, [&](const Seq&, int, int depth) {
                units += depth;
                return false;
            });
            units = warp_sum(units) * heads;
            const Spans spans(units, p.pairs);
            if (pair < spans.n) {
                unit = spans.first(pair);
                end = spans.first(pair + 1);
            }
            return;
        }
        if (!sorted) return;
        if (lane < n_seq) mine = sequence(p.g, lane);
        most = mine.nq > 0 ? mine.nk / kTileN + 1 : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        total = warp_sum(deeper(mine, -1, tokens));
    }

    /* The lane whose `own` is the next piece of the span; -1: there is none. */
    __device__ __forceinline__ int piece() {
        if (unit >= end) return -1;
        int owner = -1, done = 0, used = 0;
        walk(p, lane, [&](const Seq& s, int i, int depth) {
            int before = 0, sum = 0;
            owner = lane_holding(depth * heads, unit - done, lane, &before, &sum);
            if (owner < 0) {
                done += sum;
                return false;
            }
            const int tiles = __shfl_sync(0xffffffffu, depth, owner), in = unit - done - before, head = in / tiles;
            own = tile_of(s, i + owner, p.tokens, head, rank);
            own.first = in - head * tiles;
            own.tiles = min(tiles - own.first, end - unit);
            own.slot = own.tiles == tiles ? -1 : own.first > 0 ? 0 : 1;
            used = own.tiles;
            return true;
        });
        unit = owner < 0 ? end : unit + used;
        return owner;
    }

    /* The lane whose `own` is the pair's k-th query tile; -1: there is none. */
    __device__ __forceinline__ int find(int k) {
        if (p.partials) return piece();
        const int at = sorted && (k & 1) ? k * pairs + pairs - 1 - pair : k * pairs + pair;
        const int t = (int)((uint32_t)at / (uint32_t)heads), head = at - t * heads;
        int before = 0, sum;
        if (sorted) {
            if (t >= total) return -1;
            int lo = 0, hi = most;   /* the least depth with at most t deeper tiles: tile t has that depth */
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (warp_sum(deeper(mine, mid, tokens)) <= t) hi = mid;
                else lo = mid + 1;
            }
            const int more = deeper(mine, lo, tokens), same = deeper(mine, lo - 1, tokens) - more;
            const int in = t - warp_sum(more);
            const int owner = max(lane_holding(same, in, lane, &before, &sum), 0);
            own = tile_of(mine, deeper(mine, -1, tokens) - (more + same) + (in - before), p.tokens, head, rank);
            return owner;
        }
        for (; block < (int)p.g.n_seq; block += 32) {
            Seq q = {};
            if (block + lane < p.g.n_seq) q = sequence(p.g, block + lane);
            const int owner = lane_holding(deeper(q, -1, tokens), t - base, lane, &before, &sum);
            if (owner >= 0) {
                own = tile_of(q, t - base - before, p.tokens, head, rank);
                return owner;
            }
            base += sum;
        }
        return -1;
    }
};

/* Zeros for a query tile none of whose rows has a key: this CTA's rows of it, a row's 512 bytes an instruction. */
__device__ void clear(const Plan& p, const Shared& s, int q0, int rows, int head, int lane) {
    uint16_t* const out = p.g.o + (int64_t)q0 * p.g.o_row + (int64_t)(head * p.group) * p.g.o_head;
    for (int r = 0; r < rows * p.group; ++r) *(uint4*)(out + s.at[r] + 8 * lane) = make_uint4(0u, 0u, 0u, 0u);
}

/* Announces them in the ring; `owner`: the first one's, found before the barriers stood. A query tile without keys never
 * enters it: the products' warp looks one tile ahead, and a row of such tiles would fill the ring before the output's warps
 * have done the last one with keys, each waiting for the other. */
__device__ void announce(const Plan& p, Order& order, Shared& s, int owner) {
    for (int k = 0, n = 0;; owner = order.find(++n)) {
        if (owner >= 0 && __shfl_sync(0xffffffffu, order.own.tiles, owner) == 0) {
            clear(p, s, __shfl_sync(0xffffffffu, order.own.q0, owner), __shfl_sync(0xffffffffu, order.own.rows, owner),
                  __shfl_sync(0xffffffffu, order.own.head, owner), order.lane);
            continue;
        }
        const int slot = k % kRing;
        if (!rf::mbar_wait_warp(&s.item_empty[slot], ((k / kRing) & 1) ^ 1, &s.abort, rf::kErrAttnWait)) return;
        if (owner < 0) order.own.rows = -1;
        if (order.lane == max(owner, 0)) {
            s.item[slot] = order.own;
            rf::mbar_arrive(&s.item_full[slot]);
        }
        if (owner < 0) return;
        ++k;
    }
}

/* The query tiles as one role's warp reads them. */
struct Items {
    Shared& s;
    int k = 0;
    /* The next tile; rows < 0 at the end (or when another role gave up). All lanes read it, lane 0 hands the slot back. */
    __device__ __forceinline__ Item next(int lane) {
        const int slot = k % kRing;
        Item it = {};
        it.rows = -1;
        if (rf::mbar_wait_warp(&s.item_full[slot], (k / kRing) & 1, &s.abort, rf::kErrAttnWait)) it = s.item[slot];
        __syncwarp();
        if (lane == 0) rf::mbar_arrive(&s.item_empty[slot]);
        ++k;
        return it;
    }
};

/* ------------------------------------------------------------------ roles */

/* Both CTAs of the pair; the bytes of both complete on the first CTA's barriers, but for the V rows of a key tile cut short:
 * those complete in their own CTA (v_land), where they are zeroed past the sequence before v_clean tells the products. */
__device__ void produce(const Plan& p, Shared& s, uint8_t* qtile, uint8_t* ring, const CUtensorMap* map_q, const CUtensorMap* map_k,
                        const CUtensorMap* map_v, int rank, int lane) {
    Items items{ s };
    uint32_t use = 0, done = 0, partial = 0;   /* stages filled; query tiles with keys; those cut short */
    const uint32_t q_bytes = 2u * 4u * (uint32_t)(p.group * p.tokens) * 128u;
    bool ok = true;
    for (;;) {
        const Item it = items.next(lane);
        if (it.rows < 0) break;
        if (lane == 0 && ok) {
            /* a stage: 64 rows of two 64-element columns from element x. land 0, 1: the first and second of a V cut short */
            auto stage = [&](const CUtensorMap* map, int x, int row, int land) {
                if (ok) ok = rf::mbar_wait(&s.kv_empty[use % kStages], ((use / kStages) & 1) ^ 1, &s.abort, rf::kErrAttnWait);
                if (!ok) return;
                const uint32_t st = use % kStages;
                uint32_t bar;
                if (land < 0) {
                    bar = rf::map_rank(rf::smem_addr(&s.kv_full[st]), 0);
                    if (rank == 0) rf::mbar_arrive_expect_tx(&s.kv_full[st], 2 * kStageBytes);
                } else {
                    bar = rf::map_rank(rf::smem_addr(&s.v_land[partial & 1]), rank);
                    if (land == 0) rf::mbar_arrive_expect_tx(&s.v_land[partial & 1], 2 * kStageBytes);   /* both stages' */
                    if (rank == 0) rf::mbar_arrive(&s.kv_full[st]);
                }
                rf::tma_load_3d_pair(ring + st * kStageBytes, map, bar, x, it.head, row);
                rf::tma_load_3d_pair(ring + st * kStageBytes + kBoxBytes, map, bar, x + 64, it.head, row);
                ++use;
            };
            ok = rf::mbar_wait(&s.q_empty, (done & 1) ^ 1, &s.abort, rf::kErrAttnWait);
            if (ok) {
                const uint32_t bar = rf::map_rank(rf::smem_addr(&s.q_full), 0);
                if (rank == 0) rf::mbar_arrive_expect_tx(&s.q_full, q_bytes);
                for (int b = 0; b < D / 64; ++b)
                    rf::tma_load_3d_pair(qtile + b * kTileM * 128, map_q, bar, b * 64, it.head * p.group, it.q0);
                ++done;
            }
            for (int j = 0; j <= it.tiles; ++j) {
                if (j < it.tiles)   /* this CTA's 64 keys of the tile */
                    for (int h = 0; h < 2; ++h) stage(map_k, h * 128, it.k0 + (it.first + j) * kTileN + rank * 64, -1);
                if (j > 0)          /* the tile's keys, this CTA's 128 elements */
                    for (int h = 0; h < 2; ++h)
                        stage(map_v, rank * 128, it.k0 + (it.first + j - 1) * kTileN + h * 64, j == it.tiles && cut_short(it) ? h : -1);
            }
            partial += cut_short(it);
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok) break;
    }
    /* The products have read every stage that this CTA filled (so its copies have landed) before it leaves. */
    if (lane == 0) {
        const uint64_t t0 = rf::global_ns();
        for (uint32_t u = use > kStages ? use - kStages : 0; u < use; ++u)
            while (!rf::mbar_try_wait(&s.kv_empty[u % kStages], (u / kStages) & 1) && rf::global_ns() - t0 < rf::kWaitTimeoutNs) {
            }
        if (done)
            while (!rf::mbar_try_wait(&s.q_empty, (done - 1) & 1) && rf::global_ns() - t0 < rf::kWaitTimeoutNs) {
            }
    }
}

/* The pair's first CTA, the whole warp in step. Its barriers count both CTAs' arrivals; its commits arrive in both. Each
 * lane watches a barrier of its own, so that all that a product needs costs one wait. The scores of a query tile's first
 * key tile are issued before the last PV of the query tile before it, while that one's softmax is under way: K(0) lies
 * behind V(last) in the ring. */
__device__ void multiply(Shared& s, const uint8_t* qtile, const uint8_t* ring, uint32_t tmem, int lane) {
    Items items{ s };
    uint32_t use = 0;                                    /* the ring's next stage, counted through */
    uint32_t tile = 0, begun = 0, done = 0, partial = 0;   /* the PV's key tile; query tiles with keys begun, done; with a cut last tile */
    const uint32_t q_addr = rf::smem_addr(qtile), r_addr = rf::smem_addr(ring);
    bool ok = true;
    /* lane 0 .. 3: a barrier and its parity; the other lanes watch lane 0's */
    auto wait = [&](uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2, uint64_t* b3, uint32_t p3) {
        uint64_t* bar = lane == 1 ? b1 : lane == 2 ? b2 : lane == 3 ? b3 : b0;
        const uint32_t parity = lane == 1 ? p1 : lane == 2 ? p2 : lane == 3 ? p3 : p0;
        if (ok) ok = rf::mbar_wait_lanes(bar, parity, &s.abort, rf::kErrAttnWait);
        rf::tc_fence_after();
        return ok;
    };
    auto full = [&](uint32_t u) { return &s.kv_full[u % kStages]; };
    auto phase = [&](uint32_t u) { return (u / kStages) & 1; };
    auto commit = [&](uint64_t* bar) { rf::mma_commit_pair_warp(rf::smem_addr(bar), 3); };
    Item it = {}, ahead = {};   /* the query tiles of the PV and of the scores under way */
    int j = -1, ja = 0;         /* their key tiles; j -1: no PV yet */
    for (bool first = true; ok;) {
        /* the scores' key tile: the next of this query tile, or the first of the next */
        if (first) {
            const Item i = items.next(lane);
            ahead.rows = __shfl_sync(0xffffffffu, i.rows, 0);
            ahead.tiles = __shfl_sync(0xffffffffu, i.tiles, 0);
            ahead.keys = __shfl_sync(0xffffffffu, i.keys, 0);
            ahead.first = __shfl_sync(0xffffffffu, i.first, 0);
            ja = 0;
        }
        const bool more = ahead.rows >= 0;
        const uint32_t k = j >= 0 && first ? use + 2 : use;       /* K: behind this tile's V when it is a new query tile's */
        const uint32_t v = j >= 0 && !first ? use + 2 : use;
        if (more) {
            uint64_t* q = first ? &s.q_full : full(k);
            const uint32_t pq = first ? begun & 1 : phase(k);
            if (!wait(full(k), phase(k), full(k + 1), phase(k + 1), q, pq, q, pq)) break;
            begun += first;
            const uint32_t d = tmem + (j >= 0 ? (tile + 1) & 1 : 0) * kTileN;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint64_t a = rf::sw128_kmajor_desc(q_addr + 2 * h * kTileM * 128),
                               b = rf::sw128_kmajor_desc(r_addr + (k + h) % kStages * kStageBytes);
                rf::umma_f16_pair_warp8<kTileM * 128, kBoxBytes>(d, a, b, kIdescS, h);
                commit(&s.kv_empty[(k + h) % kStages]);
            }
            commit(&s.s_full[j >= 0 ? (tile + 1) & 1 : 0]);
            if (ja + 1 == ahead.tiles) commit(&s.q_empty);   /* Q's last product is issued */
            use += 2;
        }
        if (j >= 0) {
            const bool last = j + 1 == it.tiles, cut = last && cut_short(it);
            uint64_t* p = &s.p_full[tile & 1];
            const uint32_t pp = (tile >> 1) & 1;
            if (!wait(p, pp, full(v), phase(v), full(v + 1), phase(v + 1), j == 0 ? &s.o_empty : p, j == 0 ? (done & 1) ^ 1 : pp)) break;
            if (cut) {   /* V of both CTAs, landed and zeroed past the sequence */
                ok = rf::mbar_wait_lanes<true>(&s.v_clean[partial & 1], (partial >> 1) & 1, &s.abort, rf::kErrAttnWait);
                if (!ok) break;
                ++partial;
            }
            const uint32_t a = tmem + (tile & 1) * kTileN;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint64_t b = rf::sw128_mnmajor_desc(r_addr + (v + h) % kStages * kStageBytes, kBoxBytes);
                rf::umma_f16_ts_pair_warp4(tmem + kColO, a + h * 32, b, kIdescO, j | h);
                commit(&s.kv_empty[(v + h) % kStages]);
            }
            commit(&s.pv_done[tile & 1]);
            if (last) {
                commit(&s.o_full);
                ++done;
            }
            use += 2;
            ++tile;
        }
        if (!more) break;
        it = ahead;
        j = ja;
        first = ++ja == it.tiles;
    }
    /* every product has run before tensor memory is given up */
    rf::mma_commit_pair_warp(rf::smem_addr(&s.drain), 1);
    const uint64_t t0 = rf::global_ns();
    while (!rf::mbar_try_wait(&s.drain, 0) && rf::global_ns() - t0 < rf::kWaitTimeoutNs) {
    }
    __syncwarp();
}

__device__ void soften(const Plan& p, Shared& s, uint32_t tmem, int warp, int lane) {
    Items items{ s };
    uint32_t tile = 0;
    int buf = 2;   /* of the sums */
    const int quarter = warp & 3, half = warp >> 2;   /* 32 rows; 64 keys of the tile */
    const int row = quarter * 32 + lane, token = row / p.group;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const float sl2 = p.scale_log2;
    for (;;) {
        const Item it = items.next(lane);
        /* the two warps of these rows meet once a query tile and once a key tile, and leave together: when a wait gave up
         * neither is left at a barrier */
        if (rf::bar_any(1 + quarter, 64, it.rows < 0)) return;
        const int limit = it.limit + min(token, max(it.rows - 1, 0));   /* this row's last key */
        float m = kNone, l0 = 0.f, l1 = 0.f;
        buf = buf == 2 ? 0 : buf + 1;
        for (int j = 0; j < it.tiles; ++j, ++tile) {
            const bool ok = rf::mbar_wait(&s.s_full[tile & 1], (tile >> 1) & 1, &s.abort, rf::kErrAttnWait);
            rf::tc_fence_after();
            const uint32_t at = lanes + (tile & 1) * kTileN;
            uint32_t x[2][32];
#pragma unroll
            for (int c = 0; c < 2; ++c) rf::tmem_ld32(at + 64 * half + 32 * c, x[c]);
            rf::tmem_ld_wait();
            const int key = (it.first + j) * kTileN + 64 * half;
            if (key + 63 > it.limit) {   /* the first token does not see all of these keys */
                const int last = limit - key;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e > last) x[c][e] = __float_as_uint(kNone);
            }
            float top[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                top[c] = __uint_as_float(x[c >> 1][16 * (c & 1)]);
#pragma unroll
                for (int e = 1; e < 16; ++e) top[c] = fmaxf(top[c], __uint_as_float(x[c >> 1][16 * (c & 1) + e]));
            }
            const float own = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            s.top[tile & 1][half][row] = own;
            /* both warps have read their scores, so that P may take their place */
            if (rf::bar_any(1 + quarter, 64, !ok)) return;
            const float mt = fmaxf(own, s.top[tile & 1][half ^ 1][row]) * sl2;
            const bool grow = mt > m + kGrow;
            if (__any_sync(0xffffffffu, grow)) {
                const float up = grow ? mt : m, f = m == kNone ? 0.f : exp2_approx(m - up);
                m = up;
                l0 *= f;
                l1 *= f;
                if (j > 0) {   /* this half of O so far, in the units of the old maximum; these scores came after
                                * PV(tile - 2), so that the barrier of PV(tile - 1) is at most one phase behind */
                    const bool there = rf::mbar_wait(&s.pv_done[(tile - 1) & 1], ((tile - 1) >> 1) & 1, &s.abort, rf::kErrAttnWait);
                    if (rf::bar_any(1 + quarter, 64, !there)) return;
                    rf::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 64; ++c) {
                        uint32_t o[32];
                        rf::tmem_ld32(lanes + kColO + (D / 2) * half + 32 * c, o);
                        rf::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        rf::tmem_st32(lanes + kColO + (D / 2) * half + 32 * c, o);
                    }
                }
            }
            const float base = m == kNone ? 0.f : -m;
            uint32_t w[32];
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
                float a = base, b = base;
                rf::fma2_rn(a, b, __uint_as_float(x[e >> 5][e & 31]), __uint_as_float(x[e >> 5][(e & 31) + 1]), sl2, sl2);
                a = exp2_approx(a);
                b = exp2_approx(b);
                rf::add2_rn(l0, l1, a, b);
                w[e >> 1] = pack(a, b);
            }
            rf::tmem_st32(at + 32 * half, w);
            /* The row's sum, announced before the last P so that no warp can be a query tile ahead of another here. Three
             * buffers: these scores may come before the last PV of the query tile before, but not before that of the one
             * before it, whose first PV waited for O's reader to be done with the buffer's earlier sums. */
            if (j + 1 == it.tiles) {
                s.sum[buf][half][row] = l0 + l1;
                if (half == 0) s.top_of[buf][row] = m;
            }
            rf::tmem_st_wait();
            rf::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (j + 1 == it.tiles) rf::mbar_arrive(&s.sum_full[buf]);
                /* relaxed: P is ordered by tensor memory's own fences, and a release to the cluster costs 1,800 cycles */
                rf::mbar_arrive_cluster_relaxed(rf::map_rank(rf::smem_addr(&s.p_full[tile & 1]), 0));
            }
        }
    }
}

/* V's rows past the sequence in a last key tile cut short, zeroed in this CTA's memory. Two barriers in turn: the ring holds V
 * of two such tiles at most, the third one's first stage being the first one's, which the product has read by then. */
__device__ void clean(Shared& s, uint8_t* ring, int lane) {
    Items items{ s };
    uint32_t use = 0, partial = 0;
    for (;;) {
        const Item it = items.next(lane);
        if (it.rows < 0) return;
        use += 4 * it.tiles;   /* the last two stages: 64 rows of V each */
        if (!cut_short(it)) continue;
        if (!rf::mbar_wait_warp(&s.v_land[partial & 1], (partial >> 1) & 1, &s.abort, rf::kErrAttnWait)) return;
        /* a row's 128 bytes in each of the stage's two boxes; two rows an instruction */
        const int first = it.keys - (it.first + it.tiles - 1) * kTileN;
        for (int row = first + (lane >> 4); row < kTileN; row += 2)
            *(uint4*)(ring + ((use - 2 + (uint32_t)(row >> 6)) % kStages) * kStageBytes + (lane >> 3 & 1) * kBoxBytes + (row & 63) * 128 +
                      (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        rf::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) rf::mbar_arrive_cluster(rf::map_rank(rf::smem_addr(&s.v_clean[partial & 1]), 0));
        ++partial;
    }
}

__device__ void output(const Plan& p, Shared& s, uint8_t* turn, uint32_t tmem, int rank, int warp, int lane) {
    const RidgeFillAttnPrefill& g = p.g;
    Items items{ s };
    uint32_t done = 0;
    const int row = warp * 32 + lane;
    const uint32_t mine = tmem + kColO + ((uint32_t)(warp * 32) << 16);
    for (;;) {
        const Item it = items.next(lane);
        if (it.rows < 0) return;
        const int live = it.rows * p.group;   /* this CTA's rows */
        uint16_t* const out = g.o + (int64_t)it.q0 * g.o_row + (int64_t)(it.head * p.group) * g.o_head;
        if (!rf::mbar_wait_warp(&s.o_full, done & 1, &s.abort, rf::kErrAttnWait) ||
            !rf::mbar_wait_warp(&s.sum_full[done % 3], (done / 3) & 1, &s.abort, rf::kErrAttnWait))
            return;
        rf::tc_fence_after();
        const float sum = s.sum[done % 3][0][row] + s.sum[done % 3][1][row];
        if (it.slot >= 0) {   /* a piece: a thread its row's sums, a column's 128 rows side by side */
            Partial& part = ((Partial*)p.partials)[((int64_t)rf::cluster_id_x() * 2 + it.slot) * 2 + rank];
            if (row < live) part.ml[row] = make_float2(s.top_of[done % 3][row], sum);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                rf::tmem_ld32(mine + 32 * c, o);
                rf::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (row < live) part.o[32 * c + e][row] = __uint_as_float(o[e]);
            }
            rf::tc_fence_before();
            __syncwarp();
            if (lane == 0) rf::mbar_arrive_cluster_relaxed(rf::map_rank(rf::smem_addr(&s.o_empty), 0));
            ++done;
            continue;
        }
        const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);   /* no key: zeros; a NaN stays one */
        uint8_t* tile = turn + warp * kTurnBytes;
        uint16_t* dst[8];   /* this lane's chunk of the eight rows it writes */
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = out + s.at[warp * 32 + 4 * i + (lane >> 3)] + 8 * (lane & 7);
        const int rows = live - warp * 32 - (lane >> 3);   /* row i of them is one of the tile's while 4 i < rows */
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {   /* 64 elements of the 32 rows: 16-byte chunk v of row r at chunk v ^ (r & 7) */
            uint32_t o[2][32];
            rf::tmem_ld32(mine + 64 * c, o[0]);
            rf::tmem_ld32(mine + 64 * c + 32, o[1]);
            rf::tmem_ld_wait();
            if (c + 1 == D / 64) {   /* O's last read */
                rf::tc_fence_before();
                __syncwarp();
                if (lane == 0) rf::mbar_arrive_cluster_relaxed(rf::map_rank(rf::smem_addr(&s.o_empty), 0));
            }
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = 8 * (v & 3) + 2 * e;
                    float lo, hi;
                    rf::mul2_rn(lo, hi, __uint_as_float(o[v >> 2][x]), __uint_as_float(o[v >> 2][x + 1]), inv, inv);
                    w[e] = pack(lo, hi);
                }
                *(uint4*)(tile + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (inv == 0.f) {   /* again: where the tile's V is not finite, zero weights have left a NaN in O */
#pragma unroll 1
                for (int v = 0; v < 8; ++v) *(uint4*)(tile + lane * 128 + (v << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
            __syncwarp();
            uint4 t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + (lane >> 3);
                t[i] = *(const uint4*)(tile + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (4 * i < rows) *(uint4*)(dst[i] + 64 * c) = t[i];
            __syncwarp();   /* read before the next 64 elements take its place */
        }
        ++done;
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const Plan p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* qtile = smem;
    uint8_t* ring = smem + kQBytes;
    uint8_t* turn = ring + kStages * kStageBytes;
    Shared& s = *(Shared*)(turn + kOutWarps * kTurnBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)rf::cluster_rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            rf::mbar_init(&s.item_full[i], 1);
            /* every warp but the one that orders them, and in the second CTA the one that would issue the products */
            rf::mbar_init(&s.item_empty[i], kWarps - 1 - rank);
        }
        rf::mbar_init(&s.q_full, 1);    /* first CTA's: its producer, both CTAs' bytes */
        rf::mbar_init(&s.q_empty, 1);   /* each CTA's: the products' commits */
        for (int i = 0; i < kStages; ++i) {
            rf::mbar_init(&s.kv_full[i], 1);
            rf::mbar_init(&s.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            rf::mbar_init(&s.s_full[i], 1);
            rf::mbar_init(&s.p_full[i], 2 * kSoftWarps);   /* first CTA's: both CTAs' warps */
            rf::mbar_init(&s.pv_done[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            rf::mbar_init(&s.v_land[i], 1);    /* each CTA's: its producer, its bytes */
            rf::mbar_init(&s.v_clean[i], 2);   /* first CTA's: both CTAs' zeroing warps */
        }
        rf::mbar_init(&s.o_full, 1);
        rf::mbar_init(&s.o_empty, 2 * kOutWarps);
        for (int i = 0; i < 3; ++i) rf::mbar_init(&s.sum_full[i], kSoftWarps);
        rf::mbar_init(&s.drain, 1);
        s.abort = 0;
        rf::mbar_init_fence();
        rf::tma_prefetch_map(&map_q);
        rf::tma_prefetch_map(&map_k);
        rf::tma_prefetch_map(&map_v);
    }
    if (p.partials) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   /* the join may line up */
    /* Rows of Q that no copy fills, where 128 is no multiple of the group: zeros, since what lies there would go through the
     * softmax like a row, and its maxima would have O rescaled again and again (8,192 rows of 24 heads over 2: 631 us, 575). */
    if (const int filled = p.group * p.tokens; filled < kTileM) {
        for (int i = threadIdx.x; i < (kTileM - filled) * (D / 8); i += kThreads)
            *(uint4*)(qtile + i % 4 * (kTileM * 128) + (filled + i / 32) * 128 + i / 4 % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
        rf::fence_proxy_async_smem();
    }
    if (threadIdx.x >= 128 && threadIdx.x < 128 + kTileM) {
        const int r = threadIdx.x - 128, token = r / p.group;
        s.at[r] = (int64_t)token * p.g.o_row + (int64_t)(r - token * p.group) * p.g.o_head;
    }
    if (warp == 13) rf::tmem_alloc_pair<kTmemCols>(&s.tmem);
    if (warp == 14) {   /* the first query tile is found while the barriers are made */
        Order order(p, rank, lane);
        const int owner = order.find(0);
        rf::cluster_sync_all();
        announce(p, order, s, owner);
        rf::cluster_sync_all();
        return;
    }
    rf::tc_fence_before();
    rf::cluster_sync_all();   /* both CTAs' barriers are initialised before either signals the other's */
    rf::tc_fence_after();
    const uint32_t tmem = s.tmem;
    if (warp < 8) soften(p, s, tmem, warp, lane);
    else if (warp < 12) output(p, s, turn, tmem, rank, warp - 8, lane);
    else if (warp == 12) produce(p, s, qtile, ring, &map_q, &map_k, &map_v, rank, lane);
    else if (warp == 15) clean(s, ring, lane);
    else if (rank == 0) multiply(s, qtile, ring, tmem, lane);
    rf::tc_fence_before();
    rf::cluster_sync_all();   /* no product reads the other CTA's memory any more */
    rf::tc_fence_after();
    if (warp == 13) rf::tmem_free_pair<kTmemCols>(tmem);
}

/* A join CTA with nothing to add leaves at once, but for one: the join's end is what the stream's next kernel waits for, and
 * it must not come before the split's. */
__device__ __forceinline__ void nothing_to_join() {
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

/* The query tiles that the split cut, and those without a key (zeros): a CTA joins kCols columns of a CTA's share of one
 * query tile and kv head, a thread a row, kFlight pieces' loads in flight. */
template <int kCols, int kFlight>
__global__ void __launch_bounds__(kTileM) join_kernel(const Plan p) {
    const RidgeFillAttnPrefill& g = p.g;
    const int lane = threadIdx.x & 31, row = threadIdx.x, heads = (int)g.n_head_kv;
    constexpr int parts = D / kCols;
    const int part = blockIdx.x % parts, rank = blockIdx.x / parts % 2, item = blockIdx.x / (2 * parts);
    const int query = item / heads, head = item - query * heads;
    int seen = 0, units = 0, start = 0, tiles = -1;
    Item it = {};
    walk(p, lane, [&](const Seq& s, int i, int depth) {
        const int here = min(32, (s.nq + 2 * p.tokens - 1) / (2 * p.tokens) - i), in = query - seen;
        if (in >= 0 && in < here) {   /* the query tile is one of these 32 */
            it = tile_of(s, i + in, p.tokens, head, rank);
            tiles = it.tiles;
            start = (units + warp_sum(lane < in ? depth : 0)) * heads + head * tiles;
        }
        seen += here;
        units += warp_sum(depth);
        return false;
    });
    if (tiles < 0) return nothing_to_join();   /* fewer query tiles than the grid has places for */
    const int token = row / p.group;
    uint16_t* out = g.o + (int64_t)(it.q0 + token) * g.o_row + (int64_t)(head * p.group + row - token * p.group) * g.o_head + part * kCols;
    const bool live = token < it.rows;
    if (tiles == 0) {
        if (live)
            for (int c = 0; c < kCols / 8; ++c) *(uint4*)(out + 8 * c) = make_uint4(0u, 0u, 0u, 0u);
        return nothing_to_join();
    }
    const Spans spans(units * heads, p.pairs);
    const int c0 = spans.owner(start), n = spans.owner(start + tiles - 1) - c0 + 1;
    if (n == 1) return nothing_to_join();   /* written by its one pair */
    asm volatile("griddepcontrol.wait;" ::: "memory");   /* the split is done and its results are visible */
    if (!live) return;
    auto piece = [&](int i) -> const Partial& { return ((const Partial*)p.partials)[((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * 2 + rank]; };
    float top = kNone, sum = 0.f, acc[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] = 0.f;
    for (int i = 0; i < n; i += kFlight) {
        float2 ml[kFlight];
        float o[kFlight][kCols];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const Partial& s = piece(min(i + k, n - 1));
            ml[k] = i + k < n ? s.ml[row] : make_float2(kNone, 0.f);
#pragma unroll
            for (int c = 0; c < kCols; ++c) o[k][c] = s.o[part * kCols + c][row];
        }
        float up = top;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) up = fmaxf(up, ml[k].x);
        const float f = top == kNone ? 0.f : exp2_approx(top - up);
        sum *= f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[c] *= f;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            /* no piece, or none of its keys is the row's; by the sum, since a row of NaN scores has no maximum either (fmaxf
             * passes over them), but a NaN sum, and is NaN as it is from whole query tiles */
            if (ml[k].y == 0.f) continue;
            const float w = exp2_approx(ml[k].x - up);
            sum = fmaf(w, ml[k].y, sum);
#pragma unroll
            for (int c = 0; c < kCols; ++c) acc[c] = fmaf(w, o[k][c], acc[c]);
        }
        top = up;
    }
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int c = 0; c < kCols; c += 8)
        *(uint4*)(out + c) = make_uint4(pack(acc[c] * inv, acc[c + 1] * inv), pack(acc[c + 2] * inv, acc[c + 3] * inv),
                                        pack(acc[c + 4] * inv, acc[c + 5] * inv), pack(acc[c + 6] * inv, acc[c + 7] * inv));
}

/* How a parsed call runs: query tiles go to pairs whole, or their key tiles are split evenly and the cut ones joined. Whole,
 * the pair with the longest query tile decides, or the one with two. The split is taken
 *   with fewer query tiles than pairs, when evening them out saves the longest one kLeast key tiles, 1.4 us each (the lengths
 *   are device memory: a sequence of about twice the average stands for the longest): 16 rows over 4,096 keys 17 us, 49
 *   whole; 300 over 6,000 38, 69 whole; nine short tails, one of them over 6,193 keys, 26, 70 whole; near kLeast 64 over 1,024
 *   15, 19.6 whole, and 512 over 1,500 27.5, 26 whole; eight tails over 1,000 keys each 24.5, 19.5 whole
 *   with at most two a pair, keys from kLongKeys on and a sequence of twice the average from kLongAverage: 2,048 rows over
 *   32,768, 128 query tiles of 256 key tiles on 74 pairs, would take two rounds, 86 % of the pairs' time: 670 us, 704 whole;
 *   four times 300 over 3,000 61, 70 whole; eight times 128 over 1,200 41, 25 whole; 30 times 2 over 300 63, 14 whole: the
 *   split goes through the sequences one by one
 * The extents decide, which in a captured call may be much larger than the sequences of the moment: 2,048 rows over 2,048
 * keys in operands of 32,768 keys 55 us, 34 in their own; 37 rows in 512 and 4,096 keys 16.6 and 10.5, 16 over 500 in 32,768
 * 17.8 and 16.5 */
constexpr int kLongKeys = 8192, kLongAverage = 4096, kLeast = 6;
constexpr int64_t kMostItems = 0x3fffffff;   /* query tiles, counted in 32 bits with a turn of the pairs to spare */
struct Shape {
    int group, tokens;
    int64_t items;      /* query tiles (of all kv heads) at most: a sequence's last one may be cut short */
    int pairs;
    bool split;
    int64_t bytes;
};
Shape shape_of(const RidgeFillAttnPrefill& g) {
    Shape s;
    s.group = (int)(g.n_head / g.n_head_kv);
    s.tokens = kTileM / s.group;
    const int64_t tiles = g.T / (2 * s.tokens) + g.n_seq;
    s.items = g.n_head_kv > kMostItems / tiles ? kMostItems + 1 : tiles * g.n_head_kv;   /* a call with more is refused */
    s.pairs = rf::sm_count() / 2;
    const bool few = s.items < s.pairs && 2 * g.Tk * (s.pairs - s.items) >= (int64_t)kLeast * kTileN * s.pairs * (g.n_seq + 1);
    const bool two = s.items <= 2 * s.pairs && g.Tk >= kLongKeys && 2 * g.Tk >= (int64_t)kLongAverage * (g.n_seq + 1);
    /* the split counts key tiles in 32 bits, whatever cu_seqlens and cu_keys hold: sequences that overlap too */
    s.split = (few || two) && g.n_seq * s.items * (g.Tk / kTileN + 1) <= 0x7fffffffLL;
    s.bytes = s.split ? (int64_t)s.pairs * 4 * (int64_t)sizeof(Partial) : 0;
    return s;
}

/* Head rows [T, heads, 256] bf16 as a 3-D tensor map read in boxes of 64 elements x `heads_box` heads x `rows_box` rows,
 * 128-byte swizzle; rows past T read as zero. A row or head axis of extent 1 may have any stride: it is never stepped. */
bool head_map(CUtensorMap* map, const uint16_t* base, int64_t T, int64_t heads, int64_t row_stride, int64_t head_stride,
              int heads_box, int rows_box) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = rf::tensor_map_encoder();
    if (!enc) return false;
    if (heads == 1) head_stride = D;
    if (T == 1) row_stride = heads * D;
    const cuuint64_t dims[3] = { (cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T };
    const cuuint64_t strides[2] = { (cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2 };
    const cuuint32_t box[3] = { 64, (cuuint32_t)heads_box, (cuuint32_t)rows_box };
    const cuuint32_t estr[3] = { 1, 1, 1 };
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

/* A warp's wait of which half the lanes see their phase complete and half one that nothing completes. */
__global__ void wait_selftest_kernel(int* status) {
    __shared__ uint64_t bar;
    __shared__ int abort;
    const int lane = threadIdx.x;
    if (lane == 0) {
        rf::mbar_init(&bar, 1);
        abort = 0;
        rf::mbar_init_fence();
    }
    __syncwarp();
    if (lane == 0) rf::mbar_arrive(&bar);
    __syncwarp();
    status[lane] = rf::mbar_wait_warp(&bar, lane < 16 ? 0 : 1, &abort, rf::kErrAttnWait) ? 1 : 0;
}

}  // namespace

/* Failure detection without a fault: see include/ridgefill_serve.h. */
extern "C" int ridgefill_attn_wait_selftest(int* status, RadStream s) {
    if (!status) return RAD_E_INVAL;
    wait_selftest_kernel<<<1, 32, 0, rf::as_stream(s)>>>(status);
    return rf::launch_status();
}

/* This translation unit's copy of the device error word (sm100.cuh), for ridgefill_device_error. */
namespace rf {
int attn_device_error(int reset) { return read_device_error(reset); }
}  // namespace rf

extern "C" int64_t ridgefill_attn_prefill_scratch(const RadArgs* a) {
    RidgeFillAttnPrefill g;
    return ridgefill_attn_prefill_parse(a, &g) == RAD_OK && g.T > 0 && g.n_seq > 0 ? shape_of(g).bytes : 0;
}

extern "C" int ridgefill_attn_prefill_device(const RadArgs* a, RadStream s) {
    Plan p;
    const int rc = ridgefill_attn_prefill_parse(a, &p.g);
    if (rc != RAD_OK) return rc;
    const RidgeFillAttnPrefill& g = p.g;
    if (g.T == 0 || g.n_seq == 0) return RAD_OK;
    const Shape sh = shape_of(g);
    if (sh.items > kMostItems) return RAD_E_SHAPE;
    if (sh.split && (!a->scratch || a->scratch_bytes < sh.bytes || (uintptr_t)a->scratch % 16)) return RAD_E_INVAL;
    p.group = sh.group;
    p.tokens = sh.tokens;
    p.scale_log2 = g.scale * 1.4426950408889634f;
    p.partials = sh.split ? a->scratch : nullptr;
    p.pairs = sh.pairs;
    CUtensorMap mq, mk, mv;
    if (!head_map(&mq, g.q, g.T, g.n_head, g.q_row, g.q_head, p.group, p.tokens)) return RAD_E_DEVICE;
    /* without a key row nothing is read through the maps of k and v */
    if (!head_map(&mk, g.Tk ? g.k : g.q, g.Tk ? g.Tk : 1, g.n_head_kv, g.Tk ? g.k_row : D * g.n_head_kv, g.Tk ? g.k_head : D, 1, 64) ||
        !head_map(&mv, g.Tk ? g.v : g.q, g.Tk ? g.Tk : 1, g.n_head_kv, g.Tk ? g.v_row : D * g.n_head_kv, g.Tk ? g.v_head : D, 1, 64))
        return RAD_E_DEVICE;
    if (cudaFuncSetAttribute(prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess) {
        cudaGetLastError();
        return RAD_E_DEVICE;
    }
    const int64_t pairs = sh.split || sh.items > sh.pairs ? sh.pairs : sh.items;
    prefill_kernel<<<2 * (unsigned)pairs, kThreads, kSmemBytes, rf::as_stream(s)>>>(mq, mk, mv, p);
    if (const int launched = rf::launch_status(); launched != RAD_OK || !sh.split) return launched;
    cudaLaunchConfig_t cfg = {};
    /* The join's columns a CTA and pieces in flight, by how many pieces a query tile may have. 16 rows over 32,768 keys: 35 us
     * with 8 columns and 8 pieces, 46 with 16 and 4, 98 with 64 and one; 300 rows over 6,000: 39.4, 37.9 and 47.2; 1,024 rows
     * over 16,384: 191, 184 and 185; 2,048 over 32,768, eight launches in a row: 704, 758 and 701. */
    const int cols = 3 * sh.items <= sh.pairs ? 8 : sh.items <= sh.pairs ? 16 : 64;
    cfg.gridDim = dim3((unsigned)(sh.items * 2 * (D / cols)));
    cfg.blockDim = dim3(kTileM);
    cfg.stream = rf::as_stream(s);
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, cols == 8 ? join_kernel<8, 8> : cols == 16 ? join_kernel<16, 4> : join_kernel<64, 1>, p) != cudaSuccess) {
        cudaGetLastError();
        return RAD_E_DEVICE;
    }
    return RAD_OK;
}
