/* attn_decode.cu -- ridgefill_attn_decode: attention of one new token a sequence over the paged K/V cache, on B200
 * (ridgefill_serve.h holds the formula; ridgefill_attn_kv_fill writes the cache).
 *
 * HBM-bound: the keys and values of every sequence are read once (1 KiB a key and kv head), and all of a kv head's
 * query heads are served from that read. The arithmetic (4 D flops a key and query head) goes through mma.sync, far
 * below its rate. What decides the time is how evenly the bytes spread over the SMs and how many are in flight.
 *
 * Work. A unit is 16 keys of one item (a sequence's kv head and up to 16 of its query heads). The units of all items
 * in order -- sequence, head, position -- are cut into equal spans, one a CTA, whatever the lengths: a long sequence
 * spreads over many CTAs, short ones share one. The lengths are device memory, so every CTA finds its span from
 * kv_lens itself. A span that covers a whole item writes its output; the at most two items a span cuts leave a partial
 * result (unnormalised sum, running maximum, sum of weights) in the CTA's two scratch slots, and the join kernel, whose
 * launch overlaps this one's run, adds the pieces of each item.
 *
 * Inside a CTA four warps take 16-key blocks in turn, each with running softmax statistics of its own, and meet at the
 * piece's end. A warp streams its blocks through its own ring in shared memory by 16-byte asynchronous copies, a
 * whole 512-byte row an instruction: no barrier beyond the warp's own, and two to three 8 KiB halves in flight a warp
 * (128 KiB a SM; the 49 bytes a nanosecond of a SM's share of HBM at about a microsecond's latency need 49 KiB). The products are
 * taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the up to 8 query heads sharing a kv head fill the n of
 * m16n8k16 exactly:
 *   lane (r = lane / 4, c = lane % 4) holds keys r and r + 8, elements 32 j + 8 c .. + 7 of K: the A operand up to an
 *   order of the contracted elements that Q shares; P^T goes from accumulators to the B operand by movmatrix; V^T's A
 *   operand pairs the keys 2c, 2c+1, 2c+8, 2c+9 of elements 64 j + 8 r .. + 7 by byte permutes, and the accumulators
 *   come out as eight consecutive elements a lane and head.
 *
 * Measured, 16 query heads over 2 kv heads, replayed from a graph: 64 sequences of 1 to 32,768 keys 332 us (6.71 TB/s, the
 * measured copy rate), one of 32,768 keys 19.0 us (67 MB: 10.3 us at that rate; the rest is the lengths' and the tables' way
 * from memory, 2.5 us, the first and last rows' ramp, 2, the warps' meeting, 1, and the join, 3), 32 of 256 to 2,038 keys
 * 20.8 us (77 MB), one of 500 keys 6.4 us. Every CTA of both kernels goes through all lengths: batches of thousands of short
 * sequences pay for that (of 500 keys, 1,024 sequences 4.6 TB/s, 4,096 3.3, 8,192 2.3).
 */
#include <cuda_bf16.h>

#include "common.cuh"
#include "mma.cuh"
#include "ridgefill_serve.h"

namespace {

constexpr int D = 256;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kBlock = 16;                          /* keys a warp takes at a time */
constexpr int kRound = kWarps * kBlock;             /* keys the warps of a CTA take together */
constexpr int kHalfBytes = kBlock * D * 2;          /* a block's keys, or its values */
constexpr int kRing = 3;                            /* halves of a warp's ring */
constexpr int kStart = 4;                           /* a piece's fixed cost, in blocks */
constexpr int kSmem = kWarps * kRing * kHalfBytes;
constexpr int kCtasPerSm = 2;
constexpr float kGrow = 8.0f;                       /* a maximum may be exceeded by 2^8 before the sums are rescaled */
constexpr float kNone = -INFINITY;

/* Query heads a CTA serves at once: 8 NT (NT the n-tiles of 8 heads). */
template <int NT>
struct Partial {                                    /* one piece's result */
    float o[8 * NT][D];
    float2 ml[8 * NT];                              /* maximum (log2 units) and sum of 2^(s - m) */
};

struct Plan {
    RidgeFillAttnDecode g;
    int group, chunks;      /* query heads a kv head; items a kv head (group / heads of an item, rounded up) */
    int ctas, seats;        /* CTAs of the split kernel; how many of them run at a time */
    bool narrow;            /* its grid has CTAs for narrow spans */
    int page_shift;         /* page as a power of two; -1: it is none */
    int parts;              /* CTAs a query head's join */
    void* partials;         /* [ctas][2] Partial; null: one CTA an item, nothing to join */
    float scale_log2;
};

/* Lengths and units are 32-bit: the host refuses a call whose table could hold more (ridgefill_attn_decode_device). */
__device__ __forceinline__ int length_of(const RidgeFillAttnDecode& g, int b) {
    const int most = (int)(g.n_pages * g.page), n = g.lens[b];
    return n < 0 ? 0 : (n > most ? most : n);
}
/* The units of an item of sequence b: kStart for its beginning (what a piece costs beside its keys: its first copies'
 * latency, the warps' meeting at its end), then one a block; none without keys. */
__device__ __forceinline__ int units_of(const RidgeFillAttnDecode& g, int b) {
    const int len = length_of(g, b);
    return len ? kStart + (len + kBlock - 1) / kBlock : 0;
}

__device__ __forceinline__ int warp_sum(int x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t*)&p;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

/* One warp's walk over the 16-key blocks of a piece. */
struct Blocks {
    const uint16_t* keys;      /* cache plane 0 at the item's kv head */
    int len;                   /* the sequence's keys */
    const int32_t* table;      /* its pages */
    int page_shift;            /* as Plan's: a division is 100 cycles before a piece's first row */
};

/* The slot of key `j` (-1: past the sequence, or outside the pool), by the lane that owns it. */
__device__ __forceinline__ int slot_of(const RidgeFillAttnDecode& g, const Blocks& w, int j) {
    if (j >= w.len) return -1;
    const int page = (int)g.page, n = w.page_shift >= 0 ? j >> w.page_shift : j / page;
    const int64_t slot = (int64_t)w.table[n] * page + (j - n * page);
    return slot >= 0 && slot < g.n_slots ? (int)slot : -1;
}

/* The 16-byte chunk in whose place chunk x of a block's row i lies, so that a warp's reads below meet no bank conflict. */
__device__ __forceinline__ constexpr int key_chunk(int i, int x) { return x ^ ((i & 1) << 2); }
__device__ __forceinline__ constexpr int value_chunk(int i, int x) { return x ^ ((i >> 1 & 3) << 1); }

/* The copies of one half (K when !values, else V) of the block whose slots the lanes 0..15 hold in `slots`: a row of 512
 * bytes an instruction, in whole 128-byte lines. */
__device__ __forceinline__ void fetch(const RidgeFillAttnDecode& g, const Blocks& w, int slots, bool values, uint8_t* half, int lane) {
    const uint16_t* plane = w.keys + (values ? g.c_kv : 0) + 8 * lane;
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
        const int s = __shfl_sync(0xffffffffu, slots, i);
        const int at = values ? value_chunk(i, lane) : key_chunk(i, lane);
        rf::cp_async16(half + i * 512 + at * 16, plane + (int64_t)max(s, 0) * g.c_slot, s >= 0 ? 16 : 0);
    }
    rf::cp_async_commit();
}

/* The 16-byte chunk in whose place chunk x of head row h lies where the warps' results meet: lanes write four heads at once. */
__device__ __forceinline__ constexpr int sum_chunk(int h, int x) { return x ^ (h >> 1 & 1) ^ (h & 4); }

/* A piece's keys [from, to) of item (b, kv head, first query head h0, heads), by the whole CTA; its result to the
 * output (`out`) or to `part`. */
template <int NT>
__device__ __forceinline__ void run_piece(const Plan& p, uint8_t* smem, int b, int hkv, int h0, int heads, int from, int to,
                                          Partial<NT>* part) {
    const RidgeFillAttnDecode& g = p.g;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    uint8_t* ring = smem + warp * kRing * kHalfBytes;
    const Blocks w = { g.cache + hkv * g.c_head, length_of(g, b), g.table + b * g.t_row, p.page_shift };
    const int first = from + warp * kBlock;
    const int n = first < to ? (to - first + kRound - 1) / kRound : 0;   /* this warp's blocks */

    /* halves 2 i (keys) and 2 i + 1 (values) of block i go through slot (2 i) % kRing, ... of the ring, kRing - 1 ahead */
    int cur = -1, next = -1;   /* lanes 0..15: the slots of blocks i and i + 1 */
    if (n > 0) {
        cur = slot_of(g, w, first + (lane & 15));
        next = n > 1 ? slot_of(g, w, first + kRound + (lane & 15)) : -1;
        fetch(g, w, cur, false, ring, lane);
        fetch(g, w, cur, true, ring + kHalfBytes, lane);
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t][0] = m[t][1] = kNone;
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }
    /* Q's operand: lane's elements 32 j + 8 c .. + 7 of query heads r (+ 8 a tile); heads past the item's are zero */
    uint4 q[NT][D / 32];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int h = 8 * t + r;
        const uint16_t* src = g.q + b * g.q_row + (int64_t)(hkv * p.group + h0 + h) * g.q_head + 8 * c;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) q[t][j] = h < heads ? *(const uint4*)(src + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
    }
    int at = 0;   /* ring slot of the current half */
    for (int i = 0; i < n; ++i) {
        const int after = i + 2 < n ? slot_of(g, w, first + (i + 2) * kRound + (lane & 15)) : -1;
        /* scores of the block's 16 keys */
        int free_slot = at + 2 >= kRing ? at + 2 - kRing : at + 2;
        __syncwarp();   /* every lane has read the half that lay there */
        if (i + 1 < n) fetch(g, w, next, false, ring + free_slot * kHalfBytes, lane);
        else rf::cp_async_commit();
        rf::cp_async_wait<2>();
        __syncwarp();   /* every lane's copies have landed */
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        const uint8_t* kh = ring + at * kHalfBytes + r * 512;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int x = key_chunk(r, 4 * j + c) * 16;   /* row r + 8 alike */
            const uint4 k0 = *(const uint4*)(kh + x), k1 = *(const uint4*)(kh + 8 * 512 + x);
            const uint32_t a0[4] = { k0.x, k1.x, k0.y, k1.y }, a1[4] = { k0.z, k1.z, k0.w, k1.w };
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                rf::mma_bf16(s[t], a0, q[t][j].x, q[t][j].y);
                rf::mma_bf16(s[t], a1, q[t][j].z, q[t][j].w);
            }
        }
        at = at + 1 == kRing ? 0 : at + 1;
        const bool live0 = __shfl_sync(0xffffffffu, cur, r) >= 0, live1 = __shfl_sync(0xffffffffu, cur, r + 8) >= 0;
        uint32_t phi[NT][2], plo[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            /* heads 2 c and 2 c + 1 of the tile: keys r and r + 8 here, the others across the lanes of one c */
            float x[4], top[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (e < 2 ? live0 : live1) ? s[t][e] * p.scale_log2 : kNone;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = fmaxf(x[e], x[e + 2]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], d));
            }
            /* the maximum is followed only when it has grown by more than kGrow: until then the weights stay below 2^8 */
            const bool grow = top[0] > m[t][0] + kGrow || top[1] > m[t][1] + kGrow;
            if (__any_sync(0xffffffffu, grow)) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float up = fmaxf(m[t][e], top[e]);
                    f[e] = m[t][e] == kNone ? 0.f : exp2_approx(m[t][e] - up);
                    m[t][e] = up;
                    l[t][e] *= f[e];
                }
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    o[t][d][0] *= f[0];
                    o[t][d][1] *= f[1];
                    o[t][d][2] *= f[0];
                    o[t][d][3] *= f[1];
                }
            }
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = x[e] == kNone ? 0.f : exp2_approx(x[e] - m[t][e & 1]);
                l[t][e & 1] += y[e];
            }
            /* p as its bf16 rounding and the bf16 rounding of the rest: 16 bits of it reach the product with v */
            const uint32_t h01 = pack(y[0], y[1]), h23 = pack(y[2], y[3]);
            phi[t][0] = transpose8x8(h01);
            phi[t][1] = transpose8x8(h23);
            plo[t][0] = transpose8x8(pack(y[0] - __uint_as_float(h01 << 16), y[1] - __uint_as_float(h01 & 0xffff0000u)));
            plo[t][1] = transpose8x8(pack(y[2] - __uint_as_float(h23 << 16), y[3] - __uint_as_float(h23 & 0xffff0000u)));
        }
        /* O^T += V^T P^T */
        free_slot = at + 2 >= kRing ? at + 2 - kRing : at + 2;
        __syncwarp();
        if (i + 1 < n) fetch(g, w, next, true, ring + free_slot * kHalfBytes, lane);
        else rf::cp_async_commit();
        rf::cp_async_wait<2>();
        __syncwarp();
        const uint8_t* vh = ring + at * kHalfBytes + 2 * c * 512 + value_chunk(2 * c, r) * 16;   /* keys 2c, 2c+1, 2c+8, 2c+9 alike */
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *(const uint4*)(vh + ((e & 1) + (e >> 1) * 8) * 512 + j * 128);
            const uint32_t* v0 = &v[0].x;
            const uint32_t* v1 = &v[1].x;
            const uint32_t* v2 = &v[2].x;
            const uint32_t* v3 = &v[3].x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t a[4] = { __byte_perm(v0[e], v1[e], 0x5410), __byte_perm(v0[e], v1[e], 0x7632),
                                        __byte_perm(v2[e], v3[e], 0x5410), __byte_perm(v2[e], v3[e], 0x7632) };
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    rf::mma_bf16(o[t][4 * j + e], a, phi[t][0], phi[t][1]);
                    rf::mma_bf16(o[t][4 * j + e], a, plo[t][0], plo[t][1]);
                }
            }
        }
        at = at + 1 == kRing ? 0 : at + 1;
        cur = next;
        next = after;
    }
    rf::cp_async_wait<0>();

    /* the warps' results meet in shared memory (over the rings, once every warp is done with its own) */
    Partial<NT>* mine = (Partial<NT>*)smem;
    static_assert(kWarps * sizeof(Partial<NT>) <= (size_t)kSmem, "the warps' results fit over the rings");
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[t][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int h = 8 * t + 2 * c + e;
            if (r == 0) {
                mine[warp].ml[h] = make_float2(m[t][e], sum);
            }
            /* elements 64 j + 8 r .. + 7 of head h: tiles 4 j .. 4 j + 3, two elements each */
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    *(float4*)&mine[warp].o[h][4 * sum_chunk(h, 16 * j + 2 * r + hf)] =
                        make_float4(o[t][4 * j + 2 * hf][e], o[t][4 * j + 2 * hf][2 + e], o[t][4 * j + 2 * hf + 1][e],
                                    o[t][4 * j + 2 * hf + 1][2 + e]);
        }
    __syncthreads();
    for (int x = threadIdx.x; x < heads * (D / 4); x += kThreads) {
        const int h = x / (D / 4), d = (x % (D / 4)) * 4;
        float top = kNone, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) top = fmaxf(top, mine[i].ml[h].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float2 ml = mine[i].ml[h];
            const float f = ml.x == kNone ? 0.f : exp2_approx(ml.x - top);
            const float4 v = *(const float4*)&mine[i].o[h][4 * sum_chunk(h, d / 4)];
            sum = fmaf(f, ml.y, sum);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
        }
        if (part) {
            *(float4*)&part->o[h][d] = acc;
            if (d == 0) part->ml[h] = make_float2(top, sum);
        } else {
            const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);   /* no key: zeros; a NaN stays one */
            *(uint2*)(g.o + b * g.o_row + (int64_t)(hkv * p.group + h0 + h) * g.o_head + d) =
                make_uint2(pack(acc.x * inv, acc.y * inv), pack(acc.z * inv, acc.w * inv));
        }
    }
    __syncthreads();   /* the results are read before the next piece's copies land */
}

/* The units cut into spans, CTA i taking span i. `seats` CTAs run at a time.
 * With few units: as many CTAs as have one for each of their warps, at most one a seat, equal spans.
 * From kLong units a seat on: SMs do not get equal shares of the memory's rate, so equal spans leave some idle at the
 * end. One wide span a seat takes 7/8 of the units, and twice as many narrow ones follow, which the hardware gives to
 * whichever seat comes free: 332 us for 64 sequences of up to 32,768 keys, 347 with equal spans, 334 with 4/5 and four times
 * as many. A table wide enough for that over short sequences costs the narrow spans' CTAs, which find no work: 25 us for
 * 64 sequences of some 500 keys, 21.5 without them. */
constexpr int kLong = 128, kNarrowPerSeat = 2;
struct Spans {
    int n_wide = 0, wide = 0, n = 0, each = 0, extra = 0;   /* n equal spans after the wide ones, the first `extra` one longer */
    __device__ __forceinline__ Spans(int total, int seats, bool narrow) {
        if (narrow && total / kLong >= seats) {
            n_wide = seats;
            wide = total / seats * 7 / 8;
            n = kNarrowPerSeat * seats;
        } else {
            n = min((total + kWarps - 1) / kWarps, seats);
        }
        const int rest = total - n_wide * wide;
        each = (int)((uint32_t)rest / (uint32_t)n);
        extra = rest - each * n;
    }
    __device__ __forceinline__ int ctas() const { return n_wide + n; }
    __device__ __forceinline__ int first(int i) const {
        if (i <= n_wide) return i * wide;
        i -= n_wide;
        return n_wide * wide + i * each + min(i, extra);
    }
    __device__ __forceinline__ int owner(int u) const {
        if (u < n_wide * wide) return u / wide;
        u -= n_wide * wide;
        const int longer = extra * (each + 1);
        return n_wide + (u < longer ? u / (each + 1) : extra + (u - longer) / each);
    }
};

template <int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) decode_kernel(const Plan p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const RidgeFillAttnDecode& g = p.g;
    const int lane = threadIdx.x & 31;
    const int per_kv = p.chunks, items = (int)g.n_head_kv * per_kv;   /* items of a sequence */
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   /* the join may take its place on the SMs */
    if (!p.partials) {   /* one CTA an item */
        const int b = blockIdx.x / items, it = blockIdx.x - b * items, h0 = it % per_kv * 8 * NT;
        run_piece<NT>(p, smem, b, it / per_kv, h0, min(8 * NT, p.group - h0), 0, length_of(g, b), nullptr);
        return;
    }
    const int B = (int)g.B;
    {   /* the tables' lines on their way to L2 while the lengths come (32 short sequences: 20.9 us against 21.5) */
        const int lines = (int)((g.n_pages + 31) / 32);
        const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
        if (i < (int64_t)B * lines) {
            const int b = (int)((uint32_t)i / (uint32_t)lines), n = (int)i - b * lines;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(g.table + b * g.t_row + 32 * n));
        }
    }
    const int mine = lane < B ? units_of(g, lane) : 0;   /* the first 32 sequences', a lane each */
    int total = mine;
    for (int i = 32 + lane; i < B; i += 32) total += units_of(g, i);
    total = warp_sum(total) * items;
    if (total == 0) return;
    const Spans spans(total, p.seats, p.narrow);
    if ((int)blockIdx.x >= spans.ctas()) return;
    int u = spans.first(blockIdx.x);
    const int end = spans.first(blockIdx.x + 1);
    /* the sequence holding unit u: blocks of 32 sequences, then an inclusive scan inside the block */
    int b = 0, base = 0;
    for (;; b += 32) {
        int sum = b == 0 ? mine * items : b + lane < B ? units_of(g, b + lane) * items : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + sum > u);
        if (past) {
            const int k = __ffs(past) - 1;
            const int before = __shfl_sync(0xffffffffu, sum, k > 0 ? k - 1 : 0);
            b += k;
            base += k > 0 ? before : 0;
            break;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    Partial<NT>* slots = (Partial<NT>*)p.partials + 2 * (int64_t)blockIdx.x;
    while (u < end) {
        const int units = units_of(g, b);
        if (units > 0) {
            int rest = u - base;   /* of this sequence's units * items */
            while (rest < units * items && u < end) {
                const int it = (int)((uint32_t)rest / (uint32_t)units), kv = per_kv == 1 ? it : it / per_kv, h0 = (it - kv * per_kv) * 8 * NT;
                const int u0 = rest - it * units, n = min(units - u0, end - u), len = length_of(g, b);
                const int first = max(u0 - kStart, 0), last = u0 + n - kStart;   /* blocks; none: the item begins in the next span */
                if (last > 0)
                    run_piece<NT>(p, smem, b, kv, h0, min(8 * NT, p.group - h0), first * kBlock, min(last * kBlock, len),
                                  first == 0 && u0 + n == units ? nullptr : slots + (first > 0 ? 0 : 1));
                u += n;
                rest += n;
            }
            base += units * items;
        }
        ++b;
    }
}


struct Sums {   /* four elements of a row's sum, with the maximum and the sum of weights they go by */
    float m = kNone, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
};

/* Adds pieces first, first + step, ... below n to `s`, kFlight pieces' loads in flight. */
template <int NT, int kFlight>
__device__ __forceinline__ void add_pieces(Sums& s, const Partial<NT>* pieces, int first, int step, int n, int row, int d) {
    for (int i0 = first; i0 < n; i0 += kFlight * step) {
        float2 ml[kFlight];
        float4 po[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int i = i0 + k * step;
            const Partial<NT>& x = pieces[2 * min(i, n - 1) + (i == 0 ? 1 : 0)];
            ml[k] = i < n ? x.ml[row] : make_float2(kNone, 0.f);
            po[k] = i < n ? *(const float4*)&x.o[row][d] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float up = s.m;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) up = fmaxf(up, ml[k].x);
        const float f = s.m == kNone ? 0.f : exp2_approx(s.m - up);
        s.l *= f;
        s.o = make_float4(s.o.x * f, s.o.y * f, s.o.z * f, s.o.w * f);
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const float w = ml[k].x == kNone ? 0.f : exp2_approx(ml[k].x - up);
            s.l = fmaf(w, ml[k].y, s.l);
            s.o = make_float4(fmaf(w, po[k].x, s.o.x), fmaf(w, po[k].y, s.o.y), fmaf(w, po[k].z, s.o.z), fmaf(w, po[k].w, s.o.w));
        }
        s.m = up;
    }
}

/* A join CTA with nothing to add leaves at once, but for one: the join's end is what the stream's next kernel waits for, and
 * it must not come before the split's. */
__device__ __forceinline__ void nothing_to_join() {
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

/* The items the split kernel cut. The pieces of an item lie in the slots of the CTAs that own its first to last block:
 * slot 1 of the first, slot 0 of the others. A CTA joins D / kParts elements of one query head of a sequence: groups of
 * threads, four elements a thread, take every so-many-th piece with a running maximum of their own, and meet at the end. */
template <int NT, int kFlight, int kJoinThreads, int kParts>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Plan p) {
    __shared__ float4 sums[kJoinThreads];
    __shared__ float2 stats[kJoinThreads];
    const RidgeFillAttnDecode& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31;
    const int n_head = (int)g.n_head, B = (int)g.B;
    const int part = blockIdx.x % kParts, bh = blockIdx.x / kParts;
    const int b = bh / n_head, h = bh - b * n_head, in_group = h % p.group;
    const int items = (int)g.n_head_kv * p.chunks, it = h / p.group * p.chunks + in_group / (8 * NT), row = in_group % (8 * NT);
    constexpr int lanes = D / 4 / kParts, groups = kJoinThreads / lanes;
    const int group = tid / lanes, d = (part * lanes + tid % lanes) * 4;
    uint16_t* out = g.o + b * g.o_row + (int64_t)h * g.o_head + d;
    const int units = units_of(g, b);
    if (units == 0) {   /* no key: zeros */
        if (group == 0) *(uint2*)out = make_uint2(0u, 0u);
        return nothing_to_join();
    }
    int total = 0, before = 0;
    for (int i = lane; i < B; i += 32) {
        const int n = units_of(g, i);
        total += n;
        before += i < b ? n : 0;
    }
    const Spans spans(warp_sum(total) * items, p.seats, p.narrow);
    const int start = warp_sum(before) * items + it * units;
    const int c0 = spans.owner(start + kStart), n = spans.owner(start + units - 1) - c0 + 1;
    if (n == 1) return nothing_to_join();   /* written by its one CTA */
    asm volatile("griddepcontrol.wait;" ::: "memory");   /* the split kernel is done and its results are visible */
    const Partial<NT>* pieces = (const Partial<NT>*)p.partials + 2 * (int64_t)c0;
    Sums mine;
    add_pieces<NT, kFlight>(mine, pieces, group, groups, n, row, d);
    sums[tid] = mine.o;
    stats[tid] = make_float2(mine.m, mine.l);
    __syncthreads();
    if (group > 0) return;
    float top = kNone, sum = 0.f;
#pragma unroll
    for (int k = 0; k < groups; ++k) top = fmaxf(top, stats[tid + k * lanes].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < groups; ++k) {
        const float2 s = stats[tid + k * lanes];
        const float4 v = sums[tid + k * lanes];
        const float w = s.x == kNone ? 0.f : exp2_approx(s.x - top);
        sum = fmaf(w, s.y, sum);
        acc = make_float4(fmaf(w, v.x, acc.x), fmaf(w, v.y, acc.y), fmaf(w, v.z, acc.z), fmaf(w, v.w, acc.w));
    }
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
    *(uint2*)out = make_uint2(pack(acc.x * inv, acc.y * inv), pack(acc.z * inv, acc.w * inv));
}

/* The split of a parsed call: NT (query heads an item / 8), CTAs and scratch bytes (0: one CTA an item). */
struct Shape {
    int nt, chunks, ctas, seats;
    bool split, narrow;
    int64_t bytes;
};
Shape shape_of(const RidgeFillAttnDecode& g) {
    Shape s;
    const int group = (int)(g.n_head / g.n_head_kv);
    s.nt = group <= 8 ? 1 : 2;
    s.chunks = (group + 8 * s.nt - 1) / (8 * s.nt);
    s.split = g.n_pages * g.page > 2 * kRound;
    s.seats = rf::sm_count() * kCtasPerSm;
    /* whether the tables could hold enough for narrow spans; whether the lengths do is the kernels' to see */
    s.narrow = g.B * g.n_head_kv * s.chunks * (g.n_pages * g.page / kBlock + 1 + kStart) / kLong >= s.seats;
    s.ctas = s.narrow ? (1 + kNarrowPerSeat) * s.seats : s.seats;
    const int64_t one = s.nt == 1 ? (int64_t)sizeof(Partial<1>) : (int64_t)sizeof(Partial<2>);
    s.bytes = s.split ? 2 * one * s.ctas : 0;
    return s;
}

template <int NT>
int launch(const Plan& p, bool split, cudaStream_t s) {
    if (cudaFuncSetAttribute(decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) {
        cudaGetLastError();
        return RAD_E_DEVICE;
    }
    const int64_t grid = split ? p.ctas : p.g.B * p.g.n_head_kv * p.chunks;
    decode_kernel<NT><<<(unsigned)grid, kThreads, kSmem, s>>>(p);
    if (!split) return rf::launch_status();
    const int rc = rf::launch_status();
    if (rc != RAD_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.g.B * p.g.n_head * p.parts));
    /* Loads in flight a thread, threads and CTAs a head, by how many pieces an item may have and how many heads there are,
     * all of whose CTAs should run at once: they wait on the SMs for the split's end. One sequence of 32,768 keys, 148 pieces:
     * 19.0 us with eight CTAs a head and 8 loads, 19.5 with four and 16; of 500 keys, five pieces: 6.4 us with four CTAs and 2
     * loads, 6.8 with eight and 8. Eight sequences of up to 32,768: 17.2 us with four CTAs and 2 loads, 23.8 with eight and 8.
     * 32 short sequences, a few pieces each: 20.8 us with one CTA a head, small, and 5 loads; 21.5 with 4, 22.0 with 8, 21.9
     * with four CTAs; 16 of up to 20,000: 45.6, 60 with eight CTAs. Narrow spans and fewer items than seats, a dozen pieces
     * each: 8 loads, 1 % less than with the small CTAs for 64 long ones. */
    const bool few = p.parts > 1, many = p.narrow && p.g.B * p.g.n_head_kv * p.chunks < p.seats;
    cfg.blockDim = dim3(few || many ? 256 : 128);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, few ? (p.parts == 8 ? join_kernel<NT, 8, 256, 8> : join_kernel<NT, 2, 256, 4>)
                                     : many ? join_kernel<NT, 8, 256, 1> : join_kernel<NT, 5, 128, 1>, p) != cudaSuccess) {
        cudaGetLastError();
        return RAD_E_DEVICE;
    }
    return RAD_OK;
}

}  // namespace

/* Heads (the join's grid) and the units of all items fit 32 bits; others are refused, before their products are formed. */
static bool fits(const RidgeFillAttnDecode& g) {
    if (g.B > 0x7fffffffLL / g.n_head) return false;
    return g.B * g.n_head_kv * shape_of(g).chunks * (g.n_pages * g.page / kBlock + 1 + kStart) <= 0x7fffffffLL;
}

extern "C" int64_t ridgefill_attn_decode_scratch(const RadArgs* a) {
    RidgeFillAttnDecode g;
    return ridgefill_attn_decode_parse(a, &g) == RAD_OK && g.B > 0 && fits(g) ? shape_of(g).bytes : 0;
}

extern "C" int ridgefill_attn_decode_device(const RadArgs* a, RadStream s) {
    Plan p;
    const int rc = ridgefill_attn_decode_parse(a, &p.g);
    if (rc != RAD_OK) return rc;
    if (p.g.B == 0) return RAD_OK;
    if (!fits(p.g)) return RAD_E_SHAPE;
    const Shape sh = shape_of(p.g);
    if (sh.split && (!a->scratch || a->scratch_bytes < sh.bytes || (uintptr_t)a->scratch % 16)) return RAD_E_INVAL;
    p.group = (int)(p.g.n_head / p.g.n_head_kv);
    p.chunks = sh.chunks;
    p.ctas = sh.ctas;
    p.seats = sh.seats;
    p.narrow = sh.narrow;
    p.page_shift = -1;
    for (int i = 0; i <= 20; ++i)
        if (p.g.page == 1 << i) p.page_shift = i;
    /* few heads may have many pieces each, which several CTAs a head share; launch() has the figures */
    const int64_t heads = p.g.B * p.g.n_head;
    p.parts = 8 * heads <= sh.seats && p.g.n_pages * p.g.page > 32 * kRound ? 8 : 4 * heads <= 2 * sh.seats ? 4 : 1;
    p.partials = sh.split ? a->scratch : nullptr;
    p.scale_log2 = p.g.scale * 1.4426950408889634f;
    return sh.nt == 1 ? launch<1>(p, sh.split, rf::as_stream(s)) : launch<2>(p, sh.split, rf::as_stream(s));
}
