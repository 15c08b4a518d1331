/* gdn_step.cu -- ridgefill_gdn_step: the gated delta rule's recurrent form on B200, one new token a row
 * (ridgefill_serve.h holds the formula; ridgefill_gdn_fill is the chunked form of the same rule).
 *
 * HBM-bound: a row's state is read once and written once (8 dv dk bytes a head; 4.2 MB a row at 32 heads of 128 x 128),
 * against 7 dv dk flops. A state row S[v, :] of the rule depends on no other: with a = e^g,
 *     u = beta (v - a S.k),   S' = a S + u k,   o = scale (a S.q + u k.q)
 * so both dot products of a row are taken of the OLD row in one pass, and the new row needs only their sums: one read,
 * one write, no second sweep for o. Eight lanes hold a row (16 columns each at dk 128, 16-byte words 128 bytes apart,
 * so a warp's load covers four rows in whole 128-byte lines); the two sums take three shuffles each. All of a lane's
 * words are loaded before the first is used. Loads and stores go through L2 alone, without the streaming hint, which cost
 * 3 % (169.8 -> 164.8 us at 256 rows of 32 heads). Four warps a CTA: 161 us, 6.70 TB/s, the measured copy rate and a little
 * more; 28.9 us at 27 rows of 48 heads (5.91 TB/s), 2.9 us at one row of 32.
 *
 * Every CTA looks through all rows' slot numbers for one that names the slot it writes, so that part grows with the square of
 * the rows: nothing up to some 500 (512 rows of 32 heads of 128 6.84 TB/s), a few percent at 1,024 (6.27), a third at 4,096
 * (4.04). Heads of up to 32 stay further from the memory's rate (256 rows of 32 heads 2.9 TB/s): a CTA moves 4 KiB each way, two
 * words in flight a lane, for one look through the slots and one barrier; fewer and larger CTAs were not built.
 */
#include <cuda_bf16.h>

#include "common.cuh"
#include "ridgefill_serve.h"

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kLanes = 8;                 /* lanes a state row */
constexpr int kSub = 32 / kLanes;         /* rows a warp holds side by side */

__device__ __forceinline__ void unpack4(uint2 w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x << 16);
    f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16);
    f[3] = __uint_as_float(w.y & 0xffff0000u);
}

__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

/* NJ 16-byte words of a state row a lane (columns 4 l + 32 j), P passes of kSub rows a warp: a CTA takes
 * kWarps * kSub * P state rows of one (row, v-head). */
template <int NJ, int P>
__global__ void __launch_bounds__(kThreads) gdn_step_kernel(const RidgeFillGdnStep g, int parts) {
    const int part = blockIdx.x % parts;
    const int64_t bh = blockIdx.x / parts;
    const int64_t b = bh / g.n_head_v, h = bh - b * g.n_head_v;
    const int64_t src = g.idx[b * g.idx_pitch], dst = g.out_idx ? g.out_idx[b * g.out_pitch] : src;
    if (src < 0 || src >= g.n_states || dst < 0 || dst >= g.n_states) return;   /* the whole CTA */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, sub = lane / kLanes;
    const int dk = (int)g.dk, dv = (int)g.dv;
    const int row0 = (part * kWarps + warp) * kSub * P + sub;
    const float* from = g.state + src * g.st_slot + h * g.st_head;
    float* to = g.state + dst * g.st_slot + h * g.st_head;

    float4 S[P][NJ];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int row = row0 + p * kSub, col = 4 * l + 32 * j;
            S[p][j] = row < dv && col < dk ? __ldcg((const float4*)(from + (int64_t)row * dk + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    /* Another row naming the slot this one writes: the row is skipped (the rows have no order). */
    bool shared = false;
    for (int64_t i = threadIdx.x; i < g.B; i += kThreads)
        if (i != b) {
            const int64_t s = g.idx[i * g.idx_pitch];
            shared |= s == dst || (g.out_idx && g.out_idx[i * g.out_pitch] == dst);
        }
    const int64_t hk = h / (g.n_head_v / g.n_head_k);
    const uint16_t* kp = g.k + b * g.k_row + hk * g.k_head;
    const uint16_t* qp = g.q + b * g.q_row + hk * g.q_head;
    float k[NJ][4], q[NJ][4], kq = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int col = 4 * l + 32 * j;
        unpack4(col < dk ? *(const uint2*)(kp + col) : make_uint2(0u, 0u), k[j]);
        unpack4(col < dk ? *(const uint2*)(qp + col) : make_uint2(0u, 0u), q[j]);
    }
    float v[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int row = row0 + p * kSub;
        v[p] = row < dv ? rf::bf16_bits_to_f32(g.v[b * g.v_row + h * g.v_head + row]) : 0.f;
    }
    const float decay = expf(g.g[b * g.g_row + h]), beta = g.beta[b * g.b_row + h];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) kq = fmaf(k[j][e], q[j][e], kq);
    kq = row_sum(kq);
    if (__syncthreads_or(shared)) return;

    float out = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        float sk = 0.f, sq = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const float s[4] = { S[p][j].x, S[p][j].y, S[p][j].z, S[p][j].w };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sk = fmaf(s[e], k[j][e], sk);
                sq = fmaf(s[e], q[j][e], sq);
            }
        }
        sk = row_sum(sk);
        sq = row_sum(sq);
        const float u = beta * (v[p] - decay * sk);
        const int row = row0 + p * kSub;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int col = 4 * l + 32 * j;
            const float4 n = make_float4(fmaf(u, k[j][0], decay * S[p][j].x), fmaf(u, k[j][1], decay * S[p][j].y),
                                         fmaf(u, k[j][2], decay * S[p][j].z), fmaf(u, k[j][3], decay * S[p][j].w));
            if (row < dv && col < dk) __stcg((float4*)(to + (int64_t)row * dk + col), n);
        }
        if (l == p) out = g.scale * fmaf(u, kq, decay * sq);   /* lane p of a row group keeps pass p's o */
    }
    const int row = row0 + l * kSub;
    if (l < P && row < dv) g.o[b * g.o_row + h * g.o_head + row] = rf::f32_to_bf16_bits(out);
}

template <int NJ, int P>
int launch(const RidgeFillGdnStep& g, cudaStream_t s) {
    constexpr int rows = kWarps * kSub * P;
    const int64_t parts = (g.dv + rows - 1) / rows, ctas = g.B * g.n_head_v * parts;
    if (ctas > 0x7fffffffLL) return RAD_E_SHAPE;
    gdn_step_kernel<NJ, P><<<(unsigned)ctas, kThreads, 0, s>>>(g, (int)parts);
    return rf::launch_status();
}

}  // namespace

extern "C" int ridgefill_gdn_step_device(const RadArgs* a, RadStream s) {
    RidgeFillGdnStep g;
    const int rc = ridgefill_gdn_step_parse(a, &g);
    if (rc != RAD_OK) return rc;
    if (g.B == 0) return RAD_OK;
    if (g.B > 0x7fffffffLL / g.n_head_v) return RAD_E_SHAPE;   /* so that no product of extents below passes 64 bits */
    cudaStream_t stream = rf::as_stream(s);
    /* Several state rows a lane in flight stream best (256 rows of 32 heads: of 128, 161 us with 64-row CTAs, 208 with 16-row
     * ones; of 64, 48 us with 32-row ones, 77 with 16; of 32, 24 and 38); while a head an SM would leave SMs idle, 16-row CTAs
     * spread a head over more of them */
    const bool spread = g.B * g.n_head_v <= rf::sm_count();
    if (g.dk <= 32) return spread ? launch<1, 1>(g, stream) : launch<1, 2>(g, stream);
    if (g.dk <= 64) return spread ? launch<2, 1>(g, stream) : launch<2, 2>(g, stream);
    if (spread) return launch<4, 1>(g, stream);
    return launch<4, 4>(g, stream);
}
