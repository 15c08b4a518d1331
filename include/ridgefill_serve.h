/* ridgefill_serve.h -- the serving rows: what a program runs over the caches that the fill rows write. Attention of a
 * prompt's exact rows, attention of one new token over the paged K/V cache, and the DeltaNet layers' step for one new
 * token. No counterpart in the reference: its engine answers with its own attention and recurrent kernels, whose
 * source is not part of the checkout; here they read what ridgefill_attn_kv_fill and ridgefill_gdn_fill wrote.
 *
 * The rows are described by the plugin's own types (RadOpSchema, RadKernelInfo) and called like every row: RadArgs
 * with operands in schema order, a cudaStream_t, a workspace where the row's scratch hook asks for one. They stand in
 * a table of their own beside the plugin's, whose op list is the reference plugin's and its fill ops': a program that
 * serves reads both (ridgefill_serve_count / _at).
 *
 * Every row launches on the stream it is given, allocates nothing and never synchronises; calls may be captured into
 * a graph. Values in device memory (lengths, page and slot numbers) are read where the kernel runs, with a fail-safe:
 * cu_seqlens and lengths are clamped into their operands, a page or slot outside its pool is not read or written.
 * A call's workspace is its own until the call has run: calls that may overlap on the GPU need one each.
 * Every address is a multiple of its element's size at least (of 16 bytes where a row is read in words: the parses say where).
 * An operand with an extent of 0 still carries an address: one without it counts as not given.
 */
#ifndef RIDGEFILL_SERVE_H
#define RIDGEFILL_SERVE_H

#include "ridgefill.h"

/* Operand positions. ridgefill_attn_prefill: */
enum { AP_Q = 0, AP_K, AP_V, AP_CU_Q, AP_CU_K, AP_O };
/* ridgefill_attn_decode */
enum { AD_Q = 0, AD_CACHE, AD_TABLE, AD_LENS, AD_O };
/* ridgefill_gdn_step */
enum { GS_Q = 0, GS_K, GS_V, GS_G, GS_BETA, GS_STATE, GS_STATE_IDX, GS_OUT_IDX, GS_O };

/* ridgefill_attn_prefill: causal attention over packed prompts. Sequence i holds the rows [cu_q[i], cu_q[i+1]) of q and
 * the rows [cu_k[i], cu_k[i+1]) of k and v (cu_q's without cu_k); with nq and nk of them, row r (0 <= r < nq) sees the
 * keys 0 .. nk - nq + r: the queries are the sequence's last rows, all of a prompt or its tail. Query head h reads kv
 * head h / (Hq / Hkv):
 *     o[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[r, h] . k_j)
 * zeros for a row that sees no key; rows outside every sequence are not written. The products q . k are exact bf16
 * products summed in f32; p is rounded to bf16 for the product with v and summed in f32; o is rounded once. A value of v
 * that is not finite reaches the rows that see it and may reach earlier rows of its own sequence, those whose last key lies
 * up to 126 + 256 / (Hq / Hkv) before it (they share a query tile and a key tile with rows that see its neighbours, and
 * their weight for it is zero); no row that sees no key, and no row of another sequence. */
typedef struct RidgeFillAttnPrefill {
    const uint16_t* q;       int64_t q_row, q_head;              /* [T, Hq, D] */
    const uint16_t* k;       int64_t k_row, k_head;              /* [Tk, Hkv, D] */
    const uint16_t* v;       int64_t v_row, v_head;              /* [Tk, Hkv, D] */
    const int32_t*  cu_q;    const int32_t* cu_k;                /* [n_seq + 1] */
    uint16_t*       o;       int64_t o_row, o_head;              /* [T, Hq, D] */
    int64_t         T, Tk, n_seq, n_head, n_head_kv, head_dim;
    float           scale;
} RidgeFillAttnPrefill;

/* ridgefill_attn_decode: one new token a sequence over the paged cache. Sequence i's key j (0 <= j < lens[i]) lies in
 * slot table[i, j / page] * page + j % page of cache [2, slots, Hkv, D]; query head h reads kv head h / (Hq / Hkv):
 *     o[i, h] = sum_j p_j cache[1, slot_j] / sum_j p_j,   p_j = exp(scale q[i, h] . cache[0, slot_j])
 * over the keys whose slot lies in [0, slots); zeros when there is none. The products q . k are exact bf16 products
 * summed in f32; p is held in f32 for the sum and as a bf16 pair (its rounding and the rest) for the product with v. */
typedef struct RidgeFillAttnDecode {
    const uint16_t* q;       int64_t q_row, q_head;              /* [B, Hq, D] */
    const uint16_t* cache;   int64_t c_kv, c_slot, c_head, n_slots;   /* [2, slots, Hkv, D] */
    const int32_t*  table;   int64_t t_row, n_pages;             /* [B, n_pages] */
    const int32_t*  lens;                                        /* [B] */
    uint16_t*       o;       int64_t o_row, o_head;              /* [B, Hq, D] */
    int64_t         B, n_head, n_head_kv, head_dim, page;
    float           scale;
} RidgeFillAttnDecode;

/* ridgefill_gdn_step: the gated delta rule for one new token a row (ridgefill_gdn_fill's rule on one-row sequences).
 * Per row i and v-head h (k-head h / (Hv / Hk)), S the state in slot idx[i]:
 *     S <- exp(g[i, h]) S;  S <- S + beta[i, h] (v - S k) k^T;  o[i, h] = scale S q
 * the new S written to slot out_idx[i] (idx[i] without out_idx), in f32 throughout, o rounded once to bf16. A row is
 * skipped -- no state and no o written -- when one of its slots lies outside the pool, or when the slot it would
 * write is named by another row (written or read by it): rows that share a slot have no order among themselves. To see
 * that, all B slot numbers are read for every head of every row: meant for batches of hundreds of rows (at 4,096 rows of 32
 * heads of 128 the call runs at 0.6 of its rate at 512). */
typedef struct RidgeFillGdnStep {
    const uint16_t* q;       int64_t q_row, q_head;              /* [B, Hk, dk] */
    const uint16_t* k;       int64_t k_row, k_head;              /* [B, Hk, dk] */
    const uint16_t* v;       int64_t v_row, v_head;              /* [B, Hv, dv] */
    const float*    g;       int64_t g_row;                      /* [B, Hv] */
    const float*    beta;    int64_t b_row;
    float*          state;   int64_t st_slot, st_head, n_states; /* [slots, Hv, dv, dk] */
    const int32_t*  idx;     int64_t idx_pitch;
    const int32_t*  out_idx; int64_t out_pitch;                  /* null: in place */
    uint16_t*       o;       int64_t o_row, o_head;              /* [B, Hv, dv] */
    int64_t         B, n_head_k, n_head_v, dk, dv;
    float           scale;
} RidgeFillGdnStep;

#ifdef __cplusplus
extern "C" {
#endif

/* The serving rows' schemas and rows (null past the end). */
int                  ridgefill_serve_schema_count(void);
const RadOpSchema*   ridgefill_serve_schema_at(int i);
int                  ridgefill_serve_count(void);
const RadKernelInfo* ridgefill_serve_at(int i);

/* Parses: RAD_OK or a named refusal (null operands and missing parameters RAD_E_INVAL, types RAD_E_DTYPE, ranks and
 * extents RAD_E_SHAPE, strides and alignment RAD_E_STRIDE, geometry no kernel serves RAD_E_UNSUPPORTED). */
int ridgefill_attn_prefill_parse(const RadArgs* a, RidgeFillAttnPrefill* out);
int ridgefill_attn_decode_parse(const RadArgs* a, RidgeFillAttnDecode* out);
int ridgefill_gdn_step_parse(const RadArgs* a, RidgeFillGdnStep* out);

/* The device rows: async launches on `s` (a cudaStream_t); no allocation, no synchronisation. */
int ridgefill_attn_prefill_device(const RadArgs* a, RadStream s);
int ridgefill_attn_decode_device(const RadArgs* a, RadStream s);
int ridgefill_gdn_step_device(const RadArgs* a, RadStream s);

/* Scratch hooks: device bytes the call needs in RadArgs::scratch (16-byte aligned); 0: none. */
int64_t ridgefill_attn_prefill_scratch(const RadArgs* a);
int64_t ridgefill_attn_decode_scratch(const RadArgs* a);

/* Failure-detection self-test, as ridgefill_wait_selftest: launches, on stream `s`, one kernel whose warp waits as the
 * prompt attention's warps do, half of its lanes for a barrier phase that is complete and half for one that nothing
 * completes. The wait gives up after its limit (2 s), records its code for ridgefill_device_error and answers alike in
 * every lane: status[0 .. 31] (device memory) are 0. RAD_E_INVAL on a null pointer. */
int ridgefill_attn_wait_selftest(int* status, RadStream s);

#ifdef __cplusplus
}
#endif

#endif /* RIDGEFILL_SERVE_H */
