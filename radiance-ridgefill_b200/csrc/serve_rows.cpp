/* serve_rows.cpp -- the serving rows' table (ridgefill_serve.h): their schemas, operand checks and cold-call
 * descriptions, in the plugin's own types. Every row is a DEVICE row (sm_100a CUDA); there are no host rows and no
 * fallback. Each parse reads descriptors only: values in device memory are checked where the kernel reads them.
 */
#include "ridgefill_serve.h"
#include "ridgefill_schemas.h"

#include <cmath>
#include <initializer_list>

using namespace ridgefill_schema;

namespace {

bool packed(const RadTensor* t) { return rad_tensor_is_contiguous(t) != 0; }

/* `t` is of rank shape.size() and has these extents. */
bool is(const RadTensor* t, std::initializer_list<int64_t> shape) {
    if (t->rank != shape.size()) return false;
    uint32_t i = 0;
    for (int64_t e : shape)
        if (t->shape[i++] != e) return false;
    return true;
}

/* Head rows a kernel reads or writes in 16-byte words: a dense last axis, every other stride and the base a multiple
 * of 16 bytes. An axis of extent 1 is never stepped along, so its stride may be anything. */
bool word_rows(const RadTensor* t) {
    if (t->stride[t->rank - 1] != 1 || (uintptr_t)t->data % 16) return false;
    for (uint32_t i = 0; i + 1 < t->rank; ++i)
        if (t->shape[i] > 1 && (t->stride[i] * 2) % 16) return false;
    return true;
}

/* The base is a multiple of the element's `bytes`: what a kernel reads or writes element by element. */
bool aligned(const RadTensor* t, unsigned bytes) { return (uintptr_t)t->data % bytes == 0; }

/* A slot index operand of `n` rows: i32 [n] or [n, >= 1], its last axis dense. */
int slot_rows(const RadTensor* t, int64_t n, int64_t* pitch) {
    if (t->dtype != RAD_I32) return RAD_E_DTYPE;
    if ((t->rank != 1 && t->rank != 2) || t->shape[0] != n || (t->rank == 2 && t->shape[1] < 1)) return RAD_E_SHAPE;
    if ((t->shape[t->rank - 1] > 1 && t->stride[t->rank - 1] != 1) || !aligned(t, 4)) return RAD_E_STRIDE;
    *pitch = t->rank == 1 ? 1 : t->stride[0];
    return RAD_OK;
}

/* The optional `scale` parameter: 1 / sqrt(d) unless given; false when it is not a finite number (`positive`: above 0, and
 * finite in the attention kernels' powers of two). */
bool scale_of(const RadArgs* a, int64_t d, bool positive, float* out) {
    const double s = rad_args_getf_or(a, "scale", 1.0 / std::sqrt((double)d));
    *out = (float)s;
    return std::isfinite(*out) && (!positive || (*out > 0.0f && std::isfinite(*out * 1.4426950408889634f)));
}

/* ------------------------------------------------------------------ schemas */

const RadParamSpec pPrefill[] = { RF_P_INT("M"), RF_P_INT("n_head"), RF_P_INT("n_head_kv"), RF_P_INT("head_dim"),
                                  RF_P_OPT("scale", RAD_P_F64) };
const RadOperandSpec oPrefill[] = { RF_IN("q"), RF_IN("k"), RF_IN("v"), RF_IN("cu_seqlens"), RF_IN_OPT("cu_keys"), RF_OUT("o") };
const RadParamSpec pDecode[] = { RF_P_INT("M"), RF_P_INT("n_head"), RF_P_INT("n_head_kv"), RF_P_INT("head_dim"),
                                 RF_P_INT("page"), RF_P_OPT("scale", RAD_P_F64) };
const RadOperandSpec oDecode[] = { RF_IN("q"), RF_IN("kv_cache"), RF_IN("block_table"), RF_IN("kv_lens"), RF_OUT("o") };
const RadParamSpec pStep[] = { RF_P_INT("M"), RF_P_INT("n_head_k"), RF_P_INT("n_head_v"), RF_P_INT("head_k"),
                               RF_P_INT("head_v"), RF_P_OPT("scale", RAD_P_F64) };
const RadOperandSpec oStep[] = { RF_IN("q"), RF_IN("k"), RF_IN("v"), RF_IN("g"), RF_IN("beta"), RF_INOUT("state"),
                                 RF_IN("state_idx"), RF_IN_OPT("out_idx"), RF_OUT("o") };

const RadOpSchema kServeSchemas[] = {
{ "ridgefill_attn_prefill", RF_ARR(pPrefill), RF_ARR(oPrefill),
  "Causal attention over packed prompts: sequence i holds rows [cu_seqlens[i], cu_seqlens[i + 1]) of q and rows "
  "[cu_keys[i], cu_keys[i + 1]) of k and v (cu_seqlens' without cu_keys); with nq and nk of them, row r and query head h "
  "(kv head h / (n_head / n_head_kv)) give o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j), over the keys j <= "
  "nk - nq + r (the queries are the sequence's last rows); zeros for a row that sees no key, rows outside every sequence "
  "are not written. scale 1 / sqrt(head_dim) unless given, above 0. q and o bf16 [M, n_head, head_dim], k and v bf16 "
  "[keys, n_head_kv, head_dim]. head_dim 256." },
{ "ridgefill_attn_decode", RF_ARR(pDecode), RF_ARR(oDecode),
  "Attention of one new token a sequence over the paged cache ridgefill_attn_kv_fill writes: for sequence i (M of them) "
  "and query head h (kv head h / (n_head / n_head_kv)), o[i, h] = sum_j p_j v_j / sum_j p_j with p_j = exp(scale "
  "q[i, h] . k_j) over j < kv_lens[i] (clamped into [0, n_pages * page]), key j in slot block_table[i, j / page] * page "
  "+ j % page of kv_cache bf16 [2, slots, n_head_kv, head_dim]; keys whose slot lies outside the pool are left out, and "
  "a row without any key is zero. scale 1 / sqrt(head_dim) unless given, above 0. q and o bf16 [M, n_head, head_dim], block_table "
  "i32 [M, n_pages], kv_lens i32 [M]. head_dim 256." },
{ "ridgefill_gdn_step", RF_ARR(pStep), RF_ARR(oStep),
  "The gated delta rule for one new token a row (ridgefill_gdn_fill's rule on one-row sequences): per row i of M and "
  "v-head h (k-head h / (n_head_v / n_head_k)), S = state[state_idx[i], h]: S = exp(g) S; S += beta (v - S k) k^T; "
  "o[i, h] = scale S q; the new S goes to slot out_idx[i] (absent: state_idx[i]). A row with a slot outside the pool, "
  "or whose written slot another row names, is skipped (no state and no o written). state f32 [slots, n_head_v, head_v, "
  "head_k], q and k bf16 [M, n_head_k, head_k], v and o bf16 [M, n_head_v, head_v], g (log decay) and beta f32 "
  "[M, n_head_v]; scale 1 / sqrt(head_k) unless given." },
};

/* ------------------------------------------------------------------ cold-call descriptions */

int shape_prefill(const RadParam* p, int n_p, int operand, RadOpdDesc* out) {
    const int64_t T = dim(p, n_p, "M"), h = dim(p, n_p, "n_head"), hkv = dim(p, n_p, "n_head_kv"), D = dim(p, n_p, "head_dim");
    return pick(out, operand, { opd(RAD_BF16, { T, h, D }), opd(RAD_BF16, { T, hkv, D }), opd(RAD_BF16, { T, hkv, D }),
                                opd_idx({ 2 }, T, RAD_OPD_F_IDX_CU), opd_absent(), opd(RAD_BF16, { T, h, D }) });
}

int shape_decode(const RadParam* p, int n_p, int operand, RadOpdDesc* out) {
    const int64_t B = dim(p, n_p, "M"), h = dim(p, n_p, "n_head"), hkv = dim(p, n_p, "n_head_kv");
    const int64_t D = dim(p, n_p, "head_dim"), page = dim(p, n_p, "page"), pages = 4;
    return pick(out, operand, { opd(RAD_BF16, { B, h, D }), opd(RAD_BF16, { 2, B * pages * page, hkv, D }),
                                opd_idx({ B, pages }, B * pages), opd_idx({ B }, pages * page), opd(RAD_BF16, { B, h, D }) });
}

int shape_step(const RadParam* p, int n_p, int operand, RadOpdDesc* out) {
    const int64_t B = dim(p, n_p, "M"), hk = dim(p, n_p, "n_head_k"), hv = dim(p, n_p, "n_head_v");
    const int64_t dk = dim(p, n_p, "head_k"), dv = dim(p, n_p, "head_v"), slots = B + 2;
    return pick(out, operand, { opd(RAD_BF16, { B, hk, dk }), opd(RAD_BF16, { B, hk, dk }), opd(RAD_BF16, { B, hv, dv }),
                                opd(RAD_F32, { B, hv }, RAD_FILL_SIGMOID), opd(RAD_F32, { B, hv }, RAD_FILL_SIGMOID),
                                opd(RAD_F32, { slots, hv, dv, dk }), opd_idx({ B }, slots, RAD_OPD_F_IDX_UNIQUE),
                                opd_absent(), opd(RAD_BF16, { B, hv, dv }) });
}

/* ------------------------------------------------------------------ rows */

#define SERVE_ROW(nm, op, what, shp, dts, fn, scratchfn, shapefn)                                                        \
    { nm, op, "ridgefill", what, shp, dts, RAD_DOMAIN_DEVICE, 0, nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, fn,  \
      nullptr, scratchfn, nullptr, shapefn, nullptr, nullptr, nullptr, nullptr }

const RadKernelInfo kServeRows[] = {
    SERVE_ROW("ridgefill_attn_prefill_sm100", "ridgefill_attn_prefill",
              "tcgen05 kind::f16 over CTA pairs into tensor memory, TMA-fed: 2 x 128 rows (all query heads of a kv head side by "
              "side) x 128 keys a tile, the weights back into tensor memory as the second product's operand; persistent pairs take "
              "query tiles, longest first up to 32 sequences, else in the batch's order; few over long keys split and joined",
              "head_dim 256, up to 128 query heads a kv head", "bf16 q / k / v / o, i32 cu_seqlens / cu_keys",
              ridgefill_attn_prefill_device, ridgefill_attn_prefill_scratch, shape_prefill),
    SERVE_ROW("ridgefill_attn_decode_sm100", "ridgefill_attn_decode",
              "the keys of all sequences split evenly over the SMs, each warp streaming its 16-key blocks through its own "
              "shared-memory ring into mma.sync; the pieces of a sequence joined by a second kernel",
              "head_dim 256, any page size, up to 128 query heads a kv head", "bf16 q / cache / o, i32 table / lens",
              ridgefill_attn_decode_device, ridgefill_attn_decode_scratch, shape_decode),
    SERVE_ROW("ridgefill_gdn_step_sm100", "ridgefill_gdn_step",
              "8 lanes a state row, a head's rows in flight at once, one read and one write of the state",
              "head dims 128, or at most 64", "bf16 q / k / v / o, f32 g / beta / state, i32 slots",
              ridgefill_gdn_step_device, nullptr, shape_step),
};

}  // namespace

extern "C" int ridgefill_serve_schema_count(void) { return (int)(sizeof kServeSchemas / sizeof kServeSchemas[0]); }
extern "C" const RadOpSchema* ridgefill_serve_schema_at(int i) {
    return i >= 0 && i < ridgefill_serve_schema_count() ? &kServeSchemas[i] : nullptr;
}
extern "C" int ridgefill_serve_count(void) { return (int)(sizeof kServeRows / sizeof kServeRows[0]); }
extern "C" const RadKernelInfo* ridgefill_serve_at(int i) {
    return i >= 0 && i < ridgefill_serve_count() ? &kServeRows[i] : nullptr;
}

/* ------------------------------------------------------------------ parses */

/* ridgefill_attn_prefill: q and o bf16 [T, Hq, 256], k and v bf16 [Tk, Hkv, 256] (dense head rows, bases and other strides
 * multiples of 16 bytes; q, k and v are read through tensor maps: strides positive and below 2^40 bytes), cu_seqlens and
 * cu_keys i32 [n_seq + 1] dense. Hq a multiple of Hkv, at most 128 query heads a kv head. */
extern "C" int ridgefill_attn_prefill_parse(const RadArgs* a, RidgeFillAttnPrefill* g) {
    *g = RidgeFillAttnPrefill{};
    const RadTensor* Q = rad_arg_in(a, AP_Q);
    const RadTensor* K = rad_arg_in(a, AP_K);
    const RadTensor* V = rad_arg_in(a, AP_V);
    const RadTensor* CQ = rad_arg_in(a, AP_CU_Q);
    const RadTensor* CK = rad_arg_in(a, AP_CU_K);
    const RadTensor* O = rad_arg_in(a, AP_O);
    long long T = 0, h = 0, hkv = 0, D = 0;
    if (!Q || !K || !V || !CQ || !O || !rad_args_geti(a, "M", &T) || !rad_args_geti(a, "n_head", &h) ||
        !rad_args_geti(a, "n_head_kv", &hkv) || !rad_args_geti(a, "head_dim", &D))
        return RAD_E_INVAL;
    if (D != 256) return RAD_E_UNSUPPORTED;
    if (!scale_of(a, D, true, &g->scale)) return RAD_E_INVAL;
    if (Q->dtype != RAD_BF16 || K->dtype != RAD_BF16 || V->dtype != RAD_BF16 || O->dtype != RAD_BF16 || CQ->dtype != RAD_I32 ||
        (CK && CK->dtype != RAD_I32))
        return RAD_E_DTYPE;
    if (T < 0 || h <= 0 || hkv <= 0) return RAD_E_SHAPE;
    if (h % hkv != 0 || h / hkv > 128) return RAD_E_UNSUPPORTED;
    const int64_t most = 0x7ffffe00LL;   /* rows and keys together, with a tile's to spare, in 32 bits */
    if (!is(Q, { T, h, D }) || !is(O, { T, h, D }) || K->rank != 3 || !is(K, { K->shape[0], hkv, D }) || K->shape[0] < 0 ||
        !is(V, { K->shape[0], hkv, D }) || T > most || K->shape[0] > most - T)
        return RAD_E_SHAPE;
    if (CQ->rank != 1 || CQ->shape[0] < 1 || CQ->shape[0] > 1 << 24 || (CK && !is(CK, { CQ->shape[0] }))) return RAD_E_SHAPE;
    if (!word_rows(Q) || !word_rows(K) || !word_rows(V) || !word_rows(O) || !packed(CQ) || (CK && !packed(CK)) || !aligned(CQ, 4) ||
        (CK && !aligned(CK, 4)))
        return RAD_E_STRIDE;
    for (const RadTensor* t : { Q, K, V })
        for (int i = 0; i < 2; ++i)
            if (t->shape[i] > 1 && (t->stride[i] <= 0 || t->stride[i] >= 1LL << 39)) return RAD_E_STRIDE;
    g->q = (const uint16_t*)Q->data;
    g->q_row = Q->stride[0];
    g->q_head = Q->stride[1];
    g->k = (const uint16_t*)K->data;
    g->k_row = K->stride[0];
    g->k_head = K->stride[1];
    g->v = (const uint16_t*)V->data;
    g->v_row = V->stride[0];
    g->v_head = V->stride[1];
    g->cu_q = (const int32_t*)CQ->data;
    g->cu_k = CK ? (const int32_t*)CK->data : g->cu_q;
    g->o = (uint16_t*)O->data;
    g->o_row = O->stride[0];
    g->o_head = O->stride[1];
    g->T = T;
    g->Tk = K->shape[0];
    g->n_seq = CQ->shape[0] - 1;
    g->n_head = h;
    g->n_head_kv = hkv;
    g->head_dim = D;
    return RAD_OK;
}

/* ridgefill_attn_decode: q and o bf16 [B, Hq, 256], cache bf16 [2, slots, Hkv, 256] (all read in 16-byte words: dense
 * head rows, bases and other strides multiples of 16 bytes), block_table i32 [B, n_pages] (any row pitch), kv_lens i32
 * [B] dense. Hq a multiple of Hkv, at most 128 query heads a kv head. */
extern "C" int ridgefill_attn_decode_parse(const RadArgs* a, RidgeFillAttnDecode* g) {
    *g = RidgeFillAttnDecode{};
    const RadTensor* Q = rad_arg_in(a, AD_Q);
    const RadTensor* C = rad_arg_in(a, AD_CACHE);
    const RadTensor* T = rad_arg_in(a, AD_TABLE);
    const RadTensor* L = rad_arg_in(a, AD_LENS);
    const RadTensor* O = rad_arg_in(a, AD_O);
    long long B = 0, h = 0, hkv = 0, D = 0, page = 0;
    if (!Q || !C || !T || !L || !O || !rad_args_geti(a, "M", &B) || !rad_args_geti(a, "n_head", &h) ||
        !rad_args_geti(a, "n_head_kv", &hkv) || !rad_args_geti(a, "head_dim", &D) || !rad_args_geti(a, "page", &page))
        return RAD_E_INVAL;
    if (D != 256) return RAD_E_UNSUPPORTED;
    if (!scale_of(a, D, true, &g->scale)) return RAD_E_INVAL;
    if (Q->dtype != RAD_BF16 || C->dtype != RAD_BF16 || T->dtype != RAD_I32 || L->dtype != RAD_I32 || O->dtype != RAD_BF16)
        return RAD_E_DTYPE;
    if (B < 0 || B > 0x7fffffffLL || h <= 0 || hkv <= 0 || page <= 0 || page > 1 << 20) return RAD_E_SHAPE;
    if (h % hkv != 0 || h / hkv > 128) return RAD_E_UNSUPPORTED;
    if (!is(Q, { B, h, D }) || !is(O, { B, h, D }) || !is(L, { B })) return RAD_E_SHAPE;
    if (C->rank != 4 || !is(C, { 2, C->shape[1], hkv, D }) || C->shape[1] < 0 || C->shape[1] > 0x7fffffffLL) return RAD_E_SHAPE;
    if (T->rank != 2 || T->shape[0] != B || T->shape[1] < 0 || T->shape[1] > 0x7fffff00LL / page) return RAD_E_SHAPE;
    if (!word_rows(Q) || !word_rows(C) || !word_rows(O) || !packed(L) || (T->shape[1] > 1 && T->stride[1] != 1) ||
        !aligned(T, 4) || !aligned(L, 4))
        return RAD_E_STRIDE;
    g->q = (const uint16_t*)Q->data;
    g->q_row = Q->stride[0];
    g->q_head = Q->stride[1];
    g->cache = (const uint16_t*)C->data;
    g->c_kv = C->stride[0];
    g->c_slot = C->stride[1];
    g->c_head = C->stride[2];
    g->n_slots = C->shape[1];
    g->table = (const int32_t*)T->data;
    g->t_row = T->stride[0];
    g->n_pages = T->shape[1];
    g->lens = (const int32_t*)L->data;
    g->o = (uint16_t*)O->data;
    g->o_row = O->stride[0];
    g->o_head = O->stride[1];
    g->B = B;
    g->n_head = h;
    g->n_head_kv = hkv;
    g->head_dim = D;
    g->page = page;
    return RAD_OK;
}

/* ridgefill_gdn_step: q, k bf16 [B, Hk, dk], v, o bf16 [B, Hv, dv] (last axis dense; q, k, v rows 16-byte aligned), g
 * and beta f32 [B, Hv] (any row pitch), state f32 [slots, Hv, dv, dk] (slot and head strides free and 16-byte aligned,
 * the [dv, dk] plane packed), state_idx and out_idx i32 [B] or [B, >= 1]. Head dims as ridgefill_gdn_fill serves them:
 * 128, or at most 64 with dk a multiple of 8. Hv a multiple of Hk. */
extern "C" int ridgefill_gdn_step_parse(const RadArgs* a, RidgeFillGdnStep* g) {
    *g = RidgeFillGdnStep{};
    const RadTensor* Q = rad_arg_in(a, GS_Q);
    const RadTensor* K = rad_arg_in(a, GS_K);
    const RadTensor* V = rad_arg_in(a, GS_V);
    const RadTensor* G = rad_arg_in(a, GS_G);
    const RadTensor* Be = rad_arg_in(a, GS_BETA);
    const RadTensor* S = rad_arg_in(a, GS_STATE);
    const RadTensor* I = rad_arg_in(a, GS_STATE_IDX);
    const RadTensor* W = rad_arg_in(a, GS_OUT_IDX);
    const RadTensor* O = rad_arg_in(a, GS_O);
    long long B = 0, hk = 0, hv = 0, dk = 0, dv = 0;
    if (!Q || !K || !V || !G || !Be || !S || !I || !O || !rad_args_geti(a, "M", &B) || !rad_args_geti(a, "n_head_k", &hk) ||
        !rad_args_geti(a, "n_head_v", &hv) || !rad_args_geti(a, "head_k", &dk) || !rad_args_geti(a, "head_v", &dv))
        return RAD_E_INVAL;
    const bool wide = dk == 128 && dv == 128, small = dk >= 8 && dk <= 64 && dk % 8 == 0 && dv >= 1 && dv <= 64;
    if (hk <= 0 || hv <= 0 || hv % hk != 0 || !(wide || small)) return RAD_E_UNSUPPORTED;
    if (!scale_of(a, dk, false, &g->scale)) return RAD_E_INVAL;
    if (Q->dtype != RAD_BF16 || K->dtype != RAD_BF16 || V->dtype != RAD_BF16 || G->dtype != RAD_F32 ||
        Be->dtype != RAD_F32 || S->dtype != RAD_F32 || O->dtype != RAD_BF16)
        return RAD_E_DTYPE;
    if (B < 0) return RAD_E_SHAPE;
    int64_t ip = 0, wp = 0;
    int rc = slot_rows(I, B, &ip);
    if (rc == RAD_OK && W) rc = slot_rows(W, B, &wp);
    if (rc != RAD_OK) return rc;
    if (!is(Q, { B, hk, dk }) || !is(K, { B, hk, dk }) || !is(V, { B, hv, dv }) || !is(O, { B, hv, dv }) ||
        !is(G, { B, hv }) || !is(Be, { B, hv }) || S->rank != 4 || !is(S, { S->shape[0], hv, dv, dk }) || S->shape[0] < 0)
        return RAD_E_SHAPE;
    const bool small_head = dv > 1 && S->stride[2] != dk;   /* the plane's rows are not packed */
    if (!word_rows(Q) || !word_rows(K) || O->stride[2] != 1 || V->stride[2] != 1 || (hv > 1 && (G->stride[1] != 1 || Be->stride[1] != 1)) ||
        !aligned(V, 2) || !aligned(O, 2) || !aligned(G, 4) || !aligned(Be, 4) || S->stride[3] != 1 || small_head || !aligned(S, 16) ||
        (S->shape[0] > 1 && S->stride[0] % 4) || (hv > 1 && S->stride[1] % 4))
        return RAD_E_STRIDE;
    g->q = (const uint16_t*)Q->data;
    g->q_row = Q->stride[0];
    g->q_head = Q->stride[1];
    g->k = (const uint16_t*)K->data;
    g->k_row = K->stride[0];
    g->k_head = K->stride[1];
    g->v = (const uint16_t*)V->data;
    g->v_row = V->stride[0];
    g->v_head = V->stride[1];
    g->g = (const float*)G->data;
    g->g_row = G->stride[0];
    g->beta = (const float*)Be->data;
    g->b_row = Be->stride[0];
    g->state = (float*)S->data;
    g->st_slot = S->stride[0];
    g->st_head = S->stride[1];
    g->n_states = S->shape[0];
    g->idx = (const int32_t*)I->data;
    g->idx_pitch = ip;
    g->out_idx = W ? (const int32_t*)W->data : nullptr;
    g->out_pitch = wp;
    g->o = (uint16_t*)O->data;
    g->o_row = O->stride[0];
    g->o_head = O->stride[1];
    g->B = B;
    g->n_head_k = hk;
    g->n_head_v = hv;
    g->dk = dk;
    g->dv = dv;
    return RAD_OK;
}
