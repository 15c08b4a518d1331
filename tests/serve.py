"""Calls of the serving rows (include/ridgefill_serve.h) on torch tensors, and their definitions in 64 bits with the
error a correct kernel may have, element by element, for the device tests."""
import math

import harness as H
from harness import abi

U32 = 2.0 ** -24     # half a step of f32, relative
UB16 = 2.0 ** -8     # half a step of bf16, relative


def decode_params(B, hq, hkv, page, D=256, scale=None):
    p = [H.pint("M", B), H.pint("n_head", hq), H.pint("n_head_kv", hkv), H.pint("head_dim", D), H.pint("page", page)]
    return p + ([H.pf64("scale", scale)] if scale is not None else [])


def step_params(B, hk, hv, dk=128, dv=128, scale=None):
    p = [H.pint("M", B), H.pint("n_head_k", hk), H.pint("n_head_v", hv), H.pint("head_k", dk), H.pint("head_v", dv)]
    return p + ([H.pf64("scale", scale)] if scale is not None else [])


def parse(lib, name, tensors, params):
    """The row's operand check alone (descriptors only, no device)."""
    import ctypes as C
    args, keep = abi.Plugin.args(tensors, params)
    out = (C.c_char * 2048)()
    rc = getattr(lib.lib, name)(C.byref(args), C.byref(out))
    del keep
    return rc


def attention(torch, q, k, v, scale, keep=None):
    """Softmax attention of q [n, D] over k, v [m, D] in f64, the keys `keep` [n, m] leaves (all when None): (o, the
    weights). A row that nothing is left of is zero."""
    s = (q @ k.T) * scale
    if keep is not None:
        s = s.masked_fill(~keep, -math.inf)
    top = s.amax(1, keepdim=True) if s.shape[1] else s.new_zeros(s.shape[0], 1)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    return p @ v, p


def attention_bound(torch, q, k, v, p, o, scale, p_eps):
    """|kernel - o| at most: the score q.k in f32 (256 products, each sum off by 2^-23 of the magnitudes so far on a
    truncating adder) moves a weight by e^(that) - 1, each weight is held to p_eps, the sums of the weights and of the
    weighted v in f32, o rounded once to bf16."""
    mag = ((q.abs() @ k.abs().T) * scale).amax(1, keepdim=True) if k.shape[0] else q.new_zeros(q.shape[0], 1)
    # the score's sum, then its scaling and the subtraction of the maximum, each off by 2^-24 of a value up to `mag`
    delta = (256 * 2.0 ** -23 + 4 * U32) * mag
    weighted = p @ v.abs()
    n = max(k.shape[0], 1)
    return UB16 * o.abs() * 1.01 + weighted * (2 * torch.expm1(delta) + p_eps + 2 * (n + 64) * 2.0 ** -23) + 1e-30


def decode_reference(torch, q, cache, table, lens, page, scale=None):
    """(o, bound) f64 of ridgefill_attn_decode's formula; q [B, Hq, D], cache [2, slots, Hkv, D] bf16 tensors."""
    B, hq, D = q.shape
    slots, hkv = cache.shape[1], cache.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(B, hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    for i in range(B):
        n = max(0, min(int(lens[i]), table.shape[1] * page))
        j = torch.arange(n, device=q.device)
        at = table[i].long()[j // page] * page + j % page
        at = at[(at >= 0) & (at < slots)]
        for h in range(hkv):
            rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            qq, kk, vv = q[i, rows].double(), cache[0, at, h].double(), cache[1, at, h].double()
            out, p = attention(torch, qq, kk, vv, scale)
            o[i, rows] = out
            # weights as a bf16 pair: 2^-16 of the value, and the approximate exponential's 2^-22
            bound[i, rows] = attention_bound(torch, qq, kk, vv, p, out, scale, 2.0 ** -15)
    return o, bound


def step_reference(torch, q, k, v, g, beta, state, idx, out_idx, scale=None):
    """(o, new state [B, Hv, dv, dk], bounds of both) f64 of ridgefill_gdn_step's formula for rows whose slots are
    inside the pool and named once."""
    B, hk, dk = k.shape
    hv = v.shape[1]
    scale = 1.0 / math.sqrt(dk) if scale is None else scale
    head = torch.arange(hv, device=q.device) // (hv // hk)
    qq, kk = q.double()[:, head], k.double()[:, head]
    a, bt = torch.exp(g.double()), beta.double()
    S = state.double()[idx.long()] * a[..., None, None]
    sk = torch.einsum("bhvk,bhk->bhv", S, kk)
    mag = torch.einsum("bhvk,bhk->bhv", S.abs(), kk.abs())
    u = bt[..., None] * (v.double() - sk)
    new = S + u[..., None] * kk[..., None, :]
    # f32: the exponential to 2 steps, a dot of dk terms to (dk + 4) half steps of its magnitudes
    du = U32 * bt[..., None].abs() * ((dk + 12) * mag + 4 * v.double().abs())
    dS = U32 * (8 * S.abs() + 4 * new.abs()) + (du + 2 * U32 * u.abs())[..., None] * kk.abs()[..., None, :]
    o = scale * torch.einsum("bhvk,bhk->bhv", new, qq)
    kq, kqm = (kk * qq).sum(-1)[..., None], (kk * qq).abs().sum(-1)[..., None]
    do = scale * (U32 * (dk + 16) * torch.einsum("bhvk,bhk->bhv", S.abs(), qq.abs()) + du * kq.abs() +
                  U32 * (dk + 8) * u.abs() * kqm)
    return o, new, 1.01 * UB16 * o.abs() + 2 * do + 1e-30, dS + 1e-35


def prefill_params(T, hq, hkv, D=256, scale=None):
    p = [H.pint("M", T), H.pint("n_head", hq), H.pint("n_head_kv", hkv), H.pint("head_dim", D)]
    return p + ([H.pf64("scale", scale)] if scale is not None else [])


def prefill_reference(torch, q, k, v, cu_q, cu_k, scale=None, heads=None):
    """(o, bound, written rows) f64 of ridgefill_attn_prefill's formula for in-order cu lists; `heads`: only these."""
    T, hq, D = q.shape
    hkv = k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(T, hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    rows = torch.zeros(T, dtype=torch.bool, device=q.device)
    for q0, q1, k0, k1 in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        nq, nk = q1 - q0, k1 - k0
        rows[q0:q1] = True
        keep = torch.ones(nq, nk, dtype=torch.bool, device=q.device).tril(nk - nq)
        for h in range(hq) if heads is None else heads:
            qq, kk, vv = q[q0:q1, h].double(), k[k0:k1, h // (hq // hkv)].double(), v[k0:k1, h // (hq // hkv)].double()
            out, p = attention(torch, qq, kk, vv, scale, keep)
            o[q0:q1, h] = out
            # a weight rounded to bf16, and the approximate exponential's 2^-22
            bound[q0:q1, h] = attention_bound(torch, qq, kk, vv, p, out, scale, 1.01 * UB16)
    return o, bound, rows
