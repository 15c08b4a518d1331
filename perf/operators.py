"""The serving operators, as they are measured: causal attention over packed prompts, attention of one new token
over a paged key-value cache, and the gated delta rule's step for one new token.

Each case is one call of one operator. `run` computes it in plain torch operations, in 32 bits and rounded once at
the end; with `own` set, it makes the call that a program makes of the library's row. `exact` gives the same
outputs from the definition in 64 bits. Sizes are the served stack's: 16 query and 2 key-value heads of 256 in its
attention layers, 16 key and 32 value heads of 128 in its DeltaNet layers (48 value heads in the full model), prompts
of up to 32,768 rows, an exact tail of 2,048 rows, short prompts of 256 to 2,048 rows.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

HEAD = 256          # the attention layers' head dim
DEVICE = "cuda"


# ----------------------------------------------------------------- the cases

def listed():
    return [
        # causal attention over packed prompts. `q`: the rows of each sequence; `k`: its keys (its last rows are the
        # queries' own)
        {"name": "prompt_37", "op": "prefill", "heads": 16, "kv": 2, "q": "37", "k": "37"},              # a short question
        {"name": "prompt_2048", "op": "prefill", "heads": 16, "kv": 2, "q": "2048", "k": "2048"},        # one engine chunk
        # a ragged batch of short prompts
        {"name": "prompts_ragged", "op": "prefill", "heads": 16, "kv": 2, "q": "1733,402,256,2048,911,1290",
         "k": "1733,402,256,2048,911,1290"},
        # the exact tail of a long prompt whose bulk rows were only filled
        {"name": "tail_of_32768", "op": "prefill", "heads": 16, "kv": 2, "q": "2048", "k": "32768"},
        {"name": "prompt_16384", "op": "prefill", "heads": 16, "kv": 2, "q": "16384", "k": "16384"},     # a long prompt, exact
        # one new token over the paged cache. `lens`: each sequence's cached tokens, the new one among them
        {"name": "token_after_500", "op": "decode", "heads": 16, "kv": 2, "page": 16, "lens": "500"},    # a chat's next token
        {"name": "token_after_32768", "op": "decode", "heads": 16, "kv": 2, "page": 64, "lens": "32768"},  # after a long prompt
        # a batch of short conversations
        {"name": "tokens_batch_32", "op": "decode", "heads": 16, "kv": 2, "page": 16,
         "lens": ",".join(str(256 + (i * 977) % 1793) for i in range(32))},
        # a full server: long prompts of every length
        {"name": "tokens_batch_64_long", "op": "decode", "heads": 16, "kv": 2, "page": 64,
         "lens": ",".join(str(1 + (i * 20011 + 32767) % 32768) for i in range(64))},
        # the DeltaNet layers' step. `rows`: sequences, one new token each
        {"name": "step_1", "op": "step", "rows": 1, "hk": 16, "hv": 32, "dim": 128},                      # one conversation
        {"name": "step_27_full_model", "op": "step", "rows": 27, "hk": 16, "hv": 48, "dim": 128},          # a small batch, 48 heads
        {"name": "step_256", "op": "step", "rows": 256, "hk": 16, "hv": 32, "dim": 128},                  # a full server
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prefill", "decode", "step"))
    if op == "step":
        hk = rng.choice((1, 2, 4, 8, 16))
        return {"op": op, "rows": _log_int(rng, 1, 256), "hk": hk, "hv": hk * rng.choice((1, 2, 3) if hk < 16 else (1, 2)),
                "dim": rng.choice((32, 64, 128, 128, 128))}
    kv = rng.choice((1, 2, 2, 3, 4))
    group = rng.choice((1, 2, 4, 6, 8, 8, 16))
    if op == "prefill":
        group = min(group, 8)
        total, q, k = _log_int(rng, 16, 8192), [], []
        n = rng.choice((1, 1, 2, 5, 9))
        for _ in range(n):
            rows = rng.randint(1, max(1, 2 * total // n))
            if sum(q) + rows > 8192:
                break
            q.append(rows)
            k.append(rows)
        q, k = q or [total], k or [total]
        if rng.random() < 0.25:   # a tail: more keys than rows
            k[0] += rng.randint(1, 8191)
        return {"op": op, "heads": kv * group, "kv": kv, "q": ",".join(map(str, q)), "k": ",".join(map(str, k))}
    longest = _log_int(rng, 16, 32768)
    rows = _log_int(rng, 1, max(1, min(64, 60 * 16384 // longest)))
    return {"op": op, "heads": kv * group, "kv": kv, "page": rng.choice((16, 32, 48, 64, 128)),
            "lens": ",".join(str(rng.randint(1, longest) if i else longest) for i in range(rows))}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _ends(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _pairs(q, k):
    """(row, key) pairs of one causal sequence: row r sees keys 0 .. k - q + r."""
    return q * (k - q) + q * (q + 1) // 2


def work(case):
    if case["op"] == "prefill":
        q, k = _ints(case["q"]), _ints(case["k"])
        pairs = sum(_pairs(a, b) for a, b in zip(q, k))
        return {"bytes": 2 * HEAD * (2 * case["heads"] * sum(q) + 2 * case["kv"] * sum(k)) + 8 * (len(q) + 1),
                "flops": 4 * HEAD * case["heads"] * pairs}
    if case["op"] == "decode":
        lens = _ints(case["lens"])
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 4 * HEAD * case["kv"] * sum(lens) + 4 * HEAD * case["heads"] * len(lens) + 4 * (pages + len(lens)),
                "flops": 4 * HEAD * case["heads"] * sum(lens)}
    n, hk, hv, d = case["rows"], case["hk"], case["hv"], case["dim"]
    return {"bytes": n * (8 * hv * d * d + 4 * hk * d + 4 * hv * d + 8 * hv + 8), "flops": 7 * n * hv * d * d}


# ----------------------------------------------------------------- inputs

def _bf16(g, *shape, gain=1.0):
    return (gain * torch.randn(*shape, device=DEVICE, generator=g)).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"op": case["op"]}
    if case["op"] == "prefill":
        # q and k after their norms and rope: entries of order one, the queries' gain above the keys'
        q, k = _ints(case["q"]), _ints(case["k"])
        s["q"] = _bf16(g, sum(q), case["heads"], HEAD, gain=2.0)
        s["k"] = _bf16(g, sum(k), case["kv"], HEAD)
        s["v"] = _bf16(g, sum(k), case["kv"], HEAD)
        s["cu_q"], s["cu_k"] = _i32(_ends(q)), _i32(_ends(k))
        s["o"] = torch.zeros_like(s["q"])
    elif case["op"] == "decode":
        lens, page = _ints(case["lens"]), case["page"]
        width = -(-max(lens) // page)
        used = [-(-n // page) for n in lens]
        pages = sum(used) + 8
        s["page"] = page
        s["q"] = _bf16(g, len(lens), case["heads"], HEAD, gain=2.0)
        s["cache"] = torch.empty(2, pages * page, case["kv"], HEAD, dtype=torch.bfloat16, device=DEVICE)
        s["cache"].normal_(generator=g)
        # every sequence's pages lie anywhere in the pool; entries past its last page are not read (0)
        order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
        first = _i32(_ends(used)[:-1])[:, None]
        at = torch.arange(width, dtype=torch.int32, device=DEVICE)[None, :]
        s["table"] = torch.where(at < _i32(used)[:, None], order[(first + at).clamp_(max=pages - 1).long()], 0).contiguous()
        s["lens"] = _i32(lens)
        s["o"] = torch.zeros_like(s["q"])
    else:
        # q and k L2-normalised, beta = sigmoid(N), log decay = -softplus(N); the rows' states anywhere in the first
        # half of the pool, the new ones written to the second half in row order (the old ones are kept)
        n, hk, hv, d = case["rows"], case["hk"], case["hv"], case["dim"]
        unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(torch.bfloat16)   # noqa: E731
        s["q"] = unit(torch.randn(n, hk, d, device=DEVICE, generator=g))
        s["k"] = unit(torch.randn(n, hk, d, device=DEVICE, generator=g))
        s["v"] = _bf16(g, n, hv, d)
        s["g"] = -torch.nn.functional.softplus(torch.randn(n, hv, device=DEVICE, generator=g))
        s["beta"] = torch.sigmoid(torch.randn(n, hv, device=DEVICE, generator=g))
        s["pool"] = torch.zeros(2 * n, hv, d, d, device=DEVICE)
        s["pool"][:n].normal_(0.0, 0.3, generator=g)
        s["idx"] = torch.randperm(n, device=DEVICE, generator=g).to(torch.int32)
        s["out_idx"] = torch.arange(n, 2 * n, dtype=torch.int32, device=DEVICE)
        s["o"] = torch.zeros_like(s["v"])
    if own:
        s["call"] = _bind(s)
    return s


# ----------------------------------------------------------------- one pass

def run(s):
    if own:
        rc = s["call"](torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            raise RuntimeError(f"{s['op']}: refused with {rc}")
        return (s["o"], s["pool"][s["pool"].shape[0] // 2:]) if s["op"] == "step" else s["o"]
    return {"prefill": _plain_prefill, "decode": _plain_decode, "step": _plain_step}[s["op"]](s)


def _softmax_(x, mask):
    """Softmax over the last dimension of the entries that `mask` leaves, in place; a row without any is zero."""
    x.masked_fill_(~mask, -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    return x.div_(torch.where(total == 0, 1.0, total))


def _plain_prefill(s):
    q, k, v = (s[n].float().transpose(0, 1) for n in ("q", "k", "v"))      # [heads, rows, HEAD]
    group, rows, keys = q.shape[0] // k.shape[0], q.shape[1], k.shape[1]
    r, c = torch.arange(rows, device=q.device), torch.arange(keys, device=q.device)
    row_seq = (r[:, None] >= s["cu_q"][None, 1:]).sum(1)
    key_seq = (c[:, None] >= s["cu_k"][None, 1:]).sum(1)
    # the last key of row r: as far before its sequence's last key as r is before its last row
    last = s["cu_k"][1:][row_seq] - (s["cu_q"][1:][row_seq] - r)
    mask = (row_seq[:, None] == key_seq[None, :]) & (c[None, :] <= last[:, None])
    p = torch.matmul(q.reshape(-1, group * rows, q.shape[2]), k.transpose(1, 2)).view(-1, group, rows, keys)
    p = _softmax_(p.mul_(1.0 / math.sqrt(HEAD)), mask)
    o = torch.matmul(p.view(-1, group * rows, keys), v).view(-1, rows, HEAD)
    return o.transpose(0, 1).to(torch.bfloat16).contiguous()


def _plain_decode(s):
    n, heads = s["q"].shape[:2]
    page, kv = s["page"], s["cache"].shape[2]
    slots = s["table"].long()[:, :, None] * page + torch.arange(page, device=s["q"].device)
    k, v = (plane[slots.view(n, -1)].float() for plane in s["cache"])        # [n, keys, kv, HEAD]
    mask = torch.arange(k.shape[1], device=k.device)[None, :] < s["lens"][:, None]
    q = s["q"].float().view(n, kv, heads // kv, HEAD)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(HEAD))
    p = _softmax_(p, mask[:, None, None, :])
    return torch.matmul(p, v.transpose(1, 2)).view(n, heads, HEAD).to(torch.bfloat16)


def _plain_step(s):
    share = s["v"].shape[1] // s["k"].shape[1]
    q, k = (s[n].float().repeat_interleave(share, dim=1)[..., None] for n in ("q", "k"))   # [n, hv, dk, 1]
    state = s["pool"][s["idx"].long()].mul_(s["g"].exp()[..., None, None])
    u = s["beta"][..., None, None] * (s["v"].float()[..., None] - torch.matmul(state, k))
    state.add_(torch.matmul(u, k.transpose(2, 3)))
    o = torch.matmul(state, q)[..., 0] * (1.0 / math.sqrt(k.shape[2]))
    return o.to(torch.bfloat16), state


# ----------------------------------------------------------------- the library's calls

def _bind(s):
    package = str(Path(__file__).resolve().parent.parent / "radiance-ridgefill_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ridgefill_abi as abi

    lib = abi.product()
    codes = {torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.int32: abi.I32}
    t = lambda name: abi.tensor(codes[s[name].dtype], s[name].shape, s[name].data_ptr(), s[name].stride())   # noqa: E731
    if s["op"] == "step":
        row = lib.find_row("ridgefill_gdn_step", abi.DOMAIN_DEVICE)
        params = [abi.pint("M", s["v"].shape[0]), abi.pint("n_head_k", s["k"].shape[1]), abi.pint("n_head_v", s["v"].shape[1]),
                  abi.pint("head_k", s["k"].shape[2]), abi.pint("head_v", s["v"].shape[2])]
        operands = [t(n) for n in ("q", "k", "v", "g", "beta", "pool", "idx", "out_idx", "o")]
    else:
        heads = [abi.pint("M", s["q"].shape[0]), abi.pint("n_head", s["q"].shape[1]), abi.pint("head_dim", HEAD)]
        if s["op"] == "prefill":
            row = lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
            params = heads + [abi.pint("n_head_kv", s["k"].shape[1])]
            operands = [t(n) for n in ("q", "k", "v", "cu_q", "cu_k", "o")]
        else:
            row = lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
            params = heads + [abi.pint("n_head_kv", s["cache"].shape[2]), abi.pint("page", s["page"])]
            operands = [t(n) for n in ("q", "cache", "table", "lens", "o")]
    size = lib.scratch_bytes(row, operands, params)
    s["scratch"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEVICE)
    return lib.bind(row, operands, params, scratch=s["scratch"].data_ptr(), scratch_bytes=size)


# ----------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefill":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        group = case["heads"] // case["kv"]
        q0 = k0 = 0
        for nq, nk in zip(_ints(case["q"]), _ints(case["k"])):
            ahead = torch.ones(nq, nk, dtype=torch.bool, device=DEVICE).triu(nk - nq + 1)
            for h in range(case["heads"]):
                keys = s["k"][k0:k0 + nk, h // group].double()
                score = s["q"][q0:q0 + nq, h].double() @ keys.T / math.sqrt(HEAD)
                p = torch.softmax(score.masked_fill(ahead, -math.inf), dim=1)
                out[q0:q0 + nq, h] = p @ s["v"][k0:k0 + nk, h // group].double()
            q0, k0 = q0 + nq, k0 + nk
        return out
    if case["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        group = case["heads"] // case["kv"]
        for i, n in enumerate(_ints(case["lens"])):
            at = torch.arange(n, device=DEVICE)
            slot = s["table"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
            k, v = s["cache"][0, slot].double(), s["cache"][1, slot].double()
            for h in range(case["heads"]):
                p = torch.softmax(k[:, h // group] @ s["q"][i, h].double() / math.sqrt(HEAD), dim=0)
                out[i, h] = p @ v[:, h // group]
        return out
    n, hk, hv, d = case["rows"], case["hk"], case["hv"], case["dim"]
    o = torch.zeros(n, hv, d, dtype=torch.float64, device=DEVICE)
    new = torch.zeros(n, hv, d, d, dtype=torch.float64, device=DEVICE)
    for i in range(n):
        q, k = (s[x][i].double()[torch.arange(hv, device=DEVICE) // (hv // hk)] for x in ("q", "k"))
        S = s["pool"][s["idx"][i].long()].double() * torch.exp(s["g"][i].double())[:, None, None]
        u = s["beta"][i].double()[:, None] * (s["v"][i].double() - torch.einsum("hvk,hk->hv", S, k))
        new[i] = S + u[:, :, None] * k[:, None, :]
        o[i] = torch.einsum("hvk,hk->hv", new[i], q) / math.sqrt(d)
    return o, new
