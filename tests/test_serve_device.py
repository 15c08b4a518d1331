"""The serving rows as they are used, on B200: a prompt's layers filled by the fill rows, its exact rows answered, then new
tokens one at a time over the same caches -- attention layer and DeltaNet layer, each against the same rows answered as
one prompt, and the whole run against 64 bits."""
import math

import pytest

import harness as H
import serve as S
from harness import abi

pytestmark = pytest.mark.gpu
D = 256


class AttentionLayer:
    """One attention layer's cache and projections of a whole conversation (random), driven through the library's rows."""

    def __init__(self, torch, lib, prompts, steps, hq=16, hkv=2, page=16, seed=1):
        self.torch, self.lib, self.hq, self.hkv, self.page = torch, lib, hq, hkv, page
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)   # noqa: E731
        self.lens = list(prompts)
        total = [n + steps for n in prompts]
        self.q = [rn(n, hq, D) for n in total]
        self.k = [rn(n, hkv, D) for n in total]
        self.v = [rn(n, hkv, D) for n in total]
        self.w = torch.ones(D, device="cuda")
        used = [-(-n // page) for n in total]
        order = torch.randperm(sum(used) + 2, device="cuda", generator=g).to(torch.int32)
        self.cache = torch.full((2, (sum(used) + 2) * page, hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.table = torch.zeros(len(prompts), max(used), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n

    def slots(self, i, positions):
        return (self.table[i].long()[positions // self.page] * self.page + positions % self.page).to(self.torch.int32)

    def fill(self, rows):
        """ridgefill_attn_kv_fill over `rows`, a list of (sequence, positions): the cache, and k as it lies there."""
        torch = self.torch
        k = torch.cat([self.k[i][p] for i, p in rows])
        v = torch.cat([self.v[i][p] for i, p in rows])
        pos = torch.cat([p for _, p in rows]).to(torch.int32)
        slots = torch.cat([self.slots(i, p) for i, p in rows])
        out = torch.empty_like(k)
        params = [H.pint("M", k.shape[0]), H.pint("n_head_kv", self.hkv), H.pint("head_dim", D), H.pint("rope_dim", 64),
                  H.pf64("rope_theta", 1e7)]
        ops = [H.dev(k), H.dev(v), H.dev(self.w), H.dev(pos), H.dev(slots), H.dev(self.cache), H.dev(out)]
        assert H.launch(self.lib, "ridgefill_attn_kv_fill", ops, params) == abi.OK
        return out, v

    def prompt(self, tail=None):
        """Fill the prompts and answer their rows (the last `tail` of each)."""
        torch = self.torch
        rows = [(i, torch.arange(n, device="cuda")) for i, n in enumerate(self.lens)]
        k, v = self.fill(rows)
        first = [0 if tail is None else max(0, n - tail) for n in self.lens]
        q = torch.cat([self.q[i][f:n] for i, (f, n) in enumerate(zip(first, self.lens))])
        cu = lambda lens: torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")   # noqa: E731
        cu_q, cu_k = cu([n - f for f, n in zip(first, self.lens)]), cu(self.lens)
        o = torch.empty_like(q)
        ops = [H.dev(q), H.dev(k), H.dev(v), H.dev(cu_q), H.dev(cu_k), H.dev(o)]
        assert H.launch(self.lib, "ridgefill_attn_prefill", ops, S.prefill_params(q.shape[0], self.hq, self.hkv)) == abi.OK
        return o, cu_q.tolist()

    def token(self):
        """The next token of every sequence: its cache row, then its answer."""
        torch = self.torch
        self.fill([(i, torch.tensor([n], device="cuda")) for i, n in enumerate(self.lens)])
        q = torch.stack([self.q[i][n] for i, n in enumerate(self.lens)])
        self.lens = [n + 1 for n in self.lens]
        lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        o = torch.empty_like(q)
        ops = [H.dev(q), H.dev(self.cache), H.dev(self.table), H.dev(lens), H.dev(o)]
        assert H.launch(self.lib, "ridgefill_attn_decode", ops, S.decode_params(len(self.lens), self.hq, self.hkv, self.page)) == abi.OK
        return o

    def reference(self, i, n):
        """(o, bound) of sequence i's row at position n - 1 over the cache as it stands, in 64 bits; the bound covers both
        rows' arithmetic."""
        torch = self.torch
        slots = self.slots(i, torch.arange(n, device="cuda")).long()
        out, bound = [], []
        for h in range(self.hq):
            q, k, v = self.q[i][n - 1, h].double()[None], self.cache[0, slots, h * self.hkv // self.hq].double(), \
                self.cache[1, slots, h * self.hkv // self.hq].double()
            o, p = S.attention(torch, q, k, v, 1 / math.sqrt(D))
            out.append(o[0])
            bound.append(S.attention_bound(torch, q, k, v, p, o, 1 / math.sqrt(D), 1.01 * S.UB16)[0])
        return torch.stack(out), torch.stack(bound)


def test_attention_layer_prompt_then_tokens(cuda, product_lib):
    torch = cuda
    steps = 3
    layer = AttentionLayer(torch, product_lib, [200, 1, 131, 16], steps)
    o, cu = layer.prompt()
    for i, n in enumerate(layer.lens):
        for row in {1, n // 2 + 1, n}:
            want, bound = layer.reference(i, row)
            assert ((o[cu[i] + row - 1].double() - want).abs() <= bound).all(), (i, row)
    last = None
    for _ in range(steps):
        last = layer.token()
        for i, n in enumerate(layer.lens):
            want, bound = layer.reference(i, n)
            assert ((last[i].double() - want).abs() <= bound).all(), (i, n)
    # the whole conversation as one prompt answers its last row as the last token was answered: both within their bounds
    again, cu = layer.prompt()
    for i, n in enumerate(layer.lens):
        want, bound = layer.reference(i, n)
        assert ((again[cu[i + 1] - 1].double() - last[i].double()).abs() <= 2 * bound).all()


def test_exact_tail_of_a_filled_prompt(cuda, product_lib):
    """The tail's rows of long prompts over all their keys (split along the keys) and the same rows of the whole prompts,
    both against 64 bits; the next token follows."""
    torch = cuda
    layer = AttentionLayer(torch, product_lib, [9000, 700], 1)
    tail, cu_t = layer.prompt(tail=40)
    whole, cu_w = layer.prompt()
    for i, n in enumerate(layer.lens):
        for back in range(1, 41, 3):
            want, bound = layer.reference(i, n + 1 - back)
            assert ((tail[cu_t[i + 1] - back].double() - want).abs() <= bound).all()
            assert ((whole[cu_w[i + 1] - back].double() - want).abs() <= bound).all()
    o = layer.token()
    for i, n in enumerate(layer.lens):
        want, bound = layer.reference(i, n)
        assert ((o[i].double() - want).abs() <= bound).all()


def test_delta_net_layer_prompt_then_tokens(cuda, product_lib):
    """conv_prep and the fill over a ragged batch of prompts, then tokens by conv_prep over one-row sequences and the step:
    states and outputs of the same rows filled as longer prompts, to the fill's tolerances (state 1e-3, o 1e-2, relative
    2-norm), conv states bit for bit."""
    torch = cuda
    hk, hv, steps, prompts = 2, 4, 4, [150, 64, 7]
    C, n = (2 * hk + hv) * 128, len(prompts)
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    x = [rn(p + steps, C).to(torch.bfloat16) for p in prompts]
    ab = [rn(p + steps, 2, hv).to(torch.bfloat16) for p in prompts]
    w, a_log, dt = (0.5 * rn(C, 4)).to(torch.bfloat16), 0.3 * rn(hv), 0.3 * rn(hv)
    idx = torch.arange(n, dtype=torch.int32, device="cuda")

    def prepare(rows, conv, ctx):
        X = torch.cat([x[i][r] for i, r in enumerate(rows)])
        AB = torch.cat([ab[i][r] for i, r in enumerate(rows)])
        T = X.shape[0]
        lens = [len(range(*r.indices(1 << 20))) for r in rows]
        cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")
        q, k = (torch.empty(T, hk, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        v, o = (torch.empty(T, hv, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        gate, beta = (torch.empty(T, hv, device="cuda") for _ in range(2))
        a, b, held = AB[:, 0].contiguous(), AB[:, 1].contiguous(), torch.tensor(ctx, dtype=torch.int32, device="cuda")
        ops = [H.dev(X), H.dev(w), abi.absent(), H.dev(a_log), H.dev(dt), H.dev(conv), H.dev(cu), H.dev(a), H.dev(b), H.dev(idx),
               H.dev(held), H.dev(q), H.dev(k), H.dev(v), H.dev(gate), H.dev(beta)]
        params = [H.pint("M", T), H.pint("n_head_k", hk), H.pint("n_head_v", hv), H.pint("head_k", 128), H.pint("head_v", 128),
                  H.pint("conv", 4)]
        assert H.launch(product_lib, "ridgefill_gdn_conv_prep", ops, params) == abi.OK
        return q, k, v, gate, beta, cu, o

    def fill(rows, conv, state):
        q, k, v, gate, beta, cu, o = prepare(rows, conv, [0] * n)
        ops = [H.dev(q), H.dev(k), H.dev(v), H.dev(gate), H.dev(beta), H.dev(state), H.dev(idx), H.dev(cu), H.dev(o)]
        assert H.launch(product_lib, "ridgefill_gdn_fill", ops, H.gdn_params(k.shape[0], hk, hv)) == abi.OK
        return o, cu.tolist()

    new = lambda: (torch.zeros(n, 3, C, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, hv, 128, 128, device="cuda"))   # noqa: E731
    conv, state = new()
    fill([slice(0, p) for p in prompts], conv, state)
    for t in range(steps):
        q, k, v, gate, beta, _, o = prepare([slice(p + t, p + t + 1) for p in prompts], conv, [p + t for p in prompts])
        ops = [H.dev(q), H.dev(k), H.dev(v), H.dev(gate), H.dev(beta), H.dev(state), H.dev(idx), abi.absent(), H.dev(o)]
        assert H.launch(product_lib, "ridgefill_gdn_step", ops, S.step_params(n, hk, hv)) == abi.OK
        conv2, state2 = new()
        want, cu = fill([slice(0, p + t + 1) for p in prompts], conv2, state2)
        assert torch.equal(conv, conv2)
        rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())   # noqa: E731
        assert rel(state, state2) <= 1e-3
        assert rel(o, torch.stack([want[cu[i + 1] - 1] for i in range(n)])) <= 1e-2
