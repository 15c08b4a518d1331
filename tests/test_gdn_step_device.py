"""ridgefill_gdn_step on B200 against its formula in 64 bits, element by element within the bound of f32 arithmetic:
head dims 128 and small ones, odd batches, strided operands, in place and into other slots, skipped rows, shared
slots, and the chunked fill of the same tokens."""
import numpy as np
import pytest

import harness as H
import serve as S
from harness import abi

pytestmark = pytest.mark.gpu


def inputs(torch, seed, B, hk, hv, dk=128, dv=128, slots=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(torch.bfloat16)   # noqa: E731
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)              # noqa: E731
    slots = 2 * B + 1 if slots is None else slots
    return dict(q=unit(rn(B, hk, dk)), k=unit(rn(B, hk, dk)), v=rn(B, hv, dv).to(torch.bfloat16),
                g=-torch.nn.functional.softplus(rn(B, hv)), beta=torch.sigmoid(rn(B, hv)), state=0.3 * rn(slots, hv, dv, dk),
                idx=torch.randperm(slots, device="cuda", generator=g)[:B].to(torch.int32),
                o=torch.full((B, hv, dv), 7.0, dtype=torch.bfloat16, device="cuda"))


def call(lib, d, out_idx=None, scale=None):
    B, hk, dk = d["k"].shape
    hv, dv = d["v"].shape[1:]
    ops = [H.dev(d[n]) for n in ("q", "k", "v", "g", "beta", "state", "idx")] + [H.dev(out_idx), H.dev(d["o"])]
    return H.launch(lib, "ridgefill_gdn_step", ops, S.step_params(B, hk, hv, dk, dv, scale))


def check(torch, d, before, out_idx=None, scale=None, rows=None):
    o, new, bo, bs = S.step_reference(torch, d["q"], d["k"], d["v"], d["g"], d["beta"], before, d["idx"], out_idx, scale)
    rows = torch.arange(o.shape[0], device="cuda") if rows is None else rows
    dst = (d["idx"] if out_idx is None else out_idx).long()[rows]
    assert ((d["state"][dst].double() - new[rows]).abs() <= bs[rows]).all(), "state"
    assert ((d["o"][rows].double() - o[rows]).abs() <= bo[rows]).all(), "o"
    rest = torch.ones(before.shape[0], dtype=torch.bool, device="cuda")
    rest[dst] = False
    assert torch.equal(d["state"][rest], before[rest]), "a slot no row writes changed"


@pytest.mark.parametrize("B,hk,hv", [(1, 1, 1), (1, 16, 32), (3, 2, 6), (27, 16, 48), (130, 4, 8)])
@pytest.mark.parametrize("fork", [False, True])
def test_wide_heads(cuda, product_lib, B, hk, hv, fork):
    torch = cuda
    d = inputs(torch, B + hv, B, hk, hv)
    before = d["state"].clone()
    out = None
    if fork:   # every row to a slot of its own that no row reads
        free = torch.ones(before.shape[0], dtype=torch.bool, device="cuda")
        free[d["idx"].long()] = False
        out = free.nonzero()[:B, 0].to(torch.int32)
    assert call(product_lib, d, out) == abi.OK
    check(torch, d, before, out)


@pytest.mark.parametrize("dk,dv", [(8, 1), (16, 16), (24, 40), (32, 32), (40, 33), (64, 64), (56, 7)])
def test_small_heads(cuda, product_lib, dk, dv):
    torch = cuda
    d = inputs(torch, dk * 64 + dv, 5, 4, 8, dk, dv)
    before = d["state"].clone()
    assert call(product_lib, d, scale=0.7) == abi.OK
    check(torch, d, before, scale=0.7)


@pytest.mark.parametrize("dk,dv", [(8, 1), (32, 33), (24, 64), (64, 63), (40, 31)])
def test_small_heads_of_a_large_batch(cuda, product_lib, dk, dv):
    """More heads than SMs: the form with several state rows a lane, cut anywhere."""
    torch = cuda
    d = inputs(torch, dk + dv, 70, 2, 6, dk, dv)
    before = d["state"].clone()
    assert call(product_lib, d) == abi.OK
    check(torch, d, before)


def test_strided_operands(cuda, product_lib):
    """q, k, v as slices of one projected row, g and beta with a row pitch, slot pitch and head pitch of the pool
    above the packed ones, o into a wider row, slot numbers in a [B, 2] table's first column."""
    torch = cuda
    B, hk, hv = 9, 2, 4
    d = inputs(torch, 5, B, hk, hv)
    row = torch.randn(B, 2 * hk * 128 + hv * 128 + 8, device="cuda").to(torch.bfloat16)
    for name, at, h in (("q", 0, hk), ("k", hk * 128, hk), ("v", 2 * hk * 128, hv)):
        row[:, at:at + h * 128] = d[name].reshape(B, -1)
        d[name] = row[:, at:at + h * 128].view(B, h, 128)
    for name in ("g", "beta"):
        wide = torch.zeros(B, 3 * hv, device="cuda")
        wide[:, hv:2 * hv] = d[name]
        d[name] = wide[:, hv:2 * hv]
    pool = torch.zeros(2 * B + 1, hv + 1, 128 * 128 + 4, device="cuda")
    pool[:, :hv, :128 * 128] = d["state"].view(2 * B + 1, hv, -1)
    d["state"] = pool[:, :hv, :128 * 128].unflatten(2, (128, 128))
    table = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
    table[:, 0] = d["idx"]
    d["o"] = torch.zeros(B, hv, 136, dtype=torch.bfloat16, device="cuda")[:, :, 4:132]
    before = d["state"].clone()
    edge = pool[:, hv].clone(), pool[:, :, 128 * 128:].clone()
    idx = d["idx"]
    d["idx"] = table
    assert call(product_lib, d) == abi.OK
    d["idx"] = idx
    check(torch, d, before)
    assert torch.equal(pool[:, hv], edge[0]) and torch.equal(pool[:, :, 128 * 128:], edge[1])


def test_skipped_rows(cuda, product_lib):
    """Rows with a slot outside the pool, and rows whose written slot another row names, leave state and o as they
    were; the others are not disturbed."""
    torch = cuda
    B = 8
    d = inputs(torch, 6, B, 2, 4, slots=12)
    d["idx"] = torch.tensor([0, 1, -1, 12, 3, 3, 5, 6], dtype=torch.int32, device="cuda")      # 4 and 5 share slot 3
    before, o = d["state"].clone(), d["o"].clone()
    assert call(product_lib, d) == abi.OK
    live = torch.tensor([0, 1, 6, 7], device="cuda")
    dead = torch.tensor([2, 3, 4, 5], device="cuda")
    d2 = dict(d, idx=d["idx"].clamp(0, 11))
    check(torch, d2, before, rows=live)
    assert torch.equal(d["o"][dead], o[dead])
    # a fork: rows 0, 1 and 2 read slot 1; row 0 would write it in place, which the others read: skipped
    d = inputs(torch, 7, 4, 2, 4, slots=12)
    d["idx"] = torch.tensor([1, 1, 1, 5], dtype=torch.int32, device="cuda")
    out = torch.tensor([1, 8, 9, -3], dtype=torch.int32, device="cuda")
    before, o = d["state"].clone(), d["o"].clone()
    assert call(product_lib, d, out) == abi.OK
    check(torch, d, before, out.clamp(0), rows=torch.tensor([1, 2], device="cuda"))
    assert torch.equal(d["o"][[0, 3]], o[[0, 3]])


def test_infinite_and_nan_elsewhere(cuda, product_lib):
    """Slots that no row names may hold anything."""
    torch = cuda
    d = inputs(torch, 8, 3, 2, 4, slots=6)
    d["idx"] = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    d["state"][[1, 3, 5]] = float("nan")
    before = d["state"].clone()
    assert call(product_lib, d) == abi.OK
    used = d["idx"].long()
    o, new, bo, bs = S.step_reference(torch, d["q"], d["k"], d["v"], d["g"], d["beta"], before, d["idx"], None)
    assert ((d["state"][used].double() - new).abs() <= bs).all() and ((d["o"].double() - o).abs() <= bo).all()
    assert torch.isnan(d["state"][[1, 3, 5]]).all()


def test_decay_extremes(cuda, product_lib):
    """A decay of exactly one, and one that clears the state; beta 0 (the state only decays) and 1."""
    torch = cuda
    d = inputs(torch, 9, 4, 2, 4)
    d["g"][0], d["g"][1] = 0.0, -200.0
    d["beta"][2], d["beta"][3] = 0.0, 1.0
    before = d["state"].clone()
    assert call(product_lib, d) == abi.OK
    check(torch, d, before)


def test_large_pool_offsets(cuda, product_lib):
    """A pool of more than 2^31 elements: slots at both ends."""
    torch = cuda
    slots, hv = 2200, 64
    d = inputs(torch, 10, 3, 32, hv, slots=4)
    pool = torch.zeros(slots, hv, 128, 128, device="cuda")
    assert pool.numel() > 2 ** 31
    at = torch.tensor([slots - 1, 0, 1100], dtype=torch.int32, device="cuda")
    pool[at.long()] = d["state"][:3]
    d["state"], d["idx"] = pool, at
    before = pool[at.long()].clone()
    assert call(product_lib, d) == abi.OK
    o, new, bo, bs = S.step_reference(torch, d["q"], d["k"], d["v"], d["g"], d["beta"], before, torch.arange(3, device="cuda"), None)
    assert ((pool[at.long()].double() - new).abs() <= bs).all() and ((d["o"].double() - o).abs() <= bo).all()


def test_repeats_and_graph_on_a_side_stream(cuda, product_lib):
    """The same call gives the same bits, eagerly and replayed from a graph captured on another stream."""
    torch = cuda
    d = inputs(torch, 11, 6, 4, 8)
    out = torch.ones(13, dtype=torch.bool, device="cuda")
    out[d["idx"].long()] = False
    out = out.nonzero()[:6, 0].to(torch.int32)
    assert call(product_lib, d, out) == abi.OK
    want_o, want_s = d["o"].clone(), d["state"].clone()
    row = product_lib.find_row("ridgefill_gdn_step", abi.DOMAIN_DEVICE)
    ops = [H.dev(d[n]) for n in ("q", "k", "v", "g", "beta", "state", "idx")] + [H.dev(out), H.dev(d["o"])]
    bound = product_lib.bind(row, ops, S.step_params(6, 4, 8))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
    for _ in range(3):
        d["o"].zero_()
        d["state"][out.long()] = 0
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d["o"], want_o) and torch.equal(d["state"], want_s)


def test_steps_continue_a_fill(cuda, product_lib):
    """A prompt filled by ridgefill_gdn_fill (with o), then tokens stepped one at a time: the states and outputs of one
    fill over prompt and tokens together, to the fill's own tolerances (state 1e-3, o 1e-2 relative 2-norm)."""
    torch = cuda
    T, n, hk, hv = 200, 5, 2, 4
    q, k, v, g, beta, state = H.gdn_inputs(31, T + n, hk, hv, "slow", slots=1)
    cu16 = lambda a: torch.from_numpy(a.view(np.int16)).cuda()   # noqa: E731
    Q, K, V = cu16(q), cu16(k), cu16(v)
    G, B = torch.from_numpy(g).cuda(), torch.from_numpy(beta).cuda()
    idx = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, want_o = H.oracle_gdn(k, v, g, beta, state, [0], [0, T + n], q=q)
    ST = torch.from_numpy(state.copy()).cuda()
    O = torch.zeros(T + n, hv, 128, dtype=torch.int16, device="cuda")
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    ops = [H.dev(Q[:T]), H.dev(K[:T]), H.dev(V[:T]), H.dev(G[:T]), H.dev(B[:T]), H.dev(ST), H.dev(idx), H.dev(cu), H.dev(O[:T])]
    assert H.launch(product_lib, "ridgefill_gdn_fill", ops, H.gdn_params(T, hk, hv)) == abi.OK
    for t in range(T, T + n):
        r = slice(t, t + 1)
        ops = [H.dev(Q[r]), H.dev(K[r]), H.dev(V[r]), H.dev(G[r]), H.dev(B[r]), H.dev(ST), H.dev(idx), abi.absent(), H.dev(O[r])]
        assert H.launch(product_lib, "ridgefill_gdn_step", ops, S.step_params(1, hk, hv)) == abi.OK
    assert H.rel_l2(ST.cpu().numpy()[0], want[0]) <= 1e-3
    got = H.bf16_bits_to_f32(O.cpu().numpy().view(np.uint16))
    ref = want_o if want_o.dtype != np.uint16 else H.bf16_bits_to_f32(want_o)
    assert H.rel_l2(got[T:], ref[T:]) <= 1e-2
