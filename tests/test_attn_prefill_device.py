"""ridgefill_attn_prefill on B200 against its formula in 64 bits, element by element within the bound of its arithmetic:
rows and keys around the 128-key tiles and the query tiles, tails, rows without keys, empty and many sequences, every
kind of head group, strides, rows behind the last sequence, NaN in other sequences and behind them, offsets past 32
bits; and with the rows it is used with."""
import pytest

import harness as H
import serve as S
from harness import abi

pytestmark = pytest.mark.gpu
D = 256


def ends(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def inputs(torch, seed, nq, nk, hq, hkv, pad=0, gain=2.0):
    """Packed sequences, `pad` rows behind the last one (q: anything; k, v: NaN)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    q = (gain * rn(sum(nq) + pad, hq, D)).to(torch.bfloat16)
    k, v = (rn(sum(nk) + pad, hkv, D).to(torch.bfloat16) for _ in range(2))
    k[sum(nk):] = float("nan")
    v[sum(nk):] = float("nan")
    return dict(q=q, k=k, v=v, cu_q=ends(nq), cu_k=ends(nk), o=torch.full_like(q, 7.0))


def operands(torch, d):
    cu = [torch.tensor(d[n], dtype=torch.int32, device="cuda") for n in ("cu_q", "cu_k")]
    same = d["cu_q"] == d["cu_k"]
    return [H.dev(d["q"]), H.dev(d["k"]), H.dev(d["v"]), H.dev(cu[0]), H.dev(None if same else cu[1]), H.dev(d["o"])], cu


def call(lib, torch, d, scale=None):
    ops, keep = operands(torch, d)
    T, hq, _ = d["q"].shape
    rc = H.launch(lib, "ridgefill_attn_prefill", ops, S.prefill_params(T, hq, d["k"].shape[1], scale=scale))
    assert lib.lib.ridgefill_device_error(1) == 0
    return rc


def check(torch, d, scale=None, heads=None):
    o, bound, rows = S.prefill_reference(torch, d["q"], d["k"], d["v"], d["cu_q"], d["cu_k"], scale, heads)
    pick = slice(None) if heads is None else heads
    err = (d["o"].double() - o).abs()[rows][:, pick]
    bad = ~(err <= bound[rows][:, pick])
    assert not bad.any(), f"{int(bad.sum())} elements off, first at {bad.nonzero()[0].tolist()}, {float(err[bad][0])}"
    assert (d["o"][~rows] == 7.0).all(), "a row outside every sequence was written"


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 100, 127, 128, 129, 255, 256, 257, 700])
def test_one_prompt(cuda, product_lib, n):
    torch = cuda
    d = inputs(torch, n, [n], [n], 16, 2, pad=n % 3)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("nq,nk", [(1, 128), (1, 129), (1, 1000), (5, 384), (16, 2000), (40, 4100), (200, 257), (128, 1152)])
def test_tails(cuda, product_lib, nq, nk):
    torch = cuda
    d = inputs(torch, nq + nk, [nq], [nk], 16, 2)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("nq,nk", [(10, 0), (300, 100), (129, 128), (1, 0), (50, 1)])
def test_rows_without_keys(cuda, product_lib, nq, nk):
    """More rows than keys: the first nq - nk rows see none and are zero."""
    torch = cuda
    d = inputs(torch, 7 * nq + nk, [nq, 20], [nk, 20], 8, 1)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)
    assert (d["o"][:nq - nk] == 0).all()


@pytest.mark.parametrize("nq,nk,hq,hkv", [([1033, 1033], [443, 1033], 96, 3), ([6000], [50], 8, 1), ([3000, 100], [0, 100], 128, 1),
                                          ([200] * 40, [0, 200] * 20, 64, 2), ([900, 64] * 20, [1, 64] * 20, 32, 1)])
def test_many_query_tiles_without_keys(cuda, product_lib, nq, nk, hq, hkv):
    """Whole rows of query tiles that no key reaches, behind tiles with keys and between them: zeros, and the rest unharmed."""
    torch = cuda
    d = inputs(torch, 65, nq, nk, hq, hkv)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d, heads=[0, hq // 2, hq - 1])
    for q0, n, k in zip(d["cu_q"], nq, nk):
        assert (d["o"][q0:q0 + max(n - k, 0)] == 0).all()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (4, 1), (12, 2), (9, 3), (16, 1), (20, 1), (48, 3), (100, 1), (128, 1), (130, 2)])
def test_head_groups(cuda, product_lib, hq, hkv):
    torch = cuda
    d = inputs(torch, hq * 10 + hkv, [150, 33], [150, 290], hq, hkv, pad=2)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("nq", [[300, 0, 45, 128, 1], [0, 0, 7], [17] * 32, [5, 0, 130] * 13, [3] * 100, [0] * 40 + [200] + [0] * 30])
def test_packed_sequences(cuda, product_lib, nq):
    """Up to 32 sequences (sorted) and more, empty ones among them; some with more keys than rows."""
    torch = cuda
    nk = [n + (37 * i) % 200 if i % 3 == 0 and n else n for i, n in enumerate(nq)]
    d = inputs(torch, len(nq), nq, nk, 16, 2, pad=5)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("nq,nk", [([1], [9000]), ([40], [8192]), ([300], [20001]), ([2048], [9000]), ([100, 3, 0, 64], [5000, 3, 0, 8200]),
                                   ([50, 20, 33], [10000, 0, 20]), ([9000 - 8000, 700], [1000, 8300]), ([1] * 40, [700 + 13 * i for i in range(40)])])
def test_split_over_long_keys(cuda, product_lib, nq, nk):
    """Few rows over long keys: the key tiles cut into spans, the cut query tiles joined; rows without keys, short and empty
    sequences beside them."""
    torch = cuda
    d = inputs(torch, 80 + sum(nq), nq, nk, 16, 2, pad=3)
    ops, keep = operands(torch, d)
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
    split = product_lib.scratch_bytes(row, ops, S.prefill_params(d["q"].shape[0], 16, 2)) > 0
    assert split == (len(nq) < 40)   # many sequences of some 1,000 keys are quicker whole
    if split:
        assert product_lib.launch(row, ops, S.prefill_params(d["q"].shape[0], 16, 2)) == abi.E_INVAL      # without its workspace
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d, heads=None if sum(nq) < 500 else [0, 5, 8, 15])


@pytest.mark.parametrize("nq,nk,hq,hkv", [([16], [4096], 16, 2), ([1], [1024], 16, 2), ([300], [6000], 16, 2), ([1500], [1500], 2, 2),
                                          ([16, 1, 1, 100], [4000, 20, 90, 300], 16, 2), ([20, 20, 400], [800, 2000, 400], 8, 1),
                                          ([4] * 8, [1000, 900, 800, 700, 1200, 1000, 50, 3000], 16, 2), ([64], [20000], 8, 8)])
def test_split_of_few_query_tiles(cuda, product_lib, nq, nk, hq, hkv):
    """Fewer query tiles than pairs: cut into many pieces, a few, none."""
    torch = cuda
    d = inputs(torch, 68, nq, nk, hq, hkv, pad=2)
    params, (ops, keep) = S.prefill_params(d["q"].shape[0], hq, hkv), operands(torch, d)
    assert product_lib.scratch_bytes(product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE), ops, params) > 0
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d, heads=sorted({0, hq // 2, hq - 1}))


@pytest.mark.parametrize("hq,hkv", [(3, 1), (12, 2), (40, 1), (128, 1)])
def test_split_head_groups(cuda, product_lib, hq, hkv):
    torch = cuda
    d = inputs(torch, 90 + hq, [25, 7], [9000, 31], hq, hkv, gain=12.0)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


def test_long_prompt(cuda, product_lib):
    """Many query tiles a CTA, the ring and every barrier through many phases."""
    torch = cuda
    d = inputs(torch, 51, [6000, 1500], [6000, 3333], 16, 2)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d, heads=[0, 7, 8, 13])


def test_weights_far_apart(cuda, product_lib):
    """Scores that span hundreds, and a maximum that rises along the keys: the sums are rescaled again and again."""
    torch = cuda
    d = inputs(torch, 52, [900], [900], 16, 2, gain=40.0)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)
    d = inputs(torch, 53, [64], [1500], 8, 1)
    d["q"][:] = d["q"][0, 0]
    d["k"][:, 0] = (d["q"][0, 0].float()[None] * (torch.arange(1500, device="cuda")[:, None] / 300.0)).to(torch.bfloat16)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)
    d["k"] = d["k"].flip(0).contiguous()       # and one that falls
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


def test_strides_and_scale(cuda, product_lib):
    """q, k, v slices of one fused projection row, o into a wider row, a scale of its own; k and v as planes of a
    [rows, 2, Hkv, D] cache."""
    torch = cuda
    d = inputs(torch, 54, [140, 60], [140, 60], 12, 2)
    row = torch.full((200, 16 * D + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    for name, at, h in (("q", 0, 12), ("k", 12 * D, 2), ("v", 14 * D, 2)):
        row[:, at:at + h * D] = d[name].reshape(200, -1)
        d[name] = row[:, at:at + h * D].view(200, h, D)
    whole = torch.full((200, 13, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    d["o"] = whole[:, 1:, 8:]
    assert call(product_lib, torch, d, scale=0.02) == abi.OK
    check(torch, d, 0.02)
    whole[:, 1:, 8:] = 7.0
    assert (whole == 7.0).all()
    d = inputs(torch, 55, [90], [300], 8, 2)
    cache = torch.stack([d["k"], d["v"]], 1)
    d["k"], d["v"] = cache[:, 0], cache[:, 1]
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("T", [1, 45, 260])
def test_head_major_operands(cuda, product_lib, T):
    """q, k, v and o kept a head after the other ([heads, rows, D] seen as [rows, heads, D]), o larger than its rows."""
    torch = cuda
    d = inputs(torch, 70 + T, [T], [T], 12, 3)
    for name in ("q", "k", "v"):
        d[name] = d[name].transpose(0, 1).contiguous().transpose(0, 1)
    whole = torch.full((12, T + 2, D), 7.0, dtype=torch.bfloat16, device="cuda")
    d["o"] = whole[:, 1:T + 1].transpose(0, 1)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)
    assert (whole[:, 0] == 7.0).all() and (whole[:, T + 1] == 7.0).all()


def test_in_place(cuda, product_lib):
    """o may be q itself."""
    torch = cuda
    d = inputs(torch, 75, [300, 41], [300, 41], 16, 2)
    q = d["q"].clone()
    d["o"] = d["q"]
    assert call(product_lib, torch, d) == abi.OK
    check(torch, dict(d, q=q))


def test_nan_stays_in_its_sequence(cuda, product_lib):
    """NaN and infinities in one sequence's q, k and v reach no row of another, nor rows 128 or more before them; keys'
    NaN reach no earlier row at all."""
    torch = cuda
    nq = [100, 200, 70]
    d = inputs(torch, 56, nq, nq, 16, 2)
    d["q"][150], d["k"][160], d["v"][299] = float("nan"), float("inf"), float("nan")
    assert call(product_lib, torch, d) == abi.OK
    got = d["o"]
    clean = inputs(torch, 56, nq, nq, 16, 2)
    assert call(product_lib, torch, clean) == abi.OK
    same = (got == clean["o"]).all(dim=2).all(dim=1)
    assert same[:100].all() and same[300:].all() and same[100:150].all()
    assert torch.isnan(got[150]).all() and torch.isnan(got[299]).all()
    check(torch, clean)


@pytest.mark.parametrize("nq,nk,hq,hkv,at", [(700, 700, 16, 2, 500), (700, 700, 2, 2, 600), (300, 9000, 16, 2, 8900), (520, 6000, 3, 3, 5800),
                                             (40, 2000, 8, 1, 1970)])
def test_how_far_a_nan_value_reaches(cuda, product_lib, nq, nk, hq, hkv, at):
    """A NaN in v: every row that sees it is NaN, rows whose last key lies more than 126 + 256 / group before it are as
    without it. Whole query tiles and split ones."""
    torch = cuda
    d = inputs(torch, 67, [nq], [nk], hq, hkv)
    assert call(product_lib, torch, d) == abi.OK
    clean = d["o"].clone()
    check(torch, d)
    d["v"][at] = float("nan")
    assert call(product_lib, torch, d) == abi.OK
    first = at - (nk - nq)   # the first row that sees it
    assert torch.isnan(d["o"][max(first, 0):]).all()
    far = first - (126 + 256 // (hq // hkv))
    assert far <= 0 or torch.equal(d["o"][:far], clean[:far])


def test_more_than_32_bits_of_keys(cuda, product_lib):
    """Keys and values at the far end of operands of more than 2^31 elements."""
    torch = cuda
    rows, n = 4_300_000, 200
    k, v = (torch.empty(rows, 2, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    d = inputs(torch, 57, [n], [n], 16, 2)
    k[-n:], v[-n:] = d["k"], d["v"]
    small = dict(d)
    d["k"], d["v"], d["cu_k"] = k, v, [rows - n, rows]
    assert call(product_lib, torch, d) == abi.OK
    check(torch, dict(small, o=d["o"]))


def test_lists_out_of_order(cuda, product_lib):
    """cu lists outside their operands are clamped, a falling pair is an empty sequence: nothing out of range is read
    or written."""
    torch = cuda
    d = inputs(torch, 58, [60], [60], 8, 2, pad=4)
    d["cu_q"], d["cu_k"] = [-5, 40, 30, 1 << 30], [-7, 40, 35, 1 << 30]
    assert call(product_lib, torch, d) == abi.OK
    k = dict(d, k=torch.nan_to_num(d["k"]), v=torch.nan_to_num(d["v"]))
    o, bound, rows = S.prefill_reference(torch, k["q"], k["k"], k["v"], [0, 40], [0, 40])
    assert ((d["o"][:30].double() - o[:30]).abs() <= bound[:30]).all()


def test_repeats_streams_and_graphs(cuda, product_lib):
    """The same call gives the same bits, eagerly and from graphs of several calls, split ones with a workspace each, replayed
    side by side."""
    torch = cuda
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
    calls = []
    for seed, n, nk in ((59, [500, 33], [500, 33]), (60, [1200], [1200]), (61, [70], [9999]), (62, [200], [8500])):
        d = inputs(torch, seed, n, nk, 16, 2)
        assert call(product_lib, torch, d) == abi.OK
        check(torch, d)
        ops, keep = operands(torch, d)
        size = product_lib.scratch_bytes(row, ops, S.prefill_params(sum(n), 16, 2))
        ws = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device="cuda")
        keep.append(ws)
        bound = product_lib.bind(row, ops, S.prefill_params(sum(n), 16, 2), scratch=ws.data_ptr(), scratch_bytes=size)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
        calls.append((d, d["o"].clone(), graph, stream, keep))
    for _ in range(5):
        for d, *_ in calls:
            d["o"].zero_()
        torch.cuda.synchronize()
        for _, _, graph, stream, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for d, want, *_ in calls:
            assert torch.equal(d["o"], want)
    assert product_lib.lib.ridgefill_device_error(1) == 0


@pytest.mark.parametrize("nq,nk", [([16] * 3, [512] * 3), ([5, 16], [0, 512]), ([200], [8192])])
def test_next_kernel_sees_the_answer(cuda, product_lib, nq, nk):
    """What follows a split call on its stream, or in its graph, comes after all of it: also where every span is a whole query
    tile, so that the join, whose launch overlaps the split's run, has nothing to add."""
    torch = cuda
    d = inputs(torch, 63, nq, nk, 8, 1)
    more = 9000 - d["k"].shape[0]   # rows behind the last sequence: the call is split by the operands' extent
    if more > 0:
        d["k"], d["v"] = (torch.cat([d[x], torch.full((more, 1, D), float("nan"), dtype=d[x].dtype, device="cuda")]) for x in "kv")
    ops, keep = operands(torch, d)
    row, params = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE), S.prefill_params(sum(nq), 8, 1)
    n = product_lib.scratch_bytes(row, ops, params)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    bound = product_lib.bind(row, ops, params, scratch=ws.data_ptr(), scratch_bytes=n)
    stream, graph, seen = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(d["o"])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
        seen.copy_(d["o"])
        d["o"].fill_(7.0)
    with torch.cuda.stream(stream):
        for _ in range(20):
            graph.replay()
            stream.synchronize()
            check(torch, dict(d, o=seen))
        for _ in range(20):
            assert bound(stream.cuda_stream) == abi.OK
            seen.copy_(d["o"])
            d["o"].fill_(7.0)
            stream.synchronize()
            check(torch, dict(d, o=seen))


def test_lists_that_overlap(cuda, product_lib):
    """Sequences that share rows (a list that falls and rises again) read and write in range, and the rows that only the first
    one holds are its own."""
    torch = cuda
    d = inputs(torch, 64, [300], [9000], 8, 2)
    d["cu_q"], d["cu_k"] = [0, 200, 100, 300], [0, 9000, 0, 8900]   # rows 0 .. 199, none, and rows 100 .. 299
    assert call(product_lib, torch, d) == abi.OK
    o, bound, _ = S.prefill_reference(torch, d["q"], d["k"], d["v"], [0, 200], [0, 9000])
    assert ((d["o"][:100].double() - o[:100]).abs() <= bound[:100]).all()
    assert product_lib.lib.ridgefill_device_error(1) == 0


@pytest.mark.parametrize("keys", [700, 9000])
def test_a_replay_takes_the_lengths_of_its_moment(cuda, product_lib, keys):
    """One captured call, whole and split, replayed with other sequences in the same rows."""
    torch = cuda
    d = inputs(torch, 66, [600], [keys], 16, 2)
    cu = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2)]
    ops, params = [H.dev(d["q"]), H.dev(d["k"]), H.dev(d["v"]), H.dev(cu[0]), H.dev(cu[1]), H.dev(d["o"])], S.prefill_params(600, 16, 2)
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
    n = product_lib.scratch_bytes(row, ops, params)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    bound = product_lib.bind(row, ops, params, scratch=ws.data_ptr(), scratch_bytes=n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
    for q, k in (([0, 600, 600, 600], [0, keys, keys, keys]), ([0, 1, 400, 600], [0, 1, 500, keys]), ([0] * 4, [0] * 4),
                 ([7, 7, 300, 301], [0, 5, 290, keys]), ([0, 600, 600, 600], [0, 3, 3, 3])):
        d["cu_q"], d["cu_k"] = q, k
        for t, x in zip(cu, (q, k)):
            t.copy_(torch.tensor(x, dtype=torch.int32))
        d["o"].fill_(7.0)
        graph.replay()
        check(torch, d)
    assert product_lib.lib.ridgefill_device_error(1) == 0


@pytest.mark.parametrize("nq,nk,hq,hkv", [([40], [9000], 16, 2), ([300, 20], [6000, 400], 16, 2), ([64], [20000], 8, 8)])
def test_nan_in_a_split_call(cuda, product_lib, nq, nk, hq, hkv):
    """A NaN in a row of q, or in keys that fill whole pieces of it, makes the row NaN as it does in whole query tiles, where
    the maximum of its scores passes over it; the other rows and heads are as without it."""
    torch = cuda
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)

    def clean():
        return inputs(torch, 69, nq, nk, hq, hkv)

    d = clean()
    assert product_lib.scratch_bytes(row, operands(torch, d)[0], S.prefill_params(sum(nq), hq, hkv)) > 0
    assert call(product_lib, torch, d) == abi.OK
    want = d["o"]
    d = clean()
    d["q"][17, 3, 100] = float("nan")
    d["q"][nq[0] - 1, 0] = float("nan")
    assert call(product_lib, torch, d) == abi.OK
    assert torch.isnan(d["o"][17, 3]).all() and torch.isnan(d["o"][nq[0] - 1, 0]).all()
    d["o"][17, 3], d["o"][nq[0] - 1, 0] = want[17, 3], want[nq[0] - 1, 0]
    assert torch.equal(d["o"], want)
    group = hq // hkv
    for first, last in ((0, nk[0]), (128, 4096), (2000, 2001)):   # every key of the sequence, those of whole pieces, one key
        d = clean()
        d["k"][first:last, 1, 77] = float("nan")
        assert call(product_lib, torch, d) == abi.OK
        assert torch.isnan(d["o"][:nq[0], group:2 * group]).all(), (first, last)
        d["o"][:nq[0], group:2 * group] = want[:nq[0], group:2 * group]
        assert torch.equal(d["o"], want)


@pytest.mark.parametrize("nq,nk", [([37] * 60, [37] * 60), ([70, 1, 129] * 30, [200, 1, 129] * 30), ([30] * 3, [9001, 77, 3])])
def test_sequence_ends_beside_nan_values(cuda, product_lib, nq, nk):
    """Last key tiles that hold rows of other sequences, which a CTA clears before the pair's product reads them: the odd
    sequences' v NaN, the even ones' answers finite, within their bounds and bit for bit the same a hundred times."""
    torch = cuda
    d = inputs(torch, 71, nq, nk, 16, 2, pad=3)
    odd = torch.zeros(d["v"].shape[0], dtype=torch.bool, device="cuda")
    rows = torch.zeros(d["q"].shape[0], dtype=torch.bool, device="cuda")
    for i in range(len(nq)):
        (rows[d["cu_q"][i]:d["cu_q"][i + 1]] if i % 2 == 0 else odd[d["cu_k"][i]:d["cu_k"][i + 1]])[:] = True
    clean = dict(d, o=d["o"].clone())
    assert call(product_lib, torch, clean) == abi.OK
    check(torch, clean, heads=[0, 15])
    d["v"][odd] = float("nan")
    for _ in range(100):
        d["o"].fill_(7.0)
        assert call(product_lib, torch, d) == abi.OK
        assert torch.equal(d["o"][rows], clean["o"][rows])


def test_a_wait_gives_up_for_the_whole_warp(cuda, product_lib):
    """Failure detection without a fault: a wait that half of a warp's lanes see complete and half do not gives up after its
    limit in all of them, records its code, and the same context then answers a prompt."""
    import ctypes
    torch = cuda
    lib = product_lib.lib
    lib.ridgefill_device_error(1)
    fn = lib.ridgefill_attn_wait_selftest
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert fn(None, None) == abi.E_INVAL
    status = torch.full((32,), 7, dtype=torch.int32, device="cuda")
    assert fn(status.data_ptr(), torch.cuda.current_stream().cuda_stream) == abi.OK
    torch.cuda.synchronize()
    assert status.tolist() == [0] * 32
    assert lib.ridgefill_device_error(1) == 0x401
    assert lib.ridgefill_device_error(0) == 0
    d = inputs(torch, 72, [130, 9], [130, 200], 16, 2)
    assert call(product_lib, torch, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("nq,nk,hq,hkv", [([53], [17], 16, 2), ([300, 20], [100, 20], 8, 1), ([40] * 40, [3] * 40, 4, 1), ([129], [128], 128, 1),
                                          ([20, 64], [9000, 10], 16, 2), ([10, 40, 700], [9000, 1, 650], 16, 2)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_without_keys_beside_values_that_are_not_finite(cuda, product_lib, nq, nk, hq, hkv, value):
    """A row that sees no key is zero, whatever its sequence's keys, values and other rows hold; whole query tiles and split
    calls."""
    torch = cuda
    d = inputs(torch, 73, nq, nk, hq, hkv)
    clean = dict(d, o=d["o"].clone())
    assert call(product_lib, torch, clean) == abi.OK
    check(torch, clean, heads=[0, hq - 1])
    empty = [(q0, max(a - b, 0)) for q0, a, b in zip(d["cu_q"], nq, nk)]
    for name in ("v", "k", "q"):
        d[name][:] = value
        d["o"].fill_(7.0)
        assert call(product_lib, torch, d) == abi.OK
        for q0, n in empty:
            assert (d["o"][q0:q0 + n] == 0).all(), name
