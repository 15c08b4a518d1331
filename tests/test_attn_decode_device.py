"""ridgefill_attn_decode on B200 against its formula in 64 bits, element by element within the bound of its arithmetic:
lengths of zero, one and around the 16- and 64-key blocks, ragged batches, every kind of head group and page size,
strides, pages outside the pool, NaN in slots that no sequence owns, offsets past 32 bits, and its workspace."""
import pytest

import harness as H
import serve as S
from harness import abi

pytestmark = pytest.mark.gpu
D = 256


def inputs(torch, seed, lens, hq, hkv, page, spare=3, gain=2.0, width=None):
    """Every sequence's pages anywhere in a pool with `spare` unowned pages; unowned slots and the ends of last pages
    hold NaN, table entries past a sequence's pages lie outside the pool."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lens)
    used = [-(-max(n, 0) // page) for n in lens]
    pages = sum(used) + spare
    width = max(max(used), 1) if width is None else width
    cache = torch.full((2, pages * page, hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((B, width), 1 << 30, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        mine = order[at:at + used[i]][:width]
        at += used[i]
        table[i, :len(mine)] = mine
        j = torch.arange(min(max(n, 0), width * page), device="cuda")
        slots = mine.long()[j // page] * page + j % page
        cache[:, slots] = torch.randn(2, len(j), hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    q = (gain * torch.randn(B, hq, D, device="cuda", generator=g)).to(torch.bfloat16)
    return dict(q=q, cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                o=torch.full_like(q, 7.0), page=page)


def call(lib, d, scale=None):
    B, hq, _ = d["q"].shape
    ops = [H.dev(d[n]) for n in ("q", "cache", "table", "lens", "o")]
    return H.launch(lib, "ridgefill_attn_decode", ops, S.decode_params(B, hq, d["cache"].shape[2], d["page"], scale=scale))


def check(torch, d, scale=None):
    o, bound = S.decode_reference(torch, d["q"], d["cache"], d["table"], d["lens"].tolist(), d["page"], scale)
    err = (d["o"].double() - o).abs()
    assert (err <= bound).all(), f"{int((~(err <= bound)).sum())} elements off, at most {float((err / bound).max()):.2f} bounds"


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500]


@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 256])
def test_edge_lengths(cuda, product_lib, page):
    torch = cuda
    d = inputs(torch, page, EDGES, 16, 2, page)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("length", [0, 1, 5, 64, 65, 128])
def test_one_short_sequence(cuda, product_lib, length):
    """At most two units of keys: one CTA an item, no join, no workspace."""
    torch = cuda
    d = inputs(torch, 100 + length, [length], 16, 2, 16, width=8)
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    ops = [H.dev(d[n]) for n in ("q", "cache", "table", "lens", "o")]
    assert product_lib.scratch_bytes(row, ops, S.decode_params(1, 16, 2, 16)) == 0
    assert call(product_lib, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (8, 1), (12, 2), (15, 5), (16, 1), (24, 3), (17, 1), (40, 2), (128, 1)])
def test_head_groups(cuda, product_lib, hq, hkv):
    torch = cuda
    d = inputs(torch, hq * 10 + hkv, [777, 3, 0, 260], hq, hkv, 32)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


@pytest.mark.parametrize("lens", [[32768], [32767, 1], [5000, 9, 12345, 1, 1, 20001, 64, 700], [40] * 300, [0] * 70 + [1000]])
def test_ragged_batches(cuda, product_lib, lens):
    """One long sequence over every SM, long beside short, many short ones, empty ones before a full one."""
    torch = cuda
    d = inputs(torch, len(lens), lens, 16, 2, 64)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


def test_weights_far_apart(cuda, product_lib):
    """Scores that span hundreds: one key takes all the weight, wherever it lies; and the maximum rising along the
    sequence, which rescales the sums again and again."""
    torch = cuda
    d = inputs(torch, 41, [3000, 700], 16, 2, 16, gain=40.0)
    assert call(product_lib, d) == abi.OK
    check(torch, d)
    d = inputs(torch, 42, [2000], 8, 1, 16)
    j = torch.arange(2000, device="cuda")
    slots = d["table"][0].long()[j // 16] * 16 + j % 16
    d["cache"][0, slots, 0] = (d["q"][0, 0].float()[None] * (j[:, None] / 400.0)).to(torch.bfloat16)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


def test_strides(cuda, product_lib):
    """q a slice of a fused projection row, o into a wider row, a table wider than its row and with a pitch, the cache
    as [slots, 2, Hkv, D] seen as two planes, a scale of its own, negative and too long lengths."""
    torch = cuda
    d = inputs(torch, 43, [130, 70, 333, 0], 16, 2, 16)
    B = 4
    row = torch.zeros(B, 16, 2 * D + 8, dtype=torch.bfloat16, device="cuda")
    row[:, :, D:2 * D] = d["q"]
    d["q"] = row[:, :, D:2 * D]
    d["o"] = torch.full((B, 20, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    whole, d["o"] = d["o"], d["o"][:, 2:18, 8:]
    table = torch.full((B, 60), -5, dtype=torch.int32, device="cuda")
    table[:, :d["table"].shape[1]] = d["table"]
    d["table"] = table[:, :50]
    inter = d["cache"].permute(1, 0, 2, 3).contiguous()
    d["cache"] = inter.permute(1, 0, 2, 3)
    d["lens"][3] = -9
    assert call(product_lib, d, scale=0.11) == abi.OK
    check(torch, d, 0.11)
    whole[:, 2:18, 8:] = 7.0
    assert (whole == 7.0).all()
    d["lens"][:] = 1 << 30     # past the table: all its pages, those outside the pool left out
    d["cache"] = torch.nan_to_num(d["cache"])      # those inside it are read to their ends
    assert call(product_lib, d, scale=0.11) == abi.OK
    check(torch, dict(d, lens=torch.tensor([50 * 16] * B)), 0.11)


def test_head_major_cache(cuda, product_lib):
    """The cache kept as [Hkv, 2, slots, D], o and q a head after the other."""
    torch = cuda
    d = inputs(torch, 50, [700, 33, 128], 12, 3, 16)
    d["cache"] = d["cache"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    d["q"] = d["q"].transpose(0, 1).contiguous().transpose(0, 1)
    d["o"] = torch.full((12, 3, D), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


def test_empty_pool_and_table(cuda, product_lib):
    """No slot in the pool, or no page in the table: every row is zero."""
    torch = cuda
    d = inputs(torch, 51, [300, 40], 8, 2, 16)
    empty = dict(d, cache=d["cache"][:, :0], o=d["o"].clone())
    ops = [H.dev(d["q"]), abi.tensor(abi.BF16, (2, 0, 2, D), d["cache"].data_ptr(), (0, 512, 256, 1)), H.dev(d["table"]), H.dev(d["lens"]),
           H.dev(empty["o"])]
    assert H.launch(product_lib, "ridgefill_attn_decode", ops, S.decode_params(2, 8, 2, 16)) == abi.OK
    assert (empty["o"] == 0).all()
    ops = [H.dev(d["q"]), H.dev(d["cache"]), abi.tensor(abi.I32, (2, 0), d["table"].data_ptr()), H.dev(d["lens"]), H.dev(d["o"])]
    assert H.launch(product_lib, "ridgefill_attn_decode", ops, S.decode_params(2, 8, 2, 16)) == abi.OK
    assert (d["o"] == 0).all()


def test_pages_outside_the_pool(cuda, product_lib):
    """Keys on pages outside the pool are left out; a sequence that only has such is zero. The pool's last page may be
    cut short."""
    torch = cuda
    d = inputs(torch, 44, [200, 200, 90, 40], 16, 2, 16)
    d["table"][0, 3] = -1
    d["table"][0, 7] = d["cache"].shape[1] // 16
    d["table"][1, :] = -1
    d["table"][2, 5] = 1 << 27      # slot number past 32 bits after the product with the page
    assert call(product_lib, d) == abi.OK
    check(torch, d)
    assert (d["o"][1] == 0).all()
    d = inputs(torch, 45, [64], 8, 1, 16, spare=0)
    d["table"][0] = torch.tensor([3, 1, 2, 0])
    d["cache"] = torch.randn_like(d["cache"].float()).to(torch.bfloat16)[:, :60]
    assert call(product_lib, d) == abi.OK
    check(torch, d)


def test_infinite_scores_and_nan_inputs(cuda, product_lib):
    """A key whose score is -inf carries no weight; a NaN in one sequence and kv head reaches no other."""
    torch = cuda
    d = inputs(torch, 46, [300, 300], 4, 2, 1)
    d["q"][:] = d["q"].abs()
    d["cache"][0, d["table"][0, 37].long(), :, 0] = -float("inf")
    d["cache"][1, d["table"][1, 19].long(), 1] = float("nan")
    assert call(product_lib, d) == abi.OK
    assert torch.isnan(d["o"][1, 2:]).all()
    # without the key, and with the NaN out of the way
    without = dict(d, table=torch.cat([d["table"][:, :37], d["table"][:, 38:]], 1), lens=torch.tensor([299, 299]))
    without["table"][1] = d["table"][1, :299]
    o, bound = S.decode_reference(torch, d["q"][:1], d["cache"], without["table"][:1], [299], 1)
    assert ((d["o"][:1].double() - o).abs() <= bound).all()
    o, bound = S.decode_reference(torch, d["q"][1:, :2], d["cache"][:, :, :1], d["table"][1:], [300], 1)
    assert ((d["o"][1:, :2].double() - o).abs() <= bound).all()


def test_long_cache_offsets(cuda, product_lib):
    """A cache of more than 2^31 elements a plane, the sequence's pages at its far end."""
    torch = cuda
    page, pages, hkv = 64, 70000, 2
    g = torch.Generator(device="cuda").manual_seed(47)
    cache = torch.empty(2, pages * page, hkv, D, dtype=torch.bfloat16, device="cuda")
    assert cache[0].numel() > 2 ** 31
    table = torch.arange(pages - 12, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    cache[:, (pages - 12) * page:] = torch.randn(2, 12 * page, hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    q = torch.randn(1, 16, D, device="cuda", generator=g).to(torch.bfloat16)
    d = dict(q=q, cache=cache, table=table, lens=torch.tensor([750], dtype=torch.int32, device="cuda"), o=torch.zeros_like(q), page=page)
    assert call(product_lib, d) == abi.OK
    check(torch, d)


def test_repeats_streams_and_graphs(cuda, product_lib):
    """The same call gives the same bits; two captured graphs of different calls, each with its workspace, replayed
    side by side on two streams; the workspace's earlier contents do not matter."""
    torch = cuda
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    calls = []
    for seed, lens in ((48, [9000, 40, 3000]), (49, [100] * 40)):
        d = inputs(torch, seed, lens, 16, 2, 32)
        assert call(product_lib, d) == abi.OK
        check(torch, d)
        params = S.decode_params(len(lens), 16, 2, 32)
        ops = [H.dev(d[n]) for n in ("q", "cache", "table", "lens", "o")]
        n = product_lib.scratch_bytes(row, ops, params)
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
        bound = product_lib.bind(row, ops, params, scratch=ws.data_ptr(), scratch_bytes=n)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
        calls.append((d, d["o"].clone(), graph, stream, ws))
    for _ in range(5):
        for d, _, _, _, ws in calls:
            d["o"].zero_()
            ws.fill_(0xFF)
        torch.cuda.synchronize()
        for _, _, graph, stream, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for d, want, _, _, _ in calls:
            assert torch.equal(d["o"], want)


@pytest.mark.parametrize("lens", [[16] * 4, [60] * 300, [12, 0, 3], [2000, 7]])
def test_next_kernel_sees_the_answer(cuda, product_lib, lens):
    """What follows the call on its stream, or in its graph, comes after all of it: also where no item needs the join, whose
    launch overlaps the first kernel's run."""
    torch = cuda
    d = inputs(torch, 50, lens, 16, 2, 16, width=64)
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    params, ops = S.decode_params(len(lens), 16, 2, 16), [H.dev(d[n]) for n in ("q", "cache", "table", "lens", "o")]
    n = product_lib.scratch_bytes(row, ops, params)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
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


def test_a_replay_takes_the_lengths_of_its_moment(cuda, product_lib):
    """One captured call, replayed while the sequences grow, shrink to nothing and change places in the table."""
    torch = cuda
    top = [30000, 5000, 700, 64, 1, 0]
    d = inputs(torch, 53, top, 16, 2, 64)
    ops, params = [H.dev(d[n]) for n in ("q", "cache", "table", "lens", "o")], S.decode_params(len(top), 16, 2, 64)
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    n = product_lib.scratch_bytes(row, ops, params)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    bound = product_lib.bind(row, ops, params, scratch=ws.data_ptr(), scratch_bytes=n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert bound(torch.cuda.current_stream().cuda_stream) == abi.OK
    for i, lens in enumerate(([30000, 5000, 700, 64, 1, 0], [1, 2, 3, 4, 1, 0], [0] * 6, [29999, 0, 700, 0, 1, 0], [17, 4999, 0, 63, 0, 0])):
        order = torch.randperm(len(top), device="cuda")
        d["table"].copy_(d["table"][order].clone())
        top = [top[k] for k in order.tolist()]
        d["lens"].copy_(torch.tensor([min(a, b) for a, b in zip(lens, top)], dtype=torch.int32))
        d["o"].fill_(7.0)
        graph.replay()
        check(torch, d)
