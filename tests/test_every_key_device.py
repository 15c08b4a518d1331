"""Every key counted, on B200: with q = 0 all of a row's keys have the same weight, so that v's columns, each the indicator
of a few keys, come back as how many of them the row saw. One key lost, read twice or taken from another row, head or
sequence is off by a step of the count, where the bounds of random inputs grow with the length.

Weights are then 2^0 = 1 and every sum a whole number below 2^24, all exact in f32 (and 1 in bf16); what is left is the
division, two roundings of f32, and the output's rounding: within TOL of the count over the number of keys."""
import pytest

import harness as H
import serve as S
from harness import abi

gpu = pytest.mark.gpu
D = 256
EACH = 8                               # keys a column stands for, one run of them
WINDOW = EACH * D                      # keys that one call's columns cover
TOL = 1.01 * S.UB16 + 4 * S.U32        # relative, against steps of 1 / EACH or more


def indicator(torch, n, first, shift, device="cuda"):
    """[n, D]: key j of the window [first, first + WINDOW) is 1 in column ((j - first) // EACH + shift) % D, others 0."""
    j = torch.arange(n, device=device)
    v = torch.zeros(n, D, device=device)
    inside = (j >= first) & (j < first + WINDOW)
    v[j[inside], ((j[inside] - first) // EACH + shift) % D] = 1
    return v


def agrees(torch, o, counts, seen):
    """o [..., D] against counts [..., D] of `seen` keys; a row that saw none is zero."""
    want = counts.double() / seen.double().clamp(min=1)
    return bool(((o.double() - want).abs() <= TOL * want).all())


def test_a_key_lost_or_doubled_is_noticed():
    """The comparison itself: one key of 32,768 missing from its column, or there twice, with any rounding of the answer."""
    import torch
    n = 32768
    v = indicator(torch, n, 2048 * 7, 3, "cpu")
    counts = v.sum(0)
    for key, by in ((2048 * 7, -1), (2048 * 7 + 100, -1), (2048 * 8 - 1, 1)):
        off = counts + by * v[key]
        for nudge in (1 - S.UB16, 1, 1 + S.UB16):   # rounded down, not, up
            assert not agrees(torch, (off / (n + by) * nudge), counts, torch.tensor(n))
    assert agrees(torch, (counts / n).to(torch.bfloat16), counts, torch.tensor(n))


def launch(lib, name, tensors, params):
    assert H.launch(lib, name, tensors, params) == abi.OK
    assert lib.lib.ridgefill_device_error(1) == 0


LONG_BATCH = [1 + (i * 20011 + 32767) % 32768 for i in range(64)]


@gpu
@pytest.mark.parametrize("lens,hq,hkv,page", [
    ([32768], 16, 2, 64), ([20001], 16, 2, 16), ([32767, 1, 8191], 8, 1, 48), ([5000, 9, 12345, 1, 1, 20001, 64, 700], 16, 2, 64),
    ([256 + (i * 977) % 1793 for i in range(32)], 16, 2, 16), (LONG_BATCH, 16, 2, 64), ([9000, 0, 77], 40, 2, 32), ([2049], 128, 1, 7)])
def test_decode_sees_every_key_once(cuda, product_lib, lens, hq, hkv, page):
    """Spans, pieces and joins of every layout: short and long sequences, wide and narrow spans, several chunks of heads."""
    torch = cuda
    B, width = len(lens), max(-(-max(lens) // page), 1)
    used = [-(-n // page) for n in lens]
    g = torch.Generator(device="cuda").manual_seed(sum(lens))
    order = torch.randperm(sum(used), device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    cache = torch.ones(2, sum(used) * page, hkv, D, dtype=torch.bfloat16, device="cuda")   # what no key holds counts in every column
    slots, at = [], 0
    for i, n in enumerate(lens):
        table[i, :used[i]] = order[at:at + used[i]]
        at += used[i]
        j = torch.arange(n, device="cuda")
        slots.append(table[i].long()[j // page] * page + j % page)
    q = torch.zeros(B, hq, D, dtype=torch.bfloat16, device="cuda")
    o, seen = torch.empty_like(q), torch.tensor(lens, dtype=torch.int32, device="cuda")
    for first in range(0, max(lens), WINDOW):
        counts = torch.zeros(B, hkv, D, device="cuda")
        for i, n in enumerate(lens):
            for h in range(hkv):
                v = indicator(torch, n, first, 31 * i + 97 * h)
                cache[1, slots[i], h] = v.to(torch.bfloat16)
                counts[i, h] = v.sum(0)
        o.fill_(7.0)
        launch(product_lib, "ridgefill_attn_decode", [H.dev(q), H.dev(cache), H.dev(table), H.dev(seen), H.dev(o)],
               S.decode_params(B, hq, hkv, page))
        assert agrees(torch, o, counts.repeat_interleave(hq // hkv, dim=1), seen[:, None, None]), first


@gpu
@pytest.mark.parametrize("nq,nk,hq,hkv", [
    ([300], [20001], 16, 2), ([40], [8192], 16, 2), ([1], [9000], 16, 2), ([16], [4096], 16, 2), ([2048], [9000], 16, 2), ([64], [20000], 8, 8),
    ([100, 3, 0, 64], [5000, 3, 0, 8200], 16, 2), ([25, 7], [9000, 31], 40, 1),                                  # split
    ([700], [700], 16, 2), ([3000], [3000], 8, 1), ([300, 0, 45, 128, 1], [500, 0, 45, 128, 300], 12, 2), ([60] * 40, [90] * 40, 16, 2)])
def test_prefill_sees_every_key_once(cuda, product_lib, nq, nk, hq, hkv):
    """Whole query tiles and split ones, every row by how many of its keys each column holds."""
    torch = cuda
    T, K = sum(nq), sum(nk)
    cu = [torch.tensor([0] + list(torch.tensor(x).cumsum(0)), dtype=torch.int32, device="cuda") for x in (nq, nk)]
    q, k = torch.zeros(T, hq, D, dtype=torch.bfloat16, device="cuda"), torch.ones(K, hkv, D, dtype=torch.bfloat16, device="cuda")
    o, v = torch.empty_like(q), torch.empty_like(k)
    for first in range(0, max(nk), WINDOW):
        counts, seen = torch.zeros(T, hkv, D, device="cuda"), torch.zeros(T, device="cuda")
        q0 = k0 = 0
        for i, (a, b) in enumerate(zip(nq, nk)):
            last = torch.arange(a, device="cuda") + (b - a)   # each row's last key
            seen[q0:q0 + a] = (last + 1).clamp(min=0)
            for h in range(hkv):
                x = indicator(torch, b, first, 31 * i + 97 * h)
                v[k0:k0 + b, h] = x.to(torch.bfloat16)
                if a:
                    counts[q0:q0 + a, h] = torch.cat([x.new_zeros(1, D), x.cumsum(0)])[(last + 1).clamp(min=0)]
            q0, k0 = q0 + a, k0 + b
        o.fill_(7.0)
        launch(product_lib, "ridgefill_attn_prefill", [H.dev(q), H.dev(k), H.dev(v), H.dev(cu[0]), H.dev(cu[1]), H.dev(o)],
               S.prefill_params(T, hq, hkv))
        assert agrees(torch, o, counts.repeat_interleave(hq // hkv, dim=1), seen[:, None, None]), first
