"""The serving rows' table and operand checks, without a GPU: schemas and rows beside the plugin's own, a description
for every operand, the refusal codes of broken operand sets (parses read descriptors only), and the bound call."""
import ctypes as C
import re

import pytest

import harness as H
import serve as S
from harness import abi

OPS = {
    "ridgefill_attn_prefill": (["M", "n_head", "n_head_kv", "head_dim", "scale"],
                               ["q", "k", "v", "cu_seqlens", "cu_keys", "o"]),
    "ridgefill_attn_decode": (["M", "n_head", "n_head_kv", "head_dim", "page", "scale"],
                              ["q", "kv_cache", "block_table", "kv_lens", "o"]),
    "ridgefill_gdn_step": (["M", "n_head_k", "n_head_v", "head_k", "head_v", "scale"],
                           ["q", "k", "v", "g", "beta", "state", "state_idx", "out_idx", "o"]),
}


def cold_params(op):
    return {"ridgefill_attn_prefill": lambda: S.prefill_params(40, 16, 2),
            "ridgefill_attn_decode": lambda: S.decode_params(3, 16, 2, 16),
            "ridgefill_gdn_step": lambda: S.step_params(3, 2, 4)}[op]()


def test_table(product_lib):
    schemas = {s.op.decode(): s for s in product_lib.serve_schemas()}
    rows = {r.op.decode(): r for r in product_lib.serve_rows()}
    plugin = {s.op.decode() for s in product_lib.schemas()}
    for op, (params, operands) in OPS.items():
        assert op in schemas and op in rows and op not in plugin
        sc = schemas[op]
        assert [sc.params[i].key.decode() for i in range(sc.n_params)] == params
        assert [sc.operands[i].name.decode() for i in range(sc.n_operands)] == operands
        assert rows[op].domain == abi.DOMAIN_DEVICE
        assert product_lib.find_row(op, abi.DOMAIN_DEVICE).name == rows[op].name
        assert product_lib.schema(op).op == op.encode()
    assert set(schemas) == set(rows)
    n = product_lib.lib.ridgefill_serve_count()
    assert not product_lib.lib.ridgefill_serve_at(n) and not product_lib.lib.ridgefill_serve_at(-1)


def test_descriptions(product_lib):
    for op in OPS:
        sc, row = product_lib.schema(op), product_lib.find_row(op, abi.DOMAIN_DEVICE)
        params = cold_params(op)
        pp = (abi.RadParam * len(params))(*params)
        d = abi.RadOpdDesc()
        for i in range(sc.n_operands):
            assert row.opd_shape(pp, len(params), i, C.byref(d)) == abi.OK, (op, i)
        assert row.opd_shape(pp, len(params), sc.n_operands, C.byref(d)) == abi.E_SHAPE


def test_exports_every_declared_entry_point(product_lib):
    text = (H.ROOT / "include" / "ridgefill_serve.h").read_text()
    block = text[text.find('extern "C" {'):]
    names = set(re.findall(r"^\s*(?:const\s+)?[A-Za-z_][\w\s\*]*?\b(\w+)\s*\(", block, re.M))
    assert {"ridgefill_serve_at", "ridgefill_attn_decode_device", "ridgefill_gdn_step_device"} <= names
    assert not [n for n in sorted(names) if not hasattr(product_lib.lib, n)]


# ----------------------------------------------------------------- refusals (fake addresses: nothing is read)

BASE = 1 << 20


def T(dtype, shape, strides=None, off=0):
    return abi.tensor(dtype, shape, BASE + off, strides)


def prefill_case(T_=40, keys=70, hq=16, hkv=2, D=256, n=3):
    return dict(q=T(abi.BF16, [T_, hq, D]), k=T(abi.BF16, [keys, hkv, D]), v=T(abi.BF16, [keys, hkv, D]),
                cu_q=T(abi.I32, [n + 1]), cu_k=T(abi.I32, [n + 1]), o=T(abi.BF16, [T_, hq, D]))


def decode_case(B=3, hq=16, hkv=2, D=256, page=16, pages=5, slots=400):
    return dict(q=T(abi.BF16, [B, hq, D]), kv_cache=T(abi.BF16, [2, slots, hkv, D]), block_table=T(abi.I32, [B, pages]),
                kv_lens=T(abi.I32, [B]), o=T(abi.BF16, [B, hq, D]))


def step_case(B=3, hk=2, hv=4, dk=128, dv=128, slots=5):
    return dict(q=T(abi.BF16, [B, hk, dk]), k=T(abi.BF16, [B, hk, dk]), v=T(abi.BF16, [B, hv, dv]), g=T(abi.F32, [B, hv]),
                beta=T(abi.F32, [B, hv]), state=T(abi.F32, [slots, hv, dv, dk]), state_idx=T(abi.I32, [B]),
                out_idx=abi.absent(), o=T(abi.BF16, [B, hv, dv]))


PREFILL = [
    (abi.OK, {}, {}),
    (abi.OK, dict(cu_k=abi.absent()), {}),
    (abi.OK, dict(q=T(abi.BF16, [40, 16, 256], [20 * 256, 256, 1])), {}),
    (abi.OK, dict(k=T(abi.BF16, [70, 2, 256], [1024, 256, 1]), v=T(abi.BF16, [70, 2, 256], [1024, 256, 1], off=1024)), {}),
    (abi.E_INVAL, dict(v=abi.absent()), {}),
    (abi.E_INVAL, {}, dict(n_head_kv=None)),
    (abi.E_INVAL, {}, dict(scale=float("nan"))),
    (abi.E_INVAL, {}, dict(scale=0.0)),
    (abi.E_INVAL, {}, dict(scale=-0.1)),
    (abi.E_UNSUPPORTED, {}, dict(head_dim=64)),
    (abi.E_UNSUPPORTED, {}, dict(n_head_kv=5)),
    (abi.E_UNSUPPORTED, dict(q=T(abi.BF16, [40, 258, 256])), dict(n_head=258)),                # 129 heads a kv head
    (abi.E_DTYPE, dict(k=T(abi.F16, [70, 2, 256])), {}),
    (abi.E_DTYPE, dict(cu_q=T(abi.I64, [4])), {}),
    (abi.E_DTYPE, dict(o=T(abi.F32, [40, 16, 256])), {}),
    (abi.E_SHAPE, {}, dict(M=41)),
    (abi.E_SHAPE, dict(v=T(abi.BF16, [71, 2, 256])), {}),
    (abi.E_SHAPE, dict(cu_k=T(abi.I32, [3])), {}),
    (abi.E_SHAPE, dict(cu_q=T(abi.I32, [0])), {}),
    (abi.E_SHAPE, dict(o=T(abi.BF16, [40, 16, 128])), {}),
    (abi.E_SHAPE, dict(k=T(abi.BF16, [1 << 31, 2, 256]), v=T(abi.BF16, [1 << 31, 2, 256])), {}),
    (abi.E_STRIDE, dict(cu_q=T(abi.I32, [4], [2])), {}),
    (abi.E_STRIDE, dict(q=T(abi.BF16, [40, 16, 256], off=4)), {}),
    (abi.E_STRIDE, dict(k=T(abi.BF16, [70, 2, 256], [516, 256, 1])), {}),
    (abi.E_STRIDE, dict(v=T(abi.BF16, [70, 2, 256], [0, 256, 1])), {}),
    (abi.E_STRIDE, dict(k=T(abi.BF16, [70, 2, 256], [-512, 256, 1])), {}),
]

DECODE = [
    (abi.OK, {}, {}),
    (abi.OK, dict(block_table=T(abi.I32, [3, 5], [9, 1])), {}),
    (abi.OK, dict(q=T(abi.BF16, [3, 16, 256], [16 * 264, 264, 1])), {}),
    (abi.OK, dict(kv_cache=T(abi.BF16, [2, 400, 2, 256], [512, 1024, 256, 1])), {}),       # [slots, 2, Hkv, D] seen as planes
    (abi.E_INVAL, dict(kv_lens=abi.absent()), {}),
    (abi.E_INVAL, {}, dict(page=None)),
    (abi.E_INVAL, {}, dict(scale=float("nan"))),
    (abi.E_INVAL, {}, dict(scale=float("inf"))),
    (abi.E_INVAL, {}, dict(scale=-1.0)),
    (abi.E_UNSUPPORTED, {}, dict(head_dim=128)),
    (abi.E_UNSUPPORTED, {}, dict(n_head_kv=3)),                                            # 16 heads over 3
    (abi.E_DTYPE, dict(q=T(abi.F16, [3, 16, 256])), {}),
    (abi.E_DTYPE, dict(kv_cache=T(abi.F32, [2, 400, 2, 256])), {}),
    (abi.E_DTYPE, dict(block_table=T(abi.I64, [3, 5])), {}),
    (abi.E_SHAPE, {}, dict(page=0)),
    (abi.E_SHAPE, {}, dict(page=(1 << 20) + 1)),
    (abi.E_SHAPE, {}, dict(M=4)),
    (abi.E_SHAPE, dict(kv_cache=T(abi.BF16, [3, 400, 2, 256])), {}),
    (abi.E_SHAPE, dict(kv_cache=T(abi.BF16, [2, 400, 1, 256])), {}),
    (abi.E_SHAPE, dict(block_table=T(abi.I32, [2, 5])), {}),
    (abi.E_SHAPE, dict(block_table=T(abi.I32, [3, 1 << 28])), {}),                         # keys past 32 bits
    (abi.E_SHAPE, dict(block_table=T(abi.I32, [3, 1 << 44])), dict(page=1 << 20)),         # and past 64
    (abi.E_SHAPE, dict(q=T(abi.BF16, [1 << 31, 16, 256]), o=T(abi.BF16, [1 << 31, 16, 256]), kv_lens=T(abi.I32, [1 << 31]),
                       block_table=T(abi.I32, [1 << 31, 5])), dict(M=1 << 31)),
    (abi.E_SHAPE, dict(o=T(abi.BF16, [3, 16, 128])), {}),
    (abi.E_STRIDE, dict(block_table=T(abi.I32, [3, 5], [10, 2])), {}),
    (abi.E_STRIDE, dict(kv_lens=T(abi.I32, [3], [2])), {}),
    (abi.E_STRIDE, dict(q=T(abi.BF16, [3, 16, 256], off=8)), {}),
    (abi.E_STRIDE, dict(kv_cache=T(abi.BF16, [2, 400, 2, 256], [400 * 520, 520, 260, 1])), {}),
    (abi.E_STRIDE, dict(o=T(abi.BF16, [3, 16, 256], [16 * 512, 512, 2])), {}),
]

STEP = [
    (abi.OK, {}, {}),
    (abi.OK, dict(out_idx=T(abi.I32, [3, 2])), {}),
    (abi.OK, dict(state=T(abi.F32, [5, 4, 128, 128], [4 * 128 * 128 + 4, 128 * 128, 128, 1])), {}),
    (abi.OK, dict(g=T(abi.F32, [3, 4], [8, 1])), {}),
    (abi.E_INVAL, dict(state_idx=abi.absent()), {}),
    (abi.E_INVAL, {}, dict(head_v=None)),
    (abi.E_INVAL, {}, dict(scale=float("inf"))),
    (abi.E_UNSUPPORTED, {}, dict(head_k=96)),
    (abi.E_UNSUPPORTED, {}, dict(head_v=64)),                                              # 128 x 64
    (abi.E_UNSUPPORTED, {}, dict(n_head_k=3)),
    (abi.E_DTYPE, dict(state=T(abi.BF16, [5, 4, 128, 128])), {}),
    (abi.E_DTYPE, dict(g=T(abi.BF16, [3, 4])), {}),
    (abi.E_DTYPE, dict(out_idx=T(abi.I64, [3])), {}),
    (abi.E_SHAPE, {}, dict(M=2)),
    (abi.E_SHAPE, dict(state_idx=T(abi.I32, [4])), {}),
    (abi.E_SHAPE, dict(out_idx=T(abi.I32, [2])), {}),
    (abi.E_SHAPE, dict(state=T(abi.F32, [5, 2, 128, 128])), {}),
    (abi.E_SHAPE, dict(beta=T(abi.F32, [3, 2])), {}),
    (abi.E_STRIDE, dict(state=T(abi.F32, [5, 4, 128, 128], [4 * 128 * 132, 128 * 132, 132, 1])), {}),
    (abi.E_STRIDE, dict(state=T(abi.F32, [5, 4, 128, 128], off=4)), {}),
    (abi.E_STRIDE, dict(k=T(abi.BF16, [3, 2, 128], off=2)), {}),
    (abi.E_STRIDE, dict(beta=T(abi.F32, [3, 4], [1, 3])), {}),
    (abi.E_STRIDE, dict(state_idx=T(abi.I32, [3, 2], [1, 3])), {}),
]


def _params(base, change):
    out = []
    for p in base:
        key = p.key.decode()
        if key not in change:
            out.append(p)
        elif change[key] is not None:
            out.append(H.pint(key, change[key]))
    return out + [H.pf64("scale", change["scale"]) for _ in range("scale" in change)]


@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill_refusals(product_lib, case):
    want, operands, params = PREFILL[case]
    tensors = list((prefill_case() | operands).values())
    assert S.parse(product_lib, "ridgefill_attn_prefill_parse", tensors, _params(S.prefill_params(40, 16, 2), params)) == want


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode_refusals(product_lib, case):
    want, operands, params = DECODE[case]
    tensors = list((decode_case() | operands).values())
    assert S.parse(product_lib, "ridgefill_attn_decode_parse", tensors, _params(S.decode_params(3, 16, 2, 16), params)) == want


@pytest.mark.parametrize("case", range(len(STEP)))
def test_step_refusals(product_lib, case):
    want, operands, params = STEP[case]
    tensors = list((step_case() | operands).values())
    assert S.parse(product_lib, "ridgefill_gdn_step_parse", tensors, _params(S.step_params(3, 2, 4), params)) == want


def test_null_arguments(product_lib):
    for op in OPS:
        assert S.parse(product_lib, op + "_parse", [], []) == abi.E_INVAL


def test_no_rows_is_no_work(product_lib):
    """M = 0 with every operand given: accepted, nothing is launched (so it needs no device)."""
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
    assert product_lib.launch(row, list(prefill_case(T_=0).values()), S.prefill_params(0, 16, 2)) == abi.OK
    assert product_lib.launch(row, list(prefill_case(n=0).values()), S.prefill_params(40, 16, 2)) == abi.OK
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    assert product_lib.launch(row, list(decode_case(B=0).values()), S.decode_params(0, 16, 2, 16)) == abi.OK
    row = product_lib.find_row("ridgefill_gdn_step", abi.DOMAIN_DEVICE)
    assert product_lib.launch(row, list(step_case(B=0).values()), S.step_params(0, 2, 4)) == abi.OK
    assert product_lib.bind(row, list(step_case(B=0).values()), S.step_params(0, 2, 4))(None) == abi.OK


def test_decode_needs_its_workspace(product_lib):
    """A call without the workspace its hook asks for is refused before any launch."""
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    tensors, params = list(decode_case(pages=64, slots=4096).values()), S.decode_params(3, 16, 2, 16)
    need = product_lib.scratch_bytes(row, tensors, params)
    assert need > 0
    assert product_lib.launch(row, tensors, params) == abi.E_INVAL
    assert product_lib.launch(row, tensors, params, scratch=BASE, scratch_bytes=need - 1) == abi.E_INVAL
    assert product_lib.launch(row, tensors, params, scratch=BASE + 8, scratch_bytes=need) == abi.E_INVAL


def test_rows_found_by_several_threads():
    """A library's first lookups from two threads at once: the second one, while the first still reads the tables, finds its
    row too."""
    import threading
    H.build_product()
    lib = abi.Plugin(abi.PRODUCT_SO)
    inside, go, read = threading.Event(), threading.Event(), lib.rows

    def slow():
        lib.rows = read
        inside.set()
        assert go.wait(30)
        return read()

    lib.rows = slow
    got = []
    first = threading.Thread(target=lambda: got.append(lib.find_row("ridgefill_gdn_step", abi.DOMAIN_DEVICE)))
    first.start()
    assert inside.wait(30)
    second = lib.find_row("ridgefill_gdn_fill", abi.DOMAIN_DEVICE)
    go.set()
    first.join()
    assert second is not None and second.op == b"ridgefill_gdn_fill"
    assert got[0] is not None and got[0].op == b"ridgefill_gdn_step"
    assert lib.find_row("no_such_row", abi.DOMAIN_DEVICE) is None


# An address no kernel can read or write: not a multiple of its element's size.
UNALIGNED = [
    ("ridgefill_attn_prefill", "cu_q", abi.I32, [4], 2), ("ridgefill_attn_prefill", "cu_k", abi.I32, [4], 1),
    ("ridgefill_attn_decode", "block_table", abi.I32, [3, 5], 2), ("ridgefill_attn_decode", "kv_lens", abi.I32, [3], 3),
    ("ridgefill_gdn_step", "v", abi.BF16, [3, 4, 128], 1), ("ridgefill_gdn_step", "o", abi.BF16, [3, 4, 128], 7),
    ("ridgefill_gdn_step", "g", abi.F32, [3, 4], 2), ("ridgefill_gdn_step", "beta", abi.F32, [3, 4], 1),
    ("ridgefill_gdn_step", "state_idx", abi.I32, [3], 2), ("ridgefill_gdn_step", "out_idx", abi.I32, [3], 2),
]


@pytest.mark.parametrize("op,name,dtype,shape,off", UNALIGNED)
def test_unaligned_addresses(product_lib, op, name, dtype, shape, off):
    """Refused, and one element behind an aligned one accepted."""
    base = {"ridgefill_attn_prefill": prefill_case, "ridgefill_attn_decode": decode_case, "ridgefill_gdn_step": step_case}[op]()
    for at, want in ((off, abi.E_STRIDE), (2 if dtype == abi.BF16 else 4, abi.OK)):
        tensors = list((base | {name: T(dtype, shape, off=at)}).values())
        assert S.parse(product_lib, op + "_parse", tensors, cold_params(op)) == want


HUGE = 3074457345618258603   # 6 of them are 2 past 2^64


def test_step_extents_past_64_bits(product_lib):
    """M times n_head_v is checked before it is a grid: extents whose product passes 64 bits are refused, not wrapped."""
    row = product_lib.find_row("ridgefill_gdn_step", abi.DOMAIN_DEVICE)
    for B, hv in ((6, HUGE), (1 << 33, 4), (2, 1 << 31)):
        tensors = dict(q=T(abi.BF16, [B, 1, 128], [128, 128, 1]), k=T(abi.BF16, [B, 1, 128], [128, 128, 1]),
                       v=T(abi.BF16, [B, hv, 128], [128, 128, 1]), g=T(abi.F32, [B, hv], [1, 1]), beta=T(abi.F32, [B, hv], [1, 1]),
                       state=T(abi.F32, [5, hv, 128, 128], [1 << 14, 1 << 14, 128, 1]), state_idx=T(abi.I32, [B]),
                       out_idx=abi.absent(), o=T(abi.BF16, [B, hv, 128], [128, 128, 1]))
        assert product_lib.launch(row, list(tensors.values()), S.step_params(B, 1, hv)) == abi.E_SHAPE, (B, hv)


def test_prefill_extents_past_64_bits(product_lib):
    """The query tiles of all kv heads are counted without wrapping: too many of them are refused, and need no workspace."""
    row = product_lib.find_row("ridgefill_attn_prefill", abi.DOMAIN_DEVICE)
    for T_, h, n in ((1280, HUGE, 1), (40, 1 << 62, 1), (256, 1 << 29, 3)):
        tensors = dict(q=T(abi.BF16, [T_, h, 256], [256, 256, 1]), k=T(abi.BF16, [1 << 20, h, 256], [256, 256, 1]),
                       v=T(abi.BF16, [1 << 20, h, 256], [256, 256, 1]), cu_q=T(abi.I32, [n + 1]), cu_k=T(abi.I32, [n + 1]),
                       o=T(abi.BF16, [T_, h, 256], [256, 256, 1]))
        params = S.prefill_params(T_, h, h)
        assert product_lib.scratch_bytes(row, list(tensors.values()), params) == 0
        assert product_lib.launch(row, list(tensors.values()), params) == abi.E_SHAPE, (T_, h)


def test_decode_scratch_of_a_refused_call(product_lib):
    """Extents that the call refuses need no workspace; their products are not formed."""
    row = product_lib.find_row("ridgefill_attn_decode", abi.DOMAIN_DEVICE)
    for B, h in ((3, HUGE * 2), (1 << 30, 1 << 40)):
        tensors = dict(q=T(abi.BF16, [B, h, 256], [256, 256, 1]), kv_cache=T(abi.BF16, [2, 400, h, 256], [256, 256, 256, 1]),
                       block_table=T(abi.I32, [B, 64]), kv_lens=T(abi.I32, [B]), o=T(abi.BF16, [B, h, 256], [256, 256, 1]))
        params = S.decode_params(B, h, h, 16)
        assert product_lib.launch(row, list(tensors.values()), params) == abi.E_SHAPE
        assert product_lib.scratch_bytes(row, list(tensors.values()), params) == 0


@pytest.mark.parametrize("op,case", [("ridgefill_attn_prefill", prefill_case), ("ridgefill_attn_decode", decode_case)])
def test_scales_that_overflow(product_lib, op, case):
    """The kernels work in powers of two: a scale whose product with log2(e) is no finite f32 is refused."""
    for scale, want in ((3e38, abi.E_INVAL), (2.4e38, abi.E_INVAL), (2.3e38, abi.OK), (1e-30, abi.OK), (1e-60, abi.E_INVAL)):
        params = cold_params(op) + [H.pf64("scale", scale)]
        assert S.parse(product_lib, op + "_parse", list(case().values()), params) == want, scale


def test_prefill_rows_and_keys_in_32_bits(product_lib):
    """A query tile's last key is reckoned from rows and keys together, in 32 bits: both at their most are refused."""
    for rows, keys, want in ((1 << 30, 0x7ffffe00, abi.E_SHAPE), (1 << 30, (1 << 30) - 512, abi.OK), (1 << 30, (1 << 30) - 511, abi.E_SHAPE),
                             (40, 0x7ffffe00 - 40, abi.OK), (40, 0x7ffffe00 - 39, abi.E_SHAPE)):
        tensors = list(prefill_case(T_=rows, keys=keys, hq=2).values())
        assert S.parse(product_lib, "ridgefill_attn_prefill_parse", tensors, S.prefill_params(rows, 2, 2)) == want, (rows, keys)
