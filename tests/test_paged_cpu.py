"""The paged cache's checks of arguments, and its entry points in the C ABI; nothing here reaches a GPU."""

import ctypes as C
import os
import re

import pytest
import torch

import hyquant_b200 as hq
from hyquant_b200 import _lib
from hyquant_b200 import paged_kv

FAKE = 1 << 20


def attention_args(**fields):
    """Arguments that pass every check; the addresses are made up.  T is 0: a call that passes returns before a launch."""
    a = _lib.PagedAttentionArgs()
    a.struct_bytes = C.sizeof(a)
    a.R, a.T, a.H_Q, a.H_KV, a.head_dim, a.page_size, a.max_pages, a.max_q_len = 2, 5, 8, 2, 128, 64, 10, 4
    a.dtype, a.sm_scale, a.num_pages = _lib.HQ_BF16, 0.1, 20
    for name in ("q", "pages", "page_table", "kv_lens", "cu_q", "out", "workspace"):
        setattr(a, name, FAKE)
    a.q_st = a.o_st = 1024
    a.q_sh = a.o_sh = 128
    a.table_stride, a.workspace_bytes = 10, 1 << 40
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("fields,code,text", [
    (dict(struct_bytes=8), -1, b"struct_bytes"), (dict(R=-1), -1, b"size"), (dict(T=-1), -1, b"size"), (dict(H_Q=0), -1, b"size"),
    (dict(H_KV=0), -1, b"size"), (dict(max_q_len=0), -1, b"size"), (dict(num_pages=-1), -1, b"size"), (dict(max_pages=-1), -1, b"size"),
    (dict(head_dim=64), -2, b"head_dim"), (dict(H_Q=9), -2, b"heads"), (dict(H_Q=34), -2, b"heads"), (dict(page_size=48), -2, b"page_size"),
    (dict(page_size=256), -2, b"page_size"), (dict(max_pages=1 << 28, table_stride=1 << 28), -2, b"tables"), (dict(dtype=2), -2, b"dtype"),
    (dict(sm_scale=-1.0), -1, b"sm_scale"), (dict(sm_scale=float("nan")), -1, b"sm_scale"), (dict(sm_scale=float("inf")), -1, b"sm_scale"),
    (dict(cu_q=None), -1, b"cu_q"), (dict(q=None), -1, b"null"), (dict(out=None), -1, b"null"), (dict(kv_lens=None), -1, b"null"),
    (dict(page_table=None), -1, b"null"), (dict(pages=None), -1, b"null"), (dict(table_stride=9), -1, b"overlap"),
    (dict(o_st=0), -1, b"overlap"), (dict(o_sh=64), -1, b"overlap"),
    (dict(q=FAKE + 8), -3, b"aligned"), (dict(out=FAKE + 2), -3, b"aligned"), (dict(pages=FAKE + 4), -3, b"aligned"),
    (dict(q_st=1028), -3, b"aligned"), (dict(o_sh=129), -3, b"aligned"),
])
def test_attention_refusals(fields, code, text):
    lib, n = _lib.lib(), C.c_int64()
    a = attention_args(**fields)
    assert lib.hq_paged_attention(C.byref(a), None) == code and text in lib.hq_last_error()
    assert lib.hq_paged_attention_workspace_bytes(C.byref(a), C.byref(n)) == code


@pytest.mark.parametrize("fields", [dict(R=4000, T=4096, H_Q=32, H_KV=8, max_q_len=4096, max_pages=1 << 13, page_size=128, table_stride=1 << 13),
                                    dict(R=3, T=1 << 20, max_q_len=1 << 20, max_pages=1 << 14, table_stride=1 << 14),
                                    dict(R=1 << 15, T=1 << 15, H_KV=8, max_q_len=1, max_pages=1 << 14, table_stride=1 << 14)])
def test_more_positions_than_32_bits_hold(fields):
    lib, n = _lib.lib(), C.c_int64()
    a = attention_args(**fields)
    assert lib.hq_paged_attention_workspace_bytes(C.byref(a), C.byref(n)) == -2 and b"too much" in lib.hq_last_error()
    assert lib.hq_paged_attention(C.byref(a), None) == -2 and b"too much" in lib.hq_last_error()


def test_attention_null_block_and_nothing_to_do():
    lib, n = _lib.lib(), C.c_int64(-1)
    assert lib.hq_paged_attention(None, None) == -1
    assert lib.hq_paged_attention_workspace_bytes(None, C.byref(n)) == -1
    assert lib.hq_paged_attention_workspace_bytes(C.byref(attention_args()), None) == -1
    for fields in (dict(T=0), dict(R=0), dict(T=0, q=None, out=None, pages=None)):
        assert lib.hq_paged_attention(C.byref(attention_args(**fields)), None) == 0
    assert lib.hq_paged_attention_workspace_bytes(C.byref(attention_args()), C.byref(n)) == 0 and n.value >= 0


def advance(**fields):
    a = _lib.PageAdvanceArgs()
    a.struct_bytes, a.R, a.T, a.page_size, a.max_pages, a.free_cap, a.table_stride = C.sizeof(a), 3, 4, 16, 10, 9, 10
    for name, kind in a._fields_:
        if kind is C.c_void_p and name != "keep":
            setattr(a, name, FAKE)
    for name, value in fields.items():
        setattr(a, name, value)
    return _lib.lib().hq_page_advance(C.byref(a), None)


@pytest.mark.parametrize("fields,code", [
    (dict(struct_bytes=100), -1), (dict(R=-1), -1), (dict(T=-1), -1), (dict(free_cap=-1), -1), (dict(max_pages=-1), -1), (dict(R=8193), -2),
    (dict(page_size=8), -2), (dict(page_size=0), -2), (dict(kv_lens=None), -1), (dict(add=None), -1), (dict(slots=None), -1), (dict(cu_q=None), -1),
    (dict(status=None), -1), (dict(page_table=None), -1), (dict(free_pages=None), -1), (dict(free_count_out=None), -1), (dict(table_stride=9), -1),
    (dict(R=8192, max_pages=1 << 20, table_stride=1 << 20), -2)])
def test_advance_refusals(fields, code):
    assert advance(**fields) == code


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), -1), (dict(H=0), -1), (dict(page=17), -2), (dict(dtype=3), -2), (dict(k=None), -1), (dict(slots=None), -1), (dict(pages=None), -1),
    (dict(k=FAKE + 8), -3), (dict(k_st=1020), -3), (dict(v_sh=4), -3), (dict(pages=FAKE + 8), -3), (dict(slots=FAKE + 4), -3), (dict(T=1 << 30, H=2), -2)])
def test_append_refusals(change, code):
    a = dict(k=FAKE, v=FAKE, dtype=0, k_st=1024, k_sh=128, v_st=1024, v_sh=128, T=4, H=8, slots=FAKE, pages=FAKE, num=10, page=64)
    a.update(change)
    assert _lib.lib().hq_paged_append(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), -1), (dict(H=0), -1), (dict(page=0), -2), (dict(dtype=-1), -2), (dict(k=None), -1), (dict(v=FAKE + 2), -3), (dict(slots=None), -1),
    (dict(num=-1), -1)])
def test_read_refusals(change, code):
    a = dict(pages=FAKE, num=10, page=64, slots=FAKE, T=4, H=8, dtype=0, k=FAKE, v=FAKE)
    a.update(change)
    assert _lib.lib().hq_paged_read(*a.values(), None) == code


def test_nothing_to_do_touches_nothing():
    lib = _lib.lib()
    assert lib.hq_paged_append(None, None, 0, 0, 0, 0, 0, 0, 8, None, None, 10, 64, None) == 0
    assert lib.hq_paged_append(FAKE, FAKE, 0, 1024, 128, 1024, 128, 4, 8, FAKE, None, 0, 64, None) == 0
    assert lib.hq_paged_read(None, 10, 64, None, 0, 8, 0, None, None, None) == 0


def test_python_refusals():
    with pytest.raises(ValueError):
        hq.paged_pages(4, 2, 48, device="cpu")
    pages = hq.paged_pages(4, 2, 64, device="cpu")
    assert pages.shape == (4, 2, 4, 2112) and pages.dtype == torch.uint8
    i32 = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 128)
    with pytest.raises(hq.HyQuantError):                                    # no CPU path
        hq.paged_attention(torch.zeros(1, 4, 128, dtype=torch.bfloat16), pages, torch.zeros(1, 4, dtype=torch.int32), i32)
    with pytest.raises(hq.HyQuantError):
        hq.paged_append(pages, x, x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(hq.HyQuantError):
        hq.paged_read(pages, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(hq.HyQuantError):
        hq.page_advance(i32, i32, i32, torch.zeros(1, 4, dtype=torch.int32), i32, i32, page_size=64, max_tokens=1)
    with pytest.raises(ValueError):
        hq.PagedKVCache(0, 4, 2, max_requests=1, max_pages_per_request=4, device="cpu")
    with pytest.raises(ValueError):
        hq.PagedKVCache(1, 4, 2, max_requests=1, max_pages_per_request=4, page_size=20, device="cpu")
    cache = hq.PagedKVCache(3, 4, 2, max_requests=2, max_pages_per_request=4, device="cpu")
    assert len(cache) == 3 and cache.free_pages.tolist() == [3, 2, 1, 0] and int(cache.free_count) == 4
    cache.check()                                                           # no step yet: nothing to report
    with pytest.raises(hq.HyQuantError):
        cache.append(0, x, x)


def test_argument_blocks_as_bytes():
    assert _lib.lib().hq_page_advance(None, None) == -1
    for struct_, pack, ints in ((_lib.PageAdvanceArgs, paged_kv._pack_advance, 21), (_lib.PagedAttentionArgs, paged_kv._pack_args, 26)):
        values = [0.5 if kind is C.c_float else i + 1 for i, (_, kind) in enumerate(struct_._fields_)]
        assert len(values) == ints
        a = struct_.from_buffer_copy(pack(*values))
        assert [getattr(a, name) for name, _ in struct_._fields_] == values


def test_format_constants():
    assert paged_kv.BLOCK_BYTES == 2 * paged_kv.BLOCK * 64 + 2 * paged_kv.BLOCK * 2
    assert [f[0] for f in _lib.PagedAttentionArgs._fields_][-2:] == ["workspace", "workspace_bytes"] and C.sizeof(_lib.PagedAttentionArgs) == 160


@pytest.mark.parametrize("name,mirror", [("hq_page_advance_args", _lib.PageAdvanceArgs), ("hq_paged_attention_args", _lib.PagedAttentionArgs)])
def test_the_listed_argument_blocks_are_the_bound_ones(name, mirror):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "INTEGRATION.md")).read()
    fields = eval(re.search(r"class %s\(C\.Structure\):\n    _fields_ = (\[.*?\)\])\n" % name, text, re.S).group(1), {"C": C})
    listed = type("Listed", (C.Structure,), {"_fields_": fields})
    assert [f[0] for f in fields] == [f[0] for f in mirror._fields_] and C.sizeof(listed) == C.sizeof(mirror)
    assert all(getattr(listed, f[0]).offset == getattr(mirror, f[0]).offset for f in fields)


def test_pieces_of_query_tiles_begin_on_16_bytes():
    """A query tile's piece in the workspace (its rows of 128 sums, a maximum and a sum each) is read and written in 16-byte pieces,
    two of them one behind the other per block and 32 bytes of a merge's order: whatever the rows, odd numbers of them too."""
    lib, n = _lib.lib(), C.c_int64()

    def workspace(G, most):
        a = attention_args(H_Q=G, H_KV=1, max_q_len=most, o_st=G * 128)
        assert lib.hq_paged_attention_workspace_bytes(C.byref(a), C.byref(n)) == 0
        return n.value
    full = 2 * 256 * 130 * 4 + 32
    blocks = workspace(1, 256) // full
    assert blocks >= 1 and workspace(1, 256) == blocks * full
    for G in range(1, 17):
        for most in range(16 // G + 1, 260):
            per, rest = divmod(workspace(G, most), blocks)
            assert rest == 0 and (per - 32) % 32 == 0 and (per - 32) // 2 >= min(256, most * G) * 130 * 4, (G, most)


@pytest.mark.parametrize("fields,apart", [
    (dict(), True), (dict(o_st=128, o_sh=128), False), (dict(o_st=512, o_sh=128), False), (dict(o_st=1016, o_sh=128), False), (dict(o_st=128, o_sh=640), True),
    (dict(o_st=128, o_sh=632), False), (dict(o_st=136, o_sh=672), True), (dict(o_st=136, o_sh=664), False), (dict(o_st=1080, o_sh=136), True),
    (dict(o_st=1072, o_sh=136), False), (dict(T=1, R=1, o_st=0, o_sh=128), True), (dict(T=1, R=1, o_st=0, o_sh=120), False),
    (dict(H_Q=1, H_KV=1, o_sh=0, o_st=128), True), (dict(H_Q=1, H_KV=1, o_sh=0, o_st=120), False), (dict(o_st=-1024), False), (dict(o_sh=-128), False),
    (dict(o_st=1 << 60, o_sh=1 << 58), False), (dict(o_st=1 << 40), True)])
def test_rows_of_the_output_lie_apart(fields, apart):
    """Five tokens of eight heads: every pair of strides that puts two rows on the same elements is refused."""
    lib, n = _lib.lib(), C.c_int64()
    a = attention_args(**fields)
    rc = lib.hq_paged_attention_workspace_bytes(C.byref(a), C.byref(n))
    assert rc == 0 if apart else rc == -1 and b"overlap" in lib.hq_last_error()
    if abs(a.o_st) < 1 << 20 and abs(a.o_sh) < 1 << 20:
        at = [t * a.o_st + h * a.o_sh + c for t in range(a.T) for h in range(a.H_Q) for c in range(128)]
        assert not apart or len(set(at)) == len(at)
        assert apart or len(set(at)) < len(at) or min(at) < 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,offset,st,sh,copied", [
    (5, 2, 0, 256, 128, False), (5, 2, 1, 256, 128, True), (5, 2, 4, 256, 128, None), (5, 2, 8, 256, 128, False), (5, 2, 0, 257, 128, True), (5, 2, 0, 384, 132, True),
    (5, 2, 0, 0, 128, False), (1, 2, 0, 257, 128, False), (1, 2, 3, 257, 128, True), (5, 1, 0, 136, 3, False), (1, 1, 0, 7, 5, False), (1, 1, 1, 7, 5, True),
    (0, 2, 1, 256, 128, None)])
def test_rows_the_kernels_cannot_read_as_they_lie_are_copied(T, H, offset, st, sh, copied, dtype):
    """Views at every offset and with every stride, contiguous ones at an odd offset among them; an index of one value has no stride."""
    flat = torch.arange(3000, dtype=torch.float32).remainder(251).to(dtype)
    x = flat.as_strided((T, H, 128), (st, sh, 1), offset)
    y, address, y_st, y_sh = paged_kv._rows(x)
    assert address == y.data_ptr() and address % 16 == 0 and (y_st | y_sh) % 8 == 0
    assert torch.equal(y, x) and (copied is None or (y is not x) == copied)
    size = y.element_size()
    for t in range(T):
        for h in range(H):
            assert address + (t * y_st + h * y_sh) * size == y[t, h].data_ptr()


def test_strides_of_a_single_token_and_of_a_single_head_do_not_count():
    lib, n = _lib.lib(), C.c_int64()
    for fields in (dict(T=1, R=1, q_st=3, o_st=5), dict(H_Q=1, H_KV=1, q_sh=1, o_sh=1, q_st=128, o_st=128)):
        assert lib.hq_paged_attention_workspace_bytes(C.byref(attention_args(**fields)), C.byref(n)) == 0


@pytest.mark.parametrize("name", [n for n, kind in _lib.PageAdvanceArgs._fields_ if kind is C.c_void_p])
def test_advance_refuses_misaligned_arrays(name):
    assert advance(**{name: FAKE + (4 if name == "slots" else 2)}) == -3 and b"aligned" in _lib.lib().hq_last_error()


@pytest.mark.parametrize("name", ["page_table", "kv_lens", "cu_q"])
def test_attention_refuses_misaligned_arrays(name):
    a = attention_args(**{name: FAKE + 2})
    assert _lib.lib().hq_paged_attention(C.byref(a), None) == -3 and b"aligned" in _lib.lib().hq_last_error()
