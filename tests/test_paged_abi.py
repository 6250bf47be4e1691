"""Refusals of the paged KV cache's entry points, on the host before any launch (no GPU call is made), and their sizes."""
import ctypes

import pytest

from ameva_compute_amd._lib import PagedBatchStruct, PagedKVStruct, lib

F16, Q4_0, Q8_0 = 1, 2, 8
A = 4096  # an address that is aligned and never read


def kv(**more):
    return PagedKVStruct(**{**dict(type=F16, n_head_kv=2, D=128, page_size=16, n_pages=9, page_stride=2 * 16 * 256, k=A, v=A, bounds=A), **more})


def batch(**more):
    return PagedBatchStruct(**{**dict(n_seq=3, n_tok=3, max_q=1, max_kv=100, table_stride=7, cu_q=None, n_kv=A, table=A), **more})


def refs(k, b):
    return (None if k is None else ctypes.byref(k)), (None if b is None else ctypes.byref(b))


def attn(k, b, q=A, stride=1024, out=A, heads=8, ws=A, n=1 << 40):
    return lib().amv_paged_attn(*refs(k, b), q, stride, out, heads, 0.1, ws, n, None)


def shared(k, b, table=A, n_pre=20):
    return lib().amv_paged_attn_shared(*refs(k, b), table, n_pre, A, 1024, A, 8, 0.1, A, 1 << 40, None)


def sparse(k, b, sel=A, n_sel=4):
    return lib().amv_paged_attn_sparse(*refs(k, b), sel, n_sel, A, 1024, A, 8, 0.1, A, 1 << 40, None)


def select(k, b, n_sel=4, first=1, last=1, ws=A, n=1 << 40, sel=A):
    return lib().amv_paged_select(*refs(k, b), A, 1024, 8, n_sel, first, last, sel, ws, n, None)


def append(k, b, qkv=A, stride=12 * 128, heads=8, n_dims=128, mode=0, base=1e4, rule=0, out=A, out_stride=1024):
    return lib().amv_paged_rope_append(*refs(k, b), qkv, stride, heads, None, n_dims, mode, base, 1.0, 1.0, rule, out, out_stride, None,
                                       None)


def refused(rc, word):
    assert rc == -1 and word in lib().amv_last_error().decode(), (rc, lib().amv_last_error())


@pytest.mark.parametrize("call", [attn, shared, sparse, select, append])
def test_pools_and_batches(call):
    refused(call(None, batch()), "null pool")
    refused(call(kv(), None), "null pool")
    for bad in (dict(type=3), dict(type=0), dict(D=96), dict(D=256), dict(page_size=8), dict(page_size=48), dict(page_size=2048)):
        refused(call(kv(**bad), batch()), "not supported")
    for bad in (dict(k=None), dict(v=None), dict(n_pages=0), dict(n_pages=1 << 31)):
        refused(call(kv(**bad), batch()), "without pages")
    for bad in (dict(n_head_kv=0), dict(page_stride=2 * 16 * 256 - 16), dict(page_stride=2 * 16 * 256 + 8), dict(k=A + 2), dict(v=A + 8),
                dict(bounds=A + 4)):
        refused(call(kv(**bad), batch()), "KV heads")
    refused(call(kv(n_head_kv=3, page_stride=3 * 16 * 256), batch()), "8 heads over 3")
    for bad in (dict(n_kv=None), dict(table=None), dict(n_seq=0), dict(n_tok=-1), dict(max_q=0), dict(max_kv=-1)):
        refused(call(kv(), batch(**bad)), "null lengths or table")
    for bad in (dict(n_seq=70000, n_tok=70000), dict(n_tok=1 << 25, cu_q=A), dict(max_kv=(1 << 30) + 1)):
        refused(call(kv(), batch(**bad)), "too large")
    for bad in (dict(n_tok=4), dict(max_q=2)):
        refused(call(kv(), batch(**bad)), "one token a sequence")
    refused(call(kv(), batch(table_stride=6)), "columns of the table")
    assert call(kv(), batch(n_tok=0, cu_q=A)) == 0  # nothing to do


def test_attention():
    for bad in (dict(q=None), dict(out=None)):
        refused(attn(kv(), batch(), **bad), "null pointer")
    for bad in (dict(stride=1020), dict(stride=1026), dict(q=A + 4), dict(out=A + 8)):
        refused(attn(kv(), batch(), **bad), "16-byte aligned")
    need = lib().amv_paged_attn_workspace_bytes(*refs(kv(), batch(max_kv=100000, table_stride=6250)), 8, 0, 0)
    assert need > 0
    for bad in (dict(ws=None), dict(n=need - 1), dict(ws=A + 8)):
        refused(attn(kv(), batch(max_kv=100000, table_stride=6250), **{**dict(n=need), **bad}), "workspace")
    refused(shared(kv(), batch(), table=None), "without pages")
    refused(shared(kv(), batch(), n_pre=-1), "prefix")
    refused(sparse(kv(), batch(), sel=None), "selected")
    for n in (0, -1, 16385):
        refused(sparse(kv(), batch(), n_sel=n), "selected")


def test_select():
    refused(select(kv(bounds=None), batch()), "no bounds")
    refused(select(kv(), batch(), sel=None), "null pointer")
    for bad in (dict(n_sel=0), dict(first=-1), dict(last=-1), dict(first=3, last=2), dict(n_sel=16385)):
        refused(select(kv(), batch(), **bad), "pages with the first")
    refused(select(kv(), batch(max_kv=16 * 16385, table_stride=16385)), "more than 16384")
    long = batch(max_kv=160000, table_stride=10000)
    need = lib().amv_paged_select_workspace_bytes(*refs(kv(), long))
    assert need >= 3 * 2 * 10000 * 8
    for bad in (dict(ws=None), dict(n=need - 1), dict(ws=A + 8)):
        refused(select(kv(), long, **{**dict(n=need), **bad}), "workspace")


def test_append():
    for bad in (dict(qkv=None), dict(out=None)):
        refused(append(kv(), batch(), **bad), "null pointer")
    for bad in (dict(stride=12 * 128 - 4), dict(stride=12 * 128 + 2), dict(out_stride=1020), dict(out_stride=1025), dict(qkv=A + 8), dict(out=A + 4)):
        refused(append(kv(), batch(), **bad), "16-byte aligned")
    for m in (1, 3, -1):
        refused(append(kv(), batch(), mode=m), "rope mode")
    for n in (-2, 3, 130):
        refused(append(kv(), batch(), n_dims=n), "rotated")
    refused(append(kv(), batch(), base=0.0), "frequency base")
    for r in (-1, 3):
        refused(append(kv(), batch(), rule=r), "Q8_0 rule")


def test_sizes():
    c = lib().amv_paged_chunk_bytes
    assert (c(F16, 128, 16), c(Q8_0, 128, 64), c(Q4_0, 64, 32)) == (16 * 256, 64 * (128 + 8), 32 * (32 + 4))
    assert all(c(*a) == -1 for a in ((3, 128, 16), (F16, 96, 16), (F16, 128, 24), (F16, 128, 0), (F16, 128, -16), (Q8_0, 64, 4096)))
    w = lib().amv_paged_attn_workspace_bytes
    assert w(*refs(kv(), batch()), 8, 0, 0) == 0  # short sequences: no parts
    assert w(*refs(kv(), batch()), 8, -1, 0) == -1 and w(*refs(kv(D=100), batch()), 8, 0, 0) == -1
    empty = batch(n_tok=0, cu_q=A)
    assert [w(*refs(kv(), empty), 8, *a) for a in ((0, 0), (0, 5))] == [0, 0] and w(*refs(kv(), batch(n_tok=0, cu_q=A, max_kv=0)), 8, 9, 0) >= 0
    assert lib().amv_paged_select_workspace_bytes(*refs(kv(), empty)) == 0
    # parts of a prefix need room for every row, and the own keys' with them
    assert w(*refs(kv(), batch()), 8, 20, 0) >= 2 * 3 * 8 * (8 + 512)


def test_python_side():
    torch = pytest.importorskip("torch")
    from ameva_compute_amd import ops
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedKV(F16, *(torch.empty(2, 1, 16, 64, dtype=torch.float16) for _ in "kv"), 16, 1, 64)
    with pytest.raises(ValueError, match="not supported"):
        ops.PagedKV.alloc(F16, 2, 20, 1, 64, "cpu")
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedBatch(torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), 16)


def test_launches_that_would_be_too_large():
    """More workgroups than a grid has: sequences (even empty ones) of many KV heads, rows of many heads."""
    chunk = 16 * 256
    many = kv(n_head_kv=1024, page_stride=1024 * chunk)
    seqs = batch(n_seq=65535, n_tok=8, cu_q=A, max_q=1)
    refused(attn(many, seqs, heads=1024, stride=1024 * 128), "too large")
    refused(append(many, seqs, heads=1024, stride=3 * 1024 * 128, out_stride=1024 * 128), "too large")
    refused(attn(kv(), batch(n_seq=1, n_tok=(1 << 22) + 1, cu_q=A, max_q=9)), "too large")
    tokens = batch(n_seq=1, n_tok=(1 << 13) + 1, cu_q=A, max_q=9)
    rc = lib().amv_paged_select(*refs(many, tokens), A, 1024 * 128, 1024, 4, 1, 1, A, A, 1 << 40, None)
    refused(rc, "too large")
