"""What the paged-cache calls refuse, before they touch a device (no GPU needed)."""
import ctypes as C

import pytest
import torch

import pulsar_amd as pq
from pulsar_amd._abi import PagedKVView

ARG, ALIGN, WS = -1, -2, -3


def _view(**kw):
    c = PagedKVView()
    f = dict(k=4096, v=8192, page_stride=16 * 8 * 64, npages=4, page=16, nkv=8, hd=64, dtype=2, table=64,
             table_stride=4, table_pages=4, kv_len=64, q_start=64, nseq=2)
    f.update(kw)
    for name, x in f.items():
        setattr(c, name, x)
    return C.byref(c)


def _prep(view, qkv=64, rs=3104, q=128, qs=2048, qn=64, kn=64, cs=64, rows=64, nh=32, rot=32, T=5):
    return pq.lib().pq_paged_qk_prep(qkv, rs, q, qs, qn, kn, cs, rows, view, nh, rot, T, 1e-5, None)


def _decode(view, q=64, qs=3104, gate=64, gs=3104, out=64, os=2048, qx=None, dx=None, nh=32, win=0, sinks=0, most=64,
            ws=None, wn=0):
    return pq.lib().pq_paged_attn_decode(q, qs, view, gate, gs, out, os, qx, dx, nh, 0.125, win, sinks, most, ws, wn, None)


def _prefill(view, q=64, qs=3104, gate=64, gs=3104, out=64, os=2048, qx=None, dx=None, nh=32, T=5, win=0, sinks=0,
             most=64, ws=None, wn=0):
    return pq.lib().pq_paged_attn_prefill(q, qs, view, gate, gs, out, os, qx, dx, nh, T, 0.125, win, sinks, most, ws, wn,
                                          None)


@pytest.mark.parametrize("bad,code,word", [
    (dict(k=None), ARG, b"null"), (dict(v=None), ARG, b"null"), (dict(table=None), ARG, b"null"),
    (dict(kv_len=None), ARG, b"null"), (dict(hd=96), ARG, b"head_dim"), (dict(dtype=0), ARG, b"type"),
    (dict(page=4), ARG, b"page"), (dict(page=48), ARG, b"page"), (dict(page=131072), ARG, b"page"),
    (dict(npages=0), ARG, b"npages"), (dict(nkv=0), ARG, b"nkv"), (dict(nseq=0), ARG, b"nseq"), (dict(nseq=65536), ARG, b"nseq"),
    (dict(table_pages=0), ARG, b"table"), (dict(table_stride=3), ARG, b"table"),
    (dict(page_stride=16 * 8 * 64 - 8), ARG, b"stride"), (dict(page_stride=16 * 8 * 64 + 4), ARG, b"stride"),
    (dict(k=4104), ALIGN, b"aligned"), (dict(v=8200), ALIGN, b"aligned")])
def test_bad_caches(bad, code, word):
    for call in (_prep, _decode, _prefill):
        assert call(_view(**bad)) == code, (call.__name__, bad)
        assert word in pq.lib().pq_last_error(), (bad, pq.lib().pq_last_error())


def test_null_view():
    for call in (_prep, _decode, _prefill):
        assert call(None) == ARG


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(q=None), dict(qn=None), dict(kn=None), dict(cs=None), dict(rows=0), dict(nh=0), dict(nh=30),
    dict(nh=136), dict(rot=33), dict(rot=66), dict(rot=-2), dict(T=0), dict(rs=3000), dict(qs=2047),
    dict(q=64, qs=2048)])
def test_bad_prep(bad):
    assert _prep(_view(), **bad) == ARG, bad


def test_rows_without_q_start():
    assert _prep(_view(q_start=None), T=3) == ARG
    assert _prefill(_view(q_start=None), T=3) == ARG
    assert b"q_start" in pq.lib().pq_last_error()


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(out=None), dict(qx=64), dict(nh=0), dict(nh=30), dict(nh=136), dict(win=-1), dict(win=(1 << 30) + 1),
    dict(sinks=-1), dict(most=0), dict(qs=2047), dict(os=2047), dict(gs=31)])
def test_bad_attention(bad):
    for call in (_decode, _prefill):
        assert call(_view(), **bad) == ARG, (call.__name__, bad)
    for T in (0, (1 << 23) + 1):
        assert _prefill(_view(), T=T) == ARG and _prep(_view(), T=T) == ARG
    assert _decode(_view(nkv=1024, nseq=65535, page_stride=1 << 20), nh=1024, qs=65536, os=65536, gs=1024) == ARG


def _tensors(nseq=2, pages=3, dtype=torch.float16):
    k = torch.zeros((4, 16, 8, 64), dtype=dtype)
    return k, k.clone(), torch.zeros((nseq, pages), dtype=torch.int32), torch.zeros(nseq, dtype=torch.int32)


def test_view_refusals():
    k, v, t, n = _tensors()
    pq.PagedKV(k, v, t, n)
    for bad in ((k.float(), v.float(), t, n), (k, v.bfloat16(), t, n), (k[0], v[0], t, n), (k, v[:2], t, n),
                (k.transpose(1, 2), v.transpose(1, 2), t, n), (k[::2], v[:2], t, n), (k, v, t.long(), n), (k, v, t, n.long()),
                (k, v, t[0], n), (k, v, t.t(), n), (k, v, t, n[:1]), (k, v, t, torch.zeros(4, dtype=torch.int32)[::2]),
                (k, v, t, n, n), (k, v, t, n, torch.zeros(3, dtype=torch.int64)),
                (k, v, t[:1].expand(2, 3), n)):
        with pytest.raises(ValueError):
            pq.PagedKV(*bad)


def test_call_refusals():
    kv = pq.PagedKV(*_tensors(), torch.zeros(3, dtype=torch.int32))
    rows = torch.zeros((2, 3104), dtype=torch.bfloat16)
    w, cs = torch.ones(64), torch.zeros((40, 16, 2))
    for bad in (dict(qkv=rows.float()), dict(qkv=rows[0]), dict(qkv=rows[:, :3000]), dict(qkv=rows.t()),
                dict(q_norm=w.half()), dict(q_norm=w[:32]), dict(rope_cs=cs[..., :1]), dict(rope_cs=cs.half()),
                dict(out=rows[:1, :2048]), dict(out=rows[:, :2040])):
        kw = dict(qkv=rows, q_norm=w, k_norm=w, rope_cs=cs)
        kw.update(bad)
        with pytest.raises(ValueError):
            pq.paged_qk_prep(kv, nh=32, rot=32, **kw)
    qx, dx = torch.zeros((2, 2048), dtype=torch.int8), torch.zeros((2, 64))
    for call in (pq.paged_attn_decode, pq.paged_attn_prefill):
        for bad in (dict(q=rows.float()), dict(q=rows[:, :2040]), dict(gate=rows[:1, :32]), dict(gate=rows[:, :31]),
                    dict(out=rows[:, :2040]), dict(out=rows[:1]), dict(qx=qx), dict(qx=qx, dx=dx.half()),
                    dict(qx=qx[:, :64], dx=dx), dict(qx=qx.float(), dx=dx), dict(win=-1), dict(sinks=-1), dict(win=2 ** 32),
                    dict(max_kv=0), dict(max_kv=2 ** 31), dict(ws=torch.zeros(8, 8)[:, :4])):
            kw = dict(q=rows)
            kw.update(bad)
            with pytest.raises(ValueError):
                call(kv, nh=32, scale=0.125, **kw)
        with pytest.raises(ValueError, match="GPU"):
            call(kv, rows, 32, 0.125)
    with pytest.raises(ValueError):
        pq.paged_attn_decode(kv, rows[:1], 32, 0.125)
    with pytest.raises(ValueError, match="GPU"):
        pq.paged_qk_prep(kv, rows, w, w, cs, 32, 32)


INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("most,win,sinks", [
    (INT_MAX, 1, INT_MAX), (INT_MAX, 1, INT_MAX - 1), (INT_MAX, 30, INT_MAX), (INT_MAX - 1, 1, INT_MAX), (INT_MAX, 1, 1 << 30),
    (INT_MAX, 0, INT_MAX), (INT_MAX, 1 << 30, 0)])
def test_largest_lengths_and_sinks(most, win, sinks):
    """The tiles of a length near 2^31 are counted without a wrap: about all of them are seen here, so that the call
    is split as one of 2^30 keys that are all seen is, and needs as large a workspace."""
    need = pq.lib().pq_paged_decode_workspace_bytes
    assert need(1, 32, 8, 64, 1 << 30, 0, 0) > 0
    assert need(1, 32, 8, 64, most, win, sinks) == need(1, 32, 8, 64, 1 << 30, 0, 0)


def test_sizes_past_an_int():
    """The library's sizes are ints: a stride or a count that does not fit one is refused, not cut to its low 32 bits
    (the storage is never touched)."""
    k, v, t, n = _tensors()
    start = torch.zeros(3, dtype=torch.int32)
    kv = pq.PagedKV(k, v, t, n, start)
    rows = torch.zeros((2, 3104), dtype=torch.bfloat16)
    far = torch.empty_strided((2, 3104), ((1 << 32) + 3104, 1), dtype=torch.bfloat16)
    w, cs = torch.ones(64), torch.zeros((40, 16, 2))
    for kw in (dict(qkv=far), dict(qkv=rows, out=far)):
        with pytest.raises(ValueError, match="stride"):
            pq.paged_qk_prep(kv, q_norm=w, k_norm=w, rope_cs=cs, nh=32, rot=32, **kw)
    for call in (pq.paged_attn_decode, pq.paged_attn_prefill):
        for kw in (dict(q=far), dict(q=rows, gate=far), dict(q=rows, out=far)):
            with pytest.raises(ValueError, match="stride"):
                call(kv, nh=32, scale=0.125, **kw)
        for nh in (32 - (1 << 32), 0, -8):
            with pytest.raises(ValueError, match="nh"):
                call(kv, rows, nh, 0.125)
    with pytest.raises(ValueError, match="nh"):
        pq.paged_qk_prep(kv, rows, w, w, cs, 32 - (1 << 32), 32, out=rows)
    wide = torch.empty_strided((2, 3), ((1 << 32) + 3, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="table"):
        pq.PagedKV(k, v, wide, n, start)


def test_strides_of_dimensions_of_one():
    """The stride of a dimension of size 1 says nothing: such tensors, which contiguous() would return as they are, are
    taken."""
    n, start = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((3, 1), dtype=torch.int32).t()                   # [1][3], strides 1, 1
    pool = torch.zeros((4, 1, 16, 64), dtype=torch.float16).transpose(1, 2)   # one kv head, [4][16][1][64]
    assert pool.is_contiguous() and table.is_contiguous()
    kv = pq.PagedKV(pool, pool.clone(), table, n, start)
    assert kv.c.page_stride == 16 * 64 and kv.c.table_stride == kv.c.table_pages == 3
    one = torch.zeros((1, 16, 8, 64), dtype=torch.float16)
    one = one.as_strided(one.shape, (8, 512, 64, 1))                     # a pool of one page
    assert pq.PagedKV(one, one, table, n).c.page_stride == 16 * 8 * 64
    row = torch.zeros((64 * 4, 1), dtype=torch.bfloat16).t()             # one row, strides 1, 1
    assert row.is_contiguous()
    for call in (pq.paged_attn_decode, pq.paged_attn_prefill):
        with pytest.raises(ValueError, match="GPU"):                     # all else is in order
            call(kv, row, 4, 0.125)
    assert pq.ops._paged_rows(kv, "q", row, 256)[1:] == (256, 1)
    assert pq.ops._paged_rows(kv, "q", row[:, :192], 128)[1:] == (192, 1)
