"""What the operators on the paged cache refuse, without a GPU: the C calls
return -1 before anything is queued (the pointers are never followed), and the
Python face raises before it calls the library."""
import ctypes as ct

import pytest
import torch

import secure_infer_amd as si
from secure_infer_amd import _lib

P = 0x10000  # a 16-byte aligned stand-in for a device address
BAD = (1 << 64) - 1


def attention(**kw):
    d = dict(q=P, q_token_stride=1024, q_head_stride=128, out=P, out_token_stride=1024, out_head_stride=128, cache_k=P,
             cache_v=P, slot_bytes=2 * 128 * 2 * 128, nslots=8, tables=P, table_stride=4, kv_lens=P, q_starts=P,
             table_pages=4, tokens=5, seqs=2, q_heads=8, kv_heads=2, head_dim=128, page_tokens=128, dtype=0, causal=1,
             window=0, scale=0.1)
    d.update(kw)
    return _lib.SiPagedAttentionDesc(**d)


@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(cache_k=None), dict(cache_v=None), dict(tables=None), dict(kv_lens=None),
    dict(tokens=0), dict(seqs=0), dict(q_heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(table_pages=0),
    dict(q_starts=None), dict(tokens=1 << 28, q_heads=16), dict(head_dim=0), dict(head_dim=124), dict(head_dim=264),
    dict(dtype=2), dict(page_tokens=4), dict(page_tokens=100), dict(page_tokens=65536), dict(table_pages=1 << 24),
    dict(nslots=0), dict(nslots=1 << 31), dict(slot_bytes=2 * 128 * 2 * 128 - 16), dict(slot_bytes=65544),
    dict(q_token_stride=1020), dict(q_head_stride=4), dict(out_token_stride=7), dict(out_head_stride=129),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(q=P + 8), dict(out=P + 2), dict(cache_k=P + 4),
    dict(cache_v=P + 8)])
def test_attention_refuses(change):
    L = _lib.load()
    assert L.secure_infer_gpu_paged_attention_workspace(ct.byref(attention())) != BAD
    d = attention(**change)
    assert L.secure_infer_gpu_paged_attention_workspace(ct.byref(d)) == BAD
    assert L.secure_infer_gpu_paged_attention(None, ct.byref(d)) == -1


def test_attention_refuses_a_short_workspace():
    L = _lib.load()
    assert L.secure_infer_gpu_paged_attention(None, None) == -1
    assert L.secure_infer_gpu_paged_attention_workspace(None) == BAD
    d = attention(q_starts=None, tokens=2)
    need = L.secure_infer_gpu_paged_attention_workspace(ct.byref(d))
    for ws, have in ((None, need), (P, need - 1), (P + 8, need)):
        if need:
            d.workspace, d.workspace_bytes = ws, have
            assert L.secure_infer_gpu_paged_attention(None, ct.byref(d)) == -1


def append(**kw):
    d = dict(k=P, v=P, k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128, cache_k=P,
             cache_v=P, slot_bytes=2 * 128 * 2 * 128, nslots=8, tables=P, table_stride=4, kv_lens=P, q_starts=P,
             table_pages=4, tokens=5, seqs=2, kv_heads=2, head_dim=128, page_tokens=128)
    d.update(kw)
    return _lib.SiPagedAppendDesc(**d)


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(cache_k=None), dict(cache_v=None), dict(tables=None), dict(kv_lens=None),
    dict(tokens=0), dict(tokens=1 << 31), dict(seqs=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=12),
    dict(nslots=0), dict(nslots=1 << 31), dict(table_pages=0), dict(q_starts=None), dict(page_tokens=100),
    dict(page_tokens=4), dict(slot_bytes=65520), dict(slot_bytes=65544), dict(k_token_stride=3), dict(v_head_stride=4),
    dict(k=P + 8), dict(cache_v=P + 8)])
def test_append_refuses(change):
    L = _lib.load()
    assert L.secure_infer_gpu_paged_append(None, None) == -1
    assert L.secure_infer_gpu_paged_append(None, ct.byref(append(**change))) == -1


def pages(**kw):
    d = dict(caches=(ct.c_void_p * 2)(P, P), ncaches=2, page_tokens=16, slot_bytes=512, page_bytes=512, nslots=8,
             tables=P, kv_lens=P, refs=P, tables_out=P, kv_lens_out=P, refs_out=P, rows=3, table_pages=4, list=P, n=1,
             workspace=P, workspace_bytes=1 << 20)
    d.update(kw)
    return _lib.SiPagesDesc(**d)


@pytest.mark.parametrize("change", [
    dict(tables=None), dict(refs=None), dict(tables_out=None), dict(refs_out=None), dict(workspace=None),
    dict(workspace=P + 4), dict(workspace_bytes=16), dict(nslots=0), dict(nslots=1 << 31), dict(rows=0),
    dict(rows=1 << 31), dict(table_pages=0), dict(page_tokens=0), dict(page_tokens=12), dict(table_pages=1 << 28),
    dict(n=1 << 29)])
def test_page_calls_refuse(change):
    L = _lib.load()
    for fn in (L.secure_infer_gpu_pages_fork, L.secure_infer_gpu_pages_free, L.secure_infer_gpu_pages_compact,
               L.secure_infer_gpu_pages_reserve):
        assert fn(None, None) == -1
        assert fn(None, ct.byref(pages(**change))) == -1


@pytest.mark.parametrize("change", [
    dict(caches=None), dict(caches=(ct.c_void_p * 2)(P, None)), dict(caches=(ct.c_void_p * 2)(P, P + 8)),
    dict(page_bytes=0), dict(page_bytes=500), dict(slot_bytes=496), dict(slot_bytes=520)])
def test_page_copies_refuse(change):
    L = _lib.load()
    for fn in (L.secure_infer_gpu_pages_fork, L.secure_infer_gpu_pages_free, L.secure_infer_gpu_pages_compact):
        assert fn(None, ct.byref(pages(**change))) == -1


@pytest.mark.parametrize("change", [dict(kv_lens=None), dict(kv_lens_out=None), dict(list=None)])
def test_page_calls_with_rows_refuse(change):
    L = _lib.load()
    for fn in (L.secure_infer_gpu_pages_fork, L.secure_infer_gpu_pages_free, L.secure_infer_gpu_pages_reserve):
        assert fn(None, ct.byref(pages(**change))) == -1


def test_python_refuses_host_tensors():
    c = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16)
    t, n = torch.zeros((1, 2), dtype=torch.int64), torch.ones(1, dtype=torch.int64)
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    refs = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        si.paged_attention(q, c, c, t, n)
    with pytest.raises(ValueError, match="device tensor"):
        si.paged_append(q, q, c, c, t, n)
    for call in (lambda: si.fork_pages([c], t, n, refs, torch.zeros((1, 2), dtype=torch.int64)),
                 lambda: si.free_pages([c], t, n, refs, n), lambda: si.compact_pages([c], t, refs),
                 lambda: si.reserve_pages(t, n, refs, n, 16)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    with pytest.raises(ValueError, match=r"\[n, 2\]"):
        si.fork_pages([c], t, n, refs, n)


@pytest.mark.gpu
def test_python_refuses_device_arguments():
    dev = "cuda"
    c = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=dev)
    t, n = torch.zeros((1, 2), dtype=torch.int64, device=dev), torch.ones(1, dtype=torch.int64, device=dev)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=dev)
    good = dict(q=q, cache_k=c, cache_v=c, tables=t, kv_lens=n)
    assert si.paged_attention(**good).shape == q.shape
    assert si.paged_attention(**{**good, "q": q[:0], "tables": t[:0], "kv_lens": n[:0]}).shape == (0, 4, 64)
    for change, what in (
            (dict(q=q.half()), "bfloat16"), (dict(q=q[:, :3]), "query heads"), (dict(q=q[..., :32]), "q must be"),
            (dict(q=torch.zeros((1, 4, 65), dtype=torch.bfloat16, device=dev)[..., 1:]), "multiples of 8|boundary"),
            (dict(q=q.cpu()), "q must be"), (dict(tables=t.int()), "tables"), (dict(kv_lens=n.int()), "kv_lens"),
            (dict(kv_lens=torch.cat([n, n])), "kv_lens"), (dict(q_starts=n), "q_starts"),
            (dict(tables=t.expand(3, 2), kv_lens=n.repeat(3)), "one row per sequence"), (dict(scale=float("inf")), "scale"),
            (dict(window=-1), "window"), (dict(out=q[:, :2]), "out"), (dict(cache_v=c.half()), "cache_v"),
            (dict(cache_v=c[:1]), "cache_k and cache_v"), (dict(cache_k=c.float(), cache_v=c.float()), "bfloat16"),
            (dict(cache_k=c[:, :12], cache_v=c[:, :12]), "contiguous|power"),
            (dict(lse=torch.zeros((1, 4), dtype=torch.float64, device=dev)), "lse"),
            (dict(tables=t[:, :0]), "no pages")):
        with pytest.raises(ValueError, match=what):
            si.paged_attention(**{**good, **change})
    with pytest.raises(ValueError, match="overlap"):
        two = dict(q=q.repeat(2, 1, 1), tables=t.repeat(2, 1), kv_lens=n.repeat(2))
        si.paged_attention(**{**good, **two}, out=q.expand(2, 4, 64))
    refs = torch.zeros(2, dtype=torch.int32, device=dev)
    for call, what in (
            (lambda: si.compact_pages([c], t, refs.long()), "refs"), (lambda: si.compact_pages([], t, refs), "no caches"),
            (lambda: si.compact_pages([c], t, refs[:1]), "one entry per slot"),
            (lambda: si.compact_pages([c, c[:, :8]], t, refs), "contiguous|one shape"),
            (lambda: si.free_pages([c], t, n, refs, n.int()), "row list"),
            (lambda: si.free_pages([c], t, n, refs, n, out=(t, n)), "3 tensors"),
            (lambda: si.free_pages([c], t, n, refs, n, fail_count=n), "fail_count"),
            (lambda: si.reserve_pages(t, n, refs, n, 12), "power of two"),
            (lambda: si.reserve_pages(t, n, refs, t, 16), "counts"),
            (lambda: si.fork_pages([c], t, n, refs, torch.zeros((1, 3), dtype=torch.int64, device=dev)), "pairs")):
        with pytest.raises(ValueError, match=what):
            call()
