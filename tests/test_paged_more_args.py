"""What attention with sinks and shared prefixes and the rotated append refuse,
without a GPU: the C calls return -1 before anything is queued (the pointers are
never followed)."""
import ctypes as ct

import pytest
import torch

import secure_infer_amd as si
from secure_infer_amd import _lib
from tests.test_paged_args import BAD, P, append, attention


def more(**kw):
    d = dict(sinks=4, groups=2, group_starts=P, prefix_lens=P)
    d.update(kw)
    return _lib.SiPagedAttentionMore(**d)


def rotation(**kw):
    d = dict(freqs=P, positions=None, q=P, q_out=P, q_token_stride=1024, q_head_stride=128, q_out_token_stride=1024,
             q_out_head_stride=128, q_heads=8, rot=128, adjacent=0, dtype=0, magnitude=1.0)
    d.update(kw)
    return _lib.SiRotation(**d)


@pytest.mark.parametrize("change", [dict(sinks=(1 << 30) + 1), dict(groups=1 << 26), dict(group_starts=None),
                                    dict(prefix_lens=None)])
def test_attention_refuses(change):
    L = _lib.load()
    d = attention(window=5)
    assert L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(more())) != BAD
    m = more(**change)
    assert L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(m)) == BAD
    assert L.secure_infer_gpu_paged_attention_more(None, ct.byref(d), ct.byref(m)) == -1


def test_attention_refuses_what_the_plain_call_refuses():
    L = _lib.load()
    assert L.secure_infer_gpu_paged_attention_more(None, None, ct.byref(more())) == -1
    for change in (dict(q=None), dict(head_dim=264), dict(scale=float("nan")), dict(tokens=0)):
        d = attention(**change)
        assert L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(more())) == BAD
        assert L.secure_infer_gpu_paged_attention_more(None, ct.byref(d), ct.byref(more())) == -1


def test_attention_without_more_is_the_plain_call():
    L = _lib.load()
    d = attention(tokens=300)
    need = L.secure_infer_gpu_paged_attention_workspace(ct.byref(d))
    for m in (None, ct.byref(more(sinks=0, groups=0)), ct.byref(more(sinks=9, groups=0, group_starts=None))):
        assert L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), m) == need


def test_attention_refuses_a_short_workspace():
    L = _lib.load()
    d = attention()
    m = more()
    need = L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(m))
    assert need > 0
    for ws, have in ((None, need), (P, need - 1), (P + 8, need)):
        d.workspace, d.workspace_bytes = ws, have
        assert L.secure_infer_gpu_paged_attention_more(None, ct.byref(d), ct.byref(m)) == -1


@pytest.mark.parametrize("change", [
    dict(freqs=None), dict(rot=0), dict(rot=12), dict(rot=136), dict(dtype=2), dict(magnitude=float("nan")),
    dict(magnitude=float("inf")), dict(q=None), dict(q_out=None), dict(q=P + 8), dict(q_out=P + 2),
    dict(q_token_stride=3), dict(q_head_stride=4), dict(q_out_token_stride=5), dict(q_out_head_stride=12),
    dict(q_heads=1 << 24)])
def test_rotation_refuses(change):
    L = _lib.load()
    assert L.secure_infer_gpu_paged_append_rotated(None, ct.byref(append()), ct.byref(rotation(**change))) == -1


@pytest.mark.parametrize("change", [dict(k=None), dict(tokens=0), dict(head_dim=12), dict(v_head_stride=4),
                                    dict(page_tokens=100), dict(nslots=0), dict(q_starts=None)])
def test_rotation_refuses_what_the_append_refuses(change):
    L = _lib.load()
    assert L.secure_infer_gpu_paged_append_rotated(None, ct.byref(append(**change)), ct.byref(rotation())) == -1


def test_rotation_refuses_rot_over_256():
    L = _lib.load()
    d = append(head_dim=512, k_token_stride=1024, k_head_stride=512, slot_bytes=2 * 128 * 2 * 512)
    assert L.secure_infer_gpu_paged_append_rotated(None, ct.byref(d), ct.byref(rotation(rot=264))) == -1
    assert L.secure_infer_gpu_paged_append_rotated(None, ct.byref(d), None) == -1
    assert L.secure_infer_gpu_paged_append_rotated(None, None, ct.byref(rotation())) == -1


def test_python_refuses_host_tensors():
    c = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16)
    t, n = torch.zeros((1, 2), dtype=torch.int64), torch.ones(1, dtype=torch.int64)
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        si.paged_attention(q, c, c, t, n, window=4, sinks=1)
    with pytest.raises(ValueError, match="device tensor"):
        si.paged_append_rotated(q, q, c, c, t, n, torch.zeros(8), q=q)
