"""Operators on the paged KV cache the transfers fill and drain.

* ``paged_append`` writes new tokens' K and V rows into their pages;
  ``paged_append_rotated`` rotates K by position on the way, and the tokens' queries.
* ``paged_attention`` attends from new tokens (one per sequence, or a chunk
  of each) over their sequences' pages.
* ``fork_pages`` / ``free_pages`` / ``compact_pages`` / ``reserve_pages`` manage
  the pages of every layer at once.

Caches are the transfers' paged caches: [slots, page tokens, kv heads, head
dim] of 16-bit values.  ``tables`` [sequences, pages] int64 holds the slot of each page (an entry
outside [0, slots) is no page) and ``kv_lens`` [sequences] int64 the
tokens in a sequence's pages, the new ones included.  ``q_starts`` [sequences +
1] int64 says which rows are a sequence's new tokens (None: row b is
sequence b's one new token).  What lives on the device is not read back: the
kernels stay inside the tensors whatever it holds, and count what they cannot
serve in ``fail_count`` (an int32 tensor they add to), as the reload calls
do.  There is no backward pass: attention and append refuse tensors that
require gradients where gradients are recorded.  Every call is asynchronous on the given (default: current) stream, and
may be captured into a graph.
"""
from __future__ import annotations

import ctypes as ct
import math
from array import array

import torch

from . import _lib
from .gcm import _check, lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_REFUSED = (1 << 64) - 1
_FLOAT_MAX = torch.finfo(torch.float32).max


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream_of(stream, device: int):
    """(raw handle, the torch stream if it is not the device's current one) of
    a call's stream: a torch stream, a raw handle, or None for the current."""
    if torch.cuda.current_device() != device:
        raise ValueError(f"the tensors are on cuda:{device}, which is not the current device")
    current = torch._C._cuda_getCurrentRawStream(device)
    if stream is None:
        return current, None
    if isinstance(stream, torch.cuda.Stream):
        raw = stream.cuda_stream
    else:
        raw = stream.value or 0 if isinstance(stream, ct.c_void_p) else int(stream)
        stream = None
    if raw == current:
        return raw, None
    return raw, torch.cuda.ExternalStream(raw, device=torch.device("cuda", device)) if stream is None else stream


def _kept_by(other, tensors) -> None:
    """Tensors used on a stream other than the one they were made on are not
    reused before that stream is done with them."""
    if other is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(other)


def _empty(other, shape, dtype, device: int):
    """A tensor that belongs to the call's stream."""
    where = torch.device("cuda", device)
    if other is None:
        return torch.empty(shape, dtype=dtype, device=where)
    with torch.cuda.stream(other):
        return torch.empty(shape, dtype=dtype, device=where)


def _index(t, name: str, ndim: int, device: int, dtype=torch.int64) -> None:
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        raise ValueError(f"{name} must be a tensor on cuda:{device}")
    if t.dtype != dtype or t.ndim != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {ndim}-d {dtype} tensor")


def _fail_count(t, device: int) -> None:
    if t is not None and (t.get_device() != device or t.dtype != torch.int32 or t.numel() != 1):
        raise ValueError(f"fail_count must be one int32 on cuda:{device}")


def _aligned(t, name: str) -> None:
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must start on a 16-byte boundary")


def _tracked() -> None:
    """A tensor requires gradients.  There is no backward pass: one is refused rather than lost."""
    if torch.is_grad_enabled():
        raise ValueError("no gradient passes through the paged cache: detach its tensors or use torch.no_grad()")


def _paged_cache(t, name: str):
    """(device, dtype, slots, page tokens, heads, dim, elements from one page to the next)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    dtype = t.dtype
    if t.ndim != 4 or dtype not in _DTYPES:
        raise ValueError(f"{name} must be [slots, page tokens, kv heads, head dim] in bfloat16 or float16")
    slots, ps, heads, dim = t.shape
    page = ps * heads * dim
    if slots * page == 0:
        raise ValueError(f"{name} is empty")
    stride = t.stride()
    step = stride[0] if slots > 1 else page  # the stride of a single page is never used
    if stride[1:] != (heads * dim, dim, 1) or step < page:
        raise ValueError(f"a page of {name} must be contiguous")
    if ps & (ps - 1) or not 8 <= ps <= 32768:
        raise ValueError(f"{name} has pages of {ps} tokens: must be a power of two from 8 to 32768")
    if dim % 8:
        raise ValueError(f"{name} has head dim {dim}: must be a multiple of 8")
    if step % 8:
        raise ValueError(f"{name}'s slot stride must be a multiple of 16 bytes")
    _aligned(t, name)
    return t.get_device(), dtype, slots, ps, heads, dim, step


def _cache_pair(cache_k, cache_v):
    geometry = _paged_cache(cache_k, "cache_k")
    if geometry != _paged_cache(cache_v, "cache_v"):
        raise ValueError("cache_k and cache_v must have one shape, dtype, slot stride and device")
    return geometry


def _rows(t, name: str, heads: int, dim: int, dtype, device: int) -> tuple[int, int, int]:
    """(tokens, token stride, head stride) of [tokens, heads, dim] rows."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor on cuda:{device}")
    if t.ndim != 3 or t.shape[1:] != (heads, dim):
        raise ValueError(f"{name} must be [tokens, {heads}, {dim}], got {tuple(t.shape)}")
    token, head, one = t.stride()
    tokens = t.shape[0]
    # the stride of a single token or head is never used
    if tokens <= 1:
        token = heads * dim
    if heads == 1:
        head = dim
    if (dim > 1 and one != 1) or token % 8 or head % 8:
        raise ValueError(f"{name} needs a contiguous head dim and token / head strides that are multiples of 8")
    _aligned(t, name)
    return tokens, token, head


def _sequences(tables, kv_lens, q_starts, tokens: int, ps: int, device: int):
    """(sequences, pages of a row, row stride) of the tables."""
    if not isinstance(tables, torch.Tensor) or tables.get_device() != device:
        raise ValueError(f"tables must be a tensor on cuda:{device}")
    if tables.dtype != torch.int64 or tables.ndim != 2:
        raise ValueError("tables must be a 2-d torch.int64 tensor with contiguous rows")
    seqs, pages = tables.shape
    row, one = tables.stride()
    if pages > 1 and one != 1:
        raise ValueError("tables must be a 2-d torch.int64 tensor with contiguous rows")
    _index(kv_lens, "kv_lens", 1, device)
    if kv_lens.shape[0] != seqs:
        raise ValueError("kv_lens needs one entry per row of tables")
    if q_starts is None:
        if tokens != seqs:
            raise ValueError("without q_starts there is one row per sequence")
    else:
        _index(q_starts, "q_starts", 1, device)
        if q_starts.shape[0] != seqs + 1:
            raise ValueError("q_starts needs one entry more than tables has rows")
    if pages * ps > 1 << 30:
        raise ValueError("a table row may span at most 2**30 tokens")
    return seqs, pages, row


def paged_append(k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                 tables: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor | None = None,
                 fail_count: torch.Tensor | None = None, stream=None) -> None:
    """New tokens' K and V rows ([tokens, kv heads, head dim], any token and
    head stride in multiples of 8) into their pages.  Token i of a sequence with n new
    ones goes to position kv_len - n + i; a token whose position is
    negative, past the table or on no page is dropped and counted."""
    d, device = _append_desc(k, v, cache_k, cache_v, tables, kv_lens, q_starts, fail_count)
    if d is None:
        return
    raw, other = _stream_of(stream, device)
    _check(lib().secure_infer_gpu_paged_append(raw, ct.byref(d)), "paged_append")
    _kept_by(other, (k, v, cache_k, cache_v, tables, kv_lens, q_starts, fail_count))


def _append_desc(k, v, cache_k, cache_v, tables, kv_lens, q_starts, fail_count):
    """(the checked descriptor, or None without tokens; the device)."""
    device, dtype, slots, ps, heads, dim, step = _cache_pair(cache_k, cache_v)
    tokens, kt, kh = _rows(k, "k", heads, dim, dtype, device)
    v_tokens, vt, vh = _rows(v, "v", heads, dim, dtype, device)
    if tokens != v_tokens:
        raise ValueError("k and v must have the same tokens")
    if k.requires_grad or v.requires_grad or cache_k.requires_grad or cache_v.requires_grad:
        _tracked()
    seqs, pages, row = _sequences(tables, kv_lens, q_starts, tokens, ps, device)
    _fail_count(fail_count, device)
    if tokens == 0:
        return None, device
    if seqs == 0:
        raise ValueError("there are new tokens but no sequences")
    if pages == 0:
        raise ValueError("tables has no pages")
    return _lib.SiPagedAppendDesc(
        k=k.data_ptr(), v=v.data_ptr(), k_token_stride=kt, k_head_stride=kh, v_token_stride=vt, v_head_stride=vh,
        cache_k=cache_k.data_ptr(), cache_v=cache_v.data_ptr(), slot_bytes=2 * step, nslots=slots,
        tables=tables.data_ptr(), table_stride=row, kv_lens=kv_lens.data_ptr(), q_starts=_ptr(q_starts),
        table_pages=pages, tokens=tokens, seqs=seqs, kv_heads=heads, head_dim=dim, page_tokens=ps,
        fail_count=_ptr(fail_count)), device


def paged_append_rotated(k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                         tables: torch.Tensor, kv_lens: torch.Tensor, freqs: torch.Tensor,
                         q: torch.Tensor | None = None, q_starts: torch.Tensor | None = None,
                         positions: torch.Tensor | None = None, adjacent: bool = False, magnitude: float = 1.0,
                         q_out: torch.Tensor | None = None, fail_count: torch.Tensor | None = None,
                         stream=None) -> torch.Tensor | None:
    """paged_append with K, and the same tokens' queries ``q`` [tokens, query heads, head
    dim], rotated by position on the way.  ``freqs`` [rot / 2] float32 are the angles a position;
    with a = p * freqs[i] the dims (x, y) = (i, i + rot / 2), or (2 i, 2 i + 1) if ``adjacent``, become
    ``magnitude`` * (x cos a - y sin a, y cos a + x sin a), in float from an angle that
    is right to float accuracy at any position (for frequencies up to 2**16), rounded once; dims from rot on go as they are.  rot is a multiple of 8 up to the head
    dim and 256.  p is the token's position in its sequence, or ``positions`` [tokens] int64
    (for the rotation alone).  A token that the append drops has its query rotated all the
    same; a row of q in no sequence goes as it is.  Returns ``q_out`` (new if it is not given; q itself, if it shares no memory
    with k and v, rotates in place), or None without q."""
    d, device = _append_desc(k, v, cache_k, cache_v, tables, kv_lens, q_starts, fail_count)
    heads, dim, dtype, tokens = cache_k.shape[2], cache_k.shape[3], cache_k.dtype, k.shape[0]
    _index(freqs, "freqs", 1, device, torch.float32)
    rot = 2 * freqs.shape[0]
    if rot == 0 or rot % 8 or rot > min(dim, 256):
        raise ValueError(f"freqs must hold a multiple of 4 frequencies, at most {min(dim, 256) // 2}")
    if freqs.requires_grad:
        _tracked()
    if not abs(magnitude) <= _FLOAT_MAX:
        raise ValueError("magnitude must be finite in float32")
    if positions is not None:
        _index(positions, "positions", 1, device)
        if positions.shape[0] != tokens:
            raise ValueError("positions needs one entry per token")
    r = _lib.SiRotation(freqs=freqs.data_ptr(), positions=_ptr(positions), rot=rot, adjacent=1 if adjacent else 0,
                        dtype=_DTYPES[dtype], magnitude=magnitude)
    other = None
    if d is not None:
        raw, other = _stream_of(stream, device)
    if q is None:
        if q_out is not None:
            raise ValueError("q_out goes with q")
    else:
        if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.shape[1] == 0:
            raise ValueError(f"q must be [tokens, query heads, {dim}]")
        q_heads = q.shape[1]
        q_tokens, qt, qh = _rows(q, "q", q_heads, dim, dtype, device)
        if q_tokens != tokens:
            raise ValueError("q and k must have the same tokens")
        if q.requires_grad or (q_out is not None and q_out.requires_grad):
            _tracked()
        if q_out is None:
            q_out = q.new_empty(q.shape) if other is None else _empty(other, q.shape, dtype, device)
            ot, oh = q_heads * dim, dim
        else:
            if not isinstance(q_out, torch.Tensor) or q_out.shape != q.shape:
                raise ValueError("q_out must have q's shape")
            _, ot, oh = _rows(q_out, "q_out", q_heads, dim, dtype, device)
            _apart(ot, oh, tokens, q_heads, dim, "q_out")
            if d is not None:
                to, own = (q_out.data_ptr(), ot, oh, q_heads), (q.data_ptr(), qt, qh, q_heads)
                if to != own and _meet(to, own, tokens, dim):
                    raise ValueError("q_out must be q itself, or not overlap q")
                # (q too, where it turns in place: other waves may not have read K and V yet)
                for name, rows in (("k", (d.k, d.k_token_stride, d.k_head_stride, heads)),
                                   ("v", (d.v, d.v_token_stride, d.v_head_stride, heads))):
                    if _meet(to, rows, tokens, dim):
                        raise ValueError(f"q_out must not overlap {name}")
        r.q, r.q_out, r.q_heads = q.data_ptr(), q_out.data_ptr(), q_heads
        r.q_token_stride, r.q_head_stride, r.q_out_token_stride, r.q_out_head_stride = qt, qh, ot, oh
    if d is None:
        return q_out
    _check(lib().secure_infer_gpu_paged_append_rotated(raw, ct.byref(d), ct.byref(r)), "paged_append_rotated")
    _kept_by(other, (k, v, cache_k, cache_v, tables, kv_lens, freqs, q, q_starts, positions, q_out, fail_count))
    return q_out


def _apart(token: int, head: int, tokens: int, heads: int, dim: int, name: str) -> None:
    """The rows of an output do not overlap: the larger stride steps over the smaller
    one's rows; that of a single token or head is never used."""
    span = dim
    for stride, n in sorted((stride, n) for stride, n in ((token, tokens), (head, heads)) if n > 1):
        if stride < span:
            raise ValueError(f"{name}'s rows must not overlap")
        span += stride * (n - 1)


def _meet(a, b, tokens: int, dim: int) -> bool:
    """Whether 16-bit rows of the same tokens, (address, token stride, head stride, heads) each,
    have an element in common: exactly where the token strides are one, as in a fused buffer;
    otherwise whether the memory from the first element to the last does."""
    (at, step, a_head, a_heads), (other, b_step, b_head, b_heads) = a, b
    gap, last = (other - at) // 2, tokens - 1
    a_span, b_span = (a_heads - 1) * a_head + dim, (b_heads - 1) * b_head + dim
    if gap >= last * step + a_span or -gap >= last * b_step + b_span:
        return False
    if last and (step != b_step or step == 0):
        return True
    # a token's rows beside the other's, or a head's
    if last and a_span <= gap % step <= step - b_span:
        return False
    if a_head == b_head and a_head:
        head_span = dim if step % a_head == 0 else last * step + dim
        if head_span <= gap % a_head <= a_head - head_span:
            return False
    for x in {gap + j * b_head - i * a_head for i in range(a_heads) for j in range(b_heads)}:
        # some b token less an a token, from -last to last, brings the heads' rows within dim
        if abs(x) < dim or last and max((1 - dim - x + step - 1) // step, -last) <= min((dim - 1 - x) // step, last):
            return True
    return False


def paged_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, tables: torch.Tensor,
                    kv_lens: torch.Tensor, q_starts: torch.Tensor | None = None, scale: float | None = None,
                    causal: bool = True, window: int = 0, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                    stream=None, sinks: int = 0, prefix_groups: torch.Tensor | None = None,
                    prefix_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [tokens, query heads, head dim] over the pages:
    softmax(scale q k^T) v per token and query head (head h reads KV head
    h // (query heads / kv heads)).  Token i of a sequence with n new ones stands at p = kv_len
    - n + i; it sees the keys on held pages below kv_len, up to p
    (``causal``) and after p - window (``window`` > 0).  Where kv_len outgrows the table
    the tokens keep the positions that paged_append gives them (one over 3 * 2**29
    ends at the table instead).  Without a key to see its output is 0.  Scores
    and sums are float; the weights are rounded to q's type once, for the product with v.  ``scale`` defaults to head_dim ** -0.5.  ``lse`` [tokens, query heads]
    float32, if given, receives the log-sum-exp of the scaled scores (-inf
    without a key), with which two parts' outputs can be joined.  ``workspace`` (uint8, at least
    ``paged_attention_workspace`` bytes) saves an allocation per call.  Returns ``out``.

    ``sinks``: a token also sees the first ``sinks`` keys that its window alone would hide.

    ``prefix_groups`` [groups + 1] int64, ascending, and ``prefix_lens`` [groups] int64:
    sequences prefix_groups[g] up to prefix_groups[g + 1] share their first prefix_lens[g] keys: as far as their lengths go their
    rows hold the same K and V there, on the same pages, as fork_pages leaves them, or on copies, and the call may read them
    from any row that is long enough: once for all their tokens, where the prefix has at least 16 keys for each row (new
    token and query head of a KV head) that a sequence of the group has on average.  Beside a window each row may have given
    up pages (an entry that is no slot) that none of its own new tokens, nor any later one, sees.  What a token sees, and the
    result but for rounding, does not change; a group of one sequence, or a sequence in none, is as without groups.  A few
    sequences behind a short prefix are faster without groups, and the workspace of a call with groups holds float
    numerators of all its tokens at least twice: name them for next tokens and short chunks."""
    d, device = _attention_desc(q, cache_k, cache_v, tables, kv_lens, q_starts, scale, causal, window, out, lse)
    more = None
    if sinks or prefix_groups is not None or prefix_lens is not None:
        more = _attention_more(sinks, prefix_groups, prefix_lens, device)
    if q.requires_grad or cache_k.requires_grad or cache_v.requires_grad:
        _tracked()
    if d is None:
        return torch.empty_like(q) if out is None else out
    raw, other = _stream_of(stream, device)
    if out is None:
        out = q.new_empty(q.shape) if other is None else _empty(other, q.shape, q.dtype, device)
        d.out, d.out_token_stride, d.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
    L = lib()
    need = (L.secure_infer_gpu_paged_attention_workspace(ct.byref(d)) if more is None else
            L.secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(more)))
    if need == _REFUSED:
        raise ValueError("paged_attention refuses these arguments")
    if need:
        if workspace is None:
            workspace = _empty(other, (need,), torch.uint8, device)
        elif workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous on cuda:{device}")
        elif workspace.numel() * workspace.element_size() < need:
            raise ValueError(f"workspace needs {need} bytes")
        _aligned(workspace, "workspace")
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if more is None:
        _check(L.secure_infer_gpu_paged_attention(raw, ct.byref(d)), "paged_attention")
    else:
        _check(L.secure_infer_gpu_paged_attention_more(raw, ct.byref(d), ct.byref(more)), "paged_attention")
    _kept_by(other, (q, cache_k, cache_v, tables, kv_lens, q_starts, out, lse, workspace, prefix_groups, prefix_lens))
    return out


def paged_attention_workspace(q, cache_k, cache_v, tables, kv_lens, q_starts=None, causal: bool = True,
                              window: int = 0, sinks: int = 0, prefix_groups: torch.Tensor | None = None,
                              prefix_lens: torch.Tensor | None = None) -> int:
    """Workspace bytes of a paged_attention call with these arguments."""
    d, device = _attention_desc(q, cache_k, cache_v, tables, kv_lens, q_starts, None, causal, window, None, None)
    more = _attention_more(sinks, prefix_groups, prefix_lens, device)
    return 0 if d is None else int(lib().secure_infer_gpu_paged_attention_more_workspace(ct.byref(d), ct.byref(more)))


def _attention_more(sinks, prefix_groups, prefix_lens, device: int):
    """The checked sinks and shared prefixes."""
    if not 0 <= int(sinks) <= 1 << 30:
        raise ValueError("sinks must be 0 (none) or a number of keys up to 2**30")
    if (prefix_groups is None) != (prefix_lens is None):
        raise ValueError("prefix_groups and prefix_lens go together")
    groups = 0
    if prefix_groups is not None:
        _index(prefix_groups, "prefix_groups", 1, device)
        _index(prefix_lens, "prefix_lens", 1, device)
        groups = prefix_lens.shape[0]
        if prefix_groups.shape[0] != groups + 1:
            raise ValueError("prefix_groups needs one entry more than prefix_lens")
        if groups >= 1 << 26:
            raise ValueError("there are too many groups")
    return _lib.SiPagedAttentionMore(sinks=int(sinks), groups=groups, group_starts=_ptr(prefix_groups) if groups else None,
                                     prefix_lens=_ptr(prefix_lens) if groups else None)


def _attention_desc(q, cache_k, cache_v, tables, kv_lens, q_starts, scale, causal, window, out, lse):
    """(the checked descriptor, without an output if ``out`` is None; the
    device), or (None, the device) where there is nothing to compute."""
    device, dtype, slots, ps, heads, dim, step = _cache_pair(cache_k, cache_v)
    if dim > 256:
        raise ValueError(f"head dim {dim} is over 256")
    if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.shape[1] == 0 or q.shape[1] % heads:
        raise ValueError(f"q must be [tokens, query heads, {dim}] with a multiple of {heads} query heads")
    q_heads = q.shape[1]
    tokens, qt, qh = _rows(q, "q", q_heads, dim, dtype, device)
    if tokens * q_heads >= 1 << 26:
        raise ValueError("q has too many rows")
    seqs, pages, row = _sequences(tables, kv_lens, q_starts, tokens, ps, device)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not 0 <= int(window) < 1 << 31:
        raise ValueError("window must be 0 (none) or a positive number of keys")
    ot = oh = 0
    if out is not None:
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        _, ot, oh = _rows(out, "out", q_heads, dim, dtype, device)
        _apart(ot, oh, tokens, q_heads, dim, "out")
    if lse is not None and (lse.get_device() != device or lse.dtype != torch.float32 or lse.shape != q.shape[:2]
                            or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous float32 [tokens, query heads] tensor on cuda:{device}")
    if tokens == 0:
        return None, device
    if seqs == 0 or pages == 0:
        raise ValueError("tables has no pages")
    return _lib.SiPagedAttentionDesc(
        q=q.data_ptr(), q_token_stride=qt, q_head_stride=qh, out=q.data_ptr() if out is None else out.data_ptr(),
        out_token_stride=ot, out_head_stride=oh, lse=_ptr(lse), cache_k=cache_k.data_ptr(),
        cache_v=cache_v.data_ptr(), slot_bytes=2 * step, nslots=slots, tables=tables.data_ptr(), table_stride=row,
        kv_lens=kv_lens.data_ptr(), q_starts=_ptr(q_starts), table_pages=pages, tokens=tokens, seqs=seqs,
        q_heads=q_heads, kv_heads=heads, head_dim=dim, page_tokens=ps, dtype=_DTYPES[dtype],
        causal=1 if causal else 0, window=int(window), scale=scale), device


# ------------------------------------------------------------------ pages

class CacheSet:
    """Caches of one shape, dtype, slot stride and device (every layer's K and V),
    checked once: the page calls take it in the place of a list, which they
    check on every call (160 tensors: 43 us).  It holds the tensors; they must keep the
    memory they had, as in a captured graph."""

    def __init__(self, caches):
        self.caches = list(caches)
        self.geometry, addresses = _same_layout(self.caches)
        self.addresses = (ct.c_void_p * len(addresses))(*addresses)


def _same_layout(caches):
    """(device, dtype, slots, page tokens, heads, dim, slot stride) of caches
    that share it, and their addresses (the library checks their alignment).
    A property of all of them at a time: a check of each tensor in Python costs
    1 us a tensor, which for 160 tensors is many times the copies."""
    if not caches:
        raise ValueError("no caches given")
    geometry = _paged_cache(caches[0], "a cache")
    T = torch.Tensor
    if len(caches) > 1:
        try:
            same = (len(set(map(T.size, caches))) == 1 and len(set(map(T.get_device, caches))) == 1
                    and len({c.dtype for c in caches}) == 1)
            dense = same and all(map(T.is_contiguous, caches))
        except (TypeError, AttributeError) as e:
            raise ValueError("a cache must be a device tensor") from e
        if not same or (not dense and any([_paged_cache(c, "a cache") != geometry for c in caches])):
            raise ValueError("the caches must have one shape, dtype, slot stride and device")
    addresses = list(map(T.data_ptr, caches))
    if len(set(addresses)) != len(addresses):
        raise ValueError("a cache is given twice")
    return geometry, addresses


def _pages_call(fn_name, caches, tables, kv_lens, refs, page_tokens, rows_list, list_ndim, scrub, fail_count, out,
                stream):
    if not isinstance(refs, torch.Tensor) or not refs.is_cuda:
        raise ValueError("refs must be a device tensor")
    device = refs.get_device()
    _index(refs, "refs", 1, device, torch.int32)
    nslots = refs.shape[0]
    addresses, slot_bytes, page_bytes = None, 0, 0
    if caches is not None:
        if isinstance(caches, CacheSet):
            geometry, addresses, caches = caches.geometry, caches.addresses, caches.caches
        else:
            caches = list(caches)
            geometry, found = _same_layout(caches)
            keep = array("Q", found)
            addresses = (ct.c_void_p * len(found)).from_buffer(keep)
        where, _, slots, page_tokens, heads, dim, step = geometry
        if where != device:
            raise ValueError("the caches must be on refs' device")
        if slots != nslots:
            raise ValueError("refs needs one entry per slot")
        slot_bytes, page_bytes = 2 * step, 2 * page_tokens * heads * dim
    _index(tables, "tables", 2, device)
    rows, pages = tables.shape
    if kv_lens is not None:
        _index(kv_lens, "kv_lens", 1, device)
        if kv_lens.shape[0] != rows:
            raise ValueError("kv_lens needs one entry per row of tables")
    if page_tokens < 1 or page_tokens & (page_tokens - 1):
        raise ValueError("page_tokens must be a power of two")
    if pages * page_tokens > 1 << 30:
        raise ValueError("a table row may span at most 2**30 tokens")
    if rows_list is not None:
        _index(rows_list, "the row list", list_ndim, device)
    _fail_count(fail_count, device)
    if rows * pages * nslots == 0:
        raise ValueError("tables and refs must not be empty")
    state = (tables, refs) if kv_lens is None else (tables, kv_lens, refs)
    raw, other = _stream_of(stream, device)
    if out is None:
        out = tuple([_empty(other, t.shape, t.dtype, device) for t in state])
    else:
        if len(out) != len(state):
            raise ValueError(f"out needs {len(state)} tensors")
        for o, i in zip(out, state):
            if o.shape != i.shape or o.dtype != i.dtype or o.get_device() != device or not o.is_contiguous():
                raise ValueError("out must match the inputs in shape, dtype and device, and be contiguous")
    d = _lib.SiPagesDesc(
        caches=addresses, ncaches=0 if addresses is None else len(addresses), page_tokens=page_tokens,
        slot_bytes=slot_bytes, page_bytes=page_bytes, nslots=nslots, tables=tables.data_ptr(), kv_lens=_ptr(kv_lens),
        refs=refs.data_ptr(), tables_out=out[0].data_ptr(), kv_lens_out=None if kv_lens is None else out[1].data_ptr(),
        refs_out=out[-1].data_ptr(), rows=rows, table_pages=pages, list=_ptr(rows_list),
        n=0 if rows_list is None else rows_list.shape[0], scrub=1 if scrub else 0, fail_count=_ptr(fail_count))
    L = lib()
    workspace = _empty(other, (L.secure_infer_gpu_pages_workspace(ct.byref(d)),), torch.uint8, device)
    d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _check(getattr(L, fn_name)(raw, ct.byref(d)), fn_name.removeprefix("secure_infer_gpu_"))
    if other is not None:
        _kept_by(other, (*(caches or ()), *state, rows_list, fail_count, *out))
    return tuple(out)


def fork_pages(caches, tables: torch.Tensor, kv_lens: torch.Tensor, refs: torch.Tensor, pairs: torch.Tensor,
               fail_count: torch.Tensor | None = None, out=None, stream=None):
    """Each pair (parent row, child row) of ``pairs`` [n, 2] int64 makes the child
    the parent's copy: whole pages are shared (refs + 1), a partly filled last page is
    copied in every tensor of ``caches`` (a list, or a CacheSet of it) into the lowest
    free slots, in the list's order.  A child must be an empty row named once; a pair that cannot be served (a
    row out of range, no free slot) leaves its child as it was and is counted.
    Returns (tables, kv_lens, refs), new or written to ``out`` (which may be the
    inputs).  ``refs`` [slots] int32 counts the rows that hold a slot."""
    if not isinstance(pairs, torch.Tensor) or pairs.ndim != 2 or pairs.shape[1] != 2:
        raise ValueError("pairs must be [n, 2]")
    return _pages_call("secure_infer_gpu_pages_fork", caches, tables, kv_lens, refs, 0, pairs, 2,
                       False, fail_count, out, stream)


def free_pages(caches, tables: torch.Tensor, kv_lens: torch.Tensor, refs: torch.Tensor, rows: torch.Tensor,
               scrub: bool = True, fail_count: torch.Tensor | None = None, out=None, stream=None):
    """The rows named in ``rows`` [n] int64 give up their pages (refs - 1) and become
    empty; with ``scrub`` a page nobody holds any more is zeroed in every tensor
    of ``caches``, so a freed slot keeps no plaintext.  Returns (tables, kv_lens,
    refs) as fork_pages does."""
    return _pages_call("secure_infer_gpu_pages_free", caches, tables, kv_lens, refs, 0, rows, 1,
                       scrub, fail_count, out, stream)


def compact_pages(caches, tables: torch.Tensor, refs: torch.Tensor, scrub: bool = False, out=None, stream=None):
    """With L slots held, the held slots >= L move to the free slots < L (both
    ascending) in every tensor of ``caches``.  The pages moved from keep their contents,
    plaintext in slots that are free, unless ``scrub`` zeroes them.  Returns (tables, refs), new or written to ``out``."""
    return _pages_call("secure_infer_gpu_pages_compact", caches, tables, None, refs, 0, None, 0,
                       scrub, None, out, stream)


def reserve_pages(tables: torch.Tensor, kv_lens: torch.Tensor, refs: torch.Tensor, counts: torch.Tensor,
                  page_tokens: int, fail_count: torch.Tensor | None = None, out=None, stream=None):
    """Row b grows by counts[b] tokens (negative: by none) and takes the pages it
    then lacks from the free slots, the lowest first, rows in order.  A row
    that outgrows its table, or that needs more slots than the rows before it
    that fit theirs leave (served or not), takes none and is counted; its new length stands, so its tokens without a page are
    dropped by paged_append and unseen by paged_attention.  Returns (tables,
    kv_lens, refs) as fork_pages does."""
    if not isinstance(counts, torch.Tensor) or not isinstance(tables, torch.Tensor) \
            or counts.shape != tables.shape[:1]:
        raise ValueError("counts needs one entry per row of tables")
    return _pages_call("secure_infer_gpu_pages_reserve", None, tables, kv_lens, refs, int(page_tokens), counts, 1,
                       False, fail_count, out, stream)
