"""paged_attention and paged_append at the ends of what a call may be given: the
longest tables, rows past 32-bit offsets, lengths past the table, NaN among the
keys that are seen, outputs of any layout, keys joined from many parts.

`definition` computes chosen rows in 64 bits on the CPU, a token standing at
p = kv_len - n + i whatever its table holds.

Bound on an output element: with u the unit roundoff of the 16-bit type, A = sum_j
w_j |v_j| over the n keys seen, ds the rounding of a score ((dim + 4) 2^-24 scale sum_d
|q_d k_d|: it moves a weight and the weights' sum by a factor exp(ds) each), one
rounding of the weights to 16 bits, one of the output, and the float sums of the weights and of the
values over n keys and at most 64 parts, (n + 64) 2^-24 each in any order,
  |error| <= u |o| + (u + 4 ds + (n + 64) 2^-23) A + n 2^-25 max|v|,
the last term for fp16 weights below its normal range.  The log-sum-exp moves
by at most ds + (n + 64) 2^-24 + 2^-22 |lse|."""
import math

import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_attention import DEV, ROUND, attend, make, rand

pytestmark = pytest.mark.gpu


def definition(x, rows=None, scale=None, causal=True, window=0):
    """{row: (out, lse, bound of out, bound of lse)} of the rows of q, [heads, dim] and
    [heads] in float64."""
    q, ck, cv, tables = x["q"], x["ck"], x["cv"], x["tables"]
    hq, dim = q.shape[1:]
    slots, ps, hkv, _ = ck.shape
    scale = dim ** -0.5 if scale is None else scale
    u = ROUND[q.dtype]
    starts = x["starts"].tolist()
    found = {}
    for b in range(tables.shape[0]):
        length = int(x["kv"][b])
        for t in range(starts[b], starts[b + 1]):
            if rows is not None and t not in rows:
                continue
            p = length - starts[b + 1] + t
            pos = torch.arange(max(0, min(length, tables.shape[1] * ps)))
            if causal:
                pos = pos[pos <= p]
            if window:
                pos = pos[pos > p - window]
            slot = tables[b][pos // ps]
            keep = (slot >= 0) & (slot < slots)
            pos, slot = pos[keep], slot[keep]
            n = pos.numel()
            if n == 0:
                none = torch.zeros((hq, dim), dtype=torch.float64)
                found[t] = none, torch.full((hq,), -math.inf, dtype=torch.float64), none, none[:, 0]
                continue
            k, v = (c[slot, pos % ps].double().repeat_interleave(hq // hkv, 1) for c in (ck, cv))
            qq = q[t].double()
            s = (k * qq).sum(2) * scale                                         # [keys, heads]
            ds = (k * qq).abs().sum(2).amax(0) * abs(scale) * (dim + 4) * 2.0 ** -24  # [heads]
            lse = torch.logsumexp(s, 0)
            lse[torch.isnan(s).any(0)] = math.nan
            w = torch.exp(s - lse)[:, :, None]
            out, a = (w * v).sum(0), (w * v.abs()).sum(0)
            tol = u * out.abs() + (u + 4 * ds[:, None] + (n + 64) * 2.0 ** -23) * a
            if q.dtype == torch.float16:
                tol += n * 2.0 ** -25 * v.abs().amax(0)
            found[t] = out, lse, tol, ds + (n + 64) * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    return found


def agree(out, lse, found):
    """Outputs within their bounds, NaN where the definition has NaN."""
    for t, (want, want_lse, tol, lse_tol) in found.items():
        for got, w, bound in ((out[t].cpu().double(), want, tol), (lse[t].cpu().double(), want_lse, lse_tol)):
            assert torch.equal(torch.isnan(got), torch.isnan(w)), f"row {t}: NaN"
            near = ((got - w).abs() <= bound) | (got == w) | torch.isnan(w)
            assert near.all(), f"row {t}: off by {float((got - w).abs().nan_to_num(0).max())}"


def check(x, use_starts=True, rows=None, **kw):
    out, lse = attend(x, use_starts, lse=True, **kw)
    agree(out, lse, definition(x, rows, **kw))


def wide(x, pages):
    """The batch with table rows of `pages` entries, no page past the ones it had."""
    t = torch.full((x["tables"].shape[0], pages), -1, dtype=torch.int64)
    t[:, :x["tables"].shape[1]] = x["tables"]
    return {**x, "tables": t}


def test_a_long_chunk_under_the_longest_table():
    """Row tiles times the table's 2^30 positions pass 2^31 keys a part."""
    x = wide(make(11, [13_100], [13_000], 16, 1, 8, 32768, torch.bfloat16, spare=0), 32768)
    check(x, rows={0, 1, 6_500, 12_930, 12_999})


def test_many_sequences_under_the_longest_table():
    """2,048 sequences x 8 KV heads x 2^30 positions: every sequence has its outputs."""
    x = make(12, [900], [1], 8, 8, 8, 32768, torch.bfloat16, spare=0)
    g = torch.Generator().manual_seed(1)
    seqs = 2048
    x = dict(x, q=rand(g, seqs, 8, 8, dtype=torch.bfloat16), kv=torch.randint(0, 900, (seqs,), generator=g),
             starts=torch.arange(seqs + 1))
    x["kv"][-1] = 900
    pages = 32768
    row = wide(x, pages)["tables"].to(DEV)
    d = {k: v.to(DEV) for k, v in x.items()}
    lse = torch.full((seqs, 8), 7.0, device=DEV)
    for starts in (None, d["starts"]):
        out = si.paged_attention(d["q"], d["ck"], d["cv"], row.expand(seqs, pages), d["kv"], q_starts=starts, lse=lse)
        agree(out, lse, definition({**x, "tables": x["tables"].expand(seqs, -1)}, {0, 1, 63, 64, 65, 1000, 2046, 2047}))


@pytest.mark.parametrize("new,past", [(1, 1), (1, 40), (8, 4), (8, 8), (8, 9), (40, 3), (40, 39), (40, 200), (200, 130)])
@pytest.mark.parametrize("window,causal", [(0, True), (7, True), (100, True), (7, False), (0, False)])
def test_tokens_of_a_length_past_the_table_keep_their_places(new, past, window, causal):
    """Lengths that outgrow a table of 512 positions by `past`: a token with a place in
    the table stands there, one without sees what its position lets it see."""
    kv = [512, 512, 300]
    x = make(13, kv, [new, 2, new], 4, 2, 64, 64, torch.bfloat16, width=8)
    x["kv"] = torch.tensor([512 + past, 512 + past, 300])
    check(x, window=window, causal=causal)


def test_a_row_that_outgrows_its_table_from_reserve_to_attention():
    """60 of 64 positions are held and 8 tokens come: the first 4 are stored at 60 to 63,
    see themselves and what is before them, and the other 4 are dropped."""
    ps, width, hkv, dim = 16, 4, 2, 64
    x = make(14, [60], [8], 4, hkv, dim, ps, torch.bfloat16, width=width)
    d = {k: v.to(DEV) for k, v in x.items()}
    refs = torch.zeros(x["ck"].shape[0], dtype=torch.int32)
    refs[x["tables"][0]] = 1
    fail = torch.zeros(1, dtype=torch.int32, device=DEV)
    tables, kv, _ = si.reserve_pages(d["tables"], d["kv"], refs.to(DEV), torch.tensor([8], device=DEV), ps, fail)
    assert int(fail) == 1 and kv.tolist() == [68]
    k, v = torch.randn((2, 8, hkv, dim), device=DEV).to(torch.bfloat16)
    si.paged_append(k, v, d["ck"], d["cv"], tables, kv, q_starts=d["starts"], fail_count=fail)
    assert int(fail) == 5
    assert torch.equal(d["ck"][tables[0, 3], 12:], k[:4]) and torch.equal(d["cv"][tables[0, 3], 12:], v[:4])
    got = attend({**x, "ck": d["ck"].cpu(), "cv": d["cv"].cpu(), "kv": kv.cpu()}, lse=True)
    agree(*got, definition({**x, "ck": d["ck"].cpu(), "cv": d["cv"].cpu(), "kv": kv.cpu()}))


@pytest.mark.parametrize("new", [1, 3, 40])
def test_lengths_at_the_last_position(new):
    """Lengths up to 3 * 2^29 count as they are; a longer one ends at the table."""
    last = 3 << 29
    x = make(15, [256, 256], [new, 1], 4, 2, 64, 64, torch.bfloat16, width=4)
    for length, counts_as in ((last, last), (last + 1, 256), (1 << 40, 256)):
        for window in (0, last - 100, last - 300, (1 << 31) - 1):
            x["kv"] = torch.tensor([length, 256])
            got = attend(x, lse=True, window=window)
            agree(*got, definition({**x, "kv": torch.tensor([counts_as, 256])}, window=window))


@pytest.mark.parametrize("kv,new,bad_k,bad_v", [
    # keys whose K / V are NaN; every key of the first rows' first steps among them
    (3, 3, [0], [0]), (20, 3, range(18), [17, 18]), (200, 5, range(64), [196]), (5000, 3, range(4000, 4500), [4998]),
    (70, 70, [0], [0]), (200, 130, range(70), [70, 71]), (300, 40, range(128), [270]),
    (5000, 70, range(4610, 4900), [4935]), (9000, 30, range(8000, 8990), [8990])])
def test_what_a_token_sees_of_nan_is_nan(kv, new, bad_k, bad_v):
    """Alone and in whole steps, with NaN or a sound V beside it, in one part of many."""
    x = make(16, [kv], [new], 4, 2, 64, 64, torch.bfloat16)
    for bad, cache in ((bad_k, x["ck"]), (bad_v, x["cv"])):
        p = torch.tensor(list(bad))
        cache[x["tables"][0, p // 64], p % 64] = math.nan
    check(x)
    check(x, window=66)


@pytest.mark.parametrize("kv,new", [(20, 3), (200, 130), (4000, 4), (4000, 70)])
def test_a_nan_query_has_nan_outputs_beside_nan_values(kv, new):
    x = make(17, [kv], [new], 4, 2, 64, 64, torch.float16)
    x["q"][new - 2, 1] = math.nan
    x["cv"][x["tables"][0, (kv - 1) // 64], (kv - 1) % 64] = math.nan
    check(x)


@pytest.mark.parametrize("shape,strides", [
    ((4, 1, 64), (64, 64, 1)), ((4, 1, 64), (64, 8, 1)), ((4, 1, 64), (128, 64, 1)), ((1, 8, 64), (512, 128, 1)),
    ((1, 8, 64), (8, 72, 1)), ((1, 1, 64), (8, 8, 1)), ((4, 8, 64), (64, 256, 1)), ((4, 8, 64), (640, 72, 1)),
    ((4, 8, 64), (568, 72, 1))])
def test_outputs_of_any_layout_without_overlaps(shape, strides):
    """The stride of a single token or head is never used, so it overlaps nothing."""
    tokens, heads, dim = shape
    x = make(18, [50 + i for i in range(tokens)], [1] * tokens, heads, 1, dim, 16, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    base = torch.full((8192,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = base.as_strided(shape, strides)
    assert si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], out=out) is out
    assert torch.equal(out, attend(x, use_starts=False))
    kept = torch.ones_like(base, dtype=torch.bool)
    kept.as_strided(shape, strides)[:] = False
    assert (base[kept] == 7).all()


@pytest.mark.parametrize("shape,strides", [
    ((4, 1, 64), (0, 64, 1)), ((4, 1, 64), (56, 64, 1)), ((1, 8, 64), (512, 0, 1)), ((1, 8, 64), (512, 56, 1)),
    ((4, 8, 64), (64, 64, 1)), ((4, 8, 64), (0, 64, 1)), ((4, 8, 64), (504, 64, 1)), ((4, 8, 64), (64, 248, 1))])
def test_outputs_that_overlap_are_refused(shape, strides):
    tokens, heads, dim = shape
    x = make(19, [50] * tokens, [1] * tokens, heads, 1, dim, 16, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    out = torch.zeros(8192, dtype=torch.bfloat16, device=DEV).as_strided(shape, strides)
    with pytest.raises(ValueError, match="overlap"):
        si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], out=out)


@pytest.mark.parametrize("heads", [1, 8])
def test_workspace_of_queries_of_any_layout(heads):
    """The query is an input: its rows may be the same memory, and it is no output."""
    x = make(20, [5000, 333, 40], [1, 1, 1], heads, 1, 64, 16, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    args = (d["ck"], d["cv"], d["tables"], d["kv"])
    need = si.paged_attention_workspace(d["q"], *args)
    one = d["q"][:1].expand(3, heads, 64)
    assert si.paged_attention_workspace(one, *args) == need
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    assert torch.equal(si.paged_attention(one, *args, workspace=ws), si.paged_attention(one.contiguous(), *args))


def test_steps_of_keys_past_32_bit_offsets():
    """64 keys of 270,336 KV heads x 128 lie 4.4 GB apart from first to last."""
    heads, dim, ps, tokens = 270_336, 128, 64, 17
    g = torch.Generator(device=DEV).manual_seed(3)
    ck, cv, q = (torch.empty((n, heads, dim), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
                 for n in (ps, ps, tokens))
    lse = torch.empty((tokens, heads), device=DEV)
    out = si.paged_attention(q, ck[None], cv[None], torch.zeros((1, 1), dtype=torch.int64, device=DEV),
                             torch.tensor([ps], device=DEV), q_starts=torch.tensor([0, tokens], device=DEV), lse=lse)
    some = torch.tensor([0, 1, 2, 100_000, 262_144, heads - 1], device=DEV)
    x = dict(q=q[:, some].cpu(), ck=ck[None, :, some].cpu(), cv=cv[None, :, some].cpu(),
             tables=torch.zeros((1, 1), dtype=torch.int64), kv=torch.tensor([ps]), starts=torch.tensor([0, tokens]))
    agree(out[:, some], lse[:, some], definition(x))


def test_tensors_that_require_gradients_are_refused():
    """There is no backward pass: a result without a history is not handed out unasked."""
    x = make(21, [40, 20], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    args = dict(q=d["q"], cache_k=d["ck"], cache_v=d["cv"], tables=d["tables"], kv_lens=d["kv"])
    want = si.paged_attention(**args)
    for name in ("q", "cache_k", "cache_v"):
        tracked = {**args, name: args[name].clone().requires_grad_()}
        with pytest.raises(ValueError, match="gradient"):
            si.paged_attention(**tracked)
        with torch.no_grad():
            assert torch.equal(si.paged_attention(**tracked), want)
    k = torch.ones((2, 2, 64), dtype=torch.bfloat16, device=DEV)
    rest = (d["ck"], d["cv"], d["tables"], d["kv"])
    for kk, vv in ((k.clone().requires_grad_(), k), (k, k.clone().requires_grad_())):
        before = d["ck"].clone()
        with pytest.raises(ValueError, match="gradient"):
            si.paged_append(kk, vv, *rest)
        assert torch.equal(torch.nan_to_num(d["ck"]), torch.nan_to_num(before))
        with torch.no_grad():
            si.paged_append(kk, vv, *rest)


def test_tokens_without_any_sequence_are_refused():
    x = make(22, [40], [1], 2, 2, 64, 16, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    none = (d["ck"], d["cv"], d["tables"][:0], d["kv"][:0])
    start = torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="no sequences"):
        si.paged_append(d["q"], d["q"], *none, q_starts=start)
    si.paged_append(d["q"][:0], d["q"][:0], *none, q_starts=start)


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-33, -1e-36])
def test_scales_of_nothing_and_next_to_it(scale):
    """Products of up to 1e35 under a scale of 0 weigh the same."""
    x = make(23, [300, 70, 9], [40, 1, 3], 4, 2, 64, 32, torch.bfloat16)
    x["q"] *= 1e17
    x["ck"] *= 1e17
    check(x, scale=scale)


@pytest.mark.parametrize("hq,hkv,dim,dtype", [(8, 2, 128, torch.bfloat16), (4, 1, 64, torch.float16),
                                              (6, 2, 256, torch.bfloat16), (5, 1, 96, torch.float16)])
def test_tiles_joined_from_many_parts(hq, hkv, dim, dtype):
    """More than 2,048 (token, head) rows over keys cut into parts, beside next tokens."""
    kv, new = [7001, 5003, 2111, 40, 3000], [501, 130, 1, 1, 77]
    x = make(24, kv, new, hq, hkv, dim, 64, dtype)
    check(x, rows={0, 250, 500, 501, 600, 630, 631, 632, 633, 680, 709})
    check(x, window=1500, rows={0, 250, 500, 501, 600, 630, 631, 632, 633, 680, 709})


def test_parts_beside_infinite_and_nan_values():
    """Rows that do not see the bad keys near the diagonal of a sequence cut into parts."""
    for bad in (math.nan, math.inf):
        kv, new = [7001, 5003], [520, 130]
        x = make(25, kv, new, 8, 2, 64, 64, torch.bfloat16)
        for b, p in ((0, 6990), (0, 6700), (1, 4950)):
            x["cv"][x["tables"][b, p // 64], p % 64] = bad
        check(x, rows={0, 100, 218, 219, 400, 508, 509, 519, 520, 596, 597, 649})
