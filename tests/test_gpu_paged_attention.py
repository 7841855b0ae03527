"""paged_attention and paged_append against their definitions in 64 bits, on
the CPU: every sequence's keys are gathered page by page, a key without a held
page is not seen, and a token that sees none gives 0.

Bound on an output element, from the arithmetic: with u the unit roundoff of
the 16-bit type, A = sum_j w_j |v_j| and ds the rounding of a score
(|ds| <= (dim + 4) 2^-24 scale sum_d |q_d k_d|, which moves a weight and the
sum of weights by a factor exp(ds) each), one rounding of the weights to 16
bits and one of the output give
  |error| <= u |o| + (u + 4 ds + 2^-18) A + n 2^-25 max|v|,
the last term for fp16 weights below its normal range, and 2^-18 for the
float sums of at most 2^14 terms in any order.  The log-sum-exp moves by at
most ds + 2^-18 (1 + |lse|)."""
import math

import pytest
import torch

import secure_infer_amd as si

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rand(g, *shape, dtype=torch.float64):
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


def make(seed, kv, new, hq, hkv, dim, ps, dtype, holes=(), spare=3, stale=math.nan, width=None):
    """A batch on the CPU: sequence b has kv[b] tokens, the last new[b] new."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // ps) for n in kv]
    slots = sum(need) + spare
    order = torch.randperm(slots, generator=g)
    width = max(need + [1]) + 1 if width is None else width
    tables = torch.full((len(kv), width), -1, dtype=torch.int64)
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = order[at:at + k]
        at += k
    ck = torch.full((slots, ps, hkv, dim), stale, dtype=dtype)
    cv = ck.clone()
    for b, n in enumerate(kv):
        for j in range(need[b]):
            m = min(ps, n - j * ps)
            ck[tables[b, j], :m] = rand(g, m, hkv, dim, dtype=dtype)
            cv[tables[b, j], :m] = rand(g, m, hkv, dim, dtype=dtype)
    for b, j, e in holes:
        if e is not None and 0 <= tables[b, j] < slots:
            ck[tables[b, j]] = stale
            cv[tables[b, j]] = stale
        tables[b, j] = e
    q = rand(g, sum(new), hq, dim, dtype=dtype)
    starts = torch.tensor([0] + list(new)).cumsum(0)
    return dict(q=q, ck=ck, cv=cv, tables=tables, kv=torch.tensor(kv), starts=starts)


def expect(x, scale=None, causal=True, window=0):
    """(out, lse, bound of out, bound of lse) in float64."""
    q, ck, cv, tables = x["q"], x["ck"], x["cv"], x["tables"]
    tokens, hq, dim = q.shape
    slots, ps, hkv, _ = ck.shape
    scale = dim ** -0.5 if scale is None else scale
    u = ROUND[q.dtype]
    out = torch.zeros((tokens, hq, dim), dtype=torch.float64)
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(tables.shape[0]):
        t0, t1 = int(x["starts"][b]), int(x["starts"][b + 1])
        n = max(0, min(int(x["kv"][b]), tables.shape[1] * ps))
        pos = torch.arange(n)
        slot = tables[b][pos // ps]
        keep = (slot >= 0) & (slot < slots)
        pos, slot = pos[keep], slot[keep]
        k = ck[slot, pos % ps].double()
        v = cv[slot, pos % ps].double()
        for i in range(t1 - t0):
            p = n - (t1 - t0) + i
            seen = torch.ones_like(pos, dtype=torch.bool)
            if causal:
                seen &= pos <= p
            if window:
                seen &= pos > p - window
            if not bool(seen.any()):
                continue
            for h in range(hq):
                kk, vv = k[seen][:, h // (hq // hkv)], v[seen][:, h // (hq // hkv)]
                qq = q[t0 + i, h].double()
                s = (kk @ qq) * scale
                ds = float((kk.abs() @ qq.abs()).max() * abs(scale) * (dim + 4) * 2.0 ** -24)
                lse[t0 + i, h] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[t0 + i, h])
                out[t0 + i, h] = w @ vv
                a = w @ vv.abs()
                tol[t0 + i, h] = u * out[t0 + i, h].abs() + (u + 4 * ds + 2.0 ** -18) * a
                if q.dtype == torch.float16:
                    tol[t0 + i, h] += int(seen.sum()) * 2.0 ** -25 * vv.abs().amax(0)
                lse_tol[t0 + i, h] = ds + 2.0 ** -18 * (1 + abs(float(lse[t0 + i, h])))
    return out, lse, tol, lse_tol


def attend(x, use_starts=True, lse=False, **kw):
    d = {k: v.to(DEV) for k, v in x.items()}
    got = torch.full(x["q"].shape[:2], 7.0, dtype=torch.float32, device=DEV) if lse else None
    out = si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"],
                             q_starts=d["starts"] if use_starts else None, lse=got, **kw)
    return (out, got) if lse else out


def check(x, use_starts=True, **kw):
    out, lse = attend(x, use_starts, lse=True, **kw)
    want, want_lse, tol, lse_tol = expect(x, **kw)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(out).all()
    worst = ((out - want).abs() - tol).max()
    assert worst <= 0, f"off by {float(worst)} over the bound"
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    assert ((lse - want_lse).abs()[~none] <= lse_tol[~none]).all()
    assert (out[none] == 0).all()


KV_EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 640]


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", [
    (8, 2, 128, 128, torch.bfloat16), (7, 1, 128, 128, torch.bfloat16), (3, 3, 64, 16, torch.float16),
    (16, 2, 128, 64, torch.float16), (20, 1, 80, 32, torch.bfloat16), (4, 4, 256, 8, torch.bfloat16),
    (6, 2, 8, 128, torch.float16), (40, 1, 128, 128, torch.bfloat16), (5, 1, 40, 256, torch.float16)])
def test_one_token_of_each_sequence(hq, hkv, dim, ps, dtype):
    x = make(hq * 1000 + dim, KV_EDGES, [1] * len(KV_EDGES), hq, hkv, dim, ps, dtype)
    check(x, use_starts=False)


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", [
    (8, 2, 128, 128, torch.bfloat16), (7, 1, 128, 16, torch.bfloat16), (2, 2, 64, 32, torch.float16),
    (4, 1, 96, 64, torch.float16), (2, 1, 256, 128, torch.bfloat16), (3, 1, 72, 8, torch.bfloat16)])
def test_chunks_of_many_lengths(hq, hkv, dim, ps, dtype):
    new = [0, 1, 2, 3, 16, 17, 0, 31, 33, 64, 65, 127, 130, 1]
    kv = [5, 1, 2, 100, 16, 200, 0, 31, 130, 64, 300, 127, 131, 77]
    check(make(dim, kv, new, hq, hkv, dim, ps, dtype))


def test_tokens_before_the_first_position_see_nothing():
    # more new tokens than the sequence holds: the first stand at p < 0
    x = make(3, [0, 5, 70, 1], [3, 9, 130, 40], 4, 2, 128, 16, torch.bfloat16)
    check(x)
    check(x, causal=False)


@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 129, 4096])
def test_window(window):
    x = make(window, [300, 1, 77, 520, 130], [20, 1, 77, 1, 65], 6, 2, 128, 32, torch.bfloat16)
    check(x, window=window)
    check(x, window=window, causal=False)


def test_without_the_causal_bound():
    check(make(9, [300, 1, 77, 513], [20, 1, 70, 1], 8, 8, 64, 64, torch.float16), causal=False)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 70, 200]])
def test_pages_that_are_not_held_are_not_seen(new):
    # holes: negative, one past the last slot, a huge id; sequence 2 holds nothing
    holes = [(0, 0, -1), (0, 2, None), (1, 1, 1 << 40), (1, 3, -(1 << 62)), (2, 0, -1), (2, 1, -7)]
    x = make(21, [300, 500, 200], new, 4, 2, 128, 128, torch.bfloat16, holes=[h for h in holes if h[2] is not None])
    x["tables"][0, 2] = x["ck"].shape[0]
    check(x)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_token_does_not_see_has_no_influence(bad):
    """Rows past a sequence's end, pages of nobody, tokens after a token's
    own position and keys its window has left behind may hold anything."""
    kv, new = [200, 70, 129, 33], [50, 70, 1, 2]
    x = make(5, kv, new, 4, 2, 128, 64, torch.bfloat16, stale=bad)
    check(x)
    # the last two new tokens of sequence 0 and the last of 1 and 3: the
    # tokens before them do not see their K and V
    for b, k in ((0, 2), (1, 1), (3, 1)):
        for p in range(kv[b] - k, kv[b]):
            x["ck"][x["tables"][b, p // 64], p % 64] = bad
            x["cv"][x["tables"][b, p // 64], p % 64] = bad
    # and the first 30 keys of sequence 0, which the window has left behind
    for p in range(30):
        x["ck"][x["tables"][0, p // 64], p % 64] = bad
        x["cv"][x["tables"][0, p // 64], p % 64] = bad
    out = attend(x, window=100).cpu().double()
    clean = {k: v.clone() for k, v in x.items()}
    for c in ("ck", "cv"):
        clean[c][~torch.isfinite(clean[c])] = 0
    want, _, tol, _ = expect(clean, window=100)
    rows = [t for b, k in ((0, 2), (1, 1), (2, 0), (3, 1))
            for t in range(int(x["starts"][b]), int(x["starts"][b + 1]) - k)]
    assert ((out - want).abs()[rows] <= tol[rows]).all()


def test_scale_and_large_scores():
    x = make(31, [400, 129], [30, 1], 4, 2, 128, 128, torch.bfloat16)
    check(x, scale=0.5)
    check(x, scale=-0.2)
    check(x, scale=0.0)
    x["q"] *= 64  # weights fall to one key
    check(x)


def test_long_sequence_split_over_the_chip():
    check(make(41, [9001, 16383], [1, 1], 8, 1, 128, 128, torch.bfloat16), use_starts=False)
    check(make(42, [6007, 300], [9, 1], 4, 1, 64, 16, torch.float16))


def test_strided_queries_outputs_and_caches():
    x = make(51, [300, 77], [20, 3], 8, 2, 64, 32, torch.bfloat16)
    want, _, tol, _ = expect(x)
    d = {k: v.to(DEV) for k, v in x.items()}
    slots = d["ck"].shape[0]
    # queries inside a fused projection, outputs head-major, K and V pages side by side, tables with spare columns
    fused = torch.full((23, 12, 64), math.nan, dtype=torch.bfloat16, device=DEV)
    fused[:, 2:10] = d["q"]
    pool = torch.full((slots, 2, 32, 2, 64), math.nan, dtype=torch.bfloat16, device=DEV)
    pool[:, 0], pool[:, 1] = d["ck"], d["cv"]
    out = torch.full((8, 23, 64), 3.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    wide = torch.full((2, d["tables"].shape[1] + 5), 1 << 50, dtype=torch.int64, device=DEV)
    wide[:, :d["tables"].shape[1]] = d["tables"]
    got = si.paged_attention(fused[:, 2:10], pool[:, 0], pool[:, 1], wide[:, :d["tables"].shape[1]], d["kv"],
                             q_starts=d["starts"], out=out)
    assert got is out
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_rows_outside_every_sequence_are_zero():
    x = make(53, [50, 60], [5, 6], 2, 1, 64, 16, torch.bfloat16)
    x["q"] = torch.cat([x["q"][:2], x["q"], x["q"][:3]])
    x["starts"] = x["starts"] + 2
    check(x)


def test_starts_past_the_rows_are_bounded():
    x = make(55, [50, 60], [5, 6], 2, 1, 64, 16, torch.bfloat16)
    want, _, tol, _ = expect(x)
    x["starts"][2] = 1 << 40  # clamped to the 11 rows there are
    assert ((attend(x).cpu().double() - want).abs() <= tol).all()


def test_pages_past_32_bit_offsets():
    """A cache of more than 4 GiB a tensor, its highest slots in use."""
    slots, ps, hkv, dim = 17_000, 128, 8, 128
    x = make(61, [300, 130], [4, 1], 8, 8, dim, ps, torch.bfloat16, spare=0)
    move = torch.tensor([slots - 1, 5, slots - 2, 8192, 16383])
    d = {k: v.to(DEV) for k, v in x.items()}
    out = []
    for big in (False, True):
        if big:
            ck = torch.empty((slots, ps, hkv, dim), dtype=torch.bfloat16, device=DEV)
            cv = torch.empty_like(ck)
            ck[move.to(DEV)], cv[move.to(DEV)] = d["ck"], d["cv"]
            t = torch.where(x["tables"] >= 0, move[x["tables"].clamp_min(0)], x["tables"]).to(DEV)
            d.update(ck=ck, cv=cv, tables=t)
        out.append(si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], q_starts=d["starts"]).cpu())
        if big:
            k = torch.randn((5, hkv, dim), device=DEV).to(torch.bfloat16)
            si.paged_append(k, 2 * k, d["ck"], d["cv"], d["tables"], d["kv"], q_starts=d["starts"])
            assert torch.equal(d["ck"][d["tables"][0, 2], 296 % 128:300 % 128], k[:4])
            assert torch.equal(d["cv"][d["tables"][1, 1], 1], 2 * k[4])
    assert torch.equal(*out)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_repeats_are_identical_and_other_streams_are_ordered(new):
    x = make(71, [5000, 333], new, 8, 2, 128, 128, torch.bfloat16)
    first = attend(x)
    d = {k: v.to(DEV) for k, v in x.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (None, side, side.cuda_stream):
        out = si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], q_starts=d["starts"], stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_in_a_graph():
    x = make(81, [700, 333], [1, 1], 8, 2, 128, 128, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    k = torch.randn((2, 2, 128), device=DEV).to(torch.bfloat16)

    def step():
        si.paged_append(k, k, d["ck"], d["cv"], d["tables"], d["kv"])
        return si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        k.normal_()
        d["q"].normal_()
        d["kv"] -= 1
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()


def test_workspace_given():
    x = make(91, [5000, 333], [1, 1], 8, 2, 128, 128, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    need = si.paged_attention_workspace(d["q"], d["ck"], d["cv"], d["tables"], d["kv"])
    ws = torch.full((need + 64,), 0x7f, dtype=torch.uint8, device=DEV)
    out = si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], workspace=ws[:max(need, 16)])
    assert torch.equal(out, attend(x, use_starts=False))
    assert (ws[max(need, 16):] == 0x7f).all()
    if need:
        with pytest.raises(ValueError, match="workspace"):
            si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"], workspace=ws[:need - 16])


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("heads,dim,ps,dtype,new", [
    (8, 128, 128, torch.bfloat16, None), (1, 128, 128, torch.bfloat16, None), (3, 40, 16, torch.float16, None),
    (2, 64, 32, torch.bfloat16, [5, 0, 70, 1, 33, 0, 200]), (1, 8, 8, torch.float16, [9, 1, 0, 17, 2, 3, 40])])
def test_append_writes_only_its_rows(heads, dim, ps, dtype, new):
    kv = [77, 1, 200, 130, 33, 5, 201]
    x = make(101 + dim, kv, new or [1] * 7, heads, heads, dim, ps, dtype, stale=0.0)
    g = torch.Generator().manual_seed(7)
    tokens = x["q"].shape[0]
    fused = rand(g, tokens, 2 * heads, dim, dtype=dtype)
    k, v = fused[:, :heads], rand(g, tokens, heads, dim, dtype=dtype)
    ck, cv = x["ck"].clone(), x["cv"].clone()
    for b in range(7):
        t0, t1 = int(x["starts"][b]), int(x["starts"][b + 1])
        for i in range(t1 - t0):
            p = kv[b] - (t1 - t0) + i
            ck[x["tables"][b, p // ps], p % ps] = k[t0 + i]
            cv[x["tables"][b, p // ps], p % ps] = v[t0 + i]
    d = {n: t.to(DEV) for n, t in x.items()}
    fail = torch.zeros(1, dtype=torch.int32, device=DEV)
    si.paged_append(fused.to(DEV)[:, :heads], v.to(DEV), d["ck"], d["cv"], d["tables"], d["kv"],
                    q_starts=d["starts"] if new else None, fail_count=fail)
    assert torch.equal(d["ck"].cpu(), ck) and torch.equal(d["cv"].cpu(), cv)
    assert int(fail) == 0


def test_append_counts_what_it_drops():
    # sequence 0: 2 of 4 tokens before position 0; 1: one page missing (5 of
    # its 9 tokens there); 2: past the table's end; 3: fits
    x = make(111, [2, 69, 40, 10], [4, 9, 2, 1], 2, 2, 64, 16, torch.bfloat16, stale=0.0, width=5)
    x["tables"][1, 4] = 1 << 33
    x["kv"][2] = 81
    before = x["ck"].clone()
    d = {n: t.to(DEV) for n, t in x.items()}
    k = torch.ones((16, 2, 64), dtype=torch.bfloat16, device=DEV)
    fail = torch.full((1,), 100, dtype=torch.int32, device=DEV)
    si.paged_append(k, k, d["ck"], d["cv"], d["tables"], d["kv"], q_starts=d["starts"], fail_count=fail)
    want = before
    want[x["tables"][0, 0], :2] = 1
    want[x["tables"][1, 3], 12:] = 1
    want[x["tables"][3, 0], 9] = 1
    # position 79 of sequence 2 lies on the table's last page, which it does not hold
    assert torch.equal(d["ck"].cpu(), want)
    assert int(fail) == 100 + 2 + 5 + 2


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 70]])
def test_lengths_and_windows_past_the_table(new):
    """Lengths beyond the table's pages end there, negative ones are empty, and a
    window longer than any sequence is none."""
    x = make(71, [256, 128, 192], new, 4, 2, 64, 64, torch.bfloat16, width=4)
    x["tables"] = x["tables"][:, :4]
    x["kv"][0] = (1 << 63) - 1
    x["kv"][1] = -(1 << 63)
    check(x)
    out, lse = attend(x, lse=True)
    for window in (1 << 20, (1 << 30) + 5, (1 << 31) - 1):
        far = attend(x, lse=True, window=window)
        assert torch.equal(far[0], out) and torch.equal(far[1], lse)


@pytest.mark.parametrize("hq,hkv,new", [(40, 1, [33, 0, 2, 1]), (260, 2, [1, 3, 1, 1]), (17, 1, [1, 1, 1, 1])])
def test_groups_wider_than_a_tile_of_columns(hq, hkv, new):
    check(make(73 + hq, [300, 0, 65, 700], new, hq, hkv, 64, 32, torch.bfloat16))


@pytest.mark.parametrize("seqs,hkv,dim,window", [(64, 8, 64, 0), (64, 2, 128, 90), (65, 1, 64, 0), (130, 2, 96, 40),
                                                 (33, 16, 128, 0), (90, 9, 64, 0)])
def test_ragged_batches_over_both_ways_of_sharing_the_keys(seqs, hkv, dim, window):
    """Lengths of nothing to many steps, one or two new tokens or none: sequences that begin
    and end anywhere in a workgroup's share, and shares of one sequence."""
    g = torch.Generator().manual_seed(seqs * hkv)
    kv = [int(n) for n in torch.randint(0, 420, (seqs,), generator=g)]
    kv[3], kv[seqs - 1] = 2500, 0
    new = [int(n) for n in torch.randint(0, 3, (seqs,), generator=g)]
    x = make(seqs, kv, new, 2 * hkv, hkv, dim, 32, torch.bfloat16)
    check(x, window=window)
    one = make(seqs + 1, kv, [1] * seqs, 2 * hkv, hkv, dim, 32, torch.bfloat16)
    check(one, use_starts=False, window=window)
