"""paged_attention with sinks beside a window, and with prefixes that groups of
sequences share, against the definition in 64 bits on the CPU: every sequence
by itself, key by key.

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
from tests.test_gpu_paged_attention import DEV, KV_EDGES, ROUND, make, rand

pytestmark = pytest.mark.gpu


def definition(x, rows=None, scale=None, causal=True, window=0, sinks=0):
    """{row: (out, lse, bound of out, bound of lse)} of the rows of q, each sequence over its own row's pages,
    whichever it shares."""
    q, ck, cv, tables = x["q"], x["ck"], x["cv"], x["tables"]
    hq, dim = q.shape[1:]
    slots, ps, hkv, _ = ck.shape
    scale = dim ** -0.5 if scale is None else scale
    u = ROUND[q.dtype]
    seqs, most = tables.shape[0], tables.shape[1] * ps
    starts = x["starts"].clamp(0, q.shape[0]).tolist()
    found = {}
    for b in range(seqs):
        length = int(x["kv"][b])
        for t in range(starts[b], starts[b + 1]):
            if rows is not None and t not in rows:
                continue
            p = length - starts[b + 1] + t
            pos = torch.arange(max(0, min(length, most)))
            if causal:
                pos = pos[pos <= p]
            if window:
                pos = pos[(pos > p - window) | (pos < sinks)]
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
    out, lse = out.cpu().double(), lse.cpu().double()
    for t, (want, want_lse, tol, lse_tol) in found.items():
        for got, w, bound in ((out[t], want, tol), (lse[t], want_lse, lse_tol)):
            assert torch.equal(torch.isnan(got), torch.isnan(w)), f"row {t}: NaN"
            near = ((got - w).abs() <= bound) | (got == w) | torch.isnan(w)
            assert near.all(), f"row {t}: off by {float((got - w).abs().nan_to_num(0).max())}"


def attend(x, use_starts=True, d=None, **kw):
    d = {k: v.to(DEV) for k, v in x.items()} if d is None else d
    lse = torch.full(x["q"].shape[:2], 7.0, dtype=torch.float32, device=DEV)
    out = si.paged_attention(d["q"], d["ck"], d["cv"], d["tables"], d["kv"],
                             q_starts=d["starts"] if use_starts else None, lse=lse, prefix_groups=d.get("groups"),
                             prefix_lens=d.get("prefix"), **kw)
    return out, lse


def check(x, use_starts=True, rows=None, **kw):
    found = definition(x, rows, **kw)
    agree(*attend(x, use_starts, **kw), found)


GEOMETRIES = [
    (8, 2, 128, 128, torch.bfloat16), (7, 1, 128, 16, torch.bfloat16), (3, 3, 64, 16, torch.float16),
    (20, 1, 80, 32, torch.bfloat16), (4, 4, 256, 8, torch.bfloat16), (4, 1, 96, 64, torch.float16),
    (6, 2, 8, 128, torch.float16), (40, 1, 128, 128, torch.bfloat16)]


# ------------------------------------------------------------------ sinks

@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", GEOMETRIES)
@pytest.mark.parametrize("window,sinks", [(40, 4), (1, 1), (64, 64), (100, 33), (17, 200), (300, 5)])
def test_next_tokens_see_window_and_sinks(hq, hkv, dim, ps, dtype, window, sinks):
    x = make(hq * 1000 + dim + window, KV_EDGES, [1] * len(KV_EDGES), hq, hkv, dim, ps, dtype)
    check(x, use_starts=False, window=window, sinks=sinks)


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", GEOMETRIES[:6])
@pytest.mark.parametrize("window,sinks,causal", [(40, 4, True), (1, 65, True), (64, 64, False), (129, 1, True)])
def test_chunks_see_window_and_sinks(hq, hkv, dim, ps, dtype, window, sinks, causal):
    new = [0, 1, 2, 3, 16, 17, 0, 31, 33, 64, 65, 127, 130, 1]
    kv = [5, 1, 2, 100, 16, 200, 0, 31, 130, 64, 300, 127, 631, 77]
    check(make(dim + window, kv, new, hq, hkv, dim, ps, dtype), window=window, sinks=sinks, causal=causal)


def test_tokens_before_the_first_position_see_no_sinks():
    x = make(3, [0, 5, 70, 1], [3, 9, 130, 40], 4, 2, 128, 16, torch.bfloat16)
    check(x, window=20, sinks=4)
    check(x, window=20, sinks=4, causal=False)


@pytest.mark.parametrize("new", [1, 3, 40, 300])
def test_pages_between_sinks_and_window_given_up(new):
    """Their table entries are no pages, or hold anything: no token sees them."""
    kv, window, sinks, ps = [1000, 640, 90, 5000], 150, 20, 32
    new = [min(new, n) for n in kv]
    for entry in (-1, 1 << 40, None):
        holes = [(b, j, entry) for b, n in enumerate(kv) for j in range(-(-n // ps))
                 if entry is not None and j * ps >= sinks and (j + 1) * ps <= n - new[b] - window + 1]
        x = make(new[0], kv, new, 6, 2, 64, ps, torch.bfloat16, holes=holes, stale=math.nan)
        if entry is None:  # held, and stale
            for b, n in enumerate(kv):
                for p in range(sinks, max(sinks, n - new[b] - window + 1)):
                    x["ck"][x["tables"][b, p // ps], p % ps] = math.nan
                    x["cv"][x["tables"][b, p // ps], p % ps] = math.inf
        rows = {int(x["starts"][b]) + i for b in range(4) for i in (0, 1, new[b] // 2, new[b] - 1) if i < new[b]}
        check(x, rows=rows, window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("kv,new", [(200, 10), (700, 130), (5000, 4), (7001, 520)])
def test_values_that_some_rows_see_and_others_do_not(bad, kv, new):
    """Keys at the window's edge and near the diagonal, an infinite or NaN V among them."""
    for dim in (64, 128):
        x = make(kv, [kv], [new], 4, 2, dim, 64, torch.bfloat16)
        p_first = kv - new
        for p in (p_first - 99, kv - 2, p_first + new // 2 - 99):
            x["cv"][x["tables"][0, p // 64], p % 64] = bad
        rows = {0, 1, 2, new // 2 - 1, new // 2, new // 2 + 1, new - 2, new - 1}
        check(x, rows=rows, window=100, sinks=4)


@pytest.mark.parametrize("kv,new,bad_k,bad_v", [(3, 3, [0], [0]), (200, 5, range(10), [3]), (5000, 3, [2], []),
                                                (300, 40, [0], [1]), (7001, 530, [3], [4])])
def test_what_a_token_sees_of_nan_among_the_sinks_is_nan(kv, new, bad_k, bad_v):
    x = make(16, [kv], [new], 4, 2, 64, 64, torch.bfloat16)
    for bad, cache in ((bad_k, x["ck"]), (bad_v, x["cv"])):
        p = torch.tensor(list(bad), dtype=torch.int64)
        cache[x["tables"][0, p // 64], p % 64] = math.nan
    check(x, rows={0, 1, 2, 20, 39, 264, new - 1}, window=66, sinks=5)


@pytest.mark.parametrize("new,past", [(1, 1), (1, 40), (8, 4), (8, 9), (40, 39), (40, 200), (200, 130)])
def test_lengths_past_the_table_keep_their_sinks(new, past):
    x = make(13, [512, 512, 300], [new, 2, new], 4, 2, 64, 64, torch.bfloat16, width=8)
    x["kv"] = torch.tensor([512 + past, 512 + past, 300])
    for window, sinks, causal in ((7, 3, True), (100, 65, True), (7, 600, False)):
        check(x, window=window, sinks=sinks, causal=causal)


def test_sinks_without_a_window_change_nothing():
    x = make(31, [400, 129], [30, 1], 4, 2, 128, 128, torch.bfloat16)
    for a, b in zip(attend(x), attend(x, sinks=77)):
        assert torch.equal(a, b)
    for a, b in zip(attend(x, window=50), attend(x, window=50, sinks=0)):
        assert torch.equal(a, b)


def test_long_windows_in_parts():
    check(make(41, [9001, 16383, 300], [1, 1, 1], 8, 1, 128, 128, torch.bfloat16), use_starts=False, window=4096, sinks=4)
    check(make(42, [6007, 300], [9, 1], 4, 1, 64, 16, torch.float16), window=3000, sinks=100)
    x = make(24, [7001, 5003, 2111, 40, 3000], [501, 130, 1, 1, 77], 8, 2, 128, 64, torch.bfloat16)
    check(x, rows={0, 250, 500, 501, 600, 630, 631, 632, 633, 680, 709}, window=1500, sinks=4)


@pytest.mark.parametrize("seqs,hkv,dim,window,sinks", [(64, 8, 64, 200, 4), (64, 2, 128, 90, 40), (130, 2, 96, 40, 9),
                                                       (90, 9, 64, 333, 70)])
def test_ragged_batches(seqs, hkv, dim, window, sinks):
    g = torch.Generator().manual_seed(seqs * hkv)
    kv = [int(n) for n in torch.randint(0, 420, (seqs,), generator=g)]
    kv[3], kv[seqs - 1] = 2500, 0
    new = [int(n) for n in torch.randint(0, 3, (seqs,), generator=g)]
    x = make(seqs, kv, new, 2 * hkv, hkv, dim, 32, torch.bfloat16)
    check(x, window=window, sinks=sinks)
    one = make(seqs + 1, kv, [1] * seqs, 2 * hkv, hkv, dim, 32, torch.bfloat16)
    check(one, use_starts=False, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [1, 40])
def test_the_largest_windows_and_sinks(new):
    x = make(15, [256, 70], [new, 1], 4, 2, 64, 64, torch.bfloat16, width=4)
    out, lse = attend(x)
    agree(out, lse, definition(x))
    for window, sinks in ((1 << 30, 4), ((1 << 31) - 1, 1 << 30), (5, 1 << 30), (300, 256)):
        agree(*attend(x, window=window, sinks=sinks), definition(x, window=window, sinks=sinks))


# ------------------------------------------------------------------ shared prefixes

def share(seed, groups, hq, hkv, dim, ps, dtype, before=(), after=(), stale=math.nan):
    """A batch whose groups are (prefix, [(own keys, new tokens), ...]): the rows' pages wholly below the prefix
    are the first row's, the one at its end a copy, as a fork leaves them; sequences `before` and `after`
    them, (keys, new), are in no group.  A negative number of own keys ends the sequence inside the prefix."""
    lens, news, starts, prefix = [n for n, _ in before], [m for _, m in before], [len(before)], []
    for p, members in groups:
        lens += [p + n for n, _ in members]
        news += [m for _, m in members]
        starts.append(len(lens))
        prefix.append(p)
    lens += [n for n, _ in after]
    news += [m for _, m in after]
    hold = list(lens)
    for g, (p, members) in enumerate(groups):
        if members:
            hold[starts[g]] = max(p, hold[starts[g]])  # the first row holds the whole prefix
    x = make(seed, hold, news, hq, hkv, dim, ps, dtype, stale=stale)
    x["kv"] = torch.tensor(lens)
    for g, (p, members) in enumerate(groups):
        for b in range(starts[g] + 1, starts[g + 1]):
            x["tables"][b, :p // ps] = x["tables"][starts[g], :p // ps]
            if p % ps and x["tables"][b, p // ps] >= 0:
                for c in ("ck", "cv"):
                    x[c][x["tables"][b, p // ps], :p % ps] = x[c][x["tables"][starts[g], p // ps], :p % ps]
    x["groups"], x["prefix"] = torch.tensor(starts), torch.tensor(prefix, dtype=torch.int64)
    return x


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", GEOMETRIES)
def test_next_tokens_of_groups(hq, hkv, dim, ps, dtype):
    groups = [(257, [(1, 1), (40, 1), (3, 1)]), (ps, [(5, 1)]), (64, []), (640, [(n, 1) for n in range(1, 140, 7)]),
              (1, [(1, 1), (2, 1)]), (0, [(3, 1), (70, 1)]), (130, [(-100, 1), (-1, 1), (9, 1), (0, 1)])]
    x = share(hq + dim, groups, hq, hkv, dim, ps, dtype, before=[(33, 1), (0, 1)], after=[(200, 1)])
    check(x, use_starts=False)
    check(x)


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", GEOMETRIES[:6])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks_of_groups(hq, hkv, dim, ps, dtype, causal):
    groups = [(257, [(1, 1), (140, 130), (3, 3)]), (300, [(70, 33), (17, 16), (0, 0), (5, 5), (2, 40), (-60, 30)]),
              (64, [(64, 64)]), (31, [(n, min(n, 4)) for n in range(1, 60, 5)])]
    x = share(hq + dim, groups, hq, hkv, dim, ps, dtype, before=[(70, 20)], after=[(140, 3), (3, 3)])
    check(x, causal=causal)


@pytest.mark.parametrize("window,sinks,causal", [(1, 0, True), (50, 0, True), (200, 4, True), (90, 700, True),
                                                 (64, 64, True), (300, 40, False)])
@pytest.mark.parametrize("new", [1, 4, 50])
def test_groups_with_windows_and_sinks(window, sinks, causal, new):
    groups = [(257, [(new, new), (40 + new, new), (3 + new, new)]), (640, [(n + new, new) for n in range(0, 200, 23)])]
    x = share(window, groups, 6, 2, 64, 32, torch.bfloat16, before=[(400, new)])
    check(x, window=window, sinks=sinks, causal=causal)
    if new == 1:
        check(x, use_starts=False, window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("hq,hkv,dim,ps,dtype", GEOMETRIES[:6])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window=300, sinks=5), dict(window=3000, sinks=70)])
def test_chunks_behind_long_prefixes(hq, hkv, dim, ps, dtype, kw):
    """Groups whose tokens attend to their prefix together: a few tokens a sequence, and chunks beside single ones."""
    rows = 40 * hkv // hq  # of a chunk: about 40 rows a KV head
    groups = [(3333, [(1, 1), (rows + 70, rows), (3, 3), (-2000, 2), (0, 1)]), (2050, [(n, min(n, 2)) for n in range(1, 60, 5)]),
              (700, [(n, 1) for n in (1, 40, 200)])]
    x = share(hq + dim, groups, hq, hkv, dim, ps, dtype, before=[(70, 20)], after=[(140, 3), (3, 3)])
    tokens = x["q"].shape[0]
    check(x, rows=set(range(18, tokens, 5)) | {20, 21, tokens - 1}, **kw)


def test_groups_together_and_alone():
    """Sequences of many rows for the prefix's keys go by themselves, whether they share it or not: the same bits as
    without groups where all of a batch's do."""
    x = share(31, [(64, [(64, 64), (40, 33)]), (100, [(90, 70), (50, 50), (77, 77)])], 8, 2, 64, 32, torch.bfloat16)
    plain = {k: v for k, v in x.items() if k not in ("groups", "prefix")}
    got, want = attend(x), definition(plain)
    agree(*got, want)
    agree(*attend(plain), want)


def test_a_long_prefix_in_many_parts():
    x = share(5, [(9001, [(n, 1) for n in (1, 300, 77)]), (5000, [(40, 9), (700, 3)])], 8, 2, 128, 128, torch.bfloat16)
    check(x)
    check(x, window=4096, sinks=4)


def test_many_rows_of_a_group():
    """More rows than the row join takes, in several tiles, and more than 64 sequences."""
    groups = [(777, [(1 + n % 90, 1) for n in range(150)]), (130, [(1 + n % 50, 1) for n in range(100)])]
    x = share(6, groups, 16, 2, 64, 64, torch.float16, after=[(100, 1)] * 10)
    rows = set(range(0, 260, 9)) | {148, 149, 150, 151, 249, 250}
    check(x, use_starts=False, rows=rows)
    check(x, rows=rows)


def test_many_groups():
    g = torch.Generator().manual_seed(3)
    n = torch.randint(0, 4, (150,), generator=g).tolist()
    groups = [(int(p), [(int(k), 1) for k in torch.randint(1, 90, (m,), generator=g)])
              for p, m in zip(torch.randint(0, 300, (150,), generator=g), n)]
    x = share(7, groups, 4, 1, 64, 16, torch.bfloat16)
    check(x, use_starts=False)
    check(x, window=60, sinks=10)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_lies_behind_a_sequence_has_no_influence(bad):
    """Sequences that end inside the prefix, or see it through a window, beside infinite and NaN K and V there."""
    groups = [(300, [(-250, 1), (-100, 3), (40, 2), (1, 1)])]
    def spoil(x, caches):
        for p in (60, 299):
            for b in range(4):  # every row's copy
                if x["tables"][b, p // 64] >= 0:
                    for c in caches:
                        x[c][x["tables"][b, p // 64], p % 64] = bad
    x = share(8, groups, 4, 2, 64, 64, torch.bfloat16)
    spoil(x, ("ck", "cv"))
    out, lse = attend(x)
    clean = {k: v.clone() for k, v in x.items()}
    for c in ("ck", "cv"):
        clean[c][~torch.isfinite(clean[c])] = 0
    found = definition(clean, rows={0})  # sees 50 keys
    agree(out, lse, found)
    if math.isnan(bad):
        check(x)
        check(x, window=30, sinks=3)
    x = share(9, groups, 4, 2, 64, 64, torch.bfloat16)  # an infinite or NaN V alone
    spoil(x, ("cv",))
    check(x)
    check(x, window=45, sinks=3)


def test_groups_and_prefixes_out_of_bounds_are_clamped():
    x = share(10, [(100, [(5, 1), (9, 1)]), (200, [(4, 1), (8, 1), (30, 1)])], 4, 2, 64, 32, torch.bfloat16)
    x["groups"] = torch.tensor([-(1 << 62), 2, 1 << 62])
    check(x)
    x["prefix"] = torch.tensor([-5, 1 << 62])
    x["tables"][3:] = x["tables"][2]
    check(x)


def test_descending_groups_stay_inside_the_tensors():
    """What such groups give is not defined, but for the sequences outside them and the memory around."""
    x = share(11, [(100, [(5, 1), (9, 1)]), (200, [(4, 1), (8, 1), (30, 1)])], 4, 2, 64, 32, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    for groups in ([4, 2, 0], [5, 5, 0], [3, 1, 4]):
        d["groups"] = torch.tensor(groups, device=DEV)
        out, _ = attend(x, use_starts=False, d=d)
        assert out.shape == x["q"].shape
    torch.cuda.synchronize()


def test_groups_of_one_and_no_prefix_are_as_without():
    x = share(12, [(100, [(5, 1)]), (200, [(4, 1)]), (0, [(8, 1), (9, 1)])], 4, 2, 64, 32, torch.bfloat16)
    got = attend(x, use_starts=False)
    plain = {k: v for k, v in x.items() if k not in ("groups", "prefix")}
    agree(*got, definition(plain))
    none = dict(plain, groups=torch.zeros(1, dtype=torch.int64), prefix=torch.zeros(0, dtype=torch.int64))
    for a, b in zip(attend(none, use_starts=False), attend(plain, use_starts=False)):
        assert torch.equal(a, b)


def test_rows_outside_every_sequence_are_zero():
    x = share(13, [(100, [(5, 2), (9, 3)])], 2, 1, 64, 16, torch.bfloat16)
    x["q"] = torch.cat([x["q"][:2], x["q"], x["q"][:3]])
    x["starts"] = x["starts"] + 2
    out, lse = attend(x)
    agree(out, lse, definition(x))
    outside = [0, 1, 7, 8, 9]
    assert (out[outside] == 0).all() and torch.isinf(lse[outside]).all()


def test_scales_and_large_scores():
    x = share(14, [(300, [(5, 1), (90, 30), (9, 1)])], 4, 2, 128, 128, torch.bfloat16)
    for scale in (0.5, -0.2, 0.0):
        check(x, scale=scale)
        check(x, scale=scale, window=50, sinks=3)
    x["q"] *= 64  # weights fall to one key
    check(x)


@pytest.mark.parametrize("kw", [dict(), dict(window=100, sinks=4)])
def test_repeats_streams_and_workspaces(kw):
    x = share(15, [(5000, [(3, 1), (300, 2), (1, 1)]), (64, [(64, 64), (9, 1)])], 8, 2, 128, 128, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    first, first_lse = attend(x, d=d, **kw)
    args = (d["q"], d["ck"], d["cv"], d["tables"], d["kv"])
    more = dict(q_starts=d["starts"], prefix_groups=d["groups"], prefix_lens=d["prefix"], **kw)
    need = si.paged_attention_workspace(*args, **more)
    ws = torch.full((need + 64,), 0x7f, dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream, workspace in ((None, None), (None, ws[:need]), (side, None), (side.cuda_stream, ws[:need])):
        out = si.paged_attention(*args, stream=stream, workspace=workspace, **more)
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    assert (ws[need:] == 0x7f).all()
    with pytest.raises(ValueError, match="workspace"):
        si.paged_attention(*args, workspace=ws[:need - 16], **more)


def test_refusals():
    x = share(16, [(64, [(3, 1), (5, 1)])], 4, 2, 64, 32, torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    args = (d["q"], d["ck"], d["cv"], d["tables"], d["kv"])
    good = dict(prefix_groups=d["groups"], prefix_lens=d["prefix"])
    si.paged_attention(*args, **good)
    for change, what in (
            (dict(sinks=-1), "sinks"), (dict(sinks=(1 << 30) + 1), "sinks"), (dict(prefix_lens=None), "together"),
            (dict(prefix_groups=None), "together"), (dict(prefix_groups=d["groups"].int()), "prefix_groups"),
            (dict(prefix_lens=d["prefix"].int()), "prefix_lens"), (dict(prefix_groups=d["groups"].cpu()), "prefix_groups"),
            (dict(prefix_groups=d["groups"][:1]), "one entry more"), (dict(prefix_lens=d["prefix"][None]), "prefix_lens")):
        for fn in (si.paged_attention, si.paged_attention_workspace):
            with pytest.raises(ValueError, match=what):
                fn(*args, **{**good, **change})
    with pytest.raises(ValueError, match="gradient"):
        si.paged_attention(d["q"].requires_grad_(), *args[1:], **good)


def test_in_a_graph_and_pages_past_32_bit_offsets():
    """A cache of more than 4 GiB a tensor; lengths and prefixes change between replays."""
    slots, ps, hkv, dim = 17_000, 128, 8, 128
    x = share(17, [(300, [(5, 1), (9, 1), (200, 1)])], 8, hkv, dim, ps, torch.bfloat16, after=[(140, 1)])
    held = sorted({int(s) for s in x["tables"].flatten() if s >= 0})
    far = dict(zip(held, list(range(slots - len(held) // 2, slots)) + [7 + 1000 * i for i in range(len(held))]))
    d = {k: v.to(DEV) for k, v in x.items()}
    big = {}
    for c in ("ck", "cv"):
        big[c] = torch.empty((slots, ps, hkv, dim), dtype=torch.bfloat16, device=DEV)
        for s, f in far.items():
            big[c][f] = d[c][s]
    tables = x["tables"].clone()
    for s, f in far.items():
        tables[x["tables"] == s] = f
    b = {**d, **big, "tables": tables.to(DEV)}
    want = attend(x, use_starts=False, d=d)[0]
    assert torch.equal(attend(x, use_starts=False, d=b)[0], want)
    ws = torch.empty(si.paged_attention_workspace(b["q"], b["ck"], b["cv"], b["tables"], b["kv"],
                                                  prefix_groups=b["groups"], prefix_lens=b["prefix"]),
                     dtype=torch.uint8, device=DEV)

    def step():
        return si.paged_attention(b["q"], b["ck"], b["cv"], b["tables"], b["kv"], prefix_groups=b["groups"],
                                  prefix_lens=b["prefix"], workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        b["q"].copy_(rand(torch.Generator().manual_seed(i), *x["q"].shape, dtype=torch.bfloat16))
        b["kv"] -= 1
        b["prefix"] -= 17 * i
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, step())
            torch.cuda.synchronize()


def wide(x, pages):
    """The batch with table rows of `pages` entries, no page past the ones it had."""
    t = torch.full((x["tables"].shape[0], pages), -1, dtype=torch.int64)
    t[:, :x["tables"].shape[1]] = x["tables"]
    return {**x, "tables": t}


@pytest.mark.parametrize("new", [1, 9, 700])
def test_under_the_longest_table(new):
    """Tables of 2^30 positions: windows with sinks, and prefixes, of sequences that end long before."""
    x = share(18, [(900, [(new, new), (new + 40, new)]), (33, [(new, new), (new, new)])], 16, 1, 8, 32768, torch.bfloat16)
    x = wide(x, 32768)
    rows = {0, 1, new - 1, new, 2 * new - 1, 2 * new, 4 * new - 1}
    check(x, rows=rows)
    check(x, rows=rows, window=200, sinks=5)
    plain = {k: v for k, v in x.items() if k not in ("groups", "prefix")}
    plain["tables"][1, 0], plain["tables"][3, 0] = plain["tables"][0, 0], plain["tables"][2, 0]
    check(plain, rows=rows, window=200, sinks=5)
    check(plain, rows=rows, window=(1 << 31) - 1, sinks=1 << 30)


def test_positions_at_their_last_place():
    """Lengths up to 3 * 2^29 count as they are; the keys there are, sinks among them, end with the table."""
    last = 3 << 29
    x = share(19, [(200, [(56, 1), (60, 1)])], 4, 2, 64, 64, torch.bfloat16)
    x["tables"] = x["tables"][:, :4]
    for window, sinks in ((0, 0), (last - 100, 3), (last - 300, 70), (5, 9)):
        x["kv"] = torch.tensor([last, 256])
        check(x, window=window, sinks=sinks)
        plain = {k: v for k, v in x.items() if k not in ("groups", "prefix")}
        check(plain, window=window, sinks=sinks)


def test_many_sequences_of_one_prefix_and_one_long_tail():
    """More pairs than the even shares take, most of them short, one of many parts."""
    g = torch.Generator().manual_seed(5)
    tails = [int(n) for n in torch.randint(1, 200, (140,), generator=g)]
    tails[77] = 6000
    x = share(20, [(300, [(n, 1) for n in tails])], 8, 4, 64, 64, torch.bfloat16)
    check(x, use_starts=False, rows={0, 1, 76, 77, 78, 139})
    check(x, rows={0, 1, 76, 77, 78, 139}, window=2500, sinks=40)


@pytest.mark.parametrize("new", [[300, 1, 1], [700, 40, 3]])
def test_long_chunks_behind_a_prefix(new):
    """Sequences of a group that run in tiles of their own, their keys in several parts."""
    x = share(21, [(777, [(n + 3000 * (i == 0), n) for i, n in enumerate(new)])], 8, 2, 128, 64, torch.bfloat16)
    rows = {0, 1, 150, new[0] - 1, new[0], sum(new) - 1}
    check(x, rows=rows)
    check(x, rows=rows, causal=False)
    check(x, rows=rows, window=1000, sinks=10)


@pytest.mark.parametrize("members", [3, 90])
@pytest.mark.parametrize("use_starts", [True, False])
def test_rows_of_a_group_that_have_ended(members, use_starts):
    """Ended rows hold no page, shorter ones the first pages: the prefix is read from a row that holds it."""
    x = share(22, [(777, [(n % 50, 1) for n in range(1, members + 1)])], 4, 2, 64, 32, torch.bfloat16, after=[(100, 1)])
    whole = {k: v.clone() for k, v in x.items()}

    def cut(b, n):
        x["kv"][b] = n
        x["tables"][b, -(-n // 32):] = -1
    for kept in ([members - 1], [1], []):
        x.update({k: v.clone() for k, v in whole.items()})
        for b in range(members):
            if b not in kept:
                cut(b, 0 if b % 2 == 0 else 37 * b % 500)
        check(x, use_starts=use_starts)
        check(x, use_starts=use_starts, window=300, sinks=9)
