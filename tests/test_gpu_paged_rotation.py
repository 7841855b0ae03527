"""paged_append_rotated against the rotation in 64 bits on the CPU.

Bound on a rotated element y = m (a cos t - b sin t) with t = p f, u the unit
roundoff of the 16-bit type: the fraction of a turn is rounded to float (2^-25 of a
turn at most, 2^-22.3 radians) after 64-bit products (4 roundings of 2^-53 |t|), the
cosine and sine are within 2 units of 2^-24, times m, and the products and their
sum round 2^-24 each, so every coefficient is within m (2^-20.5 + 2^-50 |t|):
  |error| <= u |y| + 1.01 m (|a| + |b|) (2^-20 + 2^-50 |t|) + 2^-25,
the last term for fp16 results below its normal range."""
import math

import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_attention import DEV, ROUND, make, rand

pytestmark = pytest.mark.gpu


def rotated(x, at, freqs, adjacent, magnitude):
    """(rotated rows, their bounds) of x [tokens, heads, dim] in float64."""
    half, u = freqs.numel(), ROUND[x.dtype]
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    t = (at.double()[:, None] * freqs.double())[:, None, :]
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = magnitude * (a * torch.cos(t) - b * torch.sin(t))
    y[..., second] = magnitude * (b * torch.cos(t) + a * torch.sin(t))
    slack = 1.01 * abs(magnitude) * (a.abs() + b.abs()) * (2.0 ** -20 + 2.0 ** -50 * t.abs()) + 2.0 ** -25
    for d in (first, second):
        tol[..., d] = u * y[..., d].abs() + slack
    return y, tol


def frequencies(rot, base=10000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()


def batch(seed, kv, new, hq, heads, dim, ps, dtype, **kw):
    x = make(seed, kv, new, hq, heads, dim, ps, dtype, stale=0.0, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    tokens = x["q"].shape[0]
    x["k"], x["v"] = (rand(g, tokens, heads, dim, dtype=dtype) for _ in range(2))
    return x


def places(x):
    """(token, sequence, position) of every token of a sequence."""
    starts = x["starts"].tolist()
    return [(t, b, int(x["kv"][b]) - starts[b + 1] + t) for b in range(len(starts) - 1)
            for t in range(starts[b], starts[b + 1])]


def check(x, freqs, adjacent=False, magnitude=1.0, positions=None, use_starts=True, with_q=True, in_place=False):
    slots, ps, heads, dim = x["ck"].shape
    d = {n: t.to(DEV) for n, t in x.items()}
    fail = torch.full((1,), 100, dtype=torch.int32, device=DEV)
    where = places(x)
    at = torch.zeros(x["q"].shape[0], dtype=torch.int64)
    for t, _, p in where:
        at[t] = p
    if positions is not None:
        at = positions
    got = si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], freqs.to(DEV),
                                  q=d["q"] if with_q else None, q_starts=d["starts"] if use_starts else None,
                                  positions=None if positions is None else positions.to(DEV), adjacent=adjacent,
                                  magnitude=magnitude, q_out=d["q"] if in_place else None, fail_count=fail)
    k, k_tol = rotated(x["k"], at, freqs, adjacent, magnitude)
    want_k, tol_k = x["ck"].double(), torch.zeros(x["ck"].shape, dtype=torch.float64)
    want_v, dropped = x["cv"].clone(), x["q"].shape[0]
    for t, b, p in where:
        if 0 <= p < x["tables"].shape[1] * ps and 0 <= x["tables"][b, p // ps] < slots:
            s = int(x["tables"][b, p // ps])
            want_k[s, p % ps], tol_k[s, p % ps], want_v[s, p % ps] = k[t], k_tol[t], x["v"][t]
            dropped -= 1
    assert int(fail) == 100 + dropped
    assert torch.equal(d["cv"].cpu(), want_v)
    assert ((d["ck"].cpu().double() - want_k).abs() <= tol_k).all()
    if not with_q:
        assert got is None
        return
    assert not in_place or got is d["q"]
    q, q_tol = rotated(x["q"], at, freqs, adjacent, magnitude)
    owned = torch.zeros(x["q"].shape[0], dtype=torch.bool)
    for t, _, _ in where:
        owned[t] = True
    assert ((got.cpu().double() - q).abs() <= q_tol)[owned].all()
    assert torch.equal(got.cpu()[~owned], x["q"][~owned])


KV = [77, 1, 200, 130, 33, 5, 201]


@pytest.mark.parametrize("hq,heads,dim,rot,ps,dtype", [
    (8, 8, 128, 128, 128, torch.bfloat16), (28, 4, 128, 128, 128, torch.bfloat16), (3, 3, 40, 8, 16, torch.float16),
    (12, 4, 80, 32, 16, torch.float16), (1, 1, 8, 8, 8, torch.float16), (6, 2, 96, 24, 32, torch.bfloat16),
    (2, 1, 256, 256, 64, torch.bfloat16), (5, 1, 80, 40, 16, torch.bfloat16), (2, 2, 264, 256, 16, torch.float16),
    (64, 8, 64, 16, 128, torch.bfloat16), (3, 1, 72, 72, 8, torch.float16)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("new", [None, [5, 0, 70, 1, 33, 0, 200]])
def test_rotates_on_the_way(hq, heads, dim, rot, ps, dtype, adjacent, new):
    x = batch(101 + dim, KV, new or [1] * 7, hq, heads, dim, ps, dtype)
    check(x, frequencies(rot), adjacent, use_starts=new is not None)
    check(x, frequencies(rot), adjacent, magnitude=1.25, with_q=False)
    check(x, frequencies(rot), adjacent, magnitude=-0.5, in_place=True)


@pytest.mark.parametrize("at", [0, 4_000_003, (1 << 30) + 5, -(1 << 31), 1 << 40])
def test_positions_of_their_own(at):
    """Given ones turn, the sequence's own place: angles of far positions in 64 bits."""
    x = batch(7, KV, [5, 0, 70, 1, 33, 0, 200], 4, 2, 128, 32, torch.bfloat16)
    g = torch.Generator().manual_seed(at & 0xffff)
    positions = at + torch.randint(0, 1000, (x["q"].shape[0],), generator=g)
    for adjacent in (False, True):
        check(x, frequencies(128, 500000.0), adjacent, positions=positions)


def test_many_tokens():
    """More tokens than one wave a token fills the chip with."""
    x = batch(9, [6000, 300, 700], [5500, 300, 1], 2, 1, 64, 128, torch.float16)
    check(x, frequencies(64))
    check(x, frequencies(32), adjacent=True, in_place=True)


def test_tokens_that_are_dropped_have_rotated_queries():
    # sequence 0: 2 of 4 tokens before position 0; 1: one page missing; 2: past the table's end; 3: fits
    x = batch(111, [2, 69, 40, 10], [4, 9, 2, 1], 6, 2, 64, 16, torch.bfloat16, width=5)
    x["tables"][1, 4] = 1 << 33
    x["kv"][2] = 81
    for adjacent in (False, True):
        check(x, frequencies(64), adjacent)
        check(x, frequencies(24), adjacent, in_place=True)


def test_rows_in_no_sequence_go_as_they_are():
    x = batch(53, [50, 60], [5, 6], 4, 2, 64, 16, torch.bfloat16)
    for name in ("q", "k", "v"):
        x[name] = torch.cat([x[name][:2], x[name], x[name][:3]])
    x["starts"] = x["starts"] + 2
    x["q"][0, 0, :] = math.inf
    x["q"][-1, 1, :] = math.nan
    d = x["q"].clone()
    for adjacent in (False, True):
        for in_place in (False, True):
            got = {n: t.to(DEV) for n, t in x.items()}
            out = si.paged_append_rotated(got["k"], got["v"], got["ck"], got["cv"], got["tables"], got["kv"],
                                          frequencies(64).to(DEV), q=got["q"], q_starts=got["starts"], adjacent=adjacent,
                                          q_out=got["q"] if in_place else None).cpu()
            for t in (0, 1, 13, 14, 15):
                assert torch.equal(out[t].view(torch.int16), d[t].view(torch.int16))
    x["q"][0, 0, :] = 1.0
    x["q"][-1, 1, :] = 2.0
    check(x, frequencies(64))


def test_infinite_values_stay_in_their_pairs():
    x = batch(54, [50], [3], 4, 2, 64, 16, torch.bfloat16)
    x["q"][1, 2, 5] = math.inf
    x["k"][2, 0, 33] = math.nan
    d = {n: t.to(DEV) for n, t in x.items()}
    out = si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], frequencies(64).to(DEV),
                                  q=d["q"], q_starts=d["starts"])
    bad = ~torch.isfinite(out.cpu())
    assert set(map(tuple, bad.nonzero().tolist())) == {(1, 2, 5), (1, 2, 37)}
    bad = ~torch.isfinite(d["ck"].cpu())
    s = int(x["tables"][0, 3])
    assert set(map(tuple, bad.nonzero().tolist())) == {(s, 1, 0, 1), (s, 1, 0, 33)}


def test_strided_rows_out_of_a_fused_projection():
    hq, heads, dim = 6, 2, 64
    x = batch(57, [300, 77], [20, 3], hq, heads, dim, 32, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    f = frequencies(dim).to(DEV)
    want = si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], f, q=d["q"], q_starts=d["starts"])
    fused = torch.cat([d["q"], d["k"], d["v"]], 1)
    kept = fused.clone()
    pool = torch.zeros((x["ck"].shape[0], 2, 32, heads, dim), dtype=torch.bfloat16, device=DEV)
    pool[:, 0], pool[:, 1] = x["ck"].to(DEV), x["cv"].to(DEV)
    q, k, v = fused.split([hq, heads, heads], 1)
    out = torch.full((hq, 23, dim), 3.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    got = si.paged_append_rotated(k, v, pool[:, 0], pool[:, 1], d["tables"], d["kv"], f, q=q, q_starts=d["starts"], q_out=out)
    assert got is out and torch.equal(out, want) and torch.equal(fused, kept)
    assert torch.equal(pool[:, 0], d["ck"]) and torch.equal(pool[:, 1], d["cv"])
    got = si.paged_append_rotated(k, v, pool[:, 0], pool[:, 1], d["tables"], d["kv"], f, q=q, q_starts=d["starts"], q_out=q)
    assert torch.equal(fused[:, :hq], want) and torch.equal(fused[:, hq:], kept[:, hq:])


def test_refusals():
    x = batch(58, [30, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    f = frequencies(64).to(DEV)
    good = dict(k=d["k"], v=d["v"], cache_k=d["ck"], cache_v=d["cv"], tables=d["tables"], kv_lens=d["kv"], freqs=f, q=d["q"])
    si.paged_append_rotated(**good)
    fused = torch.cat([d["q"], d["k"]], 1)
    for change, what in (
            (dict(freqs=f.double()), "freqs"), (dict(freqs=f[:3]), "multiple of 4"), (dict(freqs=f[:0]), "multiple of 4"),
            (dict(freqs=torch.cat([f, f])), "at most 32"), (dict(freqs=f.cpu()), "freqs"), (dict(freqs=f[::2]), "freqs"),
            (dict(magnitude=float("nan")), "magnitude"), (dict(positions=d["kv"].int()), "positions"),
            (dict(positions=d["kv"][:1]), "positions"), (dict(q=None, q_out=d["q"]), "q_out"),
            (dict(q=d["q"].half()), "q must be"), (dict(q=d["q"][:1]), "same tokens"), (dict(q=d["q"][:, :0]), "q must be"),
            (dict(q=d["q"][..., :32]), "q must be"), (dict(q_out=d["q"][:1]), "q_out"), (dict(q_out=d["q"].float()), "q_out"),
            (dict(q_out=d["q"][:1].expand(2, 4, 64)), "overlap"), (dict(k=fused[:, 4:], q_out=fused[:, 2:]), "overlap"),
            (dict(q=fused[:, :4], q_out=fused[:, 2:]), "overlap"), (dict(v=d["v"][:1]), "same tokens"),
            (dict(cache_v=d["cv"].half()), "cache_v"), (dict(kv_lens=d["kv"].int()), "kv_lens")):
        with pytest.raises(ValueError, match=what):
            si.paged_append_rotated(**{**good, **change})
    for name in ("q", "k", "v", "freqs"):
        with pytest.raises(ValueError, match="gradient"):
            si.paged_append_rotated(**{**good, name: good[name].clone().requires_grad_()})
    none = dict(k=d["k"][:0], v=d["v"][:0], q=d["q"][:0], tables=d["tables"][:0], kv_lens=d["kv"][:0])
    assert si.paged_append_rotated(**{**good, **none}).shape == (0, 4, 64)


def test_streams_and_graphs():
    x = batch(59, [700, 333], [1, 1], 8, 2, 128, 128, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    f = frequencies(128).to(DEV)

    def step(**kw):
        return si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], f, q=d["q"], **kw)
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        out = step(stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        d["q"].normal_()
        d["k"].normal_()
        d["kv"] -= 1
        d["ck"].zero_()
        g.replay()
        torch.cuda.synchronize()
        got, cache = out.clone(), d["ck"].clone()
        d["ck"].zero_()
        assert torch.equal(got, step()) and torch.equal(cache, d["ck"])
        torch.cuda.synchronize()
