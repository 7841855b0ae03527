"""Measured cases of attention with a window and sinks, attention of batches
that share a prefix, and the append that rotates by position, all over the
paged KV cache.

`run` is one call of an operator, through the package where `own` is true and
in elementary torch operations where it is false.  Lengths follow from a case
alone (geometric ladders between its bounds); the seed gives the values, the
placement of the pages and the order of the sequences.  Cache rows that no
token may see are NaN in the attention cases, as stale memory may be.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One user's next token, 32,768 tokens into a conversation of which
        # a window of 4,096 and the first 4 are kept: where latency counts.
        dict(name="stream_one_token", op="stream", dtype="bf16", hq=32, hkv=8, dim=128, page=128, seqs=1, kv_lo=32768,
             kv_hi=32768, chunks=0, new=0, window=4096, sinks=4, dropped=True, lse=False),
        # A serving batch's next tokens, some still shorter than the window;
        # the pages between sinks and window are still held.
        dict(name="stream_batch", op="stream", dtype="bf16", hq=28, hkv=4, dim=128, page=128, seqs=64, kv_lo=130,
             kv_hi=16384, chunks=0, new=0, window=1024, sinks=4, dropped=False, lse=False),
        # A step that mixes next tokens with three prompt chunks of odd
        # lengths: fp16, head size 64, small pages, odd window and sinks.
        dict(name="stream_mixed_chunks", op="stream", dtype="fp16", hq=12, hkv=4, dim=64, page=16, seqs=27, kv_lo=77,
             kv_hi=5003, chunks=3, new=701, window=513, sinks=5, dropped=False, lse=True),
        # A load chunk of 2,048 prompt tokens at the end of 32,768, window
        # 4,096: the largest.
        dict(name="stream_chunk_32768", op="stream", dtype="bf16", hq=64, hkv=8, dim=128, page=128, seqs=1,
             kv_lo=32768, kv_hi=32768, chunks=1, new=2048, window=4096, sinks=4, dropped=True, lse=False),
        # One prompt sampled eight ways, a few hundred tokens in: the smallest.
        dict(name="shared_samples", op="shared", dtype="bf16", hq=32, hkv=8, dim=128, page=128, groups=1, seqs=8,
             prefix_lo=6144, prefix_hi=6144, tail_lo=1, tail_hi=300, new=1, window=0, sinks=0, lse=False),
        # 64 users' next tokens behind one system prompt of 8,192 tokens.
        dict(name="shared_batch", op="shared", dtype="bf16", hq=28, hkv=4, dim=128, page=128, groups=1, seqs=64,
             prefix_lo=8192, prefix_hi=8192, tail_lo=1, tail_hi=512, new=1, window=0, sinks=0, lse=False),
        # Seven documents of different lengths, asked about by one to many
        # users, four tokens a sequence (drafted ones to be checked).
        dict(name="shared_groups", op="shared", dtype="fp16", hq=12, hkv=4, dim=64, page=16, groups=7, seqs=45,
             prefix_lo=320, prefix_hi=5008, tail_lo=4, tail_hi=701, new=4, window=0, sinks=0, lse=True),
        # 256 samples of one prompt of 32,768 tokens.
        dict(name="shared_long_32768", op="shared", dtype="bf16", hq=64, hkv=8, dim=128, page=128, groups=1, seqs=256,
             prefix_lo=32768, prefix_hi=32768, tail_lo=1, tail_hi=256, new=1, window=0, sinks=0, lse=False),
        # One user's next token of one layer: the smallest append.
        dict(name="rotate_one", op="rotate", dtype="bf16", hq=32, hkv=8, dim=128, rot=128, adjacent=False,
             base=500000.0, magnitude=1.0, page=128, seqs=1, kv_lo=6144, kv_hi=6144, chunks=0, new=0, fused=True, at=0),
        # A decoding batch's next tokens.
        dict(name="rotate_tokens", op="rotate", dtype="bf16", hq=28, hkv=4, dim=128, rot=128, adjacent=False,
             base=1000000.0, magnitude=1.0, page=128, seqs=64, kv_lo=130, kv_hi=8192, chunks=0, new=0, fused=True, at=0),
        # Chunks of a smaller model that rotates 32 of 80 dims in adjacent
        # pairs, at positions of their own far out (chunks stored for reuse
        # elsewhere).
        dict(name="rotate_partial", op="rotate", dtype="fp16", hq=12, hkv=4, dim=80, rot=32, adjacent=True,
             base=10000.0, magnitude=1.1, page=16, seqs=27, kv_lo=77, kv_hi=5003, chunks=3, new=701, fused=False,
             at=1000003),
        # Prompt chunks out of a fused projection: the largest append.
        dict(name="rotate_chunks", op="rotate", dtype="bf16", hq=32, hkv=8, dim=128, rot=128, adjacent=False,
             base=500000.0, magnitude=1.0, page=128, seqs=8, kv_lo=2049, kv_hi=8192, chunks=8, new=2047, fused=True,
             at=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["stream", "shared", "rotate"])
    big = {c["name"]: c for c in listed()}
    hkv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), hkv=hkv, hq=hkv * rng.choice([1, 2, 4, 5, 7, 8]),
             dim=rng.choice([64, 80, 96, 128, 128]), page=rng.choice([16, 32, 64, 128, 128]))
    if op in ("stream", "rotate"):
        kind = rng.choice(["one", "mixed", "chunks"])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 65, 32768)
        c.update(seqs=seqs, kv_lo=_log(rng, 1, hi), kv_hi=hi,
                 chunks={"one": 0, "mixed": (seqs + 3) // 4, "chunks": seqs}[kind], new=_log(rng, 2, 2048))
    if op == "stream":
        c.update(window=_log(rng, 16, 8192), sinks=_log(rng, 1, 200), dropped=rng.random() < 0.5,
                 lse=rng.random() < 0.3)
        most = 0.5 * work(big["stream_chunk_32768"])["flops"]
        few = work(big["stream_batch"])["bytes"]
        while work(c)["flops"] > most or (c["chunks"] == 0 and work(c)["bytes"] > few):
            c["kv_hi"] = max(64, c["kv_hi"] * 2 // 3)
            c["kv_lo"] = min(c["kv_lo"], c["kv_hi"])
    elif op == "shared":
        seqs = _log(rng, 2, 200)
        hi, tail = _log(rng, 65, 32768), _log(rng, 2, 2048)
        new = rng.choice([1, 1, 1, 2, 5, _log(rng, 2, 300)])
        c.update(groups=min(seqs, _log(rng, 1, 12)), seqs=seqs, prefix_lo=_log(rng, 1, hi), prefix_hi=hi,
                 tail_lo=_log(rng, 1, tail), tail_hi=tail, new=min(new, tail),
                 window=rng.choice([0, 0, 0, _log(rng, 16, 16384)]), lse=rng.random() < 0.3)
        c.update(sinks=_log(rng, 1, 200) if c["window"] and rng.random() < 0.5 else 0)
        most = work(big["shared_long_32768"])
        while work(c)["flops"] > 0.5 * most["flops"] or work(c)["bytes"] > most["bytes"]:
            c["prefix_hi"] = max(1, c["prefix_hi"] * 2 // 3)
            c["prefix_lo"] = min(c["prefix_lo"], c["prefix_hi"])
            c["tail_hi"] = max(c["new"], c["tail_hi"] * 2 // 3)
            c["tail_lo"] = min(c["tail_lo"], c["tail_hi"])
            if c["prefix_hi"] == 1:
                c["seqs"] = max(c["groups"], c["seqs"] // 2)
    else:
        rot = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 16])
        c.update(rot=rot // 8 * 8, adjacent=rng.random() < 0.4, base=rng.choice([10000.0, 500000.0, 1000000.0]),
                 magnitude=rng.choice([1.0, 1.0, 1.2]), fused=rng.random() < 0.5,
                 at=rng.choice([0, 0, _log(rng, 1000, 4000000)]))
        while work(c)["bytes"] > work(big["rotate_chunks"])["bytes"]:
            c["new"] = max(2, c["new"] // 2)
            c["seqs"] = max(1, c["seqs"] // 2)
            c["chunks"] = min(c["chunks"], c["seqs"])
    return c


# ------------------------------------------------------------------ lengths

def _ladder(lo, hi, n):
    """n lengths from lo to hi in geometric steps."""
    if n == 1:
        return [hi]
    return [max(1, int(round(lo * (hi / lo) ** (i / (n - 1))))) for i in range(n)]


def _lengths(c):
    """(kv_len, new tokens) of each sequence of a stream or rotate case."""
    kv = _ladder(c["kv_lo"], c["kv_hi"], c["seqs"])
    step = max(1, c["seqs"] // max(1, c["chunks"]))
    out = []
    left = c["chunks"]
    for i, n in enumerate(reversed(kv)):
        new = 1
        if left and i % step == 0:
            new = c["new"] if left == c["chunks"] else max(1, c["new"] - 61 * left)
            left -= 1
        out.append((n, min(new, n)))
    return out


def _groups(c):
    """(prefix, [(tail, new), ...]) of each group of a shared case: from one
    sequence to many a group, the ladder of tails dealt out in turn."""
    n, g = c["seqs"], c["groups"]
    weight = _ladder(1, 2 * n, g)
    size = [1 + (n - g) * w // sum(weight) for w in weight]
    size[-1] += n - sum(size)
    tails = _ladder(c["tail_lo"], c["tail_hi"], n)
    tails = tails[::2] + tails[1::2]
    out, at = [], 0
    for s, p in zip(size, _ladder(c["prefix_lo"], c["prefix_hi"], g)):
        # the pages that a fork shares are whole ones
        whole = -(-p // c["page"]) * c["page"]
        out.append((whole, [(t, min(c["new"], t)) for t in tails[at:at + s]]))
        at += s
    return out


def _pairs(n, new, window, sinks, first=0):
    """(query, key) pairs of the keys from `first` on that a sequence of n keys and `new` queries sees."""
    if not window:
        return new * (n - new - first) + new * (new + 1) // 2
    total = 0
    for p in range(n - new, n):
        w = max(first, p - window + 1)
        total += p + 1 - w + max(0, min(sinks, w) - first)
    return total


def _prefix_seen(c, prefix, tails):
    """((query, key) pairs of a group's tokens with its prefix, keys that one of them sees)."""
    if not c["window"]:
        return prefix * sum(new for _, new in tails), prefix
    pairs = 0
    lowest = prefix
    for t, new in tails:
        for p in range(prefix + t - new, prefix + t):
            w = max(0, min(prefix, p - c["window"] + 1))
            lowest = min(lowest, w)
            pairs += prefix - w + min(c["sinks"], w)
    return pairs, prefix - lowest + min(c["sinks"], lowest)


def work(case):
    c = case
    row = c["hkv"] * c["dim"] * 2
    if c["op"] == "shared":
        nbytes = flops = tokens = 0
        for prefix, tails in _groups(c):
            pairs, keys = _prefix_seen(c, prefix, tails)
            tokens += sum(new for _, new in tails)
            own_pairs = sum(_pairs(prefix + t, new, c["window"], c["sinks"], prefix) for t, new in tails)
            flops += 4 * c["dim"] * c["hq"] * (pairs + own_pairs)
            kept = sum(min(t, c["window"] + new - 1) if c["window"] else t for t, new in tails)
            nbytes += 2 * row * (keys + kept) + 8 * (-(-keys // c["page"]) + sum(-(-t // c["page"]) for t, _ in tails))
        return {"bytes": nbytes + tokens * c["hq"] * (4 * c["dim"] + (4 if c["lse"] else 0)) + 16 * c["seqs"],
                "flops": flops}
    lens = _lengths(c)
    tokens = sum(new for _, new in lens)
    if c["op"] == "rotate":
        table = 8 * sum(-(-new // c["page"]) for _, new in lens) + 16 * len(lens)
        return {"bytes": 4 * tokens * row + 4 * tokens * c["hq"] * c["dim"] + table + 2 * c["rot"],
                "flops": 3 * c["rot"] * tokens * (c["hkv"] + c["hq"])}
    kept = sum(min(n, c["sinks"] + c["window"] + new - 1) for n, new in lens)
    pages = sum(-(-min(n, c["sinks"] + c["window"] + new - 1) // c["page"]) for n, new in lens)
    pairs = sum(_pairs(n, new, c["window"], c["sinks"]) for n, new in lens)
    return {"bytes": 4 * tokens * c["hq"] * c["dim"] + 2 * kept * row + 8 * pages + 16 * len(lens)
            + (4 * tokens * c["hq"] if c["lse"] else 0), "flops": 4 * c["dim"] * c["hq"] * pairs}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)


def _normal(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _fill(s, c, g, slots, spans):
    """The two caches: NaN but for the rows of `spans`, (table row, first, end) of positions."""
    shape, dtype = (c["page"], c["hkv"], c["dim"]), TYPES[c["dtype"]]
    for name in ("k_cache", "v_cache"):
        cache = torch.full((slots, *shape), math.nan, dtype=dtype, device="cuda")
        for row, lo, hi in spans:
            if hi > lo:
                at = _cache_rows(s, row, torch.arange(lo, hi, device="cuda"))
                cache.view(-1, *shape[1:])[at] = _normal(g, hi - lo, *shape[1:], dtype=dtype)
        s[name] = cache


def _cache_rows(s, b, pos):
    """Cache rows (slot * page + offset) of sequence b's positions."""
    ps = s["case"]["page"]
    return s["tables"][b][torch.div(pos, ps, rounding_mode="floor")] * ps + pos % ps


def prepare(case, seed):
    return {"stream": _prepare_stream, "shared": _prepare_shared, "rotate": _prepare_rotate}[case["op"]](
        case, _gen(seed), random.Random(seed))


def _prepare_stream(c, g, rng):
    ps, lens = c["page"], _lengths(c)
    rng.shuffle(lens)
    rows, spans, slots = [], [], 0
    for b, (n, new) in enumerate(lens):
        behind = max(0, n - new - c["window"] + 1)  # the first key that a window still holds
        pages = list(range(-(-n // ps)))
        if c["dropped"]:
            pages = [j if (j + 1) * ps > behind or j * ps < c["sinks"] else -1 for j in pages]
        rows.append(pages)
        slots += sum(j >= 0 for j in pages)
        spans += [(b, 0, min(n, c["sinks"])), (b, max(behind, min(n, c["sinks"])), n)]
    order = list(range(slots + 3))
    rng.shuffle(order)
    table = torch.full((len(lens), -(-c["kv_hi"] // ps) + 2), -1, dtype=torch.int64)
    for b, pages in enumerate(rows):
        for j in pages:
            if j >= 0:
                table[b, j] = order.pop()
    starts = _starts(new for _, new in lens)
    s = dict(case=c, lens=lens, starts=starts, tables=table.cuda(),
             kv_lens=torch.tensor([n for n, _ in lens], device="cuda"),
             q_starts=torch.tensor(starts, device="cuda") if c["chunks"] else None)
    _fill(s, c, g, slots + 3, spans)
    s["q"] = _normal(g, starts[-1], c["hq"], c["dim"], dtype=TYPES[c["dtype"]])
    return s


def _prepare_shared(c, g, rng):
    ps, groups = c["page"], _groups(c)
    rng.shuffle(groups)
    for _, tails in groups:
        rng.shuffle(tails)
    need = sum(p // ps + sum(-(-t // ps) for t, _ in tails) for p, tails in groups)
    order = list(range(need + 3))
    rng.shuffle(order)
    lens, firsts, spans = [], [0], []
    table = torch.full((c["seqs"], max(p // ps + max(-(-t // ps) for t, _ in tails) for p, tails in groups) + 2), -1,
                       dtype=torch.int64)
    for p, tails in groups:
        shared = [order.pop() for _ in range(p // ps)]
        spans.append((len(lens), 0, p))
        for t, new in tails:
            b = len(lens)
            table[b, :len(shared)] = torch.tensor(shared, dtype=torch.int64)
            for j in range(-(-t // ps)):
                table[b, len(shared) + j] = order.pop()
            spans.append((b, p, p + t))
            lens.append((p + t, new))
        firsts.append(len(lens))
    starts = _starts(new for _, new in lens)
    s = dict(case=c, lens=lens, starts=starts, firsts=firsts, prefixes=[p for p, _ in groups], tables=table.cuda(),
             kv_lens=torch.tensor([n for n, _ in lens], device="cuda"),
             q_starts=torch.tensor(starts, device="cuda") if c["new"] > 1 else None,
             prefix_groups=torch.tensor(firsts, device="cuda"),
             prefix_lens=torch.tensor([p for p, _ in groups], device="cuda"))
    _fill(s, c, g, need + 3, spans)
    s["q"] = _normal(g, starts[-1], c["hq"], c["dim"], dtype=TYPES[c["dtype"]])
    return s


def _prepare_rotate(c, g, rng):
    ps, lens, dtype = c["page"], _lengths(c), TYPES[c["dtype"]]
    rng.shuffle(lens)
    need = [-(-n // ps) for n, _ in lens]
    order = list(range(sum(need) + 3))
    rng.shuffle(order)
    table = torch.full((len(lens), max(need) + 2), -1, dtype=torch.int64)
    for b, k in enumerate(need):
        for j in range(k):
            table[b, j] = order.pop()
    starts = _starts(new for _, new in lens)
    tokens = starts[-1]
    pair = torch.arange(c["rot"] // 2, dtype=torch.float64)
    s = dict(case=c, lens=lens, starts=starts, tables=table.cuda(),
             kv_lens=torch.tensor([n for n, _ in lens], device="cuda"),
             q_starts=torch.tensor(starts, device="cuda") if c["chunks"] else None,
             freqs=(c["base"] ** (-2.0 * pair / c["rot"])).float().cuda(),
             positions=(c["at"] + torch.cat([torch.arange(n - new, n) for n, new in lens])).cuda() if c["at"] else None)
    s["k_cache"], s["v_cache"] = (_normal(g, sum(need) + 3, ps, c["hkv"], c["dim"], dtype=dtype) for _ in range(2))
    if c["fused"]:
        # [tokens, (q heads | k heads | v heads) x dim], as a fused projection leaves it
        x = _normal(g, tokens, c["hq"] + 2 * c["hkv"], c["dim"], dtype=dtype)
        s["q"], s["k"], s["v"] = x.split([c["hq"], c["hkv"], c["hkv"]], 1)
    else:
        s["q"], s["k"], s["v"] = (_normal(g, tokens, h, c["dim"], dtype=dtype) for h in (c["hq"], c["hkv"], c["hkv"]))
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


def _lse(s):
    return torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda") if s["case"]["lse"] else None


def _own_stream(s):
    import secure_infer_amd as si
    c, lse = s["case"], _lse(s)
    out = si.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], q_starts=s["q_starts"],
                             window=c["window"], sinks=c["sinks"], lse=lse)
    return (out, lse) if c["lse"] else out


def _own_shared(s):
    import secure_infer_amd as si
    c, lse = s["case"], _lse(s)
    out = si.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], q_starts=s["q_starts"],
                             window=c["window"], sinks=c["sinks"], lse=lse, prefix_groups=s["prefix_groups"],
                             prefix_lens=s["prefix_lens"])
    return (out, lse) if c["lse"] else out


def _own_rotate(s):
    import secure_infer_amd as si
    c = s["case"]
    q = si.paged_append_rotated(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["freqs"],
                                q=s["q"], q_starts=s["q_starts"], positions=s["positions"], adjacent=c["adjacent"],
                                magnitude=c["magnitude"])
    return q, s["k_cache"], s["v_cache"]


def _scores(q, k, hidden, scale):
    """(maxima, weights exp(score - maximum), their sums) of rows; a row that sees nothing has sum 0."""
    x = (q @ k.t().contiguous() * scale).masked_fill_(hidden, -math.inf)
    top = x.amax(1, keepdim=True) if x.shape[1] else x.new_full((x.shape[0], 1), -math.inf)
    w = torch.exp(x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    return top, w, w.sum(1, keepdim=True)


def _hidden(pos, key, window, sinks):
    hidden = key > pos
    if window:
        hidden = hidden | ((key <= pos - window) & (key >= sinks))
    return hidden


def _plain_stream(s):
    c = s["case"]
    group, dim = c["hq"] // c["hkv"], c["dim"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
    for b, (n, new) in enumerate(s["lens"]):
        q0, q1 = s["starts"][b], s["starts"][b + 1]
        behind = max(0, n - new - c["window"] + 1)
        key = torch.cat([torch.arange(min(c["sinks"], behind), device="cuda"),
                         torch.arange(behind, n, device="cuda")])
        rows = _cache_rows(s, b, key)
        k, v = (s[x].view(-1, c["hkv"], dim)[rows].float() for x in ("k_cache", "v_cache"))
        pos = torch.arange(n - new, n, device="cuda").repeat_interleave(group)[:, None]
        hidden = _hidden(pos, key[None, :], c["window"], c["sinks"])
        q = s["q"][q0:q1].float().view(new, c["hkv"], group, dim)
        for h in range(c["hkv"]):
            top, w, total = _scores(q[:, h].reshape(new * group, dim), k[:, h], hidden, dim ** -0.5)
            heads = slice(h * group, (h + 1) * group)
            out[q0:q1, heads] = (w @ v[:, h].contiguous() / total).view(new, group, dim).to(out.dtype)
            lse[q0:q1, heads] = (top + torch.log(total)).view(new, group)
    return (out, lse) if c["lse"] else out


def _plain_shared(s):
    c = s["case"]
    group, dim = c["hq"] // c["hkv"], c["dim"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
    for g, prefix in enumerate(s["prefixes"]):
        first, last = s["firsts"][g], s["firsts"][g + 1]
        t0, t1 = s["starts"][first], s["starts"][last]
        pos = torch.cat([torch.arange(n - new, n, device="cuda") for n, new in s["lens"][first:last]])
        key = torch.arange(prefix, device="cuda")
        rows = _cache_rows(s, first, key)
        k, v = (s[x].view(-1, c["hkv"], dim)[rows].float() for x in ("k_cache", "v_cache"))
        hidden = _hidden(pos.repeat_interleave(group)[:, None], key[None, :], c["window"], c["sinks"])
        for h in range(c["hkv"]):
            heads = slice(h * group, (h + 1) * group)
            q = s["q"][t0:t1, heads].float().reshape(-1, dim)
            # the prefix for all of the group's tokens at once
            top, w, total = _scores(q, k[:, h], hidden, dim ** -0.5)
            acc = w @ v[:, h].contiguous()
            # each sequence's own keys, joined to it
            for b in range(first, last):
                n, new = s["lens"][b]
                part = slice((s["starts"][b] - t0) * group, (s["starts"][b + 1] - t0) * group)
                mine = torch.arange(prefix, n, device="cuda")
                at = _cache_rows(s, b, mine)
                kb, vb = (s[x].view(-1, c["hkv"], dim)[at, h].float() for x in ("k_cache", "v_cache"))
                p = torch.arange(n - new, n, device="cuda").repeat_interleave(group)[:, None]
                own_top, own_w, own_total = _scores(q[part], kb, _hidden(p, mine[None, :], c["window"], c["sinks"]),
                                                    dim ** -0.5)
                both = torch.maximum(top[part], own_top)
                x, y = torch.exp(top[part] - both), torch.exp(own_top - both)
                both_total = total[part] * x + own_total * y
                o = (acc[part] * x + (own_w @ vb) * y) / both_total
                out[s["starts"][b]:s["starts"][b + 1], heads] = o.view(new, group, dim).to(out.dtype)
                lse[s["starts"][b]:s["starts"][b + 1], heads] = (both + torch.log(both_total)).view(new, group)
    return (out, lse) if c["lse"] else out


def _plain_rotate(s):
    c, ps = s["case"], s["case"]["page"]
    seq = torch.cat([torch.full((new,), b) for b, (_, new) in enumerate(s["lens"])]).cuda()
    pos = torch.cat([torch.arange(n - new, n) for n, new in s["lens"]]).cuda()
    rows = s["tables"][seq, torch.div(pos, ps, rounding_mode="floor")] * ps + pos % ps
    angle = (pos if s["positions"] is None else s["positions"]).double()[:, None] * s["freqs"].double()
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))

    def rotated(x):
        half = c["rot"] // 2
        a, b = (x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) if c["adjacent"] else (x[..., :half], x[..., half:c["rot"]])
        a, b = a.float(), b.float()
        y = [(a * cos - b * sin) * c["magnitude"], (b * cos + a * sin) * c["magnitude"]]
        y = torch.stack(y, -1).flatten(-2) if c["adjacent"] else torch.cat(y, -1)
        return torch.cat([y.to(x.dtype), x[..., c["rot"]:]], -1)

    s["k_cache"].view(-1, c["hkv"], c["dim"])[rows] = rotated(s["k"])
    s["v_cache"].view(-1, c["hkv"], c["dim"])[rows] = s["v"]
    return rotated(s["q"]), s["k_cache"], s["v_cache"]


OWN = {"stream": _own_stream, "shared": _own_shared, "rotate": _own_rotate}
PLAIN = {"stream": _plain_stream, "shared": _plain_shared, "rotate": _plain_rotate}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and token by token."""
    s = prepare(case, seed)
    return _exact_rotate(s) if case["op"] == "rotate" else _exact_attention(s)


def _exact_attention(s):
    """Every sequence by itself, over all of its keys."""
    c = s["case"]
    dim, group, ps = c["dim"], c["hq"] // c["hkv"], c["page"]
    out = torch.zeros((s["q"].shape[0], c["hq"], dim), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s["q"].shape[0], c["hq"]), dtype=torch.float64, device="cuda")
    for b, (n, new) in enumerate(s["lens"]):
        pages = s["tables"][b, :-(-n // ps)]
        here = pages.repeat_interleave(ps)[:n] >= 0
        age = torch.arange(n - new, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None, :]
        seen = age >= 0
        if c["window"]:
            seen = seen & (age < c["window"])
            seen[:, :c["sinks"]] |= (age >= 0)[:, :c["sinks"]]
        any_row = seen.any(0) & here
        index = torch.nonzero(any_row).flatten()
        k = s["k_cache"][pages.clamp_min(0)].flatten(0, 1)[:n][index]
        v = s["v_cache"][pages.clamp_min(0)].flatten(0, 1)[:n][index]
        hide = ~seen[:, index].repeat(group, 1)
        t0, t1 = s["starts"][b], s["starts"][b + 1]
        for h in range(c["hkv"]):
            # rows: the group's heads one after another
            q = s["q"][t0:t1, h * group:(h + 1) * group].double().transpose(0, 1).reshape(group * new, dim)
            weight = torch.mm(q, k[:, h].double().t().contiguous()).div_(math.sqrt(dim)).masked_fill_(hide, -math.inf)
            norm = torch.logsumexp(weight, 1)
            mean = torch.mm(weight.sub_(norm[:, None]).exp_(), v[:, h].double().contiguous())
            out[t0:t1, h * group:(h + 1) * group] = mean.view(group, new, dim).transpose(0, 1)
            lse[t0:t1, h * group:(h + 1) * group] = norm.view(group, new).t()
    return (out, lse) if c["lse"] else out


def _exact_rotate(s):
    c, ps = s["case"], s["case"]["page"]
    half = c["rot"] // 2
    first = [2 * i if c["adjacent"] else i for i in range(half)]
    second = [2 * i + 1 if c["adjacent"] else i + half for i in range(half)]
    if s["positions"] is None:
        at = torch.cat([torch.arange(n - new, n) for n, new in s["lens"]]).cuda()
    else:
        at = s["positions"]
    # a complex number a pair, turned by exp(i angle)
    turn = torch.polar(torch.full((at.numel(), half), c["magnitude"], dtype=torch.float64, device="cuda"),
                       at.double()[:, None] * s["freqs"].double()[None, :])[:, None, :]

    def turned(x):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    k, v = turned(s["k"]), s["v"].double()
    ck, cv = s["k_cache"].double(), s["v_cache"].double()
    tables, t = s["tables"].tolist(), 0
    for b, (n, new) in enumerate(s["lens"]):
        p = n - new
        while p < n:
            here = min(n - p, ps - p % ps)
            ck[tables[b][p // ps], p % ps:p % ps + here] = k[t:t + here]
            cv[tables[b][p // ps], p % ps:p % ps + here] = v[t:t + here]
            p, t = p + here, t + here
    return turned(s["q"]), ck, cv
