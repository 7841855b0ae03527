"""Measured cases of the operators on the paged KV cache: attention of new
tokens over cached pages, the writing of their K and V rows into the pages,
and forking, freeing and compacting pages.

`run` is one call of an operator, through the package where `own` is true and
in elementary torch operations where it is false.  Lengths follow from a case
alone (geometric ladders between its bounds); the seed gives the values, the
placement of the pages and the order of the sequences.  Cache rows that no
sequence holds are NaN in the attention cases, as stale memory may be.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One user's next token over a 6,144-token prefix of a layer with
        # 8 x 128 KV heads: the smallest attention call, where latency counts.
        dict(name="attend_one_token", op="attend", dtype="bf16", hq=32, hkv=8, dim=128, page=128, seqs=1, kv_lo=6144,
             kv_hi=6144, chunks=0, new=0, window=0, lse=False),
        # A serving batch's next tokens, 4 x 128 KV heads shared by 7 query
        # heads each, prefixes from a page to 8,192 tokens.
        dict(name="attend_batch", op="attend", dtype="bf16", hq=28, hkv=4, dim=128, page=128, seqs=64, kv_lo=130,
             kv_hi=8192, chunks=0, new=0, window=0, lse=False),
        # A step that mixes next tokens with three prompt chunks of odd
        # lengths: fp16, head size 64, small pages, and the log-sum-exp kept
        # for joining with another part's attention.
        dict(name="attend_mixed_chunks", op="attend", dtype="fp16", hq=12, hkv=4, dim=64, page=16, seqs=27, kv_lo=77,
             kv_hi=5003, chunks=3, new=701, window=0, lse=True),
        # A load chunk of 2,048 prompt tokens at the end of 32,768 tokens of
        # an 8 x 128 layer with 64 query heads: the largest.
        dict(name="attend_chunk_32768", op="attend", dtype="bf16", hq=64, hkv=8, dim=128, page=128, seqs=1,
             kv_lo=32768, kv_hi=32768, chunks=1, new=2048, window=0, lse=False),
        # A decoding batch's new K and V rows of one layer.
        dict(name="append_tokens", op="append", dtype="bf16", hkv=8, dim=128, page=128, seqs=64, kv_lo=130,
             kv_hi=8192, chunks=0, new=0, fused=False),
        # Prompt chunks' K and V rows, cut out of a fused projection's output.
        dict(name="append_chunks", op="append", dtype="bf16", hkv=8, dim=128, page=128, seqs=8, kv_lo=2049,
             kv_hi=8192, chunks=8, new=2047, fused=True),
        # One sequence forked: a page of each of 160 tensors (80 layers, one
        # KV head of a tensor-parallel rank) is copied.
        dict(name="fork_one", op="fork", layers=80, hkv=1, dim=128, page=128, slots=64, parents=1, each=1, kv_lo=6100,
             kv_hi=6100),
        # Eight prompts sampled four ways each, 28 layers of 4 x 128 heads.
        dict(name="fork_samples", op="fork", layers=28, hkv=4, dim=128, page=128, slots=192, parents=8, each=4,
             kv_lo=257, kv_hi=4095),
        # One short answer's pages freed and cleared on a tensor-parallel rank.
        dict(name="free_one", op="free", layers=80, hkv=1, dim=128, page=128, slots=64, rows=6, freed=1, kv_lo=700,
             kv_hi=900),
        # A third of a batch freed; every second sequence shares its first
        # half with the one before it.
        dict(name="free_batch", op="free", layers=28, hkv=4, dim=128, page=128, slots=256, rows=24, freed=8,
             kv_lo=300, kv_hi=3000),
        # A nearly compact cache: three pages move.
        dict(name="compact_few", op="compact", layers=80, hkv=1, dim=128, page=128, slots=64, rows=6, moved=3,
             kv_lo=700, kv_hi=900),
        # A fragmented cache before it is cut to half: 60 pages move.
        dict(name="compact_half", op="compact", layers=28, hkv=4, dim=128, page=128, slots=256, rows=24, moved=60,
             kv_lo=300, kv_hi=1400),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "fork", "free", "compact"])
    big = {c["name"]: c for c in listed()}
    page = rng.choice([16, 32, 64, 128, 128])
    if op in ("attend", "append"):
        hkv = rng.choice([1, 2, 4, 8])
        kind = rng.choice(["one", "mixed", "chunks"])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 65, 32768)
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), hkv=hkv, dim=rng.choice([64, 80, 96, 128, 128]),
                 page=page, seqs=seqs, kv_lo=_log(rng, 1, hi), kv_hi=hi,
                 chunks={"one": 0, "mixed": (seqs + 3) // 4, "chunks": seqs}[kind], new=_log(rng, 2, 2048))
        if op == "attend":
            c.update(hq=hkv * rng.choice([1, 2, 4, 5, 7, 8]), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                     lse=rng.random() < 0.3)
            most = 0.5 * work(big["attend_chunk_32768"])["flops"]
            few = 0.5 * work(big["attend_batch"])["bytes"]
            while work(c)["flops"] > most or (c["chunks"] == 0 and work(c)["bytes"] > few):
                c["kv_hi"] = max(64, c["kv_hi"] * 2 // 3)
                c["kv_lo"] = min(c["kv_lo"], c["kv_hi"])
        else:
            c.update(fused=rng.random() < 0.5)
            while work(c)["bytes"] > work(big["append_chunks"])["bytes"]:
                c["new"] = max(2, c["new"] // 2)
                c["seqs"] = max(1, c["seqs"] // 2)
                c["chunks"] = min(c["chunks"], c["seqs"])
        return c
    layers = _log(rng, 2, 40)
    c = dict(op=op, layers=layers, hkv=rng.choice([1, 2, 4]), dim=rng.choice([64, 128]), page=page,
             slots=rng.randint(150, 192))
    hi = page * rng.randint(2, 9) + rng.randint(0, page)
    if op == "fork":
        c.update(parents=rng.randint(1, 8), each=rng.randint(1, 4), kv_lo=rng.randint(1, hi), kv_hi=hi)
    else:
        rows = rng.randint(2, 12)
        c.update(rows=rows, kv_lo=rng.randint(1, hi), kv_hi=hi)
        if op == "free":
            c.update(freed=rng.randint(1, rows))
        else:
            held = len({p for r in _row_pages(c) for p in r})
            c.update(moved=rng.randint(1, max(1, min(held, c["slots"] - held))))
    most = work(big[{"fork": "fork_samples", "free": "free_batch", "compact": "compact_half"}[op]])["bytes"]
    while work(c)["bytes"] > most:
        c["layers"] = c["layers"] * 2 // 3
    return c


# ------------------------------------------------------------------ lengths

def _ladder(lo, hi, n):
    """n lengths from lo to hi in geometric steps."""
    if n == 1:
        return [hi]
    return [max(1, int(round(lo * (hi / lo) ** (i / (n - 1))))) for i in range(n)]


def _lengths(c):
    """(kv_len, new tokens) of each sequence of an attend or append case."""
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


def _seen(n, new, window):
    """(query, key) pairs a causal sequence of n keys and `new` queries sees."""
    total = new * (n - new) + new * (new + 1) // 2
    if window:
        total = sum(min(window, n - new + i + 1) for i in range(new))
    return total


def _row_pages(c):
    """Pages of each row of a free or compact case as numbers in order of
    their first use; every second row shares the first half of the one
    before it."""
    rows, count = [], 0
    for i, n in enumerate(_ladder(c["kv_lo"], c["kv_hi"], c["rows"])):
        need = -(-n // c["page"])
        share = rows[i - 1][:need // 2] if i % 2 else []
        rows.append(share + list(range(count, count + need - len(share))))
        count += need - len(share)
    return _fit(rows, c["slots"])


def _fit(rows, slots):
    """The rows that fit the slots, pages counted once (the last rows lose pages)."""
    return [[p for p in r if p < slots] for r in rows]


def _row_lens(c):
    return [min(n, len(r) * c["page"]) for n, r in zip(_ladder(c["kv_lo"], c["kv_hi"], c["rows"]), _row_pages(c))]


def _tensor_bytes(c):
    return c["page"] * c["hkv"] * c["dim"] * 2


def work(case):
    c = case
    if c["op"] in ("attend", "append"):
        lens = _lengths(c)
        tokens = sum(new for _, new in lens)
        row = c["hkv"] * c["dim"] * 2
        table = 8 * sum(-(-n // c["page"]) for n, _ in lens) + 16 * len(lens)
        if c["op"] == "append":
            return {"bytes": 4 * tokens * row + table, "flops": 0}
        kept = sum(min(n, c["window"] + new - 1) if c["window"] else n for n, new in lens)
        q = tokens * c["hq"] * c["dim"] * 2
        pairs = sum(_seen(n, new, c["window"]) for n, new in lens)
        return {"bytes": 2 * q + 2 * kept * row + table + (4 * tokens * c["hq"] if c["lse"] else 0),
                "flops": 4 * c["dim"] * c["hq"] * pairs}
    if c["op"] == "fork":
        part = sum(1 for n in _ladder(c["kv_lo"], c["kv_hi"], c["parents"]) if n % c["page"])
        rows = c["parents"] * (1 + c["each"])
        moved, scale = part * c["each"], 2
    elif c["op"] == "free":
        pages = _row_pages(c)
        rows = len(pages)
        moved, scale = len({p for r in pages[:c["freed"]] for p in r} - {p for r in pages[c["freed"]:] for p in r}), 1
    else:
        rows = c["rows"]
        moved, scale = c["moved"], 2
    width = _width(c)
    return {"bytes": scale * moved * 2 * c["layers"] * _tensor_bytes(c) + 2 * (8 * rows * (width + 1) + 4 * c["slots"]),
            "flops": 0}


def _width(c):
    """Columns of the page table: the longest sequence's pages and two more."""
    return -(-c["kv_hi"] // c["page"]) + 2


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)


def _normal(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    c, g, rng = case, _gen(seed), random.Random(seed)
    if c["op"] in ("attend", "append"):
        return _prepare_tokens(c, g, rng)
    return _prepare_pages(c, g, rng)


def _prepare_tokens(c, g, rng):
    dtype = TYPES[c["dtype"]]
    lens = _lengths(c)
    rng.shuffle(lens)
    ps, shape = c["page"], (c["page"], c["hkv"], c["dim"])
    need = [-(-n // ps) for n, _ in lens]
    slots = sum(need) + 3
    order = list(range(slots))
    rng.shuffle(order)
    table = torch.full((len(lens), _width(c)), -1, dtype=torch.int64)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = torch.tensor(order[at:at + k])
        at += k
    tokens = sum(new for _, new in lens)
    starts = [0]
    for _, new in lens:
        starts.append(starts[-1] + new)
    s = dict(case=c, lens=lens, starts=starts, tables=table.cuda(),
             kv_lens=torch.tensor([n for n, _ in lens], device="cuda"),
             q_starts=torch.tensor(starts, device="cuda") if c["chunks"] else None)
    if c["op"] == "append":
        s["k_cache"], s["v_cache"] = (_normal(g, slots, *shape, dtype=dtype) for _ in range(2))
        if c["fused"]:
            # [tokens, (q heads | k heads | v heads) x dim], as a fused projection leaves it
            x = _normal(g, tokens, 6 * c["hkv"], c["dim"], dtype=dtype)
            s["k"], s["v"] = x[:, 4 * c["hkv"]:5 * c["hkv"]], x[:, 5 * c["hkv"]:]
        else:
            s["k"], s["v"] = (_normal(g, tokens, c["hkv"], c["dim"], dtype=dtype) for _ in range(2))
        return s
    caches = []
    for _ in range(2):
        cache = torch.full((slots, *shape), math.nan, dtype=dtype, device="cuda")
        for b, (n, _) in enumerate(lens):
            rows = _rows(s, b)
            cache.view(-1, *shape[1:])[rows] = _normal(g, n, *shape[1:], dtype=dtype)
        caches.append(cache)
    s["k_cache"], s["v_cache"] = caches
    s["q"] = _normal(g, tokens, c["hq"], c["dim"], dtype=dtype)
    return s


def _rows(s, b):
    """Cache rows (slot * page + offset) of sequence b's tokens, in order."""
    n, ps = s["lens"][b][0], s["case"]["page"]
    pos = torch.arange(n, device="cuda")
    return s["tables"][b][torch.div(pos, ps, rounding_mode="floor")] * ps + pos % ps


def _prepare_pages(c, g, rng):
    ps = c["page"]
    # every layer's K and V cache, as one allocation's parts
    pool = torch.empty((2 * c["layers"], c["slots"], ps, c["hkv"], c["dim"]), dtype=torch.bfloat16, device="cuda")
    for part in pool:
        part.copy_(_normal(g, *part.shape, dtype=torch.bfloat16))
    refs = [0] * c["slots"]
    if c["op"] == "fork":
        lens = _ladder(c["kv_lo"], c["kv_hi"], c["parents"])
        rows, count = [], 0
        for n in lens:
            need = -(-n // ps)
            rows.append(list(range(count, count + need)))
            count += need
        rows = _fit(rows, c["slots"] - c["parents"] * c["each"])
        lens = [min(n, len(r) * ps) for n, r in zip(lens, rows)]
        rows += [[] for _ in range(c["parents"] * c["each"])]
        lens += [0] * (c["parents"] * c["each"])
    else:
        rows, lens = _row_pages(c), _row_lens(c)
    held = sorted({p for r in rows for p in r})
    if c["op"] == "compact":
        low = rng.sample(range(len(held)), len(held) - c["moved"])
        place = low + rng.sample(range(len(held), c["slots"]), c["moved"])
        rng.shuffle(place)
    else:
        place = rng.sample(range(c["slots"]), len(held))
    where = dict(zip(held, place))
    table = torch.full((len(rows), _width(c)), -1, dtype=torch.int64)
    for b, r in enumerate(rows):
        for j, p in enumerate(r):
            table[b, j] = where[p]
            refs[where[p]] += 1
    s = dict(case=c, pool=pool, caches=list(pool), tables=table.cuda(), kv_lens=torch.tensor(lens, device="cuda"),
             refs=torch.tensor(refs, dtype=torch.int32, device="cuda"))
    if c["op"] == "fork":
        p = c["parents"]
        s["pairs"] = torch.tensor([(i, p + i * c["each"] + j) for i in range(p) for j in range(c["each"])],
                                  device="cuda")
    elif c["op"] == "free":
        s["rows"] = torch.arange(c["freed"], device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


def _own_attend(s):
    import secure_infer_amd as si
    c = s["case"]
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda") if c["lse"] else None
    out = si.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], q_starts=s["q_starts"],
                             window=c["window"], lse=lse)
    return (out, lse) if c["lse"] else out


def _own_append(s):
    import secure_infer_amd as si
    si.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], q_starts=s["q_starts"])
    return s["k_cache"], s["v_cache"]


def _own_fork(s):
    import secure_infer_amd as si
    return (*si.fork_pages(s["caches"], s["tables"], s["kv_lens"], s["refs"], s["pairs"]), s["pool"])


def _own_free(s):
    import secure_infer_amd as si
    return (*si.free_pages(s["caches"], s["tables"], s["kv_lens"], s["refs"], s["rows"]), s["pool"])


def _own_compact(s):
    import secure_infer_amd as si
    return (*si.compact_pages(s["caches"], s["tables"], s["refs"]), s["pool"])


def _plain_attend(s):
    c = s["case"]
    group, dim = c["hq"] // c["hkv"], c["dim"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
    for b, (n, new) in enumerate(s["lens"]):
        q0, q1 = s["starts"][b], s["starts"][b + 1]
        first = max(0, n - new + 1 - c["window"]) if c["window"] else 0
        rows = _rows(s, b)[first:]
        k, v = (s[x].view(-1, c["hkv"], dim)[rows].float() for x in ("k_cache", "v_cache"))
        pos = torch.arange(n - new, n, device="cuda").repeat_interleave(group)[:, None]
        key = torch.arange(first, n, device="cuda")[None, :]
        hidden = key > pos
        if c["window"]:
            hidden = hidden | (key <= pos - c["window"])
        q = s["q"][q0:q1].float().view(new, c["hkv"], group, dim)
        for h in range(c["hkv"]):
            scores = q[:, h].reshape(new * group, dim) @ k[:, h].t().contiguous()
            scores = (scores * dim ** -0.5).masked_fill_(hidden, -math.inf)
            top = scores.amax(1, keepdim=True)
            p = torch.exp(scores.sub_(top))
            total = p.sum(1, keepdim=True)
            o = p @ v[:, h].contiguous() / total
            out[q0:q1, h * group:(h + 1) * group] = o.view(new, group, dim).to(out.dtype)
            lse[q0:q1, h * group:(h + 1) * group] = (top + torch.log(total)).view(new, group)
    return (out, lse) if c["lse"] else out


def _plain_append(s):
    ps = s["case"]["page"]
    seq = torch.cat([torch.full((new,), b) for b, (_, new) in enumerate(s["lens"])]).cuda()
    pos = torch.cat([torch.arange(n - new, n) for n, new in s["lens"]]).cuda()
    rows = s["tables"][seq, torch.div(pos, ps, rounding_mode="floor")] * ps + pos % ps
    for x in ("k", "v"):
        cache = s[x + "_cache"]
        cache.view(-1, *cache.shape[2:])[rows] = s[x]
    return s["k_cache"], s["v_cache"]


def _plain_fork(s):
    ps, width = s["case"]["page"], s["tables"].shape[1]
    parent, child = s["pairs"].unbind(1)
    tables, lens, refs = s["tables"].clone(), s["kv_lens"].clone(), s["refs"].clone()
    n = lens[parent]
    whole = torch.div(n, ps, rounding_mode="floor")
    part = n % ps != 0
    column = torch.arange(width, device="cuda")[None, :]
    rows = torch.where(column < whole[:, None], tables[parent], torch.full_like(tables[parent], -1))
    refs.index_put_((rows[rows >= 0],), torch.ones((), dtype=torch.int32, device="cuda"), accumulate=True)
    fresh = torch.nonzero(s["refs"] == 0).flatten()[:int(part.sum())]
    source = tables[parent[part], whole[part]]
    rows[part, whole[part]] = fresh
    refs[fresh] = 1
    tables[child] = rows
    lens[child] = n
    for cache in s["caches"]:
        cache[fresh] = cache[source]
    return (tables, lens, refs, s["pool"])


def _plain_free(s):
    tables, lens, refs = s["tables"].clone(), s["kv_lens"].clone(), s["refs"].clone()
    gone = tables[s["rows"]]
    refs.index_put_((gone[gone >= 0],), torch.full((), -1, dtype=torch.int32, device="cuda"), accumulate=True)
    tables[s["rows"]] = -1
    lens[s["rows"]] = 0
    clear = torch.nonzero((s["refs"] > 0) & (refs == 0)).flatten()
    for cache in s["caches"]:
        cache[clear] = 0
    return (tables, lens, refs, s["pool"])


def _plain_compact(s):
    live = s["refs"] > 0
    count = int(live.sum())
    slot = torch.arange(live.numel(), device="cuda")
    source, target = slot[live & (slot >= count)], slot[~live & (slot < count)]
    moved = slot.clone()
    moved[source] = target
    refs = s["refs"].clone()
    refs[target] = s["refs"][source]
    refs[source] = 0
    tables = torch.where(s["tables"] >= 0, moved[s["tables"].clamp_min(0)], s["tables"])
    for cache in s["caches"]:
        cache[target] = cache[source]
    return (tables, refs, s["pool"])


OWN = {"attend": _own_attend, "append": _own_append, "fork": _own_fork, "free": _own_free, "compact": _own_compact}
PLAIN = {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "free": _plain_free,
         "compact": _plain_compact}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, token by token and page by page."""
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "fork": _exact_pages, "free": _exact_pages,
            "compact": _exact_pages}[case["op"]](s)


def _exact_attend(s):
    c = s["case"]
    dim, group, ps = c["dim"], c["hq"] // c["hkv"], c["page"]
    tokens = s["q"].shape[0]
    out = torch.zeros((tokens, c["hq"], dim), dtype=torch.float64, device="cuda")
    lse = torch.zeros((tokens, c["hq"]), dtype=torch.float64, device="cuda")
    tables = s["tables"].tolist()
    for b, (n, new) in enumerate(s["lens"]):
        pages = torch.tensor(tables[b][:-(-n // ps)], device="cuda")
        k = s["k_cache"][pages].flatten(0, 1)[:n]
        v = s["v_cache"][pages].flatten(0, 1)[:n]
        # what token i (at n - new + i) may look at
        age = torch.arange(n - new, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None, :]
        seen = (age >= 0) & (age < c["window"]) if c["window"] else age >= 0
        for h in range(c["hq"]):
            q = s["q"][s["starts"][b]:s["starts"][b + 1], h].double()
            weight = torch.mm(q, k[:, h // group].double().t().contiguous()).div_(math.sqrt(dim))
            weight = torch.where(seen, weight, torch.full_like(weight, -math.inf))
            norm = torch.logsumexp(weight, 1)
            weight = weight.sub_(norm[:, None]).exp_()
            out[s["starts"][b]:s["starts"][b + 1], h] = torch.mm(weight, v[:, h // group].double().contiguous())
            lse[s["starts"][b]:s["starts"][b + 1], h] = norm
    return (out, lse) if c["lse"] else out


def _exact_append(s):
    ps, tables = s["case"]["page"], s["tables"].tolist()
    caches = [s[x].double() for x in ("k_cache", "v_cache")]
    new_rows = [s[x].double() for x in ("k", "v")]
    t = 0
    for b, (n, new) in enumerate(s["lens"]):
        p = n - new
        while p < n:
            here = min(n - p, ps - p % ps)
            for cache, rows in zip(caches, new_rows):
                cache[tables[b][p // ps], p % ps:p % ps + here] = rows[t:t + here]
            p, t = p + here, t + here
    return tuple(caches)


def _exact_pages(s):
    c = s["case"]
    ps, slots = c["page"], c["slots"]
    tables, lens, refs = s["tables"].tolist(), s["kv_lens"].tolist(), s["refs"].tolist()
    pool = s["pool"].double()
    if c["op"] == "fork":
        free = [i for i in range(slots) if refs[i] == 0]
        for parent, child in s["pairs"].tolist():
            lens[child] = lens[parent]
            for j in range(lens[parent] // ps):
                tables[child][j] = tables[parent][j]
                refs[tables[parent][j]] += 1
            if lens[parent] % ps:
                j, slot = lens[parent] // ps, free.pop(0)
                pool[:, slot] = pool[:, tables[parent][j]]
                tables[child][j], refs[slot] = slot, 1
    elif c["op"] == "free":
        for row in s["rows"].tolist():
            for j, slot in enumerate(tables[row]):
                if slot >= 0:
                    refs[slot] -= 1
                    if refs[slot] == 0:
                        pool[:, slot] = 0
                tables[row][j] = -1
            lens[row] = 0
    else:
        live = [i for i in range(slots) if refs[i] > 0]
        low = [i for i in range(len(live)) if refs[i] == 0]
        move = dict(zip([i for i in live if i >= len(live)], low))
        for a, b in move.items():
            pool[:, b] = pool[:, a]
            refs[a], refs[b] = 0, refs[a]
        tables = [[move.get(i, i) for i in row] for row in tables]
    whole = [torch.tensor(x, device="cuda", dtype=torch.float64) for x in (tables, lens, refs)]
    return (whole[0], whole[2], pool) if c["op"] == "compact" else (*whole, pool)
