"""fork_pages, free_pages, compact_pages and reserve_pages against their rules
in plain Python.  Everything is whole numbers or copied bytes: exact."""
import random

import pytest
import torch

import secure_infer_amd as si

pytestmark = pytest.mark.gpu

DEV = "cuda"


def make(seed, slots, rows, width, ps=16, tensors=3, hkv=2, dim=8, held=0.5, share=0.3):
    """A batch of random rows; some share pages with a row before them."""
    r = random.Random(seed)
    order = list(range(slots))
    r.shuffle(order)
    budget = int(slots * held)
    tables, lens, refs = [], [], [0] * slots
    for b in range(rows):
        row = []
        if b and r.random() < share:
            row = list(tables[r.randrange(b)])
            row = [e for e in row if e >= 0][:r.randint(0, width)]
        want = r.randint(0, width)
        while len(row) < want and budget > 0:
            row.append(order[budget - 1])
            budget -= 1
        for e in row:
            refs[e] += 1
        lens.append(max(0, len(row) * ps - r.choice([0, 1, ps - 1, r.randint(0, ps - 1)])) if row else 0)
        tables.append(row + [-1] * (width - len(row)))
    g = torch.Generator().manual_seed(seed)
    caches = [torch.randn((slots, ps, hkv, dim), generator=g).to(torch.bfloat16) for _ in range(tensors)]
    return dict(tables=tables, lens=lens, refs=refs, caches=caches, ps=ps, slots=slots, width=width)


def held(e, x):
    return 0 <= e < x["slots"]


def py_fork(x, pairs):
    T, L, R = [list(t) for t in x["tables"]], list(x["lens"]), list(x["refs"])
    C, ps, fails = [c.clone() for c in x["caches"]], x["ps"], 0
    free = [s for s in range(x["slots"]) if x["refs"][s] <= 0]
    named = set()
    for p, c in pairs:
        ok = 0 <= p < len(T) and 0 <= c < len(T) and c not in named
        if 0 <= p < len(T) and 0 <= c < len(T):
            named.add(c)
        if not ok or x["lens"][c] != 0 or any(held(e, x) for e in x["tables"][c]):
            fails += 1
            continue
        n = max(0, min(x["lens"][p], x["width"] * ps))
        row = [-1] * x["width"]
        whole = n // ps
        if n % ps and held(x["tables"][p][whole], x):
            if not free:
                fails += 1
                continue
            s = free.pop(0)
            for c_ in C:
                c_[s] = x_cache(x, c_, C)[x["tables"][p][whole]]
            row[whole] = s
            R[s] = 1
        for j in range(whole):
            row[j] = x["tables"][p][j]
            if held(row[j], x):
                R[row[j]] += 1
        T[c], L[c] = row, n
    return T, L, R, C, fails


def x_cache(x, c, C):
    return x["caches"][[c is y for y in C].index(True)]


def py_free(x, rows, scrub):
    T, L, R = [list(t) for t in x["tables"]], list(x["lens"]), list(x["refs"])
    C = [c.clone() for c in x["caches"]]
    fails = sum(not 0 <= b < len(T) for b in rows)
    gone = [0] * x["slots"]
    for b in {b for b in rows if 0 <= b < len(T)}:
        for e in T[b]:
            if held(e, x):
                gone[e] += 1
        T[b], L[b] = [-1] * x["width"], 0
    for s in range(x["slots"]):
        if not gone[s]:
            continue
        hold = max(0, R[s])
        fails += max(0, gone[s] - hold)
        R[s] = max(0, hold - gone[s])
        if hold and R[s] == 0 and scrub:
            for c in C:
                c[s] = 0
    return T, L, R, C, fails


def py_compact(x, scrub):
    R = list(x["refs"])
    live = [s for s in range(x["slots"]) if R[s] > 0]
    move = dict(zip([s for s in live if s >= len(live)], [s for s in range(len(live)) if R[s] <= 0]))
    C = [c.clone() for c in x["caches"]]
    for a, b in move.items():
        R[a], R[b] = 0, R[a]
        for c, o in zip(C, x["caches"]):
            c[b] = o[a]
    if scrub:
        for a in move:
            for c in C:
                c[a] = 0
    return [[move.get(e, e) for e in t] for t in x["tables"]], R, C


def py_reserve(x, counts):
    T, L, R = [list(t) for t in x["tables"]], list(x["lens"]), list(x["refs"])
    free = [s for s in range(x["slots"]) if R[s] <= 0]
    before = fails = 0
    for b, add in enumerate(counts):
        L[b] += max(0, add)
        if L[b] > x["width"] * x["ps"]:
            fails += 1
            continue
        lacks = [j for j in range(-(-L[b] // x["ps"])) if not held(T[b][j], x)]
        if before + len(lacks) > len(free):
            fails += 1
        else:
            for k, j in enumerate(lacks):
                T[b][j] = free[before + k]
                R[free[before + k]] = 1
        before += len(lacks)
    return T, L, R, fails


def on_device(x):
    return ([c.to(DEV) for c in x["caches"]], torch.tensor(x["tables"], device=DEV), torch.tensor(x["lens"], device=DEV),
            torch.tensor(x["refs"], dtype=torch.int32, device=DEV))


def counter():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def same(got, want):
    for g, w in zip(got, want):
        assert g.cpu().tolist() == w


def same_caches(caches, want):
    for g, w in zip(caches, want):
        assert torch.equal(g.cpu().view(torch.int16), w.view(torch.int16))


SHAPES = [(1, 6, 4), (40, 9, 5), (64, 30, 7), (700, 40, 70), (3001, 130, 40)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed,shape", list(enumerate(SHAPES)))
def test_fork(seed, shape, in_place):
    x = make(seed, *shape)
    r = random.Random(seed)
    rows = len(x["lens"])
    for b in r.sample(range(rows), rows // 2):  # empty rows to fork into
        for e in x["tables"][b]:
            if e >= 0:
                x["refs"][e] -= 1
        x["tables"][b], x["lens"][b] = [-1] * x["width"], 0
    empty = [b for b in range(rows) if x["lens"][b] == 0]
    pairs = [(r.randrange(rows), c) for c in r.sample(empty, len(empty))]
    pairs += [(r.randrange(-2, rows + 2), r.randrange(-2, rows + 2)) for _ in range(5)]
    r.shuffle(pairs)
    want = py_fork(x, pairs)
    caches, *state = on_device(x)
    fail = counter()
    got = si.fork_pages(caches, *state, torch.tensor(pairs, device=DEV), fail_count=fail,
                        out=tuple(state) if in_place else None)
    same(got, want[:3])
    same_caches(caches, want[3])
    assert int(fail) == want[4]


def test_fork_when_the_slots_run_out():
    x = make(5, 12, 3, 4, held=0.0, share=0.0)
    x["tables"][0] = [7, 2, -1, -1]
    x["lens"][0] = 17
    x["refs"] = [1] * 12
    x["refs"][9] = x["refs"][4] = 0
    x["tables"] += [[-1] * 4 for _ in range(4)]
    x["lens"] += [0] * 4
    pairs = [(0, 6), (0, 3), (0, 4), (0, 5)]  # two free slots: 6 gets slot 4, 3 gets 9
    want = py_fork(x, pairs)
    assert want[0][6] == [7, 4, -1, -1] and want[0][3] == [7, 9, -1, -1] and want[4] == 2 and want[1][4] == 0
    caches, *state = on_device(x)
    fail = counter()
    got = si.fork_pages(caches, *state, torch.tensor(pairs, device=DEV), fail_count=fail)
    same(got, want[:3])
    same_caches(caches, want[3])
    assert int(fail) == 2


def test_fork_over_missing_pages_and_of_nothing():
    x = make(6, 12, 2, 4, held=0.0, share=0.0)
    x["tables"] = [[3, -1, 99, 5], [-1] * 4, [-1] * 4, [-1] * 4]
    x["lens"] = [40, 0, 0, 0]  # pages 0, 1 whole, page 2 partial and missing
    x["refs"][3] = x["refs"][5] = 1
    for pairs in ([(0, 1), (1, 2)], []):
        want = py_fork(x, pairs)
        caches, *state = on_device(x)
        got = si.fork_pages(caches, *state, torch.tensor(pairs, dtype=torch.int64, device=DEV).reshape(-1, 2))
        same(got, want[:3])
        same_caches(caches, want[3])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("scrub", [False, True])
@pytest.mark.parametrize("seed,shape", list(enumerate(SHAPES)))
def test_free(seed, shape, scrub, in_place):
    x = make(seed + 50, *shape)
    r = random.Random(seed)
    n = len(x["lens"])
    rows = [r.randrange(n) for _ in range(n // 2)] + [-1, n, 1 << 40]
    want = py_free(x, rows, scrub)
    caches, *state = on_device(x)
    fail = counter()
    got = si.free_pages(caches, *state, torch.tensor(rows, device=DEV), scrub=scrub, fail_count=fail,
                        out=tuple(state) if in_place else None)
    same(got, want[:3])
    same_caches(caches, want[3])
    assert int(fail) == want[4] and want[4] == 3


def test_free_counts_holds_beyond_a_slots_count():
    x = make(60, 20, 3, 3, held=0.0, share=0.0)
    x["tables"] = [[4, 5, -1], [4, 6, 77], [4, 6, -1]]
    x["lens"] = [20, 20, 20]
    x["refs"][4], x["refs"][5], x["refs"][6] = 2, 1, 0
    want = py_free(x, [0, 1, 2], True)
    assert want[4] == 1 + 2
    caches, *state = on_device(x)
    fail = counter()
    got = si.free_pages(caches, *state, torch.tensor([0, 1, 2], device=DEV), fail_count=fail)
    same(got, want[:3])
    same_caches(caches, want[3])
    assert int(fail) == 3


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("scrub", [False, True])
@pytest.mark.parametrize("seed,shape", list(enumerate(SHAPES)))
def test_compact(seed, shape, scrub, in_place):
    x = make(seed + 80, *shape, tensors=5)
    want = py_compact(x, scrub)
    caches, tables, _, refs = on_device(x)
    got = si.compact_pages(caches, tables, refs, scrub=scrub, out=(tables, refs) if in_place else None)
    same(got, want[:2])
    same_caches(caches, want[2])


def test_compact_full_and_empty_caches():
    for refs in ([1, 2, 1], [0, 0, 0], [0, 0, 3]):
        x = make(90, 3, 2, 2, held=0.0)
        x["refs"], x["tables"] = refs, [[2, -1], [0, 5]]
        want = py_compact(x, True)
        caches, tables, _, r = on_device(x)
        same(si.compact_pages(caches, tables, r, scrub=True), want[:2])
        same_caches(caches, want[2])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed,shape", list(enumerate(SHAPES)))
def test_reserve(seed, shape, in_place):
    x = make(seed + 120, *shape)
    r = random.Random(seed)
    for counts in ([r.choice([0, 1, 1, x["ps"], r.randint(0, 5 * x["ps"]), -3]) for _ in x["lens"]],
                   [10 ** 9 if b == 1 else 40 for b in range(len(x["lens"]))]):
        want = py_reserve(x, counts)
        _, *state = on_device(x)
        fail = counter()
        got = si.reserve_pages(*state, torch.tensor(counts, device=DEV), x["ps"], fail_count=fail,
                               out=tuple(state) if in_place else None)
        same(got, want[:3])
        assert int(fail) == want[3]


def test_pages_of_many_tensors_and_odd_sizes():
    """More tensors than one launch takes, pages that are no multiple of a copy
    unit, page strides larger than a page, and pages over one copy unit."""
    for tensors, ps, hkv, dim, pad in ((300, 8, 1, 8, 0), (3, 128, 3, 72, 64), (2, 128, 8, 128, 0)):
        x = make(7, 24, 6, 4, ps=ps, tensors=tensors, hkv=hkv, dim=dim)
        page = ps * hkv * dim
        want = py_compact(x, True)
        _, tables, lens, refs = on_device(x)
        caches = []
        for c in x["caches"]:
            base = torch.full((24, page + pad), 5.0, dtype=torch.bfloat16, device=DEV)
            base[:, :page] = c.to(DEV).view(24, page)
            caches.append(torch.as_strided(base, c.shape, (page + pad, hkv * dim, dim, 1)))
        same(si.compact_pages(caches, tables, refs, scrub=True), want[:2])
        same_caches([c.contiguous() for c in caches], want[2])
        if pad:
            assert all((torch.as_strided(c, (24, pad), (page + pad, 1), page) == 5).all() for c in caches)


def test_on_another_stream_and_in_a_graph():
    x = make(33, 64, 12, 5)
    want = py_free(x, [1, 4], True)
    caches, *state = on_device(x)
    rows = torch.tensor([1, 4], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = si.free_pages(caches, *state, rows, stream=side)
    torch.cuda.synchronize()
    same(got, want[:3])
    same_caches(caches, want[3])
    g = torch.cuda.CUDAGraph()
    caches, *state = on_device(x)
    with torch.cuda.graph(g):
        got = si.free_pages(caches, *state, rows)
    for shift in range(3):
        for c, o in zip(caches, x["caches"]):
            c.copy_(o)
        rows.copy_(torch.tensor([1 + shift, 4], device=DEV))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = py_free(x, [1 + shift, 4], True)
        same(got, want[:3])
        same_caches(caches, want[3])


def test_a_cache_set_is_its_list():
    x = make(35, 64, 12, 5, tensors=6)
    rows = torch.tensor([1, 4, 7], device=DEV)
    caches, *state = on_device(x)
    kept = si.CacheSet(caches)
    freed = si.free_pages(kept, *state, rows)
    want = py_free(x, [1, 4, 7], True)
    same(freed, want[:3])
    same_caches(caches, want[3])
    moved = si.compact_pages(kept, freed[0], freed[2])
    again = [c.to(DEV) for c in x["caches"]]
    freed2 = si.free_pages(again, *state, rows)
    moved2 = si.compact_pages(again, freed2[0], freed2[2])
    same(moved, [t.tolist() for t in moved2])
    same_caches(caches, [c.cpu() for c in again])
    for bad, what in (([], "no caches"), ([caches[0], caches[1].half()], "one shape"),
                      ([caches[0], caches[1][:5]], "one shape"), ([caches[0].cpu()], "device tensor")):
        with pytest.raises(ValueError, match=what):
            si.CacheSet(bad)
    with pytest.raises(ValueError, match="one entry per slot"):
        si.compact_pages(kept, state[0], state[2][:-1])


def test_reserve_bounds_its_lengths():
    x = make(36, 40, 5, 4, held=0.3)
    top = (1 << 63) - 1
    counts = [top, 1 << 62, 3, -top, 0]
    want = py_reserve(x, counts)
    lens = [min(n, top) for n in want[1]]
    _, *state = on_device(x)
    fail = counter()
    got = si.reserve_pages(*state, torch.tensor(counts, device=DEV), x["ps"], fail_count=fail)
    same(got, (want[0], lens, want[2]))
    assert int(fail) == want[3] >= 2


def test_a_cache_given_twice_is_refused():
    x = make(37, 8, 2, 2, tensors=2)
    caches, tables, _, refs = on_device(x)
    twice = [caches[0], caches[1], caches[0]]
    for call in (lambda: si.CacheSet(twice), lambda: si.compact_pages(twice, tables, refs)):
        with pytest.raises(ValueError, match="twice"):
            call()
    same_caches(caches, x["caches"])
