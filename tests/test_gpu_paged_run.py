"""The operators on the paged cache as a server runs them together: prompts appended
with rotation and attended to, forked into samples that share them, and decoded, a token or
a few drafted ones a step, plain and under a window with sinks.  Every cache row is held against
the rotation in 64 bits, every output against attention in 64 bits over what the cache holds (the
bounds of the two operators' own tests)."""
import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_attention import DEV, rand
from tests.test_gpu_paged_rotation import frequencies, rotated
from tests.test_gpu_paged_sinks_prefixes import agree, definition

pytestmark = pytest.mark.gpu

PAGE, HQ, HEADS, DIM = 16, 6, 2, 64


class Run:
    def __init__(self, dtype, rows, slots, pages, window, sinks):
        self.dtype, self.kw = dtype, dict(window=window, sinks=sinks)
        self.ck, self.cv = (torch.zeros((slots, PAGE, HEADS, DIM), dtype=dtype, device=DEV) for _ in range(2))
        self.tables = torch.full((rows, pages), -1, dtype=torch.int64, device=DEV)
        self.kv = torch.zeros(rows, dtype=torch.int64, device=DEV)
        self.refs = torch.zeros(slots, dtype=torch.int32, device=DEV)
        self.fail = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.freqs = frequencies(DIM)
        self.g = torch.Generator().manual_seed(rows)

    def step(self, counts, groups=None, prefix=None):
        """counts[b] new tokens of row b; checked."""
        tokens = sum(counts)
        new = torch.tensor(counts, device=DEV)
        self.tables, self.kv, self.refs = si.reserve_pages(self.tables, self.kv, self.refs, new, PAGE, self.fail)
        starts = torch.tensor([0] + counts).cumsum(0)
        q, k, v = (rand(self.g, tokens, h, DIM, dtype=self.dtype) for h in (HQ, HEADS, HEADS))
        d = dict(q_starts=starts.to(DEV))
        turned = si.paged_append_rotated(k.to(DEV), v.to(DEV), self.ck, self.cv, self.tables, self.kv,
                                         self.freqs.to(DEV), q=q.to(DEV), fail_count=self.fail, **d)
        lse = torch.empty((tokens, HQ), device=DEV)
        out = si.paged_attention(turned, self.ck, self.cv, self.tables, self.kv, lse=lse, prefix_groups=groups,
                                 prefix_lens=prefix, **self.kw, **d)
        assert int(self.fail) == 0
        kv, tables = self.kv.tolist(), self.tables.cpu()
        where = [(b, kv[b] - n + i) for b, n in enumerate(counts) for i in range(n)]
        at = torch.tensor([p for _, p in where])
        ck, cv = self.ck.cpu(), self.cv.cpu()
        slot = torch.tensor([int(tables[b, p // PAGE]) for b, p in where])
        for x, got in ((k, ck[slot, at % PAGE]), (q, turned.cpu())):
            want, tol = rotated(x, at, self.freqs, False, 1.0)
            assert ((got.double() - want).abs() <= tol).all()
        assert torch.equal(cv[slot, at % PAGE], v)
        x = dict(q=turned.cpu(), ck=ck, cv=cv, tables=tables, kv=self.kv.cpu(), starts=starts)
        agree(out, lse, definition(x, **self.kw))  # every row's own pages: the shared ones are the same


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 4)])
def test_prompts_are_forked_and_decoded(dtype, window, sinks):
    prompts, samples = [150, 33, 260], 4
    rows = len(prompts) * samples
    run = Run(dtype, rows, 150, 24, window, sinks)
    first = [0] * rows
    for i, n in enumerate(prompts):
        first[i * samples] = n
    run.step(first)
    pairs = [(i * samples, i * samples + j) for i in range(len(prompts)) for j in range(1, samples)]
    run.tables, run.kv, run.refs = si.fork_pages([run.ck, run.cv], run.tables, run.kv, run.refs,
                                                 torch.tensor(pairs, device=DEV), run.fail)
    groups = torch.arange(0, rows + 1, samples, device=DEV)
    prefix = torch.tensor([n // PAGE * PAGE for n in prompts], device=DEV)
    for i in range(6):
        run.step([1] * rows if i % 2 == 0 else [1 + (b + i) % 4 for b in range(rows)], groups, prefix)
    # one prompt's samples end but for one: a group of one sequence
    ended = torch.tensor([1, 2, 3], device=DEV)
    run.tables, run.kv, run.refs = si.free_pages([run.ck, run.cv], run.tables, run.kv, run.refs, ended, fail_count=run.fail)
    run.tables, run.refs = si.compact_pages([run.ck, run.cv], run.tables, run.refs)
    left = [1, 0, 0, 0] + [1] * (rows - 4)
    run.step(left, groups, prefix)
    run.step(left, groups, torch.zeros_like(prefix))


def test_decode_steps_in_a_graph():
    """Append with rotation, then attention of the groups, replayed over growing sequences beside eager steps."""
    rows, width, prefix, samples = 8, 20, 96, 4
    slots = 2 * prefix // PAGE + rows * 8
    g = torch.Generator(device=DEV).manual_seed(1)
    ck, cv = (torch.randn((slots, PAGE, HEADS, DIM), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    tables = torch.full((rows, width), -1, dtype=torch.int64)
    for b in range(rows):
        tables[b, :6] = torch.arange(6) + 6 * (b // samples)
        tables[b, 6:14] = 12 + torch.arange(8) + 8 * b
    tables = tables.to(DEV)
    kv = torch.full((rows,), prefix, device=DEV) + torch.arange(rows, device=DEV)
    freqs = frequencies(DIM).to(DEV)
    q, k, v = (torch.zeros((rows, h, DIM), dtype=torch.bfloat16, device=DEV) for h in (HQ, HEADS, HEADS))
    groups, lens = torch.arange(0, rows + 1, samples, device=DEV), torch.full((2,), prefix, device=DEV)

    def step():
        turned = si.paged_append_rotated(k, v, ck, cv, tables, kv, freqs, q=q)
        return (turned, si.paged_attention(turned, ck, cv, tables, kv, prefix_groups=groups, prefix_lens=lens),
                si.paged_attention(turned, ck, cv, tables, kv, window=40, sinks=4, prefix_groups=groups, prefix_lens=lens),
                si.paged_attention(turned, ck, cv, tables, kv, window=40, sinks=4))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for x in (q, k, v):
            x.normal_()
        kv += 1 + i
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*out, ck, cv)]
        for a, b in zip(got, (*step(), ck, cv)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once():
    """Two batches over one cache, each with its own workspace, in flight together."""
    run = Run(torch.bfloat16, 6, 120, 24, 0, 0)
    run.step([120, 0, 0, 200, 0, 0])
    run.tables, run.kv, run.refs = si.fork_pages([run.ck, run.cv], run.tables, run.kv, run.refs,
                                                 torch.tensor([(0, 1), (0, 2), (3, 4), (3, 5)], device=DEV), run.fail)
    q = torch.randn((6, HQ, DIM), device=DEV).to(torch.bfloat16)
    halves = []
    for a in (0, 3):
        rows = slice(a, a + 3)
        halves.append(dict(q=q[rows], cache_k=run.ck, cache_v=run.cv, tables=run.tables[rows], kv_lens=run.kv[rows].clone(),
                           prefix_groups=torch.tensor([0, 3], device=DEV),
                           prefix_lens=torch.tensor([112 if a == 0 else 192], device=DEV)))
    want = [si.paged_attention(**h) for h in halves]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in halves]
    for _ in range(5):
        got = [si.paged_attention(**h, stream=s) for h, s in zip(halves, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
