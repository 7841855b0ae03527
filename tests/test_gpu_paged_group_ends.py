"""Ends of groups: sequences that run in tiles and have ended inside the prefix they share, and calls whose
groups are not in order (bounds as in test_gpu_paged_sinks_prefixes)."""
import math

import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_sinks_prefixes import DEV, agree, check, definition, share

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window=700, sinks=90)])
@pytest.mark.parametrize("ps", [16, 128])
def test_tiles_that_ended_inside_the_prefix(kw, ps):
    """Long prefixes for the rows, so that the groups do share."""
    groups = [(9000, [(-8900, 60), (-64, 50), (-1, 40), (-4000, 33), (5, 1), (70, 40)]),
              (5003, [(-4939, 40), (-5003, 0), (-3, 30), (-1000, 64)])]
    x = share(ps, groups, 4, 1, 64, ps, torch.bfloat16, stale=math.nan)
    tokens = x["q"].shape[0]
    check(x, rows=set(range(0, tokens, 13)) | {59, 60, 109, 110, 149, 150, tokens - 1}, **kw)


def test_descending_groups_leave_what_is_outside_them():
    """What a sequence gets inside groups out of order is not defined; the sequences outside are as ever, and
    nothing around the outputs and the workspace is written."""
    x = share(11, [(100, [(5, 1), (9, 1)]), (200, [(4, 1), (8, 1), (30, 1)])], 4, 2, 64, 32, torch.bfloat16,
              before=[(70, 1)], after=[(300, 1)])
    d = {k: v.to(DEV) for k, v in x.items()}
    args = d["q"], d["ck"], d["cv"], d["tables"], d["kv"]
    seqs, hq, dim = x["q"].shape
    found = definition({k: v for k, v in x.items() if k not in ("groups", "prefix")})
    for groups in ([4, 2, 0], [6, 6, 1], [5, 3, 6], [7, 1, 0], [1 << 40, -5, -9]):
        d["groups"] = torch.tensor(groups, device=DEV)
        more = dict(prefix_groups=d["groups"], prefix_lens=d["prefix"])
        need = si.paged_attention_workspace(*args, **more)
        ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device=DEV)
        out = torch.full((seqs + 2, hq, dim), 3.0, dtype=torch.bfloat16, device=DEV)
        lse = torch.full((seqs + 2, hq), 3.0, dtype=torch.float32, device=DEV)
        caches = d["ck"].clone(), d["cv"].clone()
        si.paged_attention(*args, out=out[1:-1], lse=lse[1:-1], workspace=ws[2048:2048 + need], **more)
        inside = {b for lo, hi in zip(groups, groups[1:]) for b in range(max(lo, 0), max(min(hi, seqs), 0))}
        agree(out[1:-1], lse[1:-1], {b: v for b, v in found.items() if b not in inside})
        for t in (out, lse):
            assert (t[[0, -1]] == 3.0).all()
        assert (ws[:2048] == 0x5a).all() and (ws[2048 + need:] == 0x5a).all()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(caches, (d["ck"], d["cv"])))
