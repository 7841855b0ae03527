"""Groups that share a prefix under a window, whose rows have given up the pages that
their own tokens no longer see: every sequence sees what its own row holds, against the
definition in 64 bits (bounds as in test_gpu_paged_sinks_prefixes)."""
import math

import pytest
import torch

from tests.test_gpu_paged_sinks_prefixes import check, share

pytestmark = pytest.mark.gpu


def give_up(x, window, sinks):
    """No page in a row's table that lies wholly between the sinks and the window of its next token."""
    ps = x["ck"].shape[1]
    starts = x["starts"].tolist()
    for b, n in enumerate(x["kv"].tolist()):
        seen_from = n - (starts[b + 1] - starts[b]) - window + 1
        for j in range(x["tables"].shape[1]):
            if j * ps >= sinks and (j + 1) * ps <= seen_from:
                x["tables"][b, j] = -1
    return x


@pytest.mark.parametrize("window,sinks,causal", [(300, 9, True), (300, 0, True), (64, 40, True), (500, 5, False), (1500, 3, True)])
@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("members", [
    [(3000, 1), (5, 1), (40, 1), (1, 1)],                   # the first, and longest, sees none of the prefix's end
    [(2000, 1), (1900, 2), (20, 3), (-200, 1), (-500, 2)],  # rows that have ended inside the prefix
    [(2500, 60), (45, 40), (-100, 20), (3, 1)],             # some that run in tiles
    [(100, 0), (90, 90), (3000, 0), (1, 1)],                # rows without new tokens
    [(-1, 1), (-300, 2), (-600, 1)]])                       # none as long as the prefix
def test_rows_hold_what_they_see(members, window, sinks, causal, dim, dtype):
    x = share(len(members) + dim + window, [(777, members), (300, [(700, 1), (2, 1)])], 4, 2, dim, 32, dtype,
              before=[(900, 3)], after=[(33, 1)], stale=math.nan)
    check(give_up(x, window, sinks), window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("use_starts", [True, False])
@pytest.mark.parametrize("members", [40, 150])
def test_many_rows(members, use_starts):
    """The row that holds the others' keys is far from the first; more than 64 sequences."""
    tails = [1000 + 7 * n for n in range(members)]
    tails[members - 2], tails[3], tails[members // 2] = 4, -170, 60
    x = give_up(share(members, [(640, [(n, 1) for n in tails])], 4, 2, 64, 32, torch.bfloat16), 200, 5)
    check(x, use_starts=use_starts, rows=set(range(0, members, 7)) | {3, members // 2, members - 2}, window=200, sinks=5)


def test_lengths_past_the_table():
    """Positions past the table move the window; the row with the first of them is the source."""
    x = share(77, [(400, [(100, 1), (112, 2), (90, 1)])], 4, 2, 64, 32, torch.bfloat16)
    x["tables"] = x["tables"][:, :16]
    x["kv"] = torch.tensor([800, 512, 490])
    check(give_up(x, 150, 4), window=150, sinks=4)
