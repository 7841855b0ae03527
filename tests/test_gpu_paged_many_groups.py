"""Hundreds and thousands of sequences in groups, long ones among them, whose own keys are shared out evenly or
cut into parts of one length (bounds as in test_gpu_paged_sinks_prefixes)."""
import pytest
import torch

from tests.test_gpu_paged_sinks_prefixes import check, share

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("use_starts", [True, False])
@pytest.mark.parametrize("kw", [dict(), dict(window=2500, sinks=40), dict(causal=False)])
def test_long_sequences_among_many(use_starts, kw):
    """In a group with a long tail, in one of their own, in none, and in one that attends by itself."""
    g = torch.Generator().manual_seed(6)
    tails = [int(n) for n in torch.randint(1, 200, (270,), generator=g)]
    tails[77], tails[200] = 6000, 1500
    groups = [(300, [(n, 1) for n in tails]), (4000, [(900, 1)]), (3, [(5200, 1), (20, 1)])]
    x = share(23, groups, 8, 2, 64, 64, torch.bfloat16, before=[(5000, 1), (3, 1)], after=[(40, 1), (4700, 1)])
    last = len(tails) + 2
    check(x, use_starts=use_starts, rows={0, 1, 2, 78, 79, 80, 202, 203, last - 1, last, last + 1, last + 2, last + 3, last + 4},
          **kw)


def test_parts_of_several_tokens():
    """Sequences of two tokens, and without new ones, between the long ones."""
    groups = [(500, [(n % 90 + 2, 2 * (n % 3)) for n in range(260)] + [(5000, 2), (0, 0), (3000, 1)])]
    x = share(24, groups, 4, 1, 128, 128, torch.float16, after=[(6000, 2)])
    tokens = x["q"].shape[0]
    check(x, rows=set(range(0, tokens - 8, 37)) | set(range(tokens - 8, tokens)))


@pytest.mark.parametrize("kw", [dict(), dict(window=2500, sinks=40)])
def test_more_than_are_shared_out_evenly(kw):
    """Parts of one length, as without groups."""
    tails = [1 + 7 * n % 50 for n in range(2100)]
    tails[2000], tails[3] = 6000, 3500
    x = share(25, [(300, [(n, 1) for n in tails]), (4000, [(900, 1)])], 2, 1, 64, 64, torch.bfloat16, after=[(4700, 1), (9, 1)])
    check(x, use_starts=False, rows={0, 3, 4, 1500, 2000, 2001, 2099, 2100, 2101, 2102}, **kw)
    check(x, rows={3, 2000, 2100, 2101, 2102}, **kw)
