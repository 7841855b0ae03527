"""Whether rows of two strided tensors share memory (secure_infer_amd.paged._meet), without a GPU: against
the sets of their elements."""
import random

import pytest
import torch

from secure_infer_amd.paged import _meet


def elements(at, token, head, heads, tokens, dim):
    return {at // 2 + t * token + h * head + d for t in range(tokens) for h in range(heads) for d in range(dim)}


def met(a, b, tokens, dim):
    return bool(elements(*a, tokens, dim) & elements(*b, tokens, dim))


def rows(t):
    return t.data_ptr(), t.stride(0), t.stride(1), t.shape[1]


def test_random_rows():
    """Exact where the token strides are one; otherwise never an overlap missed."""
    g = random.Random(7)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        dim, tokens = 8 * g.randint(1, 3), g.randint(1, 5)
        token = 8 * g.randint(1, 40)
        a = (1 << 20, token, 8 * g.randint(0, 20), g.randint(1, 4))
        other = token if g.random() < 0.8 else 8 * g.randint(0, 40)
        b = ((1 << 20) + 16 * g.randint(-60, 60), other, a[2] if g.random() < 0.4 else 8 * g.randint(0, 20), g.randint(1, 4))
        want, got = met(a, b, tokens, dim), _meet(a, b, tokens, dim)
        assert got == want if other == token or tokens == 1 else got or not want, (a, b, tokens, dim)
        assert _meet(b, a, tokens, dim) == got
        seen[want] += 1
    assert min(seen.values()) > 1000


@pytest.mark.parametrize("tokens", [1, 2, 300])
def test_fused_projections(tokens):
    """q, k and v out of one buffer do not overlap, in any of its usual orders; shifted ones do."""
    hq, h, dim = 8, 2, 64
    fused = torch.empty((tokens, hq + 2 * h, dim), dtype=torch.bfloat16)
    of_heads = torch.empty((hq + 2 * h, tokens, dim), dtype=torch.bfloat16).transpose(0, 1)
    for x in (fused, of_heads):
        q, k, v = x.split([hq, h, h], 1)
        assert not _meet(rows(q), rows(k), tokens, dim) and not _meet(rows(v), rows(q), tokens, dim)
        assert _meet(rows(q), rows(x[:, hq - 1:hq + 1]), tokens, dim) and _meet(rows(q), rows(q), tokens, dim)
    three = torch.empty((tokens, hq, 3, dim), dtype=torch.bfloat16)
    q, k, v = three.unbind(2)
    assert not _meet(rows(q), rows(k), tokens, dim) and not _meet(rows(q), rows(v), tokens, dim)
    assert _meet(rows(q), rows(three[:, 2:4, 0]), tokens, dim)
    heads = torch.empty((hq, 3, tokens, dim), dtype=torch.bfloat16)
    q, k, v = (t.transpose(0, 1) for t in heads.unbind(1))
    assert not _meet(rows(q), rows(k), tokens, dim) and not _meet(rows(v), rows(q), tokens, dim)
    assert _meet(rows(q), rows(heads[1:3, 0].transpose(0, 1)), tokens, dim)
