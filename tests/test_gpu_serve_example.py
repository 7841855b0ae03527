"""The serving example end to end: every attention output against dense
attention in 64 bits over the tokens the sequence really has (the stored
prefix, its own appended tokens, a fork's parent's), pages of ended samples
cleared, and the pages written back equal to the history."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def load():
    spec = importlib.util.spec_from_file_location("serve_prefix", ROOT / "examples" / "serve_prefix.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("prefix,samples", [(300, 2), (256, 1), (127, 0)])
def test_served_outputs_and_pages(prefix, samples):
    m = load()
    layers, heads, dim = 2, 2, 64
    srv, log, stored, back = m.serve(layers=layers, q_heads=6, heads=heads, dim=dim, prefix=prefix, chunk=45,
                                     samples=samples, steps=4, seed=prefix)
    hist = {}
    for layer, (k, v) in enumerate(stored):
        hist[layer, 0] = [k.flatten(0, 1)[:prefix].double(), v.flatten(0, 1)[:prefix].double()]
    u = 2.0 ** -8
    for entry in log:
        if entry[0] == "fork":
            for layer in range(layers):
                for c in entry[2]:
                    hist[layer, c] = list(hist[layer, entry[1]])
            continue
        layer, row, k, v, q, out = [x.cpu().double() if isinstance(x, torch.Tensor) else x for x in entry]
        h = hist[layer, row]
        h[0], h[1] = torch.cat([h[0], k]), torch.cat([h[1], v])
        n, new = h[0].shape[0], q.shape[0]
        for i in range(new):
            for head in range(6):
                kk, vv = h[0][:n - new + i + 1, head // 3], h[1][:n - new + i + 1, head // 3]
                w = torch.softmax(kk @ q[i, head] / math.sqrt(dim), 0)
                want = w @ vv
                # one rounding of the weights and one of the output to bf16,
                # and the float scores' and sums' (under 2^-13 of the weighted values)
                tol = u * want.abs() + (u + 2.0 ** -13) * (w @ vv.abs())
                assert ((out[i, head] - want).abs() <= tol).all(), (layer, row, i, head)
    # written back: sequence 0's history, page by page
    for layer in range(layers):
        for kind in range(2):
            want = hist[layer, 0][kind]
            got = back[layer][kind].flatten(0, 1)[:want.shape[0]].double()
            assert torch.equal(got, want)
    # compacted: the held slots are the lowest ones; free pages hold zeros
    refs = srv.refs.cpu()
    if samples:
        for c in srv.caches.caches:
            assert not c[refs.cuda() == 0].any()
