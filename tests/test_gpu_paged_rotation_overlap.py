"""Where paged_append_rotated's rotated queries may go: anywhere that shares no memory with an input, or into q."""
import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_attention import DEV
from tests.test_gpu_paged_rotation import batch, frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1], [20, 3]])
def test_into_rows_beside_the_inputs(new):
    """A fused buffer with room for the rotated queries."""
    hq, heads, dim = 6, 2, 64
    x = batch(61, [300, 77], new, hq, heads, dim, 32, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    f = frequencies(dim).to(DEV)
    more = dict(freqs=f, q_starts=d["starts"])
    want = si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], q=d["q"], **more)
    fused = torch.cat([d["q"], d["k"], d["v"], torch.zeros_like(d["q"])], 1)
    kept = fused[:, :hq + 2 * heads].clone()
    q, k, v, out = fused.split([hq, heads, heads, hq], 1)
    got = si.paged_append_rotated(k, v, d["ck"], d["cv"], d["tables"], d["kv"], q=q, q_out=out, **more)
    assert got is out and torch.equal(out, want) and torch.equal(fused[:, :hq + 2 * heads], kept)


def test_queries_that_share_memory_with_k_or_v_do_not_turn_in_place():
    x = batch(62, [30, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    f = frequencies(64).to(DEV)
    fused = torch.cat([d["q"], d["k"], d["v"]], 1)
    kept, caches = fused.clone(), (d["ck"].clone(), d["cv"].clone())
    q, k, v = fused.split([4, 2, 2], 1)
    for name, change in (("k", dict(k=fused[:, :2])), ("k", dict(k=fused[:, 3:5])), ("v", dict(v=fused[:, 2:4])),
                         ("k", dict(q=fused[:, 4:6], q_out=fused[:, 4:6]))):
        with pytest.raises(ValueError, match=f"not overlap {name}"):
            si.paged_append_rotated(**{**dict(k=k, v=v, cache_k=d["ck"], cache_v=d["cv"], tables=d["tables"],
                                              kv_lens=d["kv"], freqs=f, q=q, q_out=q), **change})
    torch.cuda.synchronize()
    assert torch.equal(fused, kept)
    # (NaN where the caches hold nothing)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip((d["ck"], d["cv"]), caches))
