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
