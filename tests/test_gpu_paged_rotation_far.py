"""paged_append_rotated at positions up to the ends of 64 bits, against angles reduced in whole numbers.

Bound on a rotated element y = m (a cos t - b sin t), u the unit roundoff of the 16-bit type: the fraction of
a turn is within 2^-29 (three roundings of at most 2^-53 2^(63 + 16 - 2.6 - 53) each) before it is rounded to float
(2^-26 of a turn at most; together below 2^-23.1 radians), the cosine and sine are within 2 units of 2^-24, the products and their sum round 2^-24 each, so every
coefficient is within 2^-20 m:
  |error| <= u |y| + 1.01 m (|a| + |b|) 2^-20 + 2^-25,
the last term for fp16 results below its normal range."""
import math

import pytest
import torch

import secure_infer_amd as si
from tests.test_gpu_paged_attention import DEV, ROUND
from tests.test_gpu_paged_rotation import KV, batch, frequencies

pytestmark = pytest.mark.gpu

# 2^200 / (2 pi), from pi to 75 digits
PI = 314159265358979323846264338327950288419716939937510582097494459230781640628
TURN = (10 ** 74 << 200) // (2 * PI)


def radians(p, f):
    """p * f without whole turns (p a whole number, f a float), from -pi to pi."""
    n, d = float(f).as_integer_ratio()
    x = p * n * TURN // d  # turns, in units of 2^-200
    x = (x + (1 << 199)) % (1 << 200) - (1 << 199)
    return x / (1 << 200) * 2 * math.pi


def rotated(x, positions, freqs, adjacent, magnitude):
    half, u = freqs.numel(), ROUND[x.dtype]
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    t = torch.tensor([[radians(int(p), f) for f in freqs.tolist()] for p in positions], dtype=torch.float64)[:, None, :]
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = magnitude * (a * torch.cos(t) - b * torch.sin(t))
    y[..., second] = magnitude * (b * torch.cos(t) + a * torch.sin(t))
    slack = 1.01 * abs(magnitude) * (a.abs() + b.abs()) * 2.0 ** -20 + 2.0 ** -25
    for d in (first, second):
        tol[..., d] = u * y[..., d].abs() + slack
    return y, tol


@pytest.mark.parametrize("at", [0, -500, (1 << 30) - 7, (1 << 32) - 500, -(1 << 32) - 500, 1 << 36, (1 << 40) + 12345, -(1 << 45),
                                (1 << 53) + 1, (1 << 62) + 987654321, (1 << 63) - 1001, -(1 << 63)])
@pytest.mark.parametrize("fast", [False, True])
def test_far_positions(at, fast):
    x = batch(at % 1000, KV, [5, 0, 70, 1, 33, 0, 20], 4, 2, 128, 32, torch.float16)
    g = torch.Generator().manual_seed(at & 0xffff)
    positions = torch.tensor([at + int(n) for n in torch.randint(0, 1000, (x["q"].shape[0],), generator=g)])
    freqs = frequencies(128, 500000.0)
    if fast:
        freqs = freqs * 65536
        freqs[::3] *= -1
    d = {n: t.to(DEV) for n, t in x.items()}
    for adjacent, magnitude in ((False, 1.0), (True, -1.5)):
        got = si.paged_append_rotated(d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], freqs.to(DEV), q=d["q"],
                                      q_starts=d["starts"], positions=positions.to(DEV), adjacent=adjacent,
                                      magnitude=magnitude).cpu().double()
        want, tol = rotated(x["q"], positions, freqs, adjacent, magnitude)
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("magnitude", [1e39, -1e300, 3.5e38, math.inf, math.nan])
def test_magnitudes_past_float_are_refused(magnitude):
    x = batch(63, [30, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    args = d["k"], d["v"], d["ck"], d["cv"], d["tables"], d["kv"], frequencies(64).to(DEV)
    with pytest.raises(ValueError, match="magnitude"):
        si.paged_append_rotated(*args, q=d["q"], magnitude=magnitude)
    with pytest.raises(ValueError, match="magnitude"):
        si.paged_append_rotated(*args, magnitude=magnitude)
    si.paged_append_rotated(*args, q=d["q"], magnitude=torch.finfo(torch.float32).max)
