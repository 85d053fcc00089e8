"""How the softmax weights of the 8-bit cache's attention are split, on the CPU:
the parts' bound, and what the tolerance of its tests tells apart."""

import math

import pytest

from tests import kv8_peaked_ref as VP
from tests import kv8_ref as V8

torch = pytest.importorskip("torch")


def test_split_of_every_size():
    """Weights from 0 to e5m2's largest: off by a part of themselves or by half a smallest step."""
    g = torch.Generator().manual_seed(1)
    w = torch.exp2(torch.rand(400000, generator=g) * 45 - 30 + 0.79).float()
    w = torch.cat([w, torch.zeros(1), torch.exp2(torch.arange(-30, 16).float()), torch.tensor([57343.0])])
    err = (VP.split_weights(w) - w.double()).abs()
    assert bool((err <= w.double() * VP.WEIGHT_STEP + 2.0 ** -17 + 2.0 ** -25).all())
    normal = w >= 2.0 ** -7  # nothing of nine bits falls below the smallest step
    assert bool((err[normal] <= w[normal].double() * VP.WEIGHT_STEP).all())


def emulate(q, k, v_codes, v_scales, split, top, room):
    """Rows of one head as the kernels multiply them: one reference per row, which moves
    where a weight would leave the split's range (q and k exact)."""
    t = q @ k.T / math.sqrt(q.shape[1]) * math.log2(math.e) + torch.log2(v_scales)
    o, l, m = torch.zeros(q.shape[0], v_codes.shape[1], dtype=torch.float64), torch.zeros(q.shape[0], 1, dtype=torch.float64), None
    for j in range(0, k.shape[0], 128):
        most = t[:, j:j + 128].amax(1, keepdim=True)
        new = torch.ceil(most) if m is None else torch.where(most > m + room, torch.ceil(most), m)
        f = 0.0 if m is None else torch.exp2(m - new)
        w = torch.exp2(t[:, j:j + 128] - new + top).float()
        o = o * f + split(w) @ v_codes[j:j + 128]
        l = l * f + (w.double() / v_scales[j:j + 128]).sum(1, keepdim=True)
        m = new
    return o / l


def two_parts(w):
    """The split into two e4m3 parts that end at the same smallest step."""
    x = w.to(torch.float16).float()
    hi = x.to(torch.float8_e4m3fn).float()
    return hi.double() + (x - hi).to(torch.float8_e4m3fn).double()


@pytest.mark.parametrize("weight", [0.5, 0.9, 0.97])
@pytest.mark.parametrize("keys", [4096, 32768])
def test_the_tolerance_tells_a_lost_tail(keys, weight):
    """A heavy key over a flat tail: three e5m2 parts keep within the tolerance of the
    GPU's tests, two e4m3 parts lose the tail and do not."""
    g = torch.Generator().manual_seed(keys)
    D = 64
    u = torch.sign(torch.randn(D, generator=g)).double()
    q = (2.0 * u)[None]
    k = torch.zeros(keys, D, dtype=torch.float64)
    k[0] = u * math.log(weight / (1 - weight) * keys) / (2.0 * math.sqrt(D))
    scale = torch.full((keys,), 2.0 ** -7, dtype=torch.float64)
    codes = V8.decode(V8.nearest_code((0.5 + torch.randn(keys, D, generator=g)).double() / scale[:, None]))
    o, tol = VP.attend(q, k, codes * scale[:, None], codes, scale, torch.ones(1, keys, dtype=torch.bool))
    assert bool(((emulate(q, k, codes, scale, VP.split_weights, 13, 2.75) - o).abs() <= tol).all())
    if weight > 0.5:  # (at 0.5 the tail's weights are powers of two, of which e4m3 holds these)
        assert not bool(((emulate(q, k, codes, scale, two_parts, 6, 2.75) - o).abs() <= tol).all())
