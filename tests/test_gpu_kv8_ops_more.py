"""The operators over an 8-bit cache on the GPU, at what `test_gpu_kv8_ops`
leaves out: ends of short segments, values that only a caller can have set, rows
whose softmax has one heavy key over a long tail."""

import math

import numpy as np
import pytest

from tests.test_gpu_kv8_ops import Attend, E4M3, _cuda, i32, to_gpu  # noqa: F401  (_cuda is the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("q_heads,kvh,D", [(7, 1, 128), (14, 2, 64), (16, 1, 128), (16, 1, 64)])
def test_attention_of_segments_whose_last_tile_moves_the_reference(q_heads, kvh, D):
    """A group's first tile of a segment sets its reference. With one to three tiles to
    a sequence every group's last tile does so too, and its maxima and the segment's sums
    come one after the other: many such segments, each time the same rows and right."""
    c = Attend(q_heads + D, [1 + 7 * i % 380 for i in range(300)], [1] * 300, q_heads, kvh, D, 64, q_scale=4.0)
    first = c.run()
    c.check(first, sample=range(0, 300, 9))
    for _ in range(20):
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("q_heads,kvh,D,rows", [(14, 2, 64, 2), (28, 4, 128, 2), (14, 2, 64, 12), (28, 4, 128, 16), (10, 2, 128, 37), (14, 2, 64, 200)])
@pytest.mark.parametrize("ctx", [30, 4000])
def test_attention_of_rows_beside_lanes_that_hold_none(q_heads, kvh, D, rows, ctx):
    """Items whose tile has lanes without a row, whole and cut, with a NaN in V that only
    some rows see: the lanes of a warp part between the loads of a result's columns."""
    c = Attend(rows + ctx, [ctx, ctx + 3], [rows, rows], q_heads, kvh, D, 64, extra_rows=1)
    base = c.run()
    c.check(base, sample=[0])
    group, at = q_heads // kvh, rows // 2
    for b in range(2):
        j = c.lens[b] - rows + at
        for d in (3, D - 2):
            c.v[0][c.table[b, j // 64], kvh - 1, j % 64, d] = 127
    got = c.run()
    hit = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for b in range(2):
        for d in (3, D - 2):
            hit[c.starts[b] + at:c.starts[b + 1], q_heads - group:, d] = True
    hit[c.starts[2]:] = torch.isnan(got[c.starts[2]:])  # rows behind the last sequence are not written
    assert bool(torch.isnan(got[hit]).all())
    assert torch.equal(got[:c.starts[2]][~hit[:c.starts[2]]], base[:c.starts[2]][~hit[:c.starts[2]]])
