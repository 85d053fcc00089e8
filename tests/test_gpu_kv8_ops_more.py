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
