"""Tree attention on the GPU where a tile of rows has lanes that hold none."""

import pytest

from tests.test_gpu_verify_ops import Tree, _cuda  # noqa: F401  (_cuda is the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("q_heads,kv_heads,D", [(14, 2, 64), (28, 4, 128), (10, 2, 128)])
@pytest.mark.parametrize("ctx,nodes", [([5000], [3]), ([9000, 40], [12, 5]), ([3000], [30])])
def test_tree_attention_cut_items_of_rows_beside_lanes_that_hold_none(ctx, nodes, q_heads, kv_heads, D):
    """Items that several CTAs share, of fewer rows than lanes: the lanes of a warp part
    at the stores of a part's columns, between its loads. Each time the same rows, and right."""
    case = Tree(ctx, nodes, q_heads, kv_heads, D, seed=ctx[0] + nodes[0], extra_rows=1)
    first = case.run()
    case.check(first)
    total = int(case.starts[-1])
    for _ in range(5):
        assert torch.equal(case.run()[:total], first[:total])
