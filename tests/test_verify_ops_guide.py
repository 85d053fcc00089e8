"""The guide's example of a step that verifies drafted tokens, run as it is
printed with stand-ins for the four operators: the positions of a tree's nodes
are absolute, and each layer fills and reads its own pools."""

from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest

from tests import verify_ref as V

torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parent.parent


def example():
    found = []
    for path in ROOT.glob("*.md"):
        for block in path.read_text().split("```python\n")[1:]:
            code = block.split("```")[0]
            if "page_slots(" in code and "tree_attention(" in code:
                found.append(code)
    assert len(found) == 1
    return found[0]


def test_the_example_gives_nodes_absolute_positions_and_layers_their_own_pools(monkeypatch):
    from cheetah_b200 import runtime as R
    ctx, nodes, page_tokens, rows = [40, 7, 30], [4, 3, 5], 16, 16
    trees = [[-1, 0, 0, 2], [-1, 0, 1], [-1, -1, 0, 2, 1]]
    depth = np.concatenate([V.tree_bits(t)[1] for t in trees])
    # The last sequence finds no page.
    want = V.page_slots(ctx, nodes, [], 0, np.full((3, 4), 9), 10, page_tokens, rows)
    assert want["counts"][2] == 1

    def i32(values):
        return torch.tensor(np.asarray(values), dtype=torch.int32)

    def page_slots(cached, new_tokens, free_pages, free_count, page_table, num_pages, pt, max_tokens):
        return R.PageSlots(**{name: i32(want[name]) for name in R.PageSlots._fields})

    appended, read = [], []

    def qk_norm_rope(qkv, q_heads, kv_heads, positions, slots, cos, sin, k_pool, v_pool, q_norm=None, k_norm=None):
        appended.append((positions, slots, k_pool, v_pool))
        return qkv

    def tree_attention(q, k_pool, v_pool, page_table, seq_lens, row_starts, tree_mask, positions=None, sliding_window=0):
        read.append((k_pool, v_pool, positions, sliding_window))
        return q

    for name, fake in dict(page_slots=page_slots, qk_norm_rope=qk_norm_rope, tree_attention=tree_attention,
                           token_logprobs=lambda logits, tokens, top=0: None).items():
        monkeypatch.setattr(R, name, fake)
    layers = [SimpleNamespace(qkv=lambda x: x, rest=lambda x, o: x, k_pool=object(), v_pool=object(), q_norm=None, k_norm=None)
              for _ in range(3)]
    exec(example(), dict(
        torch=torch, layers=layers, x=None, logits=None, tokens=None, q_heads=4, kv_heads=2, cached=i32(ctx), new_tokens=i32(nodes),
        free_pages=i32([]), free_count=i32([0]), page_table=None, num_pages=10, page_tokens=page_tokens, max_tokens=rows,
        depth=i32(np.concatenate([depth, np.zeros(rows - len(depth))])), rope_cos=None, rope_sin=None, tree_mask=None, qkv=None,
        k_pool=object(), v_pool=object(), q_norm=None, k_norm=None))
    absolute = [c + d for c, t in zip(ctx, trees) for d in V.tree_bits(t)[1]]
    absolute = absolute[:7] + [-1] * (rows - 7)  # refused and padding rows are skipped
    assert len(appended) == len(read) == 3
    for layer, (positions, slots, k_pool, v_pool), (k_read, v_read, seen, window) in zip(layers, appended, read):
        assert positions.dtype == torch.int32 and positions.tolist() == absolute
        assert slots.tolist() == want["slots"]
        assert k_pool is k_read is layer.k_pool and v_pool is v_read is layer.v_pool
        assert window == 0 or seen is positions
