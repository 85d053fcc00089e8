"""The guide's example of a step over an 8-bit cache, run as it is printed with
stand-ins for the operators: each layer fills and reads its own cache, and the
drafts' test sees the step's rows."""

from pathlib import Path
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parent.parent


def example():
    found = [block.split("```")[0] for path in ROOT.glob("*.md") for block in path.read_text().split("```python\n")[1:]]
    found = [code for code in found if "qk_norm_rope_kv8(" in code]
    assert len(found) == 1
    return found[0]


def test_the_example_gives_each_layer_its_own_cache(monkeypatch):
    from cheetah_b200 import runtime as R
    slots = R.PageSlots(**{name: torch.zeros(2, dtype=torch.int32) for name in R.PageSlots._fields})
    written, read, tested = [], [], []

    def append(qkv, q_heads, kv_heads, positions, slots, rope_cos, rope_sin, k_codes, v_codes, k_scales, v_scales, q_norm=None,
               k_norm=None, eps=1e-6, q_out=None, stream=None):
        written.append((k_codes, v_codes, k_scales, v_scales))
        return qkv

    def attend(q, k_codes, v_codes, k_scales, v_scales, page_table, seq_lens, row_starts, sliding_window=0, sinks=0, out=None,
               workspace=None, stream=None):
        read.append((k_codes, v_codes, k_scales, v_scales))
        assert (sliding_window, sinks) == (64, 4) and seq_lens is slots.seq_lens and row_starts is slots.row_starts
        return q

    def verify(target_probs, draft_probs, tokens, row_starts, accept_u, sample_u):
        tested.append(row_starts)
        return R.DraftVerdict(accept_u, tokens)

    for name, fake in dict(page_slots=lambda *a: slots, qk_norm_rope_kv8=append, attention_kv8=attend, verify_drafts=verify).items():
        monkeypatch.setattr(R, name, fake)
    layers = [SimpleNamespace(qkv=lambda x: x, rest=lambda x, o: x, q_norm=None, k_norm=None,
                              cache=SimpleNamespace(k_codes=object(), v_codes=object(), k_scales=object(), v_scales=object()))
              for _ in range(3)]
    names = ("cached new_tokens free_pages free_count page_table num_pages page_tokens max_tokens x q_heads kv_heads rope_cos rope_sin "
             "target_probs draft_probs tokens accept_u sample_u").split()
    exec(example(), dict({n: None for n in names}, layers=layers, window=64, sinks=4))
    assert written == read == [(c.k_codes, c.v_codes, c.k_scales, c.v_scales) for c in (layer.cache for layer in layers)]
    assert len(tested) == 1 and tested[0] is slots.row_starts
