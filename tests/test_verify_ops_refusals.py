"""Argument checks of the drafted-token operators, through the C-ABI on the
CPU: every refusal comes before any CUDA call, so the pointers here are never
read."""

import ctypes as C

import pytest

from cheetah_b200 import runtime as R

P = 0x10000  # stands for an aligned device pointer


def slots(**over):
    a = dict(cached=P, new_tokens=P, free_pages=P, free_count=P, free_capacity=4, batch=2, page_table=P,
             max_pages_per_seq=4, num_pages=8, page_tokens=16, max_tokens=32, row_starts=P, seq_lens=P, positions=P,
             seq_ids=P, slots=P, counts=P)
    return R.PageSlotsArgs(**{**a, **over}), "cheetah_cuda_op_page_slots"


def qk(**over):
    a = dict(qkv=P, qkv_stride=18 * 64, dtype=R.KV_BF16, kv_dtype=R.KV_BF16, q_norm=P, k_norm=P, eps=1e-6, rope_cos=P,
             rope_sin=P, max_positions=64, rotary_dim=64, positions=P, slots=P, tokens=3, q_heads=14, kv_heads=2,
             head_dim=64, q_out=P, k_pool=P, v_pool=P, num_pages=8, page_tokens=16)
    return R.QkNormRopeArgs(**{**a, **over}), "cheetah_cuda_op_qk_norm_rope"


def tree(**over):
    a = dict(q=P, q_stride=14 * 64, rows=5, k_pool=P, v_pool=P, page_table=P, max_pages_per_seq=4, num_pages=8,
             page_tokens=16, seq_lens=P, row_starts=P, batch=2, tree_mask=P, mask_words=1, positions=P,
             sliding_window=0, q_heads=14, kv_heads=2, head_dim=64, out=P, workspace=P, workspace_bytes=1 << 40)
    return R.TreeAttentionArgs(**{**a, **over}), "cheetah_cuda_op_tree_attention"


def logprobs(**over):
    a = dict(logits=P, row_stride=100, dtype=R.KV_F32, rows=3, vocab=100, tokens=P, top=2, logprob=P, rank=P,
             entropy=P, top_ids=P, top_logprobs=P)
    return R.TokenLogprobsArgs(**{**a, **over}), "cheetah_cuda_op_token_logprobs"


CASES = [
    (slots, dict(cached=None), "null"), (slots, dict(counts=None), "null"), (slots, dict(free_pages=None), "null free"),
    (slots, dict(batch=0), "batch"), (slots, dict(batch=16385), "batch"), (slots, dict(max_tokens=0), "max_tokens"),
    (slots, dict(max_tokens=1 << 31), "max_tokens"), (slots, dict(page_tokens=0), "pool"),
    (slots, dict(num_pages=1 << 28), "pool"), (slots, dict(max_pages_per_seq=0), "table"),
    (qk, dict(qkv=None), "null"), (qk, dict(slots=None), "null"), (qk, dict(dtype=7), "dtype"),
    (qk, dict(kv_dtype=-1), "dtype"), (qk, dict(head_dim=96), "head_dim"), (qk, dict(rotary_dim=24), "rotary_dim"),
    (qk, dict(rotary_dim=128), "rotary_dim"), (qk, dict(tokens=0), "empty"), (qk, dict(kv_heads=0), "head counts"),
    (qk, dict(qkv_stride=17 * 64), "overlap"), (qk, dict(qkv_stride=18 * 64 + 4), "aligned"),
    (qk, dict(qkv=P + 8), "aligned"), (qk, dict(q_norm=P + 4), "aligned"), (qk, dict(num_pages=0), "pool"),
    (tree, dict(q=None), "null"), (tree, dict(head_dim=80), "head_dim"), (tree, dict(q_heads=15), "multiple"),
    (tree, dict(q_heads=66, q_stride=66 * 64), "group"), (tree, dict(batch=0), "batch"), (tree, dict(rows=0), "rows"),
    (tree, dict(page_tokens=24), "page_tokens"), (tree, dict(mask_words=0), "mask_words"),
    (tree, dict(mask_words=17), "mask_words"), (tree, dict(sliding_window=8, positions=None), "positions"),
    (tree, dict(q_stride=13 * 64), "overlap"), (tree, dict(q_stride=14 * 64 + 4), "aligned"),
    (tree, dict(out=P + 8), "aligned"), (tree, dict(tree_mask=P + 4), "mask"), (tree, dict(num_pages=1 << 30), "pool"),
    (logprobs, dict(logits=None), "null"), (logprobs, dict(dtype=2), "dtype"), (logprobs, dict(rows=0), "empty"),
    (logprobs, dict(vocab=0), "empty"), (logprobs, dict(top=33), "top"), (logprobs, dict(vocab=1, top=2), "top"),
    (logprobs, dict(top_ids=None), "top_ids"), (logprobs, dict(row_stride=99), "overlap"),
    (logprobs, dict(logits=P + 2), "aligned"), (logprobs, dict(vocab=(1 << 30) + 1, row_stride=1 << 31), "2^30"),
    (tree, dict(max_pages_per_seq=(1 << 27) - 1), "table row"),
]


@pytest.mark.parametrize("make,over,message", CASES)
def test_bad_arguments_are_refused(make, over, message):
    args, name = make(**over)
    assert getattr(R.lib(), name)(C.byref(args), None) != 0
    assert message in R.lib().cheetah_cuda_last_error().decode()


def test_null_structs_are_refused():
    for name in ("page_slots", "qk_norm_rope", "tree_attention", "token_logprobs"):
        assert getattr(R.lib(), "cheetah_cuda_op_" + name)(None, None) != 0
        assert b"null" in R.lib().cheetah_cuda_last_error()
    assert R.lib().cheetah_cuda_op_tree_attention_workspace(None, None) != 0


def test_workspace_query_refuses_what_the_call_refuses():
    n = C.c_size_t(0)
    args, _ = tree(head_dim=80)
    assert R.lib().cheetah_cuda_op_tree_attention_workspace(C.byref(args), C.byref(n)) != 0
