"""Argument checks of the operators over an 8-bit cache, through the C-ABI on
the CPU: every refusal comes before any CUDA call, so the pointers here are
never read; and the references' own rules on small cases."""

import ctypes as C
import math

import numpy as np
import pytest

from cheetah_b200 import runtime as R
from tests import kv8_ref as V8

torch = pytest.importorskip("torch")

P = 0x10000  # stands for an aligned device pointer


def append(**over):
    a = dict(qkv=P, qkv_stride=18 * 64, dtype=R.KV_BF16, q_norm=P, k_norm=P, eps=1e-6, rope_cos=P, rope_sin=P,
             max_positions=64, rotary_dim=64, positions=P, slots=P, tokens=3, q_heads=14, kv_heads=2, head_dim=64, q_out=P,
             k_codes=P, v_codes=P, k_scales=P, v_scales=P, num_pages=8, page_tokens=16)
    return R.QkNormRopeKv8Args(**{**a, **over}), "cheetah_cuda_op_qk_norm_rope_kv8"


def read(**over):
    a = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, num_pages=8, page_tokens=16, slots=P, tokens=3, kv_heads=2,
             head_dim=64, dtype=R.KV_BF16, k_out=P, v_out=P)
    return R.Kv8ReadArgs(**{**a, **over}), "cheetah_cuda_op_kv8_read"


def attend(**over):
    a = dict(q=P, q_stride=14 * 64, rows=5, k_codes=P, v_codes=P, k_scales=P, v_scales=P, page_table=P, max_pages_per_seq=4,
             num_pages=8, page_tokens=16, seq_lens=P, row_starts=P, batch=2, sliding_window=0, sinks=0, q_heads=14,
             kv_heads=2, head_dim=64, out=P, workspace=P, workspace_bytes=1 << 40)
    return R.AttentionKv8Args(**{**a, **over}), "cheetah_cuda_op_attention_kv8"


def verify(**over):
    a = dict(target_probs=P, target_stride=100, draft_probs=P, draft_stride=100, rows=3, vocab=100, tokens=P, row_starts=P,
             batch=1, accept_u=P, sample_u=P, accepted=P, out_tokens=P)
    return R.VerifyDraftsArgs(**{**a, **over}), "cheetah_cuda_op_verify_drafts"


CASES = [
    (append, dict(qkv=None), "null"), (append, dict(slots=None), "null"), (append, dict(v_scales=None), "null"),
    (append, dict(dtype=7), "dtype"), (append, dict(head_dim=96), "head_dim"), (append, dict(rotary_dim=24), "rotary_dim"),
    (append, dict(rotary_dim=128), "rotary_dim"), (append, dict(tokens=0), "empty"), (append, dict(tokens=1 << 31), "empty"),
    (append, dict(max_positions=0), "empty"), (append, dict(kv_heads=0), "head counts"), (append, dict(q_heads=1025), "head counts"),
    (append, dict(qkv_stride=17 * 64), "overlap"), (append, dict(qkv_stride=18 * 64 + 4), "aligned"),
    (append, dict(qkv=P + 8), "aligned"), (append, dict(k_codes=P + 8), "aligned"), (append, dict(k_scales=P + 2), "aligned"),
    (append, dict(q_norm=P + 4), "aligned"), (append, dict(num_pages=0), "pool"), (append, dict(page_tokens=24), "pool"),
    (append, dict(num_pages=1 << 27), "pool"),
    (read, dict(k_codes=None), "null"), (read, dict(k_out=None), "null"), (read, dict(dtype=2), "dtype"),
    (read, dict(head_dim=32), "head_dim"), (read, dict(tokens=0), "empty"), (read, dict(kv_heads=0), "kv_heads"),
    (read, dict(page_tokens=8), "pool"), (read, dict(num_pages=1 << 27), "pool"), (read, dict(v_out=P + 8), "aligned"),
    (read, dict(v_scales=P + 1), "aligned"),
    (attend, dict(q=None), "null"), (attend, dict(workspace=None), "null"), (attend, dict(k_scales=None), "null"),
    (attend, dict(head_dim=80), "head_dim"), (attend, dict(q_heads=15), "multiple"), (attend, dict(kv_heads=0), "multiple"),
    (attend, dict(q_heads=66, q_stride=66 * 64), "group"), (attend, dict(batch=0), "batch"), (attend, dict(batch=4097), "batch"),
    (attend, dict(rows=0), "rows"), (attend, dict(rows=(1 << 24) + 1), "rows"), (attend, dict(page_tokens=24), "pages"),
    (attend, dict(num_pages=1 << 30), "pool"), (attend, dict(max_pages_per_seq=0), "table row"),
    (attend, dict(max_pages_per_seq=(1 << 27) - 1), "table row"), (attend, dict(sliding_window=1 << 31), "sliding_window"),
    (attend, dict(sinks=1 << 31), "sinks"), (attend, dict(q_stride=13 * 64), "overlap"), (attend, dict(q_stride=14 * 64 + 4), "aligned"),
    (attend, dict(out=P + 8), "aligned"), (attend, dict(v_codes=P + 8), "aligned"), (attend, dict(workspace=P + 16), "aligned"),
    (attend, dict(rows=1 << 20, max_pages_per_seq=1 << 21), "too many"), (attend, dict(rows=4096, batch=4096, max_pages_per_seq=1 << 23), "too many"),
    (verify, dict(target_probs=None), "null"), (verify, dict(out_tokens=None), "null"), (verify, dict(rows=0), "rows"),
    (verify, dict(vocab=0), "vocab"), (verify, dict(vocab=(1 << 30) + 1, target_stride=1 << 31, draft_stride=1 << 31), "vocab"),
    (verify, dict(batch=0), "batch"), (verify, dict(batch=65536), "batch"), (verify, dict(target_stride=99), "overlap"),
    (verify, dict(draft_stride=99), "overlap"), (verify, dict(target_probs=P + 2), "aligned"), (verify, dict(draft_probs=P + 1), "aligned"),
    (verify, dict(out_tokens=P + 8), "overlap tokens"), (verify, dict(tokens=P + 4, out_tokens=P), "overlap tokens"),
]


@pytest.mark.parametrize("make,over,message", CASES)
def test_bad_arguments_are_refused(make, over, message):
    args, name = make(**over)
    assert getattr(R.lib(), name)(C.byref(args), None) != 0
    error = R.lib().cheetah_cuda_last_error().decode()
    assert message in error and name in error


def test_null_structs_are_refused():
    for name in ("qk_norm_rope_kv8", "kv8_read", "attention_kv8", "verify_drafts"):
        assert getattr(R.lib(), "cheetah_cuda_op_" + name)(None, None) != 0
        assert b"null" in R.lib().cheetah_cuda_last_error()
    assert R.lib().cheetah_cuda_op_attention_kv8_workspace(None, None) != 0


def test_workspace_query_refuses_what_the_call_refuses():
    n = C.c_size_t(0)
    args, _ = attend(head_dim=80)
    assert R.lib().cheetah_cuda_op_attention_kv8_workspace(C.byref(args), C.byref(n)) != 0


def test_tensors_that_are_not_on_a_gpu_are_refused():
    codes, scales = torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn), torch.ones(2, 1, 1)
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: R.qk_norm_rope_kv8(torch.zeros(1, 3, 64), 1, 1, i, i, scales, scales, codes, codes, scales, scales),
                 lambda: R.kv8_read(codes, codes, scales, scales, i), lambda: R.attention_kv8(q, codes, codes, scales, scales, i, i, i),
                 lambda: R.verify_drafts(torch.zeros(1, 4), None, i, i, scales, scales)):
        with pytest.raises(R.CheetahCudaError):
            call()


def test_reference_codes():
    """The reference's rounding to e4m3: every value, its neighbours' middles, and what lies beside them."""
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(V8.nearest_code(V8.VALUES), codes)
    middle = (V8.VALUES[1:] + V8.VALUES[:-1]) / 2
    even = codes[:-1] + codes[:-1] % 2
    assert torch.equal(V8.nearest_code(middle), even)
    assert torch.equal(V8.nearest_code(middle * (1 - 1e-12)), codes[:-1]) and torch.equal(V8.nearest_code(-middle * (1 + 1e-12)), codes[1:] | 128)
    assert torch.equal(V8.nearest_code(V8.VALUES), V8.VALUES.float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert V8.nearest_code(torch.tensor([math.nan, math.inf], dtype=torch.float64)).tolist() == [127, 127]


@pytest.mark.parametrize("top,scale", [(0.0, -64), (448.0, 0), (448.0000001, 1), (224.0, -1), (1e-30, -64), (3.4e38, 120)])
def test_reference_scales(top, scale):
    assert V8.scale_for(top) == 2.0 ** scale


def test_reference_draws_what_the_target_says():
    """p = 0.5, 0.25, 0.25 and q = 0.25, 0.75, 0: a draft 1 is kept with probability 1/3, else 0 or 2 follow equally."""
    p, q = np.array([[0.5, 0.25, 0.25]] * 2, np.float32), np.array([[0.25, 0.75, 0.0]] * 2, np.float32)
    seen = []
    for u, s in ((0.3, 0.0), (0.34, 0.49), (0.9, 0.51)):
        seen.append(V8.verify(p, q, [0, 1], [0, 2], [u, 0.0], [s], [9, 9]))
    assert seen == [([1], [1, 0]), ([0], [0, -1]), ([0], [2, -1])]
