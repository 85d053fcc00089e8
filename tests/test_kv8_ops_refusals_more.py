"""More argument checks of the operators over an 8-bit cache, through the C-ABI on
the CPU (as test_kv8_ops_refusals)."""

import ctypes as C

import pytest

from cheetah_b200 import runtime as R
from tests.test_kv8_ops_refusals import P, verify


@pytest.mark.parametrize("rows", [(1 << 30) + 1, (1 << 31) - 1, 1 << 31])
def test_drafts_beyond_the_rows_that_are_counted_are_refused(rows):
    """The walk over a sequence's rows passes its end by up to a block: near 2^31 that was read."""
    args, name = verify(rows=rows, vocab=1, target_stride=1, draft_stride=1, out_tokens=P + (1 << 40))
    assert getattr(R.lib(), name)(C.byref(args), None) != 0
    error = R.lib().cheetah_cuda_last_error().decode()
    assert "rows" in error and name in error
