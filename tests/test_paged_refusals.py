"""Refusals of the paged-cache operators at the C entries; no GPU."""
import ctypes as C

import pytest

from tests.test_paged_host import NULL, _attention


@pytest.mark.parametrize("kw", [dict(batch=2), dict(batch=0)])
def test_rows_cannot_be_cleared_in_no_output(built_library, kw):
    from eptq_b200 import _lib
    assert _lib.load().eptq_ragged_attention(C.byref(_attention(clear_rest=1, out=None, **kw)), 4096, 1 << 40, None) == NULL
