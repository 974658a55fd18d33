"""The scratch of the attention over a shared prefix, without a GPU: what of it is refused."""
import ctypes as C

import pytest

from test_block8_args import L  # noqa: F401  (the library, as a fixture)
from test_block8_shared_args import _shared


@pytest.mark.parametrize("offset", [1, 4, 8, 16, 48])
@pytest.mark.parametrize("sizes", [dict(B=2, max_S=100, blocks=4), dict(B=64, max_S=20000, blocks=1000)])
def test_scratch_that_is_not_aligned_to_32_bytes_is_refused(L, offset, sizes):
    """Partial outputs go out 32 bytes at a time; of calls that have none the same is asked."""
    a = _shared(L, **sizes, workspace=4096 + offset, workspace_bytes=2 ** 40)
    assert L.lib.jf_block8_shared_attn(C.byref(a), None) == L.JF_ERR_WORKSPACE
