"""CPU: unaligned page tables, offsets and lengths are refused before any launch."""

import pytest

from tests.test_kvcache_host import P, append, attend, read
from xanosmerks_b200 import _lib


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("kw", [dict(table=P + 1), dict(table=P + 2), dict(lens=P + 2), dict(cu=P + 2), dict(cu=P + 3, T=5)])
def test_unaligned_indices_are_refused(call, kw):
    assert call(**kw) == _lib.XM_ERR_INVALID, kw
    assert b"unaligned" in _lib.lib.xm_last_error()
