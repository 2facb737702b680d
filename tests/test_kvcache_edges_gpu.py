"""GPU: attention over the paged cache at the edges of what it allows."""

import numpy as np
import pytest
import torch

from tests.test_kvcache_gpu import check_attention, dev, filled_cache, layout
from xanosmerks_b200 import _lib
from xanosmerks_b200.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("n", [96, 102, 80])            # of the spoilt key's unit all is seen, all but for the first rows, a part
@pytest.mark.parametrize("rows", [1, 2, 60])
def test_a_spoilt_value_of_a_key_of_vanishing_weight(kv, n, rows):
    """A visible key takes part with a positive weight, however small: its NaN is every row's that sees it."""
    d, page, kl = 128, 32, [n]
    table, lens, cu, pages = layout([rows], kl, page, seed=221)
    c, _ = filled_cache(pages, 1, d, page, kv, seed=222, scale=0.25)
    q = torch.ones(rows, 2, d, dtype=torch.float16, device="cuda")
    p = 66                                               # the key: -4 in every dimension, scores some 2000 below the others
    row = torch.full((1, 3 * d), -4.0, device="cuda")
    at = dev(np.array([p + 1], np.int32))
    c.append(row, 1, dev(table), at)
    page_at, half = int(table[0, p // page]), c.pool.shape[2] // 2
    lo, width = (half, 2 * d) if kv == "F16" else (half + page * d // 2, d // 16)
    lo += (p % page) * width
    want = c.attend(q, dev(table), dev(lens), dev(cu), scale=4.0)
    assert torch.isfinite(want).all()
    c.pool[page_at, :, lo:lo + width] = torch.tensor([0xff, 0x7f] * (width // 2), dtype=torch.uint8, device="cuda")
    out = c.attend(q, dev(table), dev(lens), dev(cu), scale=4.0)
    first = max(0, p - (kl[0] - rows))                   # the first row that sees the key
    assert torch.equal(out[:first], want[:first])
    assert torch.isnan(out[first:]).all()
    assert _lib.lib.xm_device_status(0) == 0


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("ql,kl,less", [([3, 5], [40, 50], 2), ([3, 5], [40, 700], 4), ([3, 5], [40, 50], 6),
                                        ([20, 200], [90, 300], 37), ([20, 200], [90, 300], 205), ([3, 70], [9, 4000], 11)])
def test_fewer_rows_than_the_offsets_name(kv, ql, kl, less):
    """The first rows of a step: each keeps the position that the offsets and lengths give it."""
    page, n = 16, sum(ql)
    table, lens, cu, pages = layout(ql, kl, page, seed=231)
    c, pool = filled_cache(pages, 2, 64, page, kv, seed=232)
    q = torch.randn(n, 4, 64, generator=torch.Generator().manual_seed(233)).half().cuda()
    whole = c.attend(q, dev(table), dev(lens), dev(cu))
    check_attention(c, pool, q, whole, table, ql, kl, 0, 0)
    got = c.attend(q[:n - less], dev(table), dev(lens), dev(cu)).double()
    # another number of rows may take other parts of the keys: both within the bounds of a row (see check_attention),
    # values of order 1
    assert (got - whole[:n - less].double()).abs().max() <= 2 * (2.0 ** -11 * 2 + 2.0 ** -10)
    a, b = (PagedKVCache(pages, 2, 64, page, kv) for _ in range(2))
    qkv = torch.randn(n, 8 * 64, generator=torch.Generator().manual_seed(234)).cuda()
    qa, qb = (x.append(r, 4, dev(table), dev(lens), dev(cu)) for x, r in ((a, qkv), (b, qkv[:n - less])))
    assert torch.equal(qa[:n - less], qb)
    assert _lib.lib.xm_device_status(0) == 0


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_queries_near_the_smallest_numbers(kv, rows):
    """bf16 reaches far below fp16 and, with its subnormals, below 2^-126: all scores are nearly 0, no row is spoilt."""
    table, lens, cu, pages = layout([rows], [90], 16, seed=241)
    c, pool = filled_cache(pages, 1, 128, 16, kv, seed=242)
    q = torch.randn(rows, 4, 128, generator=torch.Generator().manual_seed(243))
    q *= torch.tensor([1e-30, 1e-35, 3e-38, 5e-40])[None, :, None]
    q[:, :, ::5] = 0.0
    q = q.to(torch.bfloat16).cuda()
    assert (q[0, 3] != 0).any()
    out = c.attend(q, dev(table), dev(lens), dev(cu))
    check_attention(c, pool, q, out, table, [rows], [90], 0, 0)
