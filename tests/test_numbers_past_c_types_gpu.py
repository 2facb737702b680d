"""GPU: counts larger than the C types that carry them mean what they say."""

import pytest
import torch

from tests.test_kvcache_gpu import dev, filled_cache, layout
from xanosmerks_b200.sampling import sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k", [1000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 64 + 3])
def test_top_k_of_more_than_the_row(top_k):
    x = torch.randn(7, 1000, generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.rand(7, generator=torch.Generator().manual_seed(2)).cuda()
    for kw in ({}, {"top_p": 0.9}):
        for a, b in zip(sample(x, u, top_k=top_k, **kw), sample(x, u, **kw)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("top_k", [-1, -2 ** 31, -(2 ** 32) + 2])
def test_negative_top_k_keeps_all(top_k):
    x = torch.randn(7, 1000, generator=torch.Generator().manual_seed(3)).cuda()
    u = torch.rand(7, generator=torch.Generator().manual_seed(4)).cuda()
    for a, b in zip(sample(x, u, top_k=top_k), sample(x, u)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [2 ** 30, 2 ** 31, 2 ** 64 + 5])
def test_windows_and_sinks_longer_than_any_context(n):
    table, lens, cu, pages = layout([3], [90], 16, seed=251)
    c, _ = filled_cache(pages, 1, 64, 16, "F16", seed=252)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(253)).half().cuda()
    want = c.attend(q, dev(table), dev(lens), dev(cu))
    assert torch.equal(c.attend(q, dev(table), dev(lens), dev(cu), window=n), want)
    got = c.attend(q, dev(table), dev(lens), dev(cu), window=20, sinks=n)      # every key is a sink
    # (the same keys in another order of the sums: fp16 outputs of order 1, weights rounded to 2^-11)
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -9
