"""GPU: log-probabilities of rows of which a mask leaves a few tokens, none of them where a kernel looks first.

The tokens lie far below zero: log2(e) x / T goes from -90 to -135, across the exponents at which weights about a reference of
zero lose what is below them (2^-100 to 2^-126) and vanish.  Tolerances: those derived in tests/test_logprobs_gpu.py."""

import math

import pytest
import torch

from tests.test_logprobs_gpu import compare
from xanosmerks_b200.sampling import logprobs

pytestmark = pytest.mark.gpu


def masked(rows, v, allowed, dtype, seed):
    """Rows of -inf but for the `allowed` indices; row b has log2(e) x between -90 - 45 b / rows and a little below."""
    x = torch.full((rows, v), float("-inf"))
    g = torch.Generator().manual_seed(seed)
    base = -(90 + 45 * torch.arange(rows)[:, None] / rows) / math.log2(math.e)
    x[:, allowed] = base - torch.rand(rows, len(allowed), generator=g) * 1.2
    return x.to(dtype).cuda(), torch.tensor(allowed)[torch.arange(rows) % len(allowed)].cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,v,allowed", [
    (300, 32000, [500, 600]),                  # a CTA a row
    (40, 32000, [500, 600]),                   # some CTAs a row
    (46, 128000, [5000, 5100, 5205]),          # a cluster
    (300, 32000, list(range(500, 530))),       # more tokens than alternatives
    (300, 5003, [4999, 5001]),                 # the row's end
])
def test_few_tokens_far_below_zero(rows, v, allowed, dtype):
    x, t = masked(rows, v, allowed, dtype, seed=v + len(allowed))
    compare(x, t, top=2)
    compare(x * 0.1, t, temperature=0.1)


def test_two_tokens_at_a_low_temperature():
    x = torch.full((300, 32000), float("-inf"), device="cuda")
    x[:, 500], x[:, 600] = -8.6, -8.75
    r = compare(x, torch.full((300,), 500, device="cuda"), temperature=0.1)
    # -ln(1 + e^-1.5), and its entropy; 2^-16: as above for |x| / T near 87
    assert float((r.logprob + 0.2014133).abs().max()) < 2.0 ** -16 and float((r.entropy - 0.4750515).abs().max()) < 2.0 ** -14


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,count", [(0, 3), (50000, 5), (50001, 19), (50000, 1000), (127990, 10), (3, 20000), (0, 40000)])
def test_a_mask_that_leaves_a_range(first, count, dtype):
    """Fewer tokens than alternatives, as many, more, in one place of the row; the alternatives behind them are those of -inf by
    their index."""
    for rows in (1, 40, 300):
        x = torch.full((rows, 128000), float("-inf"), device="cuda", dtype=dtype)
        g = torch.Generator(device="cuda").manual_seed(first + count)
        x[:, first:first + count] = torch.randn(rows, count, device="cuda", generator=g).to(dtype)
        t = torch.full((rows,), first, device="cuda")
        if rows == 300:                                # (the rows' order is enough for a few of them)
            few = [0, 7, 299]
            got = logprobs(x, t, top=20)
            for a, b in zip(got, logprobs(x[few].contiguous(), t[few].contiguous(), top=20)):
                assert torch.allclose(a[few], b, rtol=2.0 ** -15, atol=0)
        else:
            for top in (1, 20, 64):
                compare(x[:3], t[:3], top=top)
        want = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :64]
        assert torch.equal(logprobs(x, t, top=64).top_ids.long(), want)
