"""GPU: entropies and log-probabilities of confident rows, relative to themselves.

With the largest logit M outside of the sums, S = sum w and E = sum w t over the others (t = c (x - M), w = 2^t) have terms of
one sign each, logprob = ln 2 t - ln(1 + S) and entropy = ln(1 + S) - ln 2 E / (1 + S) too: a result is off by no more than its
worst term, relative to itself.  A term: t is rounded to half a step of fp32 three times (c, the product less the reference, and
that reference less M), which moves w by 3 * 2^-24 |t| ln 2, at most 2^-17.9 for |t| <= 32; the exponential is good to 2^-22; sums
of 64 and of some 16 to 64 numbers in fp32, by roundings of one sign at worst, to 128 * 2^-24 = 2^-17.  Together below 2^-16; where
|t| <= 32 does not hold (results below 2^-31), at most 3 * 2^-24 * 126 ln 2 = 2^-16 for the first: 2^-15 covers |t| <= 126, beyond
which a weight counts as 0."""

import numpy as np
import pytest
import torch

from xanosmerks_b200.sampling import logprobs

pytestmark = pytest.mark.gpu


def want(x, t, T, top):
    """(logprob, entropy, the top ones' logprobs) in 64 bits, without cancellation."""
    x = x.astype(np.float64)
    out = []
    for row, token in zip(x, t):
        order = np.argsort(-row, kind="stable")
        z = (row - row[order[0]]) / T
        w = np.exp(z)
        w[order[0]] = 0.0
        s, e = w.sum(), (w[w > 0] * z[w > 0]).sum()
        out.append((z[token] - np.log1p(s), np.log1p(s) - e / (1 + s), z[order[:top]] - np.log1p(s)))
    return [np.array(v) for v in zip(*out)]


def compare(x, t, T=1.0, top=3):
    r = logprobs(x, t, temperature=T, top=top)
    check((r.logprob, r.entropy, r.top_logprobs), x, t, T, top)


def check(results, x, t, T, top):
    ref = want(x.float().cpu().numpy(), t.cpu().numpy(), float(np.float32(T)), top)
    for got, v in zip(results, ref):
        rel = np.where(np.abs(v) < 2.0 ** -31, 2.0 ** -15, 2.0 ** -16)
        off = np.abs(got.double().cpu().numpy() - v)
        bad = off > rel * np.abs(v) + 2.0 ** -100
        assert not bad.any(), (np.argwhere(bad)[:4], got.cpu().numpy()[bad][:4], v[bad][:4])


def peaked(rows, v, lift, dtype, seed, spread=0.0, where=None):
    """A flat row, or one of deviation `spread`, with a logit `lift` (a tensor, one a row) above the others' level."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * spread
    at = torch.randint(0, v, (rows,), generator=g) if where is None else torch.full((rows,), where)
    x[torch.arange(rows), at] = lift
    t = torch.where(torch.arange(rows) % 2 == 0, at, torch.randint(0, v, (rows,), generator=g))
    return x.to(dtype).cuda(), t.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,v", [(1, 32000), (1, 40), (2, 5003), (300, 4097), (40, 128001), (600, 32000), (1, 1 << 20)])
def test_from_even_to_certain(rows, v, dtype):
    lift = torch.linspace(0, 40, rows) if rows > 1 else torch.tensor([18.0])
    for spread in (0.0, 1.0):
        x, t = peaked(rows, v, lift, dtype, seed=rows + v, spread=spread)
        compare(x, t)
        compare(x, t, T=0.6)


@pytest.mark.parametrize("where", [0, 1, 7, 31999, 31990, 16001])
def test_where_the_peak_lies(where):
    """In vectors at the row's ends, in the first round and behind it; and the only large logit in a row of -inf."""
    for rows in (1, 300):
        x, t = peaked(rows, 32000, torch.full((rows,), 20.0), torch.float32, seed=where, spread=1.0, where=where)
        compare(x, t)
        x[:, where] += 100                             # (all else vanishes, or nearly)
        compare(x, t)
        alone = torch.full_like(x, float("-inf"))
        alone[:, where] = -50.0
        r = logprobs(alone, torch.full((rows,), where, device="cuda"), top=1)
        assert bool((r.logprob == 0).all()) and bool((r.entropy == 0).all()) and bool((r.top_logprobs == 0).all())


def test_rows_that_rise_and_several_peaks():
    """Every logit above all before it; two and more equal largest ones, in one thread's part and in others'."""
    v = 32000
    x = torch.linspace(-30, 0, v, device="cuda").repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = -40
    x[2, [3, 4, 8000, 31999]] = 1.0
    for rows in (1, 120):
        compare(x.repeat(rows, 1), torch.tensor([v - 1, 0, 8000], device="cuda").repeat(rows))
        compare(x.repeat(rows, 1).half(), torch.tensor([5, 5, 5], device="cuda").repeat(rows), T=1.7)


def test_a_first_round_far_below_the_peak():
    for dtype in (torch.float32, torch.bfloat16):
        for lift in (30.0, 80.0, 120.0, 300.0):        # (weights about the first round's largest logit overflow)
            x, t = peaked(300, 32000, torch.full((300,), lift), dtype, seed=3, spread=1.0, where=500)
            x[:, 600] = lift - 1.5
            compare(x, t)
            compare(x[:2], t[:2])


def test_many_logits_above_what_was_seen():
    """So many vectors reach the largest logit seen that the row is taken again: a flat rest, each thread's in one long sum."""
    for v, dtype in ((1 << 18, torch.float32), (260001, torch.bfloat16)):
        x = torch.zeros(300, v, dtype=dtype, device="cuda")
        lift = torch.linspace(7, 14, 300, device="cuda")[:, None]
        x[:, 1000:3000:8] = (lift - torch.linspace(6, 0, 250, device="cuda")).to(dtype)
        t = torch.arange(300, device="cuda") + 900
        r = logprobs(x, t, top=3)                      # (300 rows: one CTA each)
        some = [0, 100, 299]
        check([v[some] for v in (r.logprob, r.entropy, r.top_logprobs)], x[some], t[some], 1.0, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_whose_first_round_is_far_below_their_own_largest(dtype):
    """A cluster's part with a largest logit far above what it sees first, and far below another part's."""
    for most, second in ((100.0, 60.0), (80.0, 66.0), (140.0, 68.0), (60.0, 59.0)):
        x = torch.randn(2, 128000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * 0.5
        x[:, 5] = most
        x[:, 16400:16460:7] = second + torch.linspace(-1, 1, 9, device="cuda")
        x[1, 70000] = second - 0.5
        compare(x.to(dtype), torch.tensor([5, 16400], device="cuda"))
        compare((x * 0.1).to(dtype), torch.tensor([16407, 5], device="cuda"), T=0.1)
