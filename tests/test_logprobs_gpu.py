"""GPU: log-probabilities, ranks, entropies and alternatives against numpy in 64 bits.

Ranks and alternatives are whole numbers and equal.  A weight 2^(c x - r) has an exponent rounded to 2^-24 of its own size
(up to 200 where it counts for nothing, some 30 where it counts), a c good to 2^-24 of that again, and an exponential good to
2^-22: sums are good to 2^-18; the logarithm of a sum to 2^-18 absolute.  A log-probability adds 2^-23 of c x and of itself.
The entropy is a mean of -log p: 2^-17 of 1 + itself and the largest |log p| that counts (30)."""

import numpy as np
import pytest
import torch

from xanosmerks_b200.sampling import MAX_TOP, logprobs

pytestmark = pytest.mark.gpu


def want_row(x, token, T, top):
    """(logprob, entropy, rank, ids, their logprobs) of one row in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    v = len(x)
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        lp = np.full(v, -np.inf)
        if x[order[0]] > -np.inf:
            lp[order[0]] = 0.0
        ent = 0.0
    elif not (x > -np.inf).any():
        lp, ent = np.full(v, -np.inf), 0.0
    else:
        m = x.max()
        if m == np.inf:
            w = (x == np.inf).astype(np.float64)
            z = np.where(x == np.inf, 0.0, -np.inf)
        else:
            z = (x - m) / T
            w = np.exp(z)
        lp = z - np.log(w.sum())
        p = w / w.sum()
        ent = -(p[p > 0] * lp[p > 0]).sum()
    rank = -1
    one = np.nan
    if 0 <= token < v:
        rank = int((x > x[token]).sum() + (x[:token] == x[token]).sum())
        one = lp[token]
    return one, ent, rank, order[:top], lp[order[:top]]


def compare(logits, tokens, temperature=1.0, top=0):
    r = logprobs(logits, tokens, temperature=temperature, top=top)
    x, t = logits.float().cpu().numpy(), tokens.cpu().numpy()
    lp, ent, rank = (v.double().cpu().numpy() for v in (r.logprob, r.entropy, r.rank))
    if top:
        ids, tops = r.top_ids.cpu().numpy(), r.top_logprobs.double().cpu().numpy()
    for b in range(len(x)):
        T = float(temperature[b]) if isinstance(temperature, torch.Tensor) else float(np.float32(temperature))
        one, e, k, want_ids, want_tops = want_row(x[b], t[b], T, top)
        finite = x[b][np.isfinite(x[b])]
        size = (float(np.abs(finite).max()) if finite.size else 0.0) / (T if T > 0 else 1.0)
        tol = 2.0 ** -18 + 2.0 ** -22 * size

        def near(got, ref):
            if abs(ref) > np.finfo(np.float32).max:             # (no number of fp32: its rounding is -inf)
                ref = -np.inf
            if np.isfinite(ref):
                assert abs(got - ref) <= tol + 2.0 ** -23 * abs(ref), (b, got, ref)
            else:
                assert np.array_equal(got, ref, equal_nan=True), (b, got, ref)
        near(lp[b], one)
        assert abs(ent[b] - e) <= 2.0 ** -17 * (31 + e) + 2.0 ** -21 * size, (b, ent[b], e)
        assert rank[b] == k, (b, rank[b], k)
        if top:
            assert np.array_equal(ids[b], want_ids), (b, ids[b], want_ids)
            for got, ref in zip(tops[b], want_tops):
                near(got, ref)
    return r


def make(rows, v, seed, dtype=torch.float32, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, v, generator=g) * spread).to(dtype)
    hot = x.argmax(-1)
    t = torch.randint(0, v, (rows,), generator=g)
    return x.cuda(), torch.where(torch.arange(rows) % 2 == 0, t, hot).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 7, 33, 500, 2049, 4097, 8200, 32000])
def test_sizes_and_types(v, dtype):
    x, t = make(6, v, seed=v, dtype=dtype)
    for top in sorted({0, 1, min(5, v), min(MAX_TOP, v)}):
        compare(x, t, top=top)
    compare(x, t.int(), temperature=0.6, top=min(3, v))


@pytest.mark.parametrize("v", [128001, 300001, 1 << 20])
def test_large_vocabularies(v):
    for dtype in (torch.float32, torch.bfloat16):
        x, t = make(2, v, seed=1, dtype=dtype)
        compare(x, t, top=20)
        compare(x, t, top=MAX_TOP, temperature=1.5)


def test_many_rows():
    x, t = make(700, 5003, seed=2, dtype=torch.bfloat16)
    compare(x, t, top=4)


def test_views_with_a_pitch_and_unaligned_rows():
    wide, _ = make(5, 9001, seed=3, dtype=torch.float16)
    x, t = wide[:, 3:8004], torch.tensor([0, 8000, 17, 4000, 2], device="cuda")
    r = compare(x, t, top=9)
    whole = logprobs(x.contiguous(), t, top=9)
    assert all(torch.equal(p.view(torch.int32), q.view(torch.int32)) or torch.allclose(p, q, rtol=0, atol=1e-5)
               for p, q in zip(r, whole))


def test_temperatures_of_their_own():
    x, t = make(9, 3001, seed=4)
    compare(x, t, temperature=torch.tensor([0.0, 1.0, 0.01, 100.0, 0.5, -1.0, 1e-38, 3e-5, 2.0], device="cuda"), top=6)
    compare(x, t, temperature=0.0, top=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 5000, 70000])
def test_rows_at_the_edges(v, dtype):
    """Masked logits, NaN, infinities, equal logits, ascending rows, rows far from zero, tokens outside of the vocabulary."""
    n = 14
    x, _ = make(n, v, seed=5, dtype=dtype)
    inf = float("inf")
    x[0] = -inf                                                # nothing to choose from
    x[1, 3:] = -inf                                            # three tokens, fewer than the alternatives
    x[2, ::2] = float("nan")
    x[3, 11] = inf
    x[4, [5, v - 1]] = inf                                     # they share the mass
    x[5] = 1.25                                                # all equal
    x[6] = torch.linspace(-8, 8, v, device="cuda").to(dtype)   # every logit above all before it
    x[7] = x[7] + 1e4
    x[8] = x[8] * 100
    x[9, :v // 2] = -300.0                                     # what is seen first is far below the maximum
    x[9, v - 2] = 900.0
    x[10] = float("nan")
    x[11] = torch.finfo(dtype).min                             # the type's lowest value as a mask
    x[11, v // 3] = 0.5
    x[12, : v - 1] = torch.finfo(dtype).min
    x[13] = 0.0
    x[13, 1::2] = -0.0                                         # equal
    for token in (0, 2, 5, 11, v - 1, -1, v):
        compare(x, torch.full((n,), token, device="cuda"), top=7)
    compare(x, torch.arange(n, device="cuda"), top=0, temperature=0.3)


def test_same_bits_whatever_runs_beside_it_and_in_a_graph():
    x, t = make(3, 32000, seed=6)
    want = logprobs(x, t, top=8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = logprobs(x, t, top=8)
    x2, t2 = make(400, 32000, seed=7)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            logprobs(x2, t2, top=8)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    x, t = make(3, 100, seed=8)
    assert logprobs(x[:0], t[:0], top=2).top_ids.shape == (0, 2)
    for a, kw in (((x.double(), t), {}), ((x[0], t), {}), ((x, t[:2]), {}), ((x, t.float()), {}), ((x.cpu(), t), {}),
                  ((x, t.cpu()), {}), ((x, t), {"top": 101}), ((x, t), {"top": 65}), ((x, t), {"top": -1}),
                  ((x.t(), t), {}), ((x, t), {"temperature": t})):
        with pytest.raises(ValueError):
            logprobs(*a, **kw)


def test_rows_behind_two_to_the_31_logits():
    v = 1 << 20
    x = torch.zeros(2053, v, dtype=torch.bfloat16, device="cuda")
    x[2046:] = torch.randn(7, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    t = torch.arange(2053, device="cuda")
    whole, few = logprobs(x, t, top=3), logprobs(x[2046:].clone(), t[2046:].clone(), top=3)
    # The number of rows decides how many CTAs share one, and with it the order of a sum.  Each sum is within 2^-18 (relative; as
    # derived above) of the exact one, so two logarithms of it differ by at most 2 * 2^-18, with the logarithm's own 2^-18 each
    # by 2^-16; entropies, each within 2^-17 (1 + 14 + 30), by twice that.
    for a, b, tol in zip(whole, few, (2.0 ** -16, 45 * 2.0 ** -16, 0, 0, 2.0 ** -16)):
        assert float((a[2046:].double() - b.double()).abs().max()) <= tol
    assert torch.equal(whole.top_ids[0], torch.arange(3, device="cuda", dtype=torch.int32))
    assert abs(float(whole.logprob[5]) + 20 * 0.6931471805599453) < 2.0 ** -17         # (ln 2^20)
