"""GPU: sampling against the 64-bit oracle.  Tokens are equal; log-probabilities are rounded once to fp32 from
64-bit sums whose terms are whole multiples of 2^-44 of the largest weight (2^-24 of the value, and V 2^-44
absolute in the logarithm)."""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from xanosmerks_b200.sampling import sample

pytestmark = pytest.mark.gpu


def compare(logits, u, **kw):
    ids, logp = sample(logits, u, **kw)
    x, un = logits.float().cpu().numpy(), u.cpu().numpy()
    got, lp = ids.cpu().numpy(), logp.double().cpu().numpy()
    pick = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for r in range(len(x)):
        ref, want = O.sample_row(x[r], un[r], **{k: np.float32(pick(v, r)) if k != "top_k" else int(pick(v, r))
                                                 for k, v in kw.items()})
        assert got[r] == ref, (r, got[r], ref)
        if np.isinf(want):
            assert lp[r] == want
        else:
            assert abs(lp[r] - want) <= 2.0 ** -23 * abs(want) + x.shape[1] * 2.0 ** -43 + 1e-12, (r, lp[r], want)
    return ids, logp


def make(rows, v, seed, dtype=torch.float32, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, v, generator=g) * spread).to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 31, 33, 1000, 4097, 32000])
def test_filters_over_sizes_and_types(v, dtype):
    x, u = make(8, v, seed=v, dtype=dtype)
    compare(x, u)
    compare(x, u, temperature=0.7, top_k=20)
    compare(x, u, temperature=1.3, top_p=0.9)
    compare(x, u, min_p=0.05)
    compare(x, u, temperature=0.8, top_k=50, top_p=0.8, min_p=0.02)


@pytest.mark.parametrize("v", [128000, 151937, 300001])
def test_large_vocabularies(v):
    x, u = make(3, v, seed=1)
    compare(x, u)
    compare(x, u, top_k=1000, top_p=0.95)
    compare(x, u, top_p=0.999, temperature=2.0)


def test_parameters_of_their_own_for_each_row():
    rows, v = 40, 5003
    x, u = make(rows, v, seed=5)
    g = torch.Generator().manual_seed(6)
    compare(x, u, temperature=(torch.rand(rows, generator=g) * 1.5 * (torch.arange(rows) % 5 > 0)).cuda(),
            top_k=torch.randint(-1, 60, (rows,), generator=g, dtype=torch.int32).cuda(),
            top_p=(0.5 + 0.6 * torch.rand(rows, generator=g)).cuda(),
            min_p=(0.1 * torch.rand(rows, generator=g)).cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(dtype):
    rows, v = 16, 777
    g = torch.Generator().manual_seed(7)
    x = torch.randint(-3, 4, (rows, v), generator=g).to(dtype).cuda()        # seven different logits
    u = torch.rand(rows, generator=g).cuda()
    compare(x, u, top_k=100)
    compare(x, u, top_p=0.4)
    compare(x, u, top_k=300, top_p=0.7)
    flat = torch.zeros(rows, v, dtype=dtype, device="cuda")
    compare(flat, u, top_k=10)
    compare(flat, u, top_p=0.31)
    ids, _ = sample(flat, u, temperature=0.0)
    assert (ids == 0).all()
    signed = torch.tensor([[0.0, -0.0, 0.0, -1.0]], dtype=dtype, device="cuda")
    compare(signed, torch.tensor([0.6], device="cuda"), top_k=2)


def test_greedy_and_extreme_parameters():
    x, u = make(6, 999, seed=9)
    ids, logp = sample(x, u, temperature=0.0, top_p=0.5, top_k=7)
    assert torch.equal(ids.long(), x.argmax(-1)) and (logp == 0).all()
    for kw in (dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0), dict(min_p=5.0), dict(temperature=1e-30)):
        ids, logp = sample(x, u, **kw)
        assert torch.equal(ids.long(), x.argmax(-1)), kw
        assert (logp == 0).all()
    compare(x, u, temperature=1e30)
    compare(x, u, temperature=float("inf"))
    compare(x, u, top_k=10 ** 6, top_p=1.5, min_p=-1.0)
    compare(x, torch.zeros(6, device="cuda"), top_p=0.9)
    last = torch.full((6,), float(np.nextafter(np.float32(1), np.float32(0))), device="cuda")
    compare(x, last, top_k=5)
    ids, _ = sample(x, torch.full((6,), 1.0, device="cuda"), top_k=5)         # past the end: the last kept token
    top = x.topk(5, -1).indices.amax(-1)
    assert torch.equal(ids.long(), top)
    ids, _ = sample(x, torch.full((6,), float("nan"), device="cuda"), top_k=5)
    assert torch.equal(ids.long(), x.topk(5, -1).indices.amin(-1))


def test_masked_nan_and_infinite_logits():
    v = 500
    x, _ = make(9, v, seed=11)
    u = torch.linspace(0, 0.99, 9).cuda()
    x[0, :] = float("-inf")
    x[1, :] = float("nan")
    x[2, 1:] = float("-inf")
    x[3, :499] = float("-inf")
    x[4, ::2] = float("nan")
    x[5, [7, 300]] = float("inf")
    x[6, :] = torch.finfo(torch.float32).min                                 # masked by the type's lowest value
    x[6, [3, 400]] = 1.0
    x[7, 10:] = float("-inf")
    x[8, 100] = float("inf")
    x[8, 101:] = float("nan")
    compare(x, u)
    compare(x, u, top_k=20)
    compare(x, u, top_p=0.6, min_p=0.1)
    ids, logp = sample(x, u)
    assert ids[0] == 0 and ids[1] == 0 and torch.isneginf(logp[:2]).all()


def test_row_pitch_out_and_streams():
    wide, u = make(5, 1203, seed=13)
    x = wide[:, 2:1003]
    want, lp = compare(x, u, top_p=0.9)
    got, lq = sample(x.contiguous(), u, top_p=0.9)
    assert torch.equal(want, got) and torch.equal(lp, lq)
    out = torch.full((7,), -5, dtype=torch.int32, device="cuda")
    sample(x, u, top_p=0.9, out=out[1:6])
    assert torch.equal(out[1:6], want) and out[0] == -5 and out[6] == -5
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, _ = sample(x, u, top_p=0.9)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b, _ = sample(x, u, top_p=0.9)
        b.zero_()
        g.replay()
    s.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_the_share_of_each_token():
    """20000 draws of one row: every token's count is within six deviations of its probability."""
    n, v = 20000, 7
    row = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -20.0, 1.5])
    x = row.repeat(n, 1).cuda()
    u = ((torch.arange(n) + 0.5) / n)[torch.randperm(n, generator=torch.Generator().manual_seed(1))].cuda()
    ids, _ = sample(x, u, top_k=5)
    p = torch.softmax(row.double()[[0, 1, 3, 4, 6]], 0)
    count = torch.bincount(ids.cpu().long(), minlength=v).double()
    assert count[2] == 0 and count[5] == 0
    assert ((count[[0, 1, 3, 4, 6]] - n * p).abs() <= 2).all()               # evenly spread numbers: at most one off at each end


@pytest.mark.parametrize("v", [9001, 40000])
def test_more_tokens_than_a_list_holds_above_the_cut(v):
    g = torch.Generator().manual_seed(v)
    u = torch.rand(12, generator=g).cuda()
    two = torch.where(torch.rand(12, v, generator=g) < 0.5, 0.0, -2.0).cuda()          # two values only
    near = (torch.randn(12, v, generator=g) * 1e-3).cuda()
    steps = (-torch.logspace(-6, 6, v)[torch.randperm(v, generator=g)]).repeat(12, 1).cuda()   # evenly spaced in the exponent
    for x in (two, near, steps):
        compare(x, u, top_k=10)
        compare(x, u, top_k=512, top_p=0.6)
        compare(x, u, top_k=513, min_p=0.3)
        compare(x, u, top_k=v - 1, top_p=0.5, min_p=0.2)
        compare(x, u, top_p=0.99, min_p=0.5)           # min_p leaves out what top_p would, and more than 512 are left
        compare(x, u, top_p=0.2, min_p=0.5)
        compare(x, u, top_p=0.99999)


@pytest.mark.parametrize("count", [1, 3, 700])
def test_infinite_logits_among_many(count):
    """All of the mass lies on the infinite ones, evenly."""
    v, rows = 30000, 6
    x, u = make(rows, v, seed=77)
    at = torch.randperm(v, generator=torch.Generator().manual_seed(78))[:count].sort().values
    x[:, at.cuda()] = float("inf")
    at = at.numpy()
    un = u.cpu().numpy().astype(np.float64)
    for kw, share in ((dict(), 1.0), (dict(top_p=0.9), 0.9), (dict(top_k=2000, top_p=0.5), 0.5), (dict(top_k=400), None),
                      (dict(top_p=0.5, min_p=0.1), 0.5)):
        kept = min(count, 400) if share is None else max(1, int(np.ceil(np.float64(np.float32(share)) * count)))
        ids, logp = sample(x, u, **kw)
        want = at[np.minimum(np.floor(un * kept).astype(int), kept - 1)]
        assert (ids.cpu().numpy() == want).all(), kw
        assert (logp.cpu() + np.log(kept)).abs().max() <= 1e-6


def test_two_streams_and_a_captured_call():
    x, u = make(20, 33000, seed=101)
    kw = dict(temperature=0.9, top_p=0.95)
    want = sample(x, u, **kw), sample(x, u, top_k=40, **kw)
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), []
    torch.cuda.synchronize()
    for _ in range(5):
        for st, w, k in zip(streams, want, (0, 40)):
            with torch.cuda.stream(st):
                got.append((sample(x, u, top_k=k, **kw), w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in got for a, b in zip(g, w))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        ids, logp = sample(x, u, **kw)
    y, un = make(20, 33000, seed=102)
    x.copy_(y), u.copy_(un)
    g.replay()
    torch.cuda.synchronize()
    now = sample(x, u, **kw)
    assert torch.equal(ids, now[0]) and torch.equal(logp, now[1])
    compare(x, u, **kw)
