"""GPU: sampling by clusters of CTAs that start at different times.  A CTA may only be reached through its shared memory
once it runs, so every cluster size is drawn from rows that fill the device several times over, on two streams at once,
and every row of every call has to be the call's that ran alone (sums of whole numbers: equal bits)."""

import pytest
import torch

from tests.test_sampling_gpu import compare, make
from xanosmerks_b200.sampling import sample

pytestmark = pytest.mark.gpu


# (few rows: larger clusters for shorter rows; many rows: by the bytes of a row; 8 CTAs a cluster above 1 MB)
@pytest.mark.parametrize("rows,v", [(1, 2049), (2, 4100), (3, 20000), (18, 20000), (300, 20000), (300, 40000),
                                    (150, 100000), (40, 300001)])
def test_every_cluster_size_beside_other_work(rows, v):
    x, u = make(rows, v, seed=rows + v)
    kw = dict(temperature=0.9, top_k=30, top_p=0.9)
    want = sample(x, u, **kw), sample(x, u)
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(20):
        for st, w, k in zip(streams, want, (kw, {})):
            with torch.cuda.stream(st):
                got.append((sample(x, u, **k), w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in got for a, b in zip(g, w))
    few = slice(0, 4)
    compare(x[few], u[few], **kw)
    for a, b in zip(want[0], sample(x[few], u[few], **kw)):
        assert torch.equal(a[few], b)
