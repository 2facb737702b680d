"""GPU: page tables whose entries are gone where no row looks (pages behind a window, given back to the pool), and pages
outside the pool that rows do look at.

A page none of whose keys is seen by any row of its sequence is not needed: the outputs are the ones with the page
present, bit for bit (a masked key takes no part whatever its bytes are), and no error is reported.  Where a needed page
is missing its keys, and no others, are left out, and the error word says so."""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_kvcache_gpu import check_attention, dev, filled_cache, layout
from xanosmerks_b200 import _lib

pytestmark = pytest.mark.gpu


def seen_by(m, n, window, sinks):
    ok = np.zeros(n, bool)
    for j in range(m):
        ok |= O.visible(n - m + j, n, window, sinks)
    return ok


def released(table, ql, kl, page, window, sinks):
    """The table without the pages that no row of their sequence needs, and their number."""
    t, gone = table.copy(), 0
    for s, (m, n) in enumerate(zip(ql, kl)):
        ok = seen_by(m, n, window, sinks)
        for i in range(-(-n // page)):
            if not ok[i * page:(i + 1) * page].any():
                t[s, i] = -1
                gone += 1
    return t, gone


# one token each; a few; more than a decode step takes, keys in parts; enough rows for whole tiles
QL = [None, [2, 1, 3, 5], [40, 1, 70, 33], [300, 1, 200, 129]]


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("ql", QL, ids=["step", "few", "rows", "prompt"])
@pytest.mark.parametrize("window,sinks", [(250, 4), (250, 20), (100, 0), (16, 1)])
def test_pages_that_no_row_sees_may_be_gone(kv, page, ql, window, sinks):
    kl = [700, 717, 331, 460]                           # the window's lower edge in either half of a unit of 32 keys
    qls = ql or [1] * 4
    table, lens, cu, pages = layout(qls, kl, page, seed=201)
    c, pool = filled_cache(pages, 2, 128, page, kv, seed=202)
    q = torch.randn(sum(qls), 8, 128, generator=torch.Generator().manual_seed(203)).half().cuda()
    co = None if ql is None else dev(cu)
    want = c.attend(q, dev(table), dev(lens), co, window=window, sinks=sinks)
    assert _lib.lib.xm_device_status(1) == 0
    less, gone = released(table, qls, kl, page, window, sinks)
    assert gone > 4
    got = c.attend(q, dev(less), dev(lens), co, window=window, sinks=sinks)
    assert _lib.lib.xm_device_status(1) == 0
    assert torch.equal(got, want)
    if sum(qls) < 20:
        check_attention(c, pool, q, got, table, qls, kl, window, sinks)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("ql", QL, ids=["step", "few", "rows", "prompt"])
@pytest.mark.parametrize("bad", [-1, None])
def test_a_missing_page_hides_its_own_keys_only(kv, page, ql, bad):
    kl = [70 + m for m in (ql or [1] * 4)]
    qls = ql or [1] * 4
    table, lens, cu, pages = layout(qls, kl, page, seed=211)
    c, pool = filled_cache(pages, 1, 64, page, kv, seed=212)
    heads = 4
    q = torch.randn(sum(qls), heads, 64, generator=torch.Generator().manual_seed(213)).half().cuda()
    t = table.copy()
    lost = {0: 1, 1: 0, 3: 1}                            # sequence: page
    for s, i in lost.items():
        t[s, i] = pages if bad is None else bad
    out = c.attend(q, dev(t), dev(lens), None if ql is None else dev(cu))
    assert _lib.lib.xm_device_status(1) == _lib.ERR_PAGE
    out = out.double().cpu().numpy()
    at = 0
    for s, (m, n) in enumerate(zip(qls, kl)):
        k, v = pool.keys_values(table[s], n, 0)
        for j in range(m):
            if j < 3 or j > m - 3 or j % 29 == 0:
                seen = O.visible(n - m + j, n, 0, 0)
                if s in lost:
                    seen[lost[s] * page:(lost[s] + 1) * page] = False
                for e in range(heads):
                    ref, mag, qk, floor = O.attention_row(q[at + j, e].double().cpu().numpy(), k, v, seen, 64 ** -0.5)
                    # weights, values and keys rounded to fp16, and the output (half a step is 2^-11 each; a key's counts
                    # twice: in the numerator and in the denominator); scores in fp32
                    bound = 2.0 ** -11 * (np.abs(ref) + 2 * mag + 2 * qk * mag) + 2 * 72 * 2.0 ** -24 * max(qk, 1) * mag
                    bound += 2.0 ** -25 * (floor + 1)
                    assert (np.abs(out[at + j, e] - ref) <= bound * 1.001).all(), (s, j, e)
        at += m
