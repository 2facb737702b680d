"""CPU: refusals of the paged cache and of sampling, reported before any launch, and the layout."""

import numpy as np
import pytest
import torch

from oracle import gguf_dequant_oracle as G
from oracle import kv_oracle as O
from xanosmerks_b200 import _lib
from xanosmerks_b200.kvcache import PagedKVCache, rope_table
from xanosmerks_b200.sampling import sample

L = _lib.lib
P = 4096          # an aligned address that no refused call reads


def append(**kw):
    a = dict(qkv=P, dt=0, T=2, stride=6144, hq=32, hk=8, d=128, rope=P, rows=10, qn=None, kn=None, eps=1e-5, pool=P,
             pages=4, kv=1, page=64, table=P, tstride=4, width=4, cu=None, lens=P, B=2, q=P, qdt=1, qstride=4096)
    a.update(kw)
    return L.xm_kv_append(*a.values(), None)


def read(**kw):
    a = dict(pool=P, pages=4, kv=1, hk=8, d=128, page=64, table=P, tstride=4, width=4, cu=None, lens=P, B=2, T=2, k=P, v=P)
    a.update(kw)
    return L.xm_kv_read(*a.values(), None)


def attend(**kw):
    a = dict(q=P, dt=1, T=2, stride=4096, hq=32, hk=8, d=128, scale=0.1, window=0, sinks=0, pool=P, pages=4, kv=1,
             page=64, table=P, tstride=4, width=4, cu=None, lens=P, B=2, out=P, ostride=4096, ws=P, wsb=1 << 40)
    a.update(kw)
    return L.xm_kv_attention(*a.values(), None)


def draw(**kw):
    a = dict(x=P, dt=0, B=2, V=100, stride=100, u=P, t=1.0, tp=None, k=0, kp=None, p=1.0, pp=None, m=0.0, mp=None, ids=P, lp=P)
    a.update(kw)
    return L.xm_sample(*a.values(), None)


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("kw", [dict(page=48), dict(page=8), dict(page=2048), dict(hk=0), dict(pages=0), dict(B=0),
                                dict(width=0), dict(pool=None), dict(pool=P + 8), dict(table=None), dict(lens=None),
                                dict(T=-1), dict(T=3), dict(tstride=-1), dict(width=1 << 40)])
def test_cache_arguments_are_refused(call, kw):
    assert call(**kw) == _lib.XM_ERR_INVALID, kw
    assert L.xm_last_error()


@pytest.mark.parametrize("call", [append, read, attend])
def test_unsupported_forms(call):
    assert call(kv=2) == _lib.XM_ERR_UNSUPPORTED
    assert call(d=96) == _lib.XM_ERR_UNSUPPORTED
    assert call(d=256) == _lib.XM_ERR_UNSUPPORTED


def test_calls_without_rows_do_nothing():
    assert append(T=0, cu=P) == 0 and read(T=0, cu=P) == 0 and attend(T=0, cu=P) == 0
    assert draw(B=0) == 0


@pytest.mark.parametrize("kw", [dict(hq=31), dict(hq=0), dict(dt=7), dict(qdt=0), dict(stride=6143), dict(qstride=4095),
                                dict(qkv=None), dict(q=None), dict(rows=0), dict(qkv=P + 2), dict(q=P + 1),
                                dict(rope=P + 4), dict(qn=P + 2), dict(kn=P + 1)])
def test_append_arguments_are_refused(kw):
    assert append(**kw) == _lib.XM_ERR_INVALID, kw


@pytest.mark.parametrize("kw", [dict(hq=31), dict(hq=0), dict(hq=520), dict(dt=0), dict(stride=4095), dict(ostride=4095), dict(q=None),
                                dict(out=None), dict(window=-1), dict(sinks=-1), dict(ws=None, width=4096), dict(wsb=4096, width=4096),
                                dict(ws=P + 8, width=4096), dict(q=P + 1),
                                dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attention_arguments_are_refused(kw):
    assert attend(**kw) == _lib.XM_ERR_INVALID, kw


@pytest.mark.parametrize("kw", [dict(dt=5), dict(B=-1), dict(V=0), dict(stride=99), dict(x=None), dict(u=None),
                                dict(ids=None), dict(x=P + 2), dict(u=P + 1), dict(mp=P + 2), dict(V=1 << 31, stride=1 << 31)])
def test_sample_arguments_are_refused(kw):
    assert draw(**kw) == _lib.XM_ERR_INVALID, kw


def test_page_bytes():
    assert L.xm_kv_page_bytes(0, 8, 128, 64) == 2 * 8 * 64 * 256
    assert L.xm_kv_page_bytes(1, 8, 128, 64) == 2 * 8 * 64 * 72
    assert L.xm_kv_page_bytes(1, 1, 64, 16) == 2 * 16 * 36
    for bad in ((2, 8, 128, 64), (1, 8, 96, 64), (1, 0, 128, 64), (1, 8, 128, 63)):
        assert L.xm_kv_page_bytes(*bad) == 0


def test_python_refusals_need_no_gpu():
    with pytest.raises(NotImplementedError):
        PagedKVCache(4, 8, 128, 64, "Q8_0")
    with pytest.raises(NotImplementedError):
        PagedKVCache(4, 8, 80)
    for kw in (dict(page_size=24), dict(num_pages=0), dict(num_kv_heads=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(num_pages=4, num_kv_heads=8), **kw})
    good = torch.zeros(4, 8, 2 * 64 * 72, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache(4, 8, 128, 64, "Q4_0", pool=good)
    with pytest.raises(ValueError, match="uint8"):
        PagedKVCache(4, 8, 128, 64, "Q4_0", pool=good[:3])
    with pytest.raises(ValueError):
        rope_table(0, 128)
    with pytest.raises(ValueError):
        rope_table(4, 63)
    with pytest.raises(ValueError, match="CUDA"):
        sample(torch.zeros(2, 10), torch.zeros(2))


def test_rope_table_on_the_host():
    t = rope_table(1000, 64, 5e5, device="cpu").numpy()
    ang = np.arange(1000)[:, None] / 5e5 ** (np.arange(32) / 32.0)
    assert t.shape == (1000, 32, 2)
    assert np.abs(t[..., 0] - np.cos(ang)).max() <= 2.0 ** -24 and np.abs(t[..., 1] - np.sin(ang)).max() <= 2.0 ** -24


def test_oracle_blocks_are_gguf_q4_0_blocks():
    """The codes and scales of the cache, written as GGUF Q4_0 records, are what the reference's format reads."""
    x = np.random.default_rng(3).standard_normal((5, 64)).astype(np.float32)
    codes, d = O.q4_blocks(x)
    rec = []
    for r in range(5):
        for g in range(2):
            c = codes[r, 32 * g:32 * g + 32]
            rec.append(d[r, g:g + 1].view(np.uint8).tobytes() + (c[0::2] | (c[1::2] << 4)).tobytes())
    got = G.dequantize(b"".join(rec), "Q4_0", (5, 64))
    assert np.array_equal(np.asarray(got), O.q4_values(codes, d).astype(np.float16))
    assert np.abs(O.q4_values(codes, d) - x).max() < np.abs(x).max() / 7
    for dd in (64, 128):
        for values in (False, True):
            assert sorted(O.nibble_dims(dd, values)) == list(range(dd))
