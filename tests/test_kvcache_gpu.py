"""GPU: the paged key/value cache (append, read, attention) against the 64-bit oracle.

Tolerances, from the roundings.  Queries: fp32 normalisation and rotation of O(1) terms (at most a dozen
roundings of 2^-24 relative to |a| + |b|), then one rounding to the output type.  fp16 cache: the same with
fp16.  4-bit cache: codes and scales are decided exactly, so the bytes are equal.  Attention, against the
values that the cache holds: the softmax weights are rounded to fp16 (2^-11 each, so 2^-11 of sum p |v|; below
fp16's normal numbers half a subnormal step, 2^-25 of the largest weight, which is at least 1: 2^-25 sum |v|); a
score is an fp32 sum of D products (D + 8 roundings of 2^-24 relative to sum |q||k| scale, base-2 scaled),
which moves each weight by as much relative to itself, numerator and denominator (twice); then one rounding
to the output type.  Prompts (more than 16 rows of a KV head per sequence) over a 4-bit cache round its values
to fp16: 2^-11 of each value, and 2^-11 of sum |q||k| scale in a score.  Those are worst cases; the errors
of a whole output, taken together, are independent roundings, so its relative 2-norm is held to a step of the
output type's rounding in the mean square (half a step / sqrt 3) and 2^-10 for the rest.
"""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from xanosmerks_b200 import _lib
from xanosmerks_b200.kvcache import PagedKVCache, rope_table

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}      # half a step of the subnormals


def layout(q_lens, kv_lens, page_size, seed, spare=2, extra_width=1):
    """Random page table of sequences: (block_table, kv_lens, cu, pages) with unused entries out of the pool."""
    rng = np.random.default_rng(seed)
    need = [-(-k // page_size) for k in kv_lens]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.full((len(kv_lens), max(1, max(need)) + extra_width), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    return table, np.asarray(kv_lens, np.int32), cu, pages


def dev(x):
    return torch.as_tensor(x).cuda()


def positions(q_lens, kv_lens):
    return [(s, k - q + j) for s, (q, k) in enumerate(zip(q_lens, kv_lens)) for j in range(q)]


def filled_cache(pages, hk, d, page_size, kv_type, seed, scale=1.0):
    """A cache of normal values in every slot, and its view."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((2, pages, hk, page_size, d)) * scale).astype(np.float32)
    c = PagedKVCache(pages, hk, d, page_size, kv_type)
    pool = np.zeros(tuple(c.pool.shape), np.uint8)
    half = pool.shape[2] // 2
    for i, values in enumerate((False, True)):
        if kv_type == "F16":
            raw = x[i].astype(np.float16).reshape(pages, hk, -1).view(np.uint8)
        else:
            codes, sc = O.q4_blocks(x[i])
            nib = codes[..., O.nibble_dims(d, values)]
            rows = (nib[..., 0::2] | (nib[..., 1::2] << 4)).reshape(pages, hk, -1)
            raw = np.concatenate([rows, np.ascontiguousarray(sc).reshape(pages, hk, -1).view(np.uint8)], -1)
        pool[:, :, i * half:(i + 1) * half] = raw
    c.pool.copy_(torch.from_numpy(pool))
    return c, O.PoolView(pool, kv_type, d, page_size)


APPEND = [
    # kv, d, dtype, out, hq, hk, page, norm, rope, q_lens, kv_lens
    ("Q4_0", 128, "float32", "float16", 32, 8, 64, False, True, [1], [640]),
    ("Q4_0", 128, "float32", "bfloat16", 4, 2, 16, True, True, [1, 17, 0, 40], [33, 17, 5, 200]),
    ("Q4_0", 64, "bfloat16", "bfloat16", 5, 1, 32, True, True, [3, 70], [3, 131]),
    ("Q4_0", 64, "float16", "float16", 2, 2, 128, False, False, [9], [9]),
    ("Q4_0", 128, "float16", "float16", 2, 2, 16, False, True, [50], [50]),
    ("F16", 128, "float32", "float16", 8, 1, 16, False, True, [5, 1], [5, 70]),
    ("F16", 64, "bfloat16", "float16", 7, 7, 64, True, True, [2, 30], [65, 30]),
    ("F16", 128, "float16", "bfloat16", 3, 3, 1024, True, False, [4], [1030]),
]


@pytest.mark.parametrize("kv,d,dtype,out,hq,hk,page,norm,rope,ql,kl", APPEND)
def test_append_and_read(kv, d, dtype, out, hq, hk, page, norm, rope, ql, kl):
    dt, odt = getattr(torch, dtype), getattr(torch, out)
    table, lens, cu, pages = layout(ql, kl, page, seed=1)
    g = torch.Generator().manual_seed(2)
    qkv = (torch.randn(sum(ql), (hq + 2 * hk) * d, generator=g) * 1.7).to(dt)
    qkv[0, hq * d:hq * d + 32] = 0.0                                  # a block of zeros
    qkv[0, (hq + hk) * d] = 3.0
    qkv[0, (hq + hk) * d + 1] = -3.0                                  # equal magnitudes: the first counts
    cs = rope_table(max(kl), d, 1e4) if rope else None
    qn = (1 + 0.2 * torch.randn(d, generator=g)) if norm else None
    kn = (1 + 0.2 * torch.randn(d, generator=g)) if norm else None
    c = PagedKVCache(pages, hk, d, page, kv)
    before = torch.randint(0, 256, tuple(c.pool.shape), generator=g).to(torch.uint8)
    c.pool.copy_(before)
    q = c.append(qkv.cuda(), hq, dev(table), dev(lens), dev(cu), rope=cs, q_norm=None if qn is None else qn.cuda(),
                 k_norm=None if kn is None else kn.cuda(), eps=1e-6, out_dtype=odt)
    k, v = c.read(dev(table), dev(lens), dev(cu), num_tokens=sum(ql))
    torch.cuda.synchronize()
    assert _lib.lib.xm_device_status(0) == 0
    assert q.dtype == odt and tuple(q.shape) == (sum(ql), hq, d)

    x = qkv.float().numpy().reshape(sum(ql), hq + 2 * hk, d)
    where = positions(ql, kl)
    pos = np.array([p for _, p in where])
    csn = None if cs is None else cs.cpu().numpy()
    fix = lambda w: None if w is None else w.numpy()  # noqa: E731
    qr = O.norm_rotate(x[:, :hq], pos, csn, fix(qn), 1e-6)
    kr = O.norm_rotate(x[:, hq:hq + hk], pos, csn, fix(kn), 1e-6)
    vr = x[:, hq + hk:].astype(np.float64)

    def near(got, ref, dt_):
        pair = np.abs(ref) + np.abs(np.roll(ref, d // 2, -1))
        bound = HALF_STEP[dt_] * np.abs(ref) + 32 * 2.0 ** -24 * pair + TINY[dt_]
        assert (np.abs(got.double().cpu().numpy() - ref) <= bound * (1 + 1e-6)).all()

    near(q, qr, odt)
    pool = O.PoolView(c.pool.cpu().numpy(), kv, d, page)
    rest = before.numpy().copy()
    for t, (s, p) in enumerate(where):
        pg, slot = int(table[s, p // page]), p % page
        for h in range(hk):
            for values, ref in ((False, kr), (True, vr)):
                got = pool.row(pg, h, slot, values)
                if kv == "F16":
                    near(torch.from_numpy(got)[None], ref[t, h][None], torch.float16)
                    val = got
                else:
                    codes, sc = O.q4_blocks(ref[t, h].astype(np.float32))
                    assert np.array_equal(got[0], codes)
                    assert np.array_equal(got[1].view(np.uint16) & 0x7fff, sc.view(np.uint16) & 0x7fff)
                    assert np.array_equal(got[1], sc)
                    val = O.q4_values(codes, sc).astype(np.float16)
                assert np.array_equal((v if values else k)[t, h].cpu().numpy(), val)
    # every other slot keeps its bytes
    keep = O.PoolView(rest, kv, d, page)
    written = {(int(table[s, p // page]), p % page) for s, p in where}
    for pg in range(pages):
        for slot in range(page):
            if (pg, slot) not in written and (slot < 20 or slot % 37 == 0):
                for values in (False, True):
                    a, b = pool.row(pg, 0, slot, values), keep.row(pg, 0, slot, values)
                    a, b = (a, b) if kv == "Q4_0" else ((a.view(np.uint16),), (b.view(np.uint16),))
                    for m, n in zip(a, b):
                        assert np.array_equal(m.view(np.uint8), n.view(np.uint8)), (pg, slot, values)


def test_append_borders_between_codes():
    """Values exactly on, and one step of fp32 beside, every border between two codes."""
    d = 128
    rows = []
    for scale in (1.0, 0.3, 7e-4, 3e-7, 900.0, 1.7e5):
        for sign in (1.0, -1.0):
            dd = np.float32(np.float16(sign * scale / -8 * 8 / 8))
            a = np.float32(-8) * dd
            border = [np.float32((j - 8.5) * np.float64(dd)) for j in range(1, 16)]
            near = border + [np.nextafter(b, np.float32(np.inf), dtype=np.float32) for b in border]
            near += [np.nextafter(b, np.float32(-np.inf), dtype=np.float32) for b in border]
            near = [np.float32(x) for x in near]
            for i in range(0, len(near), 31):
                block = [a] + near[i:i + 31]
                rows.append(np.array(block + [0.0] * (32 - len(block)), np.float32))
    while len(rows) % 4:
        rows.append(np.zeros(32, np.float32))
    x = np.stack(rows).reshape(-1, d)
    n = len(x)
    table, lens, cu, pages = layout([n], [n], 16, seed=3)
    qkv = np.zeros((n, 3, d), np.float32)
    qkv[:, 1], qkv[:, 2] = x, x
    c = PagedKVCache(pages, 1, d, 16, "Q4_0")
    c.append(dev(qkv.reshape(n, -1)), 1, dev(table), dev(lens), dev(cu))
    pool = O.PoolView(c.pool.cpu().numpy(), "Q4_0", d, 16)
    codes, sc = O.q4_blocks(x)
    for t in range(n):
        for values in (False, True):
            got = pool.row(int(table[0, t // 16]), 0, t % 16, values)
            assert np.array_equal(got[0], codes[t]), t
            assert np.array_equal(got[1], sc[t])


def test_append_non_finite_values_spoil_their_block():
    d = 64
    x = np.random.default_rng(4).standard_normal((4, 3, d)).astype(np.float32)
    x[0, 2, 3], x[1, 2, 40], x[2, 2, 5] = np.nan, np.inf, -np.inf
    x[3, 2, 0] = 2e6                                   # its scale is past fp16
    table, lens, cu, pages = layout([4], [4], 16, seed=5)
    c = PagedKVCache(pages, 1, d, 16, "Q4_0")
    c.append(dev(x.reshape(4, -1)), 1, dev(table), dev(lens), dev(cu))
    _, v = c.read(dev(table), dev(lens), dev(cu), num_tokens=4)
    v = v[:, 0].cpu().numpy()
    for t, lo in ((0, 0), (1, 32), (2, 0), (3, 0)):
        assert np.isnan(v[t, lo:lo + 32]).all()
        assert np.isfinite(np.delete(v[t], np.s_[lo:lo + 32])).all()


def test_append_strides_rows_behind_and_negative_positions():
    """Rows of a wider tensor at an odd pitch, an odd start, rows behind the last sequence, more rows than tokens."""
    d, hq, hk, page = 128, 2, 1, 16
    ql, kl = [3, 2], [2, 20]                           # sequence 0: its first row would be position -1
    table, lens, cu, pages = layout(ql, kl, page, seed=6)
    wide = torch.randn(8, (hq + 2 * hk) * d + 3, generator=torch.Generator().manual_seed(7)).cuda()
    qkv = wide[:7, 1:1 + (hq + 2 * hk) * d]
    cs = rope_table(64, d, 1e4)
    big = torch.full((7, 3 * hq * d + 1), 9.0, dtype=torch.float16, device="cuda")
    out = big[:, 1:1 + hq * d].unflatten(1, (hq, d))
    c, ref = PagedKVCache(pages, hk, d, page, "F16"), PagedKVCache(pages, hk, d, page, "F16")
    c.append(qkv, hq, dev(table), dev(lens), dev(cu), rope=cs, out=out)
    q = ref.append(qkv[:5].contiguous(), hq, dev(table), dev(lens), dev(cu), rope=cs)
    assert torch.equal(out[1:5], q[1:5])
    assert (out[0] == 0).all() and (q[0] == 0).all()
    assert (out[5:] == 9).all() and (big[:, 0] == 9).all() and (big[:, 1 + hq * d:] == 9).all()
    assert torch.equal(c.pool, ref.pool)
    k, v = c.read(dev(table), dev(lens), dev(cu), num_tokens=7)
    assert (k[0] == 0).all() and (k[5:] == 0).all() and (v[5:] == 0).all() and (k[1] != 0).any()
    assert _lib.lib.xm_device_status(0) == 0


ATTEND = [
    # kv, d, dtype, hq, hk, page, window, sinks, q_lens (None: one each), kv_lens
    ("Q4_0", 128, "float16", 32, 8, 64, 0, 0, None, [640]),
    ("Q4_0", 128, "bfloat16", 8, 2, 16, 0, 0, None, [1, 15, 16, 17, 63, 64, 65, 300]),
    ("Q4_0", 64, "float16", 7, 1, 32, 0, 0, None, [1, 33, 250]),
    ("F16", 128, "bfloat16", 8, 1, 16, 0, 0, None, [2, 129, 1000]),
    ("F16", 64, "float16", 5, 5, 128, 0, 0, None, [127, 128, 129]),
    ("Q4_0", 128, "float16", 16, 1, 64, 0, 0, None, [200, 31]),
    ("Q4_0", 128, "bfloat16", 20, 1, 64, 0, 0, None, [70]),
    ("Q4_0", 128, "float16", 4, 2, 16, 50, 0, None, [40, 51, 300]),
    ("F16", 64, "bfloat16", 4, 4, 16, 33, 5, None, [3, 39, 40, 200]),
    ("Q4_0", 128, "float16", 4, 1, 16, 1, 0, None, [100]),
    ("Q4_0", 128, "float16", 8, 2, 64, 0, 0, [0, 3, 1, 20], [9, 3, 70, 90]),
    ("F16", 128, "bfloat16", 3, 3, 16, 0, 0, [130], [130]),
    ("Q4_0", 128, "bfloat16", 4, 1, 32, 0, 0, [200, 1], [333, 40]),
    ("Q4_0", 64, "float16", 14, 2, 16, 64, 4, [70, 33], [70, 200]),
    ("F16", 64, "bfloat16", 28, 4, 32, 40, 3, [90, 5], [300, 77]),
    ("Q4_0", 128, "float16", 64, 1, 64, 0, 0, [5], [70]),
    ("F16", 128, "float16", 2, 2, 1024, 100, 0, [300], [300]),
]


def check_attention(c, pool, q, out, table, ql, kl, window, sinks, scale=None):
    hk, d = c.num_kv_heads, c.head_dim
    hq = q.shape[1]
    scale = d ** -0.5 if scale is None else scale
    qn, on = q.double().cpu().numpy(), out.double().cpu().numpy()
    rounded = c.kv_type == "Q4_0" and sum(ql) > len(ql) and sum(ql) * (hq // hk) > 16 * len(ql)
    t, want = 0, np.zeros_like(on)
    for s, (m, n) in enumerate(zip(ql, kl)):
        for h in range(hk):
            k, v = pool.keys_values(table[s], n, h)
            for j in range(m):
                seen = O.visible(n - m + j, n, window, sinks)
                for e in range(h * hq // hk, (h + 1) * hq // hk):
                    ref, mag, qk, floor = O.attention_row(qn[t + j, e], k, v, seen, scale)
                    weight = 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * max(qk, 1.0)
                    if rounded:
                        weight += 2.0 ** -11 + 2 * 2.0 ** -11 * qk
                    want[t + j, e] = ref
                    bound = HALF_STEP[q.dtype] * np.abs(ref) + weight * mag + 2.0 ** -25 * floor + TINY[q.dtype]
                    err = np.abs(on[t + j, e] - ref)
                    assert (err <= bound * 1.001).all(), (s, h, j, e, float((err / np.maximum(bound, 1e-30)).max()))
        t += m
    norm = np.linalg.norm(want)
    if norm > 1e-3:                                     # (outputs in the subnormals are held to their own step above)
        rel = np.linalg.norm(on - want) / norm
        assert rel <= 2 * HALF_STEP[q.dtype] / 3 ** 0.5 + 2.0 ** -10, rel


@pytest.mark.parametrize("kv,d,dtype,hq,hk,page,window,sinks,ql,kl", ATTEND)
def test_attention(kv, d, dtype, hq, hk, page, window, sinks, ql, kl):
    dt = getattr(torch, dtype)
    qls = ql or [1] * len(kl)
    table, lens, cu, pages = layout(qls, kl, page, seed=11)
    c, pool = filled_cache(pages, hk, d, page, kv, seed=12)
    q = (torch.randn(sum(qls), hq, d, generator=torch.Generator().manual_seed(13)) * 2).to(dt).cuda()
    out = c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu), window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert _lib.lib.xm_device_status(0) == 0
    check_attention(c, pool, q, out, table, qls, kl, window, sinks)


@pytest.mark.parametrize("kv,d,dtype,hq,hk,page,window,sinks,ql,kl", [
    ("Q4_0", 128, "float16", 4, 1, 64, 0, 0, [17], [3001]),
    ("F16", 128, "bfloat16", 8, 2, 16, 0, 0, [40, 0, 3, 20], [2600, 0, 513, 20]),       # parts of their own number
    ("Q4_0", 64, "bfloat16", 7, 1, 32, 0, 0, [33, 5], [1025, 4000]),
    ("F16", 64, "float16", 5, 1, 32, 700, 4, [30, 9], [4000, 3100]),
    ("Q4_0", 128, "float16", 3, 3, 16, 2000, 70, [20, 90], [30, 4001]),                 # fewer tokens than rows: nothing to see
])
def test_few_rows_behind_long_contexts(kv, d, dtype, hq, hk, page, window, sinks, ql, kl):
    """More rows than a decode step and fewer than fill the device: the keys are split."""
    kl = [max(k, 0) for k in kl]
    assert _lib.lib.xm_kv_attention_workspace_size(sum(ql), len(ql), hq, hk, d, max(kl)) > 0
    dt = getattr(torch, dtype)
    table, lens, cu, pages = layout(ql, kl, page, seed=14)
    c, pool = filled_cache(pages, hk, d, page, kv, seed=15)
    q = (torch.randn(sum(ql) + 2, hq, d, generator=torch.Generator().manual_seed(16)) * 2).to(dt).cuda()
    out = torch.full_like(q, 7.0)
    c.attend(q, dev(table), dev(lens), dev(cu), window=window, sinks=sinks, out=out)
    assert (out[sum(ql):] == 7).all()
    check_attention(c, pool, q[:-2], out[:-2], table, ql, kl, window, sinks)
    again = torch.full_like(q, 7.0)
    c.attend(q, dev(table), dev(lens), dev(cu), window=window, sinks=sinks, out=again)
    assert torch.equal(out, again) and _lib.lib.xm_device_status(0) == 0


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("qscale,kscale", [(1e-4, 1e-3), (30.0, 1.0), (200.0, 50.0), (1.0, 3e-6)])
def test_attention_magnitudes(kv, qscale, kscale):
    """Tiny and large queries, keys and values: one-hot softmaxes, subnormal scales."""
    table, lens, cu, pages = layout([1, 40], [70, 90], 16, seed=21)
    c, pool = filled_cache(pages, 2, 128, 16, kv, seed=22, scale=kscale)
    q = (torch.randn(41, 8, 128, generator=torch.Generator().manual_seed(23)) * qscale).to(torch.bfloat16).cuda()
    out = c.attend(q, dev(table), dev(lens), dev(cu))
    check_attention(c, pool, q, out, table, [1, 40], [70, 90], 0, 0)


def test_attention_blocks_of_very_different_scales():
    """Values whose blocks differ by 2^20 in scale: each block's output is right relative to its own values."""
    table, lens, cu, pages = layout([1, 30], [50, 60], 16, seed=25)
    c, pool = filled_cache(pages, 1, 128, 16, "Q4_0", seed=26)
    half = c.pool.shape[2] // 2
    sc = c.pool[:, :, half + 16 * 64:].view(torch.float16).unflatten(2, (16, 4))
    sc *= torch.tensor([2.0 ** -10, 1.0, 2.0 ** 10, 2.0 ** -4], device="cuda", dtype=torch.float16)
    pool.p = c.pool.cpu().numpy()
    q = torch.randn(31, 4, 128, generator=torch.Generator().manual_seed(27)).half().cuda()
    for cu_, ql, kl, rows in ((dev(cu), [1, 30], [50, 60], q),):
        out = c.attend(rows, dev(table), dev(lens), cu_)
        check_attention(c, pool, rows, out, table, ql, kl, 0, 0)
    out = c.attend(q[:2], dev(table), dev(lens))
    check_attention(c, pool, q[:2], out, table, [1, 1], [50, 60], 0, 0)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("ql", [None, [3, 2, 0, 40], [3, 2, 0, 200]])
def test_rows_that_see_nothing_and_empty_sequences(kv, ql):
    """Empty sequences, and sequences with fewer tokens than rows, give zeros; rows behind the last are left."""
    kl = [0, 1, 70, 5]
    qls = ql or [1] * 4
    table, lens, cu, pages = layout(qls, kl, 16, seed=31)
    c, pool = filled_cache(pages, 2, 128, 16, kv, seed=32)
    n = sum(qls)
    rows = n + (3 if ql else 0)
    q = torch.randn(rows, 4, 128, generator=torch.Generator().manual_seed(33)).half().cuda()
    out = torch.full((rows, 4, 128), 7.0, dtype=torch.float16, device="cuda")
    c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu), out=out)
    check_attention(c, pool, q[:n], out[:n], table, qls, kl, 0, 0)
    assert (out[0] == 0).all()
    assert (out[n:] == 7).all()
    assert _lib.lib.xm_device_status(0) == 0


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("ql", [None, [1, 50]])
def test_nan_and_inf_behind_the_mask_do_not_matter(kv, ql):
    """Slots behind a sequence's last token, and keys behind the window, hold NaN and infinities."""
    kl = [70, 90]
    qls = ql or [1, 1]
    page, hk, d = 32, 1, 128
    table, lens, cu, pages = layout(qls, kl, page, seed=41)
    c, pool = filled_cache(pages, hk, d, page, kv, seed=42)
    q = torch.randn(sum(qls), 4, d, generator=torch.Generator().manual_seed(43)).half().cuda()
    want = [c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu), window=w).clone() for w in (0, 30)]
    half = c.pool.shape[2] // 2
    width = 2 * d if kv == "F16" else d // 16
    at = 0 if kv == "F16" else page * d // 2

    def spoil(s, p, byte):
        pg = int(table[s, p // page])
        for o in (0, half):
            b = o + at + (p % page) * width
            c.pool[pg, :, b:b + width] = torch.tensor([byte[0], byte[1]] * (width // 2), dtype=torch.uint8, device="cuda")

    nan, inf = (0xff, 0x7f), (0x00, 0x7c)
    for s, n in enumerate(kl):
        for i, p in enumerate(range(n, -(-n // page) * page)):
            spoil(s, p, nan if i % 2 else inf)
    got = c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu))
    assert torch.equal(got, want[0])
    for s, (m, n) in enumerate(zip(qls, kl)):
        for p in range(0, max(0, n - m + 1 - 30)):
            spoil(s, p, nan)
    got = c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu), window=30)
    assert torch.equal(got, want[1])


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
def test_nan_in_a_visible_key_spoils_the_rows_that_see_it(kv):
    table, lens, cu, pages = layout([20], [60], 16, seed=51)
    c, _ = filled_cache(pages, 1, 128, 16, kv, seed=52)
    q = torch.randn(20, 2, 128, generator=torch.Generator().manual_seed(53)).half().cuda()
    p = 50                                              # row 10 is position 50
    at = 0 if kv == "F16" else 16 * 64
    width = 256 if kv == "F16" else 8
    c.pool[int(table[0, p // 16]), 0, at + (p % 16) * width:at + (p % 16) * width + width] = torch.tensor(
        [0xff, 0x7f] * (width // 2), dtype=torch.uint8, device="cuda")
    out = c.attend(q, dev(table), dev(lens), dev(cu))
    assert torch.isfinite(out[:10]).all() and torch.isnan(out[10:]).all()
    one = c.attend(q[:1], dev(table), dev(lens))
    assert torch.isnan(one).all()


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
def test_nan_in_any_column_of_a_prompt(kv):
    """A key that every later row sees whole: the rows in front of it keep their values, the others are NaN."""
    n, page = 300, 16
    table, lens, cu, pages = layout([n], [n], page, seed=54)
    c, pool = filled_cache(pages, 1, 128, page, kv, seed=55)
    q = torch.randn(n, 2, 128, generator=torch.Generator().manual_seed(56)).half().cuda()
    want = c.attend(q, dev(table), dev(lens), dev(cu))
    at = 0 if kv == "F16" else page * 64
    width = 256 if kv == "F16" else 8
    for p in (0, 1, 6, 7, 13, 62, 70, 127):
        before = c.pool.clone()
        o = at + (p % page) * width
        c.pool[int(table[0, p // page]), 0, o:o + width] = torch.tensor([0xff, 0x7f] * (width // 2), dtype=torch.uint8,
                                                                       device="cuda")
        out = c.attend(q, dev(table), dev(lens), dev(cu))
        assert torch.equal(out[:p], want[:p]) and torch.isnan(out[p:]).all(), p
        c.pool.copy_(before)


def test_attention_strides_and_scale():
    """Queries and outputs inside wider tensors at an odd pitch; a scale of one's own."""
    table, lens, cu, pages = layout([1, 35], [40, 50], 16, seed=61)
    c, pool = filled_cache(pages, 2, 64, 16, "Q4_0", seed=62)
    wide = torch.randn(36, 4 * 64 + 5, generator=torch.Generator().manual_seed(63)).half().cuda()
    q = wide[:, 3:3 + 256].unflatten(1, (4, 64))
    big = torch.full((36, 4 * 64 + 7), 5.0, dtype=torch.float16, device="cuda")
    out = big[:, 5:5 + 256].unflatten(1, (4, 64))
    c.attend(q, dev(table), dev(lens), dev(cu), scale=0.3, out=out)
    check_attention(c, pool, q.contiguous(), out, table, [1, 35], [40, 50], 0, 0, scale=0.3)
    assert (big[:, :5] == 5).all() and (big[:, 261:] == 5).all()
    same = c.attend(q.contiguous(), dev(table), dev(lens), dev(cu), scale=0.3)
    assert torch.equal(same, out)
    two = wide[:2, 3:3 + 256].unflatten(1, (4, 64))
    o2 = big[:2, 5:5 + 256].unflatten(1, (4, 64))
    c.attend(two, dev(table), dev(lens), out=o2)
    check_attention(c, pool, two.contiguous(), o2, table, [1, 1], [40, 50], 0, 0)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
def test_bad_pages_set_the_error_word(kv):
    """Pages outside the pool and positions past the table: nothing is read or written there."""
    table, lens, cu, pages = layout([2, 30], [40, 50], 16, seed=71, extra_width=0)
    c, _ = filled_cache(pages, 1, 128, 16, kv, seed=72)
    was = c.pool.clone()
    qkv = torch.randn(32, 4 * 128, generator=torch.Generator().manual_seed(73)).cuda()
    for bad in (-1, pages, 2 ** 31 - 1):
        t = table.copy()
        t[0, 2], t[1, 1] = bad, bad
        q = c.append(qkv, 2, dev(t), dev(lens), dev(cu))
        assert (q[0] == 0).all()                        # position 38 is on the bad page
        assert _lib.lib.xm_device_status(1) == _lib.ERR_PAGE
        out = c.attend(q, dev(t), dev(lens), dev(cu))
        assert _lib.lib.xm_device_status(1) == _lib.ERR_PAGE
        assert torch.isfinite(out).all()
        k, _ = c.read(dev(t), dev(lens), dev(cu), num_tokens=32)
        assert (k[0] == 0).all()
        assert _lib.lib.xm_device_status(1) == _lib.ERR_PAGE
        c.pool.copy_(was)
    long = dev(np.array([200, 50], np.int32))           # past the table's width
    q = c.append(qkv, 2, dev(table), long, dev(cu))
    assert (q[:2] == 0).all()
    c.attend(q, dev(table), long, dev(cu))
    with pytest.raises(_lib.XMError, match="without a page"):
        _lib.check_device("test")
    assert _lib.lib.xm_device_status(1) == 0


def test_long_context_offsets_past_32_bits():
    """A pool of more than 4 GB: pages whose byte offsets pass 32 bits."""
    page, hk, d = 1024, 8, 128
    c = PagedKVCache(1100, hk, d, page, "F16")           # 4.6 GB
    assert c.pool.numel() > 2 ** 32
    table = dev(np.array([[1099, 0], [1098, 1097]], np.int32))
    lens = dev(np.array([1030, 1024], np.int32))
    cu = dev(np.array([0, 1030, 2054], np.int32))
    qkv = torch.randn(2054, 3 * hk * d, generator=torch.Generator().manual_seed(82)).half().cuda()
    q = c.append(qkv, hk, table, lens, cu)
    k, v = c.read(table, lens, cu, num_tokens=2054)
    rows = qkv.unflatten(1, (3 * hk, d))
    assert torch.equal(k, rows[:, hk:2 * hk]) and torch.equal(v, rows[:, 2 * hk:])
    out = c.attend(q[[1029, 2053]], table, lens).float()
    for i, (lo, hi) in enumerate(((0, 1030), (1030, 2054))):
        s = torch.einsum("hd,thd->ht", rows[hi - 1, :hk].double(), k[lo:hi].double()) / d ** 0.5
        ref = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v[lo:hi].double())
        assert (out[i].double() - ref).abs().max() < 2e-3   # |ref| < 1: 2^-11 twice and the scores


def test_two_streams_and_a_captured_graph():
    """The same calls eagerly, on two streams at once, and replayed from two graphs at once."""
    kl = [700, 1, 333, 90]
    table, lens, cu, pages = layout([1] * 4, kl, 64, seed=91)
    tb, ln = dev(table), dev(lens)
    c, _ = filled_cache(pages, 2, 128, 64, "Q4_0", seed=92)
    qa = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(93)).half().cuda()
    qb = (qa * 0.5).contiguous()
    want = c.attend(qa, tb, ln), c.attend(qb, tb, ln)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((c.attend(qa, tb, ln), want[0]))
        with torch.cuda.stream(s2):
            got.append((c.attend(qb, tb, ln), want[1]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    graphs = []
    for q in (qa, qb):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s1):
            o = c.attend(q, tb, ln)
        graphs.append((g, o))
    for _ in range(3):
        for (g, o), s in zip(graphs, (s1, s2)):
            o.zero_()
        torch.cuda.synchronize()
        for (g, o), s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want[0]) and torch.equal(graphs[1][1], want[1])


def test_split_prompts_on_two_streams_and_in_graphs():
    """More rows than a step, keys in parts: each call has its own workspace, in graphs too, and a replay follows the
    lengths on the device."""
    ql, kl = [40, 30], [3000, 1500]
    table, lens, cu, pages = layout(ql, kl, 64, seed=94)
    tb, ln, co = dev(table), dev(lens), dev(cu)
    c, _ = filled_cache(pages, 1, 128, 64, "Q4_0", seed=95)
    assert _lib.lib.xm_kv_attention_workspace_size(70, 2, 4, 1, 128, table.shape[1] * 64) > 0
    qa = torch.randn(70, 4, 128, generator=torch.Generator().manual_seed(96)).half().cuda()
    qb = (qa * 0.5).contiguous()
    want = c.attend(qa, tb, ln, co), c.attend(qb, tb, ln, co)
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(5):
        for st, q, w in zip(streams, (qa, qb), want):
            with torch.cuda.stream(st):
                got.append((c.attend(q, tb, ln, co), w))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for x, w in got)
    graphs = []
    for st, q in zip(streams, (qa, qb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            graphs.append((g, c.attend(q, tb, ln, co)))
    shorter = c.attend(qa, tb, ln - 700, co)
    for less, expect in ((0, want[0]), (700, shorter)):
        ln.copy_(dev(lens) - less)
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], expect)
        if not less:
            assert torch.equal(graphs[1][1], want[1])


@pytest.mark.parametrize("kv,norm", [("Q4_0", True), ("F16", False)])
def test_prompt_then_steps_as_a_decoder_uses_them(kv, norm):
    """Append a prompt, attend, then append and attend token by token: the same rows as attending everything
    at once, and right against the values that the cache holds."""
    hq, hk, d, page, n, p = 8, 2, 128, 16, 37, 30
    table, lens, cu, pages = layout([n], [n], page, seed=95)
    g = torch.Generator().manual_seed(96)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).cuda()
    w = (1 + 0.1 * torch.randn(d, generator=g)).cuda() if norm else None
    cs = rope_table(64, d, 1e4)
    kw = dict(rope=cs, q_norm=w, k_norm=w)
    whole, parts = (PagedKVCache(pages, hk, d, page, kv) for _ in range(2))
    tb = dev(table)
    qa = whole.append(qkv, hq, tb, dev(lens), dev(cu), **kw)
    oa = whole.attend(qa, tb, dev(lens), dev(cu))
    ln = dev(np.array([p], np.int32))
    c0 = dev(np.array([0, p], np.int32))
    rows = [parts.attend(parts.append(qkv[:p], hq, tb, ln, c0, **kw), tb, ln, c0)]
    for t in range(p, n):
        ln = dev(np.array([t + 1], np.int32))
        rows.append(parts.attend(parts.append(qkv[t:t + 1], hq, tb, ln, **kw), tb, ln))
    assert torch.equal(whole.pool, parts.pool)
    view = O.PoolView(parts.pool.cpu().numpy(), kv, d, page)
    check_attention(parts, view, qa, oa, table, [n], [n], 0, 0)
    check_attention(parts, view, qa, torch.cat(rows), table, [n], [n], 0, 0)
