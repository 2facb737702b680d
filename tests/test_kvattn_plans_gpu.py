"""GPU: attention over the paged cache in every plan that sizes lead to: row tiles of 256, many units and many steps of a
warp, more parts than a cluster joins, tables wider than their sequences, steps and prompts in one call.

Bounds of single outputs: the softmax weights are rounded to fp16 (2^-11 of sum p |v|, and, where a weight is subnormal,
2^-25 of the largest weight, at least 1: 2^-25 sum |v|), scores are fp32 sums of D products (D + 8 roundings of
2^-24 of sum |q||k| scale, which count twice: numerator and denominator), and the output is rounded.  More than 32 rows
(token, query head) of a KV head a sequence, in the mean, over a 4-bit cache round its keys and values to fp16 too: 2^-11 of a
value, and 2^-11 sum |q||k| scale of a score, twice.  Steps over a 4-bit cache multiply whole bytes and subtract: an
output is A - B - C with A = sum p d (c + 16 c'), B = sum p d 16 c', C = sum p d 8 in fp32, of magnitudes up to 255, 240
and 8 times S = sum p |d|, each rounded or cut (2^-23 of its magnitude) once for each 16 keys that a warp takes, at least
once for each of the two products of a unit, and once in the end: 2^-23 503 S (n / 64 + 3), where 8 |d| is the largest
value of the block, whose code is 0.

All outputs together, for zero-mean values: each rounding is at most half a step, 2^-11 in fp16 (2^-8 for bf16 outputs),
and uniform within it, so at most that / sqrt 3 of the 2-norm; the weights' and the values' move the outputs by as
much as the outputs' own, the keys' by the spread s of the scores (the deviation of q . k scale, 2 here), once in the
numerator and once in the denominator.  They are independent: their squares add up."""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests.test_kvcache_gpu import HALF_STEP, TINY, dev, filled_cache, layout
from xanosmerks_b200 import _lib

pytestmark = pytest.mark.gpu


def check(c, pool, q, out, table, ql, kl, window, sinks, tokens, rounded, heads=None):
    """Rows `tokens(s, m)` of each sequence against softmax(q K^T scale) V in 64 bits."""
    hk, d, hq = c.num_kv_heads, c.head_dim, q.shape[1]
    g, scale = hq // hk, c.head_dim ** -0.5
    total, off, at = 0.0, 0.0, 0
    cached = {}
    for s, (m, n) in enumerate(zip(ql, kl)):
        rows = tokens(s, m)
        for h in heads or range(hk):
            if not len(rows):
                continue
            key = (table[s, :-(-n // c.page_size)].tobytes(), n, h)
            if key not in cached:
                cached[key] = [torch.from_numpy(x).cuda() for x in pool.keys_values(table[s], n, h)]
            k, v = cached[key]
            i = torch.as_tensor(rows).cuda()
            qs = q[at + i, h * g:(h + 1) * g].double()                      # [rows, g, d]
            got = out[at + i, h * g:(h + 1) * g].double()
            seen = dev(np.stack([O.visible(n - m + j, n, window, sinks) for j in rows]))[:, None]
            x = (qs @ k.T * scale).masked_fill(~seen, float("-inf"))
            p = torch.softmax(x, -1)
            ref = p @ v
            qk = ((qs.abs() @ k.abs().T) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            weight = 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * qk.clamp(min=1.0)
            if rounded:
                weight = weight + 2.0 ** -11 + 2 * 2.0 ** -11 * qk
            floor = seen.double() @ v.abs()
            if c.kv_type == "Q4_0" and not rounded:
                block = v.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2) / 8
                floor = floor + 2.0 ** 25 * 2.0 ** -23 * 503 * (n / 64 + 3) * (p @ block)
            bound = HALF_STEP[q.dtype] * ref.abs() + weight * (p @ v.abs()) + 2.0 ** -25 * floor + TINY[q.dtype]
            err = (got - ref).abs()
            assert (err <= bound * 1.001).all(), (s, h, float((err / bound).max()))
            total += float((ref ** 2).sum())
            off += float((err ** 2).sum())
        at += m
    # (weights and output; 4-bit prompts: values and, through scores of deviation 2 or less, keys)
    half = 2.0 ** -11
    limit = HALF_STEP[q.dtype] ** 2 + half ** 2 + ((1 + 2 * 2 ** 2) * half ** 2 if rounded else 0.0)
    assert off ** 0.5 <= (limit / 3) ** 0.5 * total ** 0.5, (off / total) ** 0.5


def run(kv, d, dtype, hq, hk, page, window, sinks, ql, kl, tokens, extra_width=1, seed=300, heads=None):
    dt = getattr(torch, dtype)
    qls = ql or [1] * len(kl)
    table, lens, cu, pages = layout(qls, kl, page, seed=seed, extra_width=extra_width)
    c, pool = filled_cache(pages, hk, d, page, kv, seed=seed + 1)
    q = (torch.randn(sum(qls), hq, d, generator=torch.Generator().manual_seed(seed + 2)) * 2).to(dt).cuda()
    out = c.attend(q, dev(table), dev(lens), None if ql is None else dev(cu), window=window, sinks=sinks)
    assert _lib.lib.xm_device_status(1) == 0
    rounded = kv == "Q4_0" and sum(qls) * (hq // hk) > 32 * len(qls) and sum(qls) > len(qls)
    check(c, pool, q, out, table, qls, kl, window, sinks, tokens, rounded, heads)
    return c, table, lens, cu, q, out


def some(s, m):
    """The first and last tokens of a prompt, and some of every row tile."""
    rows = set(range(min(m, 3))) | set(range(max(0, m - 40), m)) | set(range(0, m, 23))
    return sorted(rows)


def every(s, m):
    return list(range(m))


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("d,dtype,hq,hk,page,window,sinks,ql,kl", [
    (128, "float16", 32, 8, 64, 0, 0, [1203], [1203]),
    (128, "bfloat16", 32, 8, 16, 0, 0, [1203], [3001]),
    (128, "float16", 32, 8, 32, 700, 70, [1203], [2400]),
    (64, "bfloat16", 28, 4, 32, 0, 0, [1500], [1777]),
    (64, "float16", 28, 4, 16, 1024, 4, [700, 1, 850], [2500, 130, 850]),
    (128, "float16", 8, 8, 128, 0, 0, [4800], [4800]),
])
def test_row_tiles_of_256(kv, d, dtype, hq, hk, page, window, sinks, ql, kl):
    assert (sum(ql) * (hq // hk) // 256 + len(ql)) * hk >= 148        # the rule that takes them
    run(kv, d, dtype, hq, hk, page, window, sinks, ql, kl, some, heads=[0, hk - 1])


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("d,g,page,width,kl", [(128, 4, 64, 130, [5003]), (64, 7, 16, 4, [3001, 64, 900]),
                                              (128, 1, 128, 800, [1000, 20000])])
def test_steps_of_many_parts(kv, d, g, page, width, kl):
    """More parts than one cluster joins; in tables wider than the sequences some of them are empty."""
    n = len(kl)
    max_keys = (max(-(-k // page) for k in kl) + width) * page
    assert _lib.lib.xm_kv_attention_workspace_size(n, n, g, 1, d, max_keys) > 0
    run(kv, d, "float16", g, 1, page, 0, 0, None, kl, every, extra_width=width)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("n", [20000, 15011])
def test_many_steps_of_a_warp(kv, n):
    """512 sequences over the same pages (a shared prefix): parts so long that a warp looks its pages up again."""
    b, hq, d, page = 512, 64, 64, 64
    table, _, _, pages = layout([1], [20000], page, seed=311, extra_width=0)
    c, pool = filled_cache(pages, 1, d, page, kv, seed=312)
    lens = np.full(b, n, np.int32) - np.arange(b, dtype=np.int32) % 100
    q = (torch.randn(b, hq, d, generator=torch.Generator().manual_seed(313)) * 2).half().cuda()
    tb = dev(table).expand(b, -1)
    out = c.attend(q, tb, dev(lens))
    assert _lib.lib.xm_device_status(1) == 0
    for s in (0, 1, 99, 300, 511):
        check(c, pool, q[s:s + 1], out[s:s + 1], table, [1], [int(lens[s])], 0, 0, every, False)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("hq,hk,ql,kl", [
    (8, 2, [0, 3, 1, 20], [9, 3, 70, 90]),               # 24 rows a sequence: steps
    (4, 2, [3, 2, 0, 40], [70, 2, 5, 90]),
    (32, 8, [8], [1000]),                                # 32: the last that are steps
    (32, 8, [9], [1000]),                                # 36: prompts
    (32, 2, [2], [333]),
    (32, 2, [3], [333]),
])
def test_both_sides_of_the_border_between_the_kernels(kv, hq, hk, ql, kl):
    run(kv, 128, "float16", hq, hk, 16, 0, 0, ql, kl, every)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
@pytest.mark.parametrize("chunk", [80, 100, 400])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_steps_and_a_prompt_in_one_call(kv, chunk, window, sinks):
    ql = [1] * 5 + [chunk] + [1] * 6
    kl = [1, 900, 33, 64, 1501, chunk + 700, 128, 65, 7, 512, 300, 1000]
    run(kv, 128, "bfloat16", 16, 4, 32, window, sinks, ql, kl, some)


@pytest.mark.parametrize("kv", ["Q4_0", "F16"])
def test_prompts_past_the_table(kv):
    """Positions that the table has no entry for: reported, and the rows in front of them keep their values."""
    ql, kl, page = [70], [100], 16
    table, lens, cu, pages = layout(ql, kl, page, seed=321, extra_width=0)
    c, pool = filled_cache(pages, 1, 64, page, kv, seed=322)
    q = torch.randn(70, 4, 64, generator=torch.Generator().manual_seed(323)).half().cuda()
    want = c.attend(q, dev(table), dev(lens), dev(cu))
    assert _lib.lib.xm_device_status(1) == 0
    out = c.attend(q, dev(table)[:, :5], dev(lens), dev(cu))                 # 80 positions
    assert _lib.lib.xm_device_status(1) == _lib.ERR_PAGE
    assert torch.equal(out[:50], want[:50]) and torch.isfinite(out).all()
