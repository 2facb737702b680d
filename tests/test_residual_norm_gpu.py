"""GPU: norm, gate, residual add and norm between two blocks against torch in 64 bits.

Tolerance.  A sum of squares of D values in fp32: fewer than 40 roundings on the way of a value (32 values a thread, ten steps
of a tree, 32 warps), all of one sign, so 80 * 2^-24 of it, and half of that behind the root; v = y r w takes three more
roundings, the gate, scale and add three more.  So v is good to 48 * 2^-24 of itself, h to that of |scale gate v| and 2^-24 of
|h| (and half a step of its type), next to 48 * 2^-24 of itself, what h's error is of it, and half a step."""

import pytest
import torch

from xanosmerks_b200.ops import residual_norm

pytestmark = pytest.mark.gpu
E = 48 * 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def compare(stream, y, post=None, gate=None, scale=1.0, pre=None, eps=1e-5, out_dtype=None, out=None):
    want_in = stream.double()
    v = y.double()
    if post is not None:
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        v = v * gate.double()
    v = float(torch.tensor(scale, dtype=torch.float32)) * v
    h = want_in + v
    dh = E * v.abs() + 2.0 ** -24 * h.abs()
    got, after = residual_norm(stream, y, post_weight=post, gate=gate, scale=scale, pre_weight=pre, eps=eps,
                               out_dtype=out_dtype, out=out)
    f = torch.finfo(stream.dtype)
    tiny = f.smallest_normal * f.eps
    assert got.dtype == stream.dtype and got.shape == stream.shape
    assert bool(((got.double() - h).abs() <= dh + HALF[stream.dtype] * h.abs() * (1 + 2.0 ** -10) + tiny).all())
    if pre is None:
        assert after is None
        return got, after
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    n = h * r * pre.double()
    # (the mean square is off by the mean of 2 |h| dh)
    ds = (h.abs() * dh).mean(-1, keepdim=True) * r * r
    dn = (dh * r * pre.double().abs()) + n.abs() * (E + ds)
    t = out_dtype or y.dtype
    assert after.dtype == t and after.shape == stream.shape
    assert bool(((after.double() - n).abs() <= dn * 1.01 + HALF[t] * n.abs() * (1 + 2.0 ** -10)
                 + torch.finfo(t).smallest_normal * torch.finfo(t).eps).all())
    return got, after


def make(shape, seed=0, stream=torch.float32, y=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = shape[-1]
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return (n(*shape) * 2).to(stream), n(*shape).to(y), 1 + 0.1 * n(d), 1 + 0.1 * n(d)


@pytest.mark.parametrize("d", [1, 2, 31, 64, 255, 256, 258, 1000, 1024, 1030, 2048, 4096, 5001, 8192, 10000, 16384, 32768, 32767])
def test_widths(d):
    for rows in (1, 5):
        s, y, post, pre = make((rows, d), seed=d)
        compare(s, y, post=post, pre=pre, scale=0.22)
        s, y, post, pre = make((rows, d), seed=d, y=torch.bfloat16)
        compare(s, y, post=post, pre=pre)


@pytest.mark.parametrize("st", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("yt", [torch.float32, torch.float16, torch.bfloat16])
def test_types_and_parts(st, yt):
    for d in (770, 4096):
        s, y, post, pre = make((7, d), seed=1, stream=st, y=yt)
        compare(s, y)
        compare(s, y, post=post)
        compare(s, y, pre=pre)
        compare(s, y, post=post, pre=pre, scale=-1.5, eps=1e-6)
        for ot in HALF:
            compare(s, y, post=post, pre=pre, out_dtype=ot)


@pytest.mark.parametrize("gt", [torch.float32, torch.bfloat16])
def test_gates(gt):
    b, t, d = 3, 5, 1152
    s, y, post, pre = make((b, t, d), seed=2, stream=torch.bfloat16, y=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((d,), (1,), (b, 1, d), (b, t, 1), (b, t, d), (b, 1, 1), (t, d), (1, t, d), (t, 1), (1, 1, d), (1, 1, 1)):
        gate = torch.randn(*shape, device="cuda", generator=g).to(gt)
        compare(s, y, post=post, gate=gate, pre=pre, scale=0.5)
    six = torch.randn(b, 6 * d, device="cuda", generator=g).to(gt)      # one of six parts of a modulation
    for gate in (six[:, None, d:2 * d], six[:, None, 1:d + 1]):
        compare(s, y, gate=gate, pre=pre)


def test_in_place_views_and_unaligned_rows():
    s, y, post, pre = make((9, 1030), seed=4, y=torch.float16)
    big = torch.full((9, 2000), 3.0, device="cuda")
    for at in (0, 1, 2):
        big[:] = 3.0
        view = big[:, at:at + 1030]
        view.copy_(s)
        first, n1 = compare(s, y, post=post, pre=pre)
        got, n2 = residual_norm(view, y, post_weight=post, pre_weight=pre, out=view)
        assert got.data_ptr() == view.data_ptr()
        assert torch.allclose(view, first, rtol=1e-5, atol=1e-6)
        assert bool((big[:, :at] == 3).all()) and bool((big[:, at + 1030:] == 3).all())
    t = y.t().contiguous().t()                       # another order of strides: copied
    compare(s, t, post=post, pre=pre)
    compare(s.view(3, 3, 1030).transpose(0, 1), y.view(3, 3, 1030), pre=pre)


def test_rows_that_are_not_numbers_stay_apart_and_zeros():
    s, y, post, pre = make((6, 512), seed=5)
    clean = residual_norm(s, y, post_weight=post, pre_weight=pre)
    y[1, 3], y[4, 500] = float("nan"), float("inf")
    got = residual_norm(s, y, post_weight=post, pre_weight=pre)
    for a, c in zip(got, clean):
        assert torch.equal(a[[0, 2, 3, 5]], c[[0, 2, 3, 5]])
        assert not bool(torch.isfinite(a[1]).any()) and not bool(torch.isfinite(a[4]).all())
    zero = torch.zeros(2, 512, device="cuda")
    h, n = residual_norm(zero, zero, post_weight=post, pre_weight=pre)
    assert bool((h == 0).all()) and bool((n == 0).all())


def test_many_rows_streams_and_graphs():
    s, y, post, pre = make((70001, 64), seed=6, stream=torch.bfloat16, y=torch.bfloat16)
    want = compare(s, y, post=post, pre=pre)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = residual_norm(s, y, post_weight=post, pre_weight=pre)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    s, y, post, pre = make((4, 256), seed=7)
    assert residual_norm(s[:0], y[:0], pre_weight=pre)[1].shape == (0, 256)
    for a, kw in (((s.cpu(), y), {}), ((s.double(), y), {}), ((s, y[:3]), {}), ((s, y.cpu()), {}), ((s, y), {"post_weight": pre[:5]}),
                  ((s, y), {"pre_weight": pre.half()}), ((s, y), {"gate": pre[:7]}), ((s, y), {"gate": pre.cpu()}),
                  ((s, y), {"gate": pre.view(1, 1, 256)}), ((s, y), {"out": s.half()}), ((s, y), {"out_dtype": torch.float64}),
                  ((torch.zeros(1, 32769, device="cuda"),) * 2, {})):
        with pytest.raises(ValueError):
            residual_norm(*a, **kw)


def test_broadcast_inputs():
    """One row, or one sequence, for all of them: rows that lie on one another are read as such, never written."""
    s, y, post, pre = make((3, 5, 512), seed=4)
    compare(s, y[:1, :1].expand(3, 5, 512), post=post, pre=pre)
    compare(s[:1].expand(3, 5, 512), y, pre=pre)
    compare(s[0, :1].expand(5, 512), y[0, :1].expand(5, 512), post=post, pre=pre)
    flat = s[0, :1].expand(5, 512)
    with pytest.raises((ValueError, RuntimeError)):
        residual_norm(flat, y[0], out=flat)
    one, z, post, pre = make((4, 1), seed=5)
    compare(one[:1].expand(4, 1), z, pre=pre)


def test_rows_behind_two_to_the_31_values():
    s, y, post, pre = make((8, 32768), seed=6, stream=torch.float16, y=torch.bfloat16)
    n = 65540
    h, z = s[:1].repeat(n, 1), y[:1].repeat(n, 1)
    h[-8:], z[-8:] = s, y
    got, after = residual_norm(h, z, post_weight=post, pre_weight=pre, out=h)
    want, following = compare(s, y, post=post, pre=pre)
    assert torch.equal(got[-8:], want) and torch.equal(after[-8:], following)
    assert torch.equal(got[:8], want[:1].expand(8, -1)) and torch.equal(after[1000], following[0])
