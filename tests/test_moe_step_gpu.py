"""GPU: the mixture-of-experts layer for a few tokens against the oracle's weights in 64 bits.

Tolerance, element by element.  Activations keep 22 bits (2^-22 of the largest magnitude of 16 bits below them, so 2^-22 of
the value or less); a sum runs through some 16 truncated additions inside a matrix instruction and up to 64 of fp32 behind
it, one step of 2^-23 each: a product W x is off by at most EPS |W| |x|, EPS = 2^-22 + 80 * 2^-23.  The activation passes
that on (slopes up to 1.13), and its own exponential and division are good to a few 2^-23 of the result; the weights of the
experts to 2^-21 (an exponential of a difference of logits)."""

import numpy as np
import pytest
import torch

from oracle import gguf_dequant_oracle as O
from xanosmerks_b200 import _lib
from xanosmerks_b200.moe import MoELayer
from xanosmerks_b200.ops import GGUFTensor
from xanosmerks_b200.synth import make_weight_device

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -22 + 80 * 2.0 ** -23
OWN = ("Q4_K", "Q5_K", "Q6_K", "Q8_0")
SCALE = {"Q4_K": 6.75e-5, "Q6_K": 1.45e-5, "Q5_K": 3.5e-5, "Q8_0": 1.6e-4, "Q2_K": 1e-3, "Q3_K": 4e-4, "Q8_K": 1.6e-4}
ACT = {"silu": lambda g: g * torch.sigmoid(g), "relu": torch.relu, "identity": lambda g: g,
       "gelu": lambda g: 0.5 * g * (1 + torch.tanh(0.7978845608 * (g + 0.044715 * g ** 3)))}


class Block:
    """A layer and its weights in 64 bits."""

    def __init__(self, qtype, E, k, H, F, seed=0, act="silu", gate=None):
        shape = {"w1": (F, H), "w3": (F, H), "w2": (H, F)}
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.gate = torch.randn(E, H, device="cuda", generator=g) / H ** 0.5 if gate is None else gate
        self.w, experts = [], {}
        for e in range(E):
            exp = {}
            for i, (n, s) in enumerate(shape.items()):
                raw = make_weight_device(qtype, *s, seed=1000 * seed + 3 * e + i, scale=SCALE.get(qtype, 5e-4))
                exp[n] = {"weight": GGUFTensor(raw, qtype, s)}
            experts[str(e)] = exp
        self.layer = MoELayer({"num_experts": E, "num_experts_per_tok": k, "hidden_act": act},
                              {"gate": {"weight": self.gate}, "experts": experts})
        self.experts, self.qtype, self.act, self.k, self.E = experts, qtype, act, k, E
        self.cache = {}

    def weights(self, e):
        if e not in self.cache:
            got = []
            for n in ("w1", "w3", "w2"):
                t = self.experts[str(e)][n]["weight"]
                raw = t.data.cpu().numpy()
                v = (O.dequant_f32(raw, self.qtype, t.shape[0] * t.shape[1]).reshape(t.shape) if self.qtype in OWN
                     else O.dequantize(raw, self.qtype, t.shape))
                got.append(torch.from_numpy(np.asarray(v, np.float64)).cuda())
            self.cache[e] = got
        return self.cache[e]

    def want(self, x, norm=None, eps=1e-5, residual=None):
        """(result, tolerance) in 64 bits."""
        v = x.double()
        if norm is not None:
            v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * norm.double()
        logit = v @ self.gate.double().T
        top, at = logit.sort(dim=-1, descending=True, stable=True)
        p, at = torch.softmax(top[:, :self.k], -1), at[:, :self.k]
        out, tol = torch.zeros_like(v), torch.zeros_like(v)
        for e in at.unique().tolist():
            t, j = (at == e).nonzero(as_tuple=True)
            w1, w3, w2 = self.weights(e)
            g, u = v[t] @ w1.T, v[t] @ w3.T
            # (the norm's own roundings: a few 2^-24 of v)
            dg, du = (EPS + 2.0 ** -22) * (v[t].abs() @ w1.abs().T), (EPS + 2.0 ** -22) * (v[t].abs() @ w3.abs().T)
            f = ACT[self.act](g)
            a = f * u
            da = u.abs() * 1.13 * dg + f.abs() * du + 1.13 * dg * du + 2.0 ** -19 * a.abs()
            y, dy = a @ w2.T, (da + EPS * a.abs()) @ w2.abs().T
            out.index_add_(0, t, p[t, j][:, None] * y)
            tol.index_add_(0, t, p[t, j][:, None] * (dy + 2.0 ** -21 * y.abs()))
        if residual is not None:
            out += residual.double()
        return out, tol + 2.0 ** -22 * out.abs()


def check(got, want):
    ref, tol = want
    off = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    bad = off > tol
    assert not bool(bad.any()), (float((off / tol).max()), float((off.norm() / ref.norm())))


def rows(T, H, seed, dtype=torch.float32):
    return torch.randn(T, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("qtype", ["Q4_K", "Q5_K", "Q6_K", "Q8_0", "Q4_0", "Q4_1", "Q5_0", "Q5_1", "Q8_1", "Q2_K", "Q3_K", "Q8_K"])
def test_every_type(qtype):
    b = Block(qtype, 4, 2, 512, 768, seed=3)
    for T in (1, 6):
        x = rows(T, 512, T)
        check(b.layer.step(x), b.want(x))


@pytest.mark.parametrize("qtype,E,k,H,F", [
    ("Q4_K", 8, 2, 4096, 1024),      # sixteen 256-blocks a row
    ("Q4_K", 3, 3, 256, 256),        # one block a row, every expert
    ("Q6_K", 5, 1, 1280, 2816),      # odd numbers of blocks; rows that are no multiple of 16 bytes
    ("Q6_K", 4, 2, 768, 4352),       # the second products' rows in two parts
    ("Q5_K", 6, 2, 4608, 512),       # the first products' rows in two parts
    ("Q8_0", 2, 1, 8448, 8448),      # three parts each
    ("Q3_K", 3, 2, 5376, 1792),      # parts and unaligned rows
    ("Q4_K", 160, 8, 512, 256),      # many small experts
    ("Q4_K", 256, 16, 256, 256),     # the limits
])
def test_shapes(qtype, E, k, H, F):
    b = Block(qtype, E, k, H, F, seed=4)
    for T in (1, 5):
        x = rows(T, H, 10 + T)
        check(b.layer.step(x), b.want(x))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 17, 33, 64])
def test_numbers_of_tokens(T):
    b = Block("Q4_K", 6, 2, 512, 512, seed=5)
    x = rows(T, 512, T)
    check(b.layer.step(x), b.want(x))


@pytest.mark.parametrize("act", ["gelu", "relu", "identity"])
def test_activations(act):
    b = Block("Q4_K", 4, 2, 512, 768, seed=6, act=act)
    x = rows(7, 512, 1)
    check(b.layer.step(x), b.want(x))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_residual_strides_and_in_place(dtype):
    H = 1024
    b = Block("Q4_K", 8, 2, H, 512, seed=7)
    x, norm = rows(5, H, 1, dtype), 1 + 0.1 * rows(1, H, 2)[0]
    res = rows(5, H, 3) * 10
    want = b.want(x, norm, 1e-5, res)
    check(b.layer.step(x, norm_weight=norm, residual=res), want)
    wide = torch.full((5, H + 17), 7.0, dtype=dtype, device="cuda")
    wide[:, 3:3 + H] = x
    big = torch.full((5, 2 * H), 9.0, device="cuda")
    big[:, :H] = res
    got = b.layer.step(wide[:, 3:3 + H], norm_weight=norm, residual=big[:, :H], out=big[:, :H])
    check(got, want)
    assert got.data_ptr() == big.data_ptr() and bool((big[:, H:] == 9).all())
    if dtype == torch.float32:                       # a residual stream in place
        h = x.clone()
        want = b.want(x, norm, 1e-5, x)
        b.layer.step(h, norm_weight=norm, residual=h, out=h)
        check(h, want)


def test_all_tokens_to_one_expert_and_equal_logits():
    """Experts with many tokens take several passes; equal logits go to the lower experts."""
    H = 512
    gate = torch.zeros(7, H, device="cuda")
    gate[5] = 1.0
    b = Block("Q4_K", 7, 2, H, 512, seed=8, gate=gate)
    x = rows(19, H, 4).abs()                         # every token: expert 5, then 0 (of equal ones)
    check(b.layer.step(x), b.want(x))
    b = Block("Q4_K", 7, 3, H, 512, seed=8, gate=torch.zeros(7, H, device="cuda"))
    check(b.layer.step(x), b.want(x))


def test_large_and_small_rows():
    """Rows far from 1 keep their bits: each has a power of two of its own."""
    b = Block("Q4_K", 4, 2, 512, 512, seed=9, act="identity")
    x = rows(6, 512, 5) * torch.tensor([1e-12, 1e-3, 1.0, 1e4, 1e9, 0.0], device="cuda")[:, None]
    b.gate.mul_(0)                                   # (no softmax of logits of 1e9)
    b.layer.gate.copy_(b.gate)
    check(b.layer.step(x), b.want(x))


def test_rows_that_are_not_numbers_stay_apart():
    b = Block("Q4_K", 4, 2, 512, 512, seed=10)
    x = rows(6, 512, 6)
    clean = b.layer.step(x)
    x[2, 7], x[4, 100] = float("nan"), float("inf")
    got = b.layer.step(x)
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], clean[keep])
    assert not bool(torch.isfinite(got[2]).any()) and not bool(torch.isfinite(got[4]).all())
    torch.cuda.synchronize()
    assert _lib.lib.xm_device_status(1) == 0


def test_same_bits_again_in_graphs_and_on_streams():
    """Two captured steps and two streams at once: each call has its own workspace."""
    H = 1024
    b = Block("Q4_K", 16, 4, H, 512, seed=11)
    xs = [rows(T, H, T) for T in (1, 6)]
    want = [b.layer.step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs = []
    torch.cuda.synchronize()
    for x, s in zip(xs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = b.layer.step(x)
        graphs.append((g, out))
    for _ in range(5):
        for (g, out), s in zip(graphs, streams):
            out.zero_()
        torch.cuda.synchronize()
        for (g, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (g, out), w in zip(graphs, want):
            assert torch.equal(out, w)
    for x, w, s in zip(xs, want, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = [b.layer.step(x) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o in got)


def test_close_to_the_block_for_many_tokens():
    b = Block("Q4_K", 8, 2, 1024, 2048, seed=12)
    x = rows(12, 1024, 1)
    a, c = b.layer.step(x), b.layer.forward_device(x)
    assert float((a - c).norm() / c.norm()) < 2e-3     # (forward_device: fp16 weights and activations)


def test_nothing_to_do_and_refusals():
    b = Block("Q4_K", 4, 2, 512, 256, seed=13)
    assert b.layer.step(rows(0, 512, 1)).shape == (0, 512)
    good = rows(2, 512, 1)
    for bad in (rows(65, 512, 1), rows(2, 256, 1), good.double(), good.cpu(), good[0], good.t().contiguous().t()):
        with pytest.raises(ValueError):
            b.layer.step(bad)
    for kw in ({"norm_weight": rows(1, 256, 1)[0]}, {"residual": rows(3, 512, 1)}, {"residual": good.half()},
               {"out": good.half()}, {"norm_weight": good[0].half()}):
        with pytest.raises(ValueError):
            b.layer.step(good, **kw)


class Sparse(Block):
    """Weights that are 0 but for one in 64, which are 1: codes of little and of the middle of their range."""

    def __init__(self, qtype, H, F, seed=0):
        shape = {"w1": (F, H), "w3": (F, H), "w2": (H, F)}
        rng = np.random.default_rng(seed)
        exp = {}
        for n, s in shape.items():
            one = rng.random((s[0] * s[1] // 64, 64)).argmin(1)             # the place in 64 values
            if qtype == "Q8_0":
                raw = np.zeros((s[0] * s[1] // 32, 34), np.uint8)
                raw[:, 1] = 0x3C                                             # fp16 1.0
                at = 64 * np.arange(len(one)) + one
                raw[at // 32, 2 + at % 32] = 1
            else:                                                            # code 32 is 0: two upper bits 10, four lower ones 0
                raw = np.zeros((s[0] * s[1] // 256, 210), np.uint8)
                raw[:, 128:192] = 0xAA
                raw[:, 192:208] = 1
                raw[:, 209] = 0x3C
                raw[np.arange(len(one)) // 4, 32 * (np.arange(len(one)) % 4) + one % 32] |= np.where(one < 32, 1, 16).astype(np.uint8)
            exp[n] = {"weight": GGUFTensor(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, s)}
        self.gate = torch.zeros(1, H, device="cuda")
        self.layer = MoELayer({"num_experts": 1, "num_experts_per_tok": 1, "hidden_act": "identity"},
                              {"gate": {"weight": self.gate}, "experts": {"0": exp}})
        self.experts, self.qtype, self.act, self.k, self.E, self.cache = {"0": exp}, qtype, "identity", 1, 1, {}


@pytest.mark.parametrize("tokens", [1, 3, 16])
@pytest.mark.parametrize("qtype", ["Q8_0", "Q6_K"])
def test_few_weights_of_small_codes(qtype, tokens):
    """What a sum loses is measured by its weights, not by the range of their codes."""
    b = Sparse(qtype, 1024, 512)
    assert 0 < float(b.weights(0)[0].sum()) <= 1024 * 512 / 64 and float(b.weights(0)[0].max()) == 1
    x = rows(tokens, 1024, 7)
    check(b.layer.step(x), b.want(x))
