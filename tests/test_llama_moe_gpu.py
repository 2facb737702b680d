"""GPU: decoders with mixture-of-experts layers, norms behind the blocks and residual scales, and the scoring of sequences,
against the numpy oracle on the same GGUF weights.  Logits: the contiguous decoder's tolerance (fp16 keys and values, 16-bit
activation split, fp16 weights and activations where many rows go through the grouped products).  A log-probability is a logit
less a logarithm of a sum of exponentials of logits, which is off by no more than the logits: twice the tolerance of the
largest logit.  The weights are made on the host, and their seed is such that no token of the oracle's has two experts nearer
than MARGIN in the choice: the decoder's router logits, some units at most, are off by the tolerance."""

import numpy as np
import pytest
import torch

from oracle import gguf_dequant_oracle as GO
from oracle.llama_oracle import LlamaOracle, rms_norm, silu
from oracle.moe_oracle import softmax
from tests.helpers import rel_err
from tests.test_llama_gpu import LOGIT_TOL
from xanosmerks_b200.llama import _WEIGHT_SCALE, LlamaConfig
from xanosmerks_b200.synth import make_weight_device

pytestmark = pytest.mark.gpu
MARGIN = 2e-2


def config(**kw):
    base = dict(num_layers=2, hidden_size=512, num_heads=4, num_kv_heads=2, intermediate_size=768, vocab_size=1000)
    return LlamaConfig(**{**base, **kw})


def host_weights(cfg, seed):
    """(the dict of LlamaWeights.from_full with (raw bytes, type, shape) for tensors, the oracle's weights)."""
    D, F, V, hd = cfg.hidden_size, cfg.intermediate_size, cfg.vocab_size, cfg.head_dim
    g = torch.Generator().manual_seed(seed)
    count = [1000 * seed]

    def w(qt, n, k):
        count[0] += 1
        raw = make_weight_device(qt, n, k, seed=count[0], device="cpu", scale=_WEIGHT_SCALE[qt])
        return (raw, qt, (n, k)), GO.dequantize(raw.numpy(), qt, (n, k)).astype(np.float32)

    def norm(n=D):
        v = 1 + 0.1 * torch.randn(n, generator=g)
        return v, v.numpy()

    layers = []
    for _ in range(cfg.num_layers):
        lw = {"wq": w(cfg.attn_qtype, cfg.num_heads * hd, D), "wk": w(cfg.attn_qtype, cfg.num_kv_heads * hd, D),
              "wv": w(cfg.attn_qtype, cfg.num_kv_heads * hd, D), "wo": w(cfg.attn_qtype, D, cfg.num_heads * hd),
              "n1": norm(), "n2": norm()}
        if cfg.num_experts:
            gate = torch.randn(cfg.num_experts, D, generator=g) * 2 / D ** 0.5
            ex = [{n: w(cfg.expert_qtype, *s) for n, s in (("w1", (F, D)), ("w2", (D, F)), ("w3", (F, D)))}
                  for _ in range(cfg.num_experts)]
            lw["moe"] = ({"gate": {"weight": gate},
                          "experts": {str(i): {n: {"weight": v[0]} for n, v in e.items()} for i, e in enumerate(ex)}},
                         (gate.numpy(), [{n: v[1] for n, v in e.items()} for e in ex]))
        else:
            lw.update(wg=w(cfg.gate_up_qtype, F, D), wu=w(cfg.gate_up_qtype, F, D), wd=w(cfg.down_qtype, D, F))
        if cfg.post_norms:
            lw.update(pn1=norm(), pn2=norm())
        layers.append(lw)
    top = {"embed": w(cfg.embed_qtype, V, D), "norm": norm(), "output": w(cfg.output_qtype, V, D)}
    full = {"layers": [{n: v[0] for n, v in lw.items()} for lw in layers], **{n: v[0] for n, v in top.items()}}
    ora = {"layers": [{n: v[1] for n, v in lw.items()} for lw in layers], "embed": top["embed"][1], "norm": top["norm"][1],
           "lm_head": top["output"][1]}
    return full, ora


def to_device(v):
    from xanosmerks_b200.ops import GGUFTensor
    if isinstance(v, dict):
        return {k: to_device(x) for k, x in v.items()}
    if isinstance(v, list):
        return [to_device(x) for x in v]
    return GGUFTensor(v[0].cuda(), v[1], v[2]) if isinstance(v, tuple) else v.cuda()


class Oracle(LlamaOracle):
    """The oracle with experts, norms behind blocks and a residual scale; remembers the narrowest choice of experts."""

    def __init__(self, cfg, weights, batch, max_ctx):
        super().__init__(cfg.reference_config(), weights, batch, max_ctx)
        self.more, self.margin = cfg, np.inf

    def mlp(self, w, h):
        if "moe" not in w:
            return (silu(h @ w["wg"].T) * (h @ w["wu"].T)) @ w["wd"].T
        gate, experts = w["moe"]
        x = h.reshape(-1, h.shape[-1])
        logit, k, out = x @ gate.T, self.more.num_experts_per_tok, np.zeros_like(x)
        order = np.sort(logit, -1)[:, ::-1]
        if k < logit.shape[1]:
            self.margin = min(self.margin, float((order[:, k - 1] - order[:, k]).min()))
        for t in range(len(x)):
            at = np.argsort(-logit[t], kind="stable")[:k]
            p = softmax(logit[t, at])
            for e, q in zip(at, p):
                ex = experts[e]
                out[t] += q * ((silu(x[t] @ ex["w1"].T) * (x[t] @ ex["w3"].T)) @ ex["w2"].T)
        return out.reshape(h.shape)

    def forward(self, ids, pos):
        eps, s = self.cfg["norm_eps"], np.float32(self.more.residual_scale)
        x = self.w["embed"][ids].astype(np.float32)
        for layer in range(self.cfg["num_layers"]):
            w = self.w["layers"][layer]
            y = self._attn(layer, rms_norm(x, w["n1"], eps), pos)
            x = x + s * (rms_norm(y, w["pn1"], eps) if "pn1" in w else y)
            y = self.mlp(w, rms_norm(x, w["n2"], eps))
            x = x + s * (rms_norm(y, w["pn2"], eps) if "pn2" in w else y)
        return rms_norm(x, self.w["norm"], eps) @ self.w["lm_head"].T


# config, batch, prompt, kv_type, seed (of weights and prompt)
CASES = [
    (dict(num_experts=4), 1, 5, None, 1),                                  # a prompt of a few tokens: steps
    (dict(num_experts=8, expert_qtype="Q6_K", post_norms=True, residual_scale=0.5), 3, 12, "F16", 1),
    (dict(num_experts=4, num_experts_per_tok=1), 2, 40, None, 1),            # more rows than a step takes
    (dict(num_experts=40, num_experts_per_tok=4, intermediate_size=256, num_layers=1), 2, 36, "F16", 1),   # several steps
    (dict(num_experts=3, num_experts_per_tok=3, residual_scale=1.5), 9, 9, "F16", 1),        # every expert; two steps
    (dict(post_norms=True, residual_scale=0.7), 2, 12, None, 1),             # no experts
    (dict(post_norms=True), 1, 6, "F16", 1),
]
STEPS = 4


def decoder(case):
    from xanosmerks_b200.llama import LlamaDecoder, LlamaWeights
    kw, batch, prompt, kv, seed = case
    cfg = config(**kw)
    full, ow = host_weights(cfg, seed)
    dec = LlamaDecoder(LlamaWeights.from_full(cfg, to_device(full)), batch=batch, max_ctx=64, kv_type=kv)
    ids = np.random.default_rng(seed).integers(0, cfg.vocab_size, size=(batch, prompt))
    return cfg, dec, Oracle(cfg, ow, batch, 64), ids


@pytest.mark.parametrize("case", CASES)
def test_decoder_matches_oracle(case):
    cfg, dec, ora, ids = decoder(case)
    nxt = dec.prefill(torch.from_numpy(ids)).cpu().numpy()
    ref = ora.forward(ids, 0)[:, -1, :]
    assert rel_err(dec.logits.cpu().numpy(), ref) < LOGIT_TOL, "prefill"
    pos = ids.shape[1]
    for step in range(STEPS):
        if step == 0:
            dec.decode_step()
            dec.length += 1
            dec.capture()
        else:
            dec.replay(1)
        ref = ora.forward(nxt[:, None], pos)[:, -1, :]
        pos += 1
        assert rel_err(dec.logits.cpu().numpy(), ref) < LOGIT_TOL, step
        got = dec.token_logprobs(top=3)
        nxt = dec.next_ids.cpu().numpy()
        assert np.array_equal(got.top_ids[:, 0].cpu().numpy(), nxt) and bool((got.rank == 0).all())
        assert torch.equal(got.top_logprobs[:, 0], got.logprob)
    assert ora.margin > MARGIN
    dec.check()


@pytest.mark.parametrize("case", [CASES[1], CASES[2], CASES[5]])
def test_score_matches_oracle(case):
    cfg, dec, ora, ids = decoder(case)
    logits = ora.forward(ids, 0).astype(np.float64)
    dec.SCORE_ROWS = 17                                      # several portions of logits
    got = dec.score(ids, top=4)
    B, S = ids.shape
    assert got.logprob.shape == got.entropy.shape == got.rank.shape == (B, S - 1) and got.top_ids.shape == (B, S - 1, 4)
    m = logits.max(-1, keepdims=True)
    lp = logits - m - np.log(np.exp(logits - m).sum(-1, keepdims=True))
    want = np.take_along_axis(lp[:, :-1], ids[:, 1:, None], -1)[..., 0]
    tol = 2 * LOGIT_TOL * np.abs(logits).max() + 1e-5
    assert np.abs(got.logprob.cpu().numpy() - want).max() < tol
    top = np.take_along_axis(lp[:, :-1], got.top_ids.cpu().numpy().astype(np.int64), -1)
    assert np.abs(got.top_logprobs.cpu().numpy() - top).max() < tol
    assert np.abs(top[..., 0] - lp[:, :-1].max(-1)).max() < tol
    # as a prompt goes on, and again with alternatives left out
    assert dec.length == 0
    again = dec.score(torch.from_numpy(ids))
    assert torch.equal(again.logprob, got.logprob) and again.top_ids is None
    with pytest.raises(ValueError):
        dec.score(ids[:, :1])


def test_tensor_parallel_shards_of_these_are_refused():
    from xanosmerks_b200.llama import LlamaWeights
    cfg = config(post_norms=True)
    full, _ = host_weights(cfg, 1)
    with pytest.raises(NotImplementedError):
        LlamaWeights.from_full(cfg, to_device(full), rank=0, world=2)
