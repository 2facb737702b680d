"""GPU: the decoder on a paged cache (fp16 and 4-bit, normalised heads), and sampled decoding, against the numpy
oracle on the same GGUF weights.  fp16 cache: the contiguous decoder's logit tolerance (fp16 keys, values and
attention output, 16-bit activation split).  4-bit cache: the oracle stores the values of Q4_0 blocks; the decoder's
keys and values differ from the oracle's by some 1e-4 of a block's range before they are rounded to codes, so one
in some 500 codes goes to the neighbour, a step of 1/8 of the block's largest value each: 0.6 % of the keys and values
in the mean square, a third of that in an attention output that averages them, and less in logits: 2e-2."""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as KO
from oracle.llama_oracle import LlamaOracle
from tests.helpers import rel_err
from tests.test_llama_gpu import LOGIT_TOL, oracle_weights
from xanosmerks_b200 import _lib
from xanosmerks_b200.llama import LlamaConfig, LlamaDecoder, LlamaWeights, synth_llama_weights

pytestmark = pytest.mark.gpu


class Q4Oracle(LlamaOracle):
    def stored(self, x):
        return KO.q4_values(*KO.q4_blocks(x)).astype(np.float32)


def make(cfg, seed=7):
    full = synth_llama_weights(cfg, seed=seed, device="cuda")
    w = oracle_weights(full)
    if cfg.qk_norm:
        for lw, src in zip(w["layers"], full["layers"]):
            lw["q_norm"], lw["k_norm"] = src["qn"].cpu().numpy(), src["kn"].cpu().numpy()
    return full, w


@pytest.mark.parametrize("kv,qk_norm,batch,layers,prompt,page", [
    ("F16", False, 1, 2, 11, 64), ("F16", True, 3, 1, 40, 16), ("Q4_0", False, 2, 1, 100, 64),
    ("Q4_0", True, 1, 2, 5, 32), ("Q4_0", False, 8, 1, 20, 16)])
def test_paged_decoder_matches_oracle(kv, qk_norm, batch, layers, prompt, page):
    cfg = LlamaConfig(num_layers=layers, vocab_size=4096, qk_norm=qk_norm)
    full, w = make(cfg)
    dec = LlamaDecoder(LlamaWeights.from_full(cfg, full), batch=batch, max_ctx=120, kv_type=kv, page_size=page)
    ora = (LlamaOracle if kv == "F16" else Q4Oracle)(cfg.reference_config(), w, batch=batch, max_ctx=120)
    tol = LOGIT_TOL if kv == "F16" else 2e-2
    ids = np.random.default_rng(8).integers(0, cfg.vocab_size, size=(batch, prompt))
    nxt = dec.prefill(torch.from_numpy(ids)).cpu().numpy()
    got, pos = dec.logits.cpu().numpy(), prompt
    assert rel_err(got, ora.forward(ids, 0)[:, -1, :]) < tol, "prefill"
    assert np.array_equal(nxt, got.argmax(-1))
    dec.decode_step()
    dec.length += 1
    for step in range(4):
        if step == 1:
            dec.capture()
        if step:
            dec.replay(1)
        ref = ora.forward(nxt[:, None], pos)[:, -1, :]
        pos += 1
        assert rel_err(dec.logits.cpu().numpy(), ref) < tol, step
        nxt = dec.next_ids.cpu().numpy()
    assert int(dec.pos0[0]) == pos and _lib.lib.xm_device_status(0) == 0


def test_paged_and_contiguous_decoders_agree():
    cfg = LlamaConfig(num_layers=2, vocab_size=4096)
    full = synth_llama_weights(cfg, seed=3, device="cuda")
    w = LlamaWeights.from_full(cfg, full)
    prompt = np.random.default_rng(4).integers(0, cfg.vocab_size, size=(2, 33))
    logits = []
    for kv in (None, "F16"):
        dec = LlamaDecoder(w, batch=2, max_ctx=64, kv_type=kv)
        dec.prefill(torch.from_numpy(prompt))
        logits.append(dec.logits.cpu().numpy().copy())
    assert rel_err(logits[1], logits[0]) < LOGIT_TOL


def test_heads_of_64_on_a_paged_cache():
    cfg = LlamaConfig(num_layers=1, vocab_size=2048, hidden_size=1024, num_heads=16, num_kv_heads=8, head_dim=64,
                      intermediate_size=2048)
    full, w = make(cfg)
    dec = LlamaDecoder(LlamaWeights.from_full(cfg, full), batch=2, max_ctx=64, kv_type="F16", page_size=16)
    ora = LlamaOracle(cfg.reference_config(), w, batch=2, max_ctx=64)
    ids = np.random.default_rng(5).integers(0, cfg.vocab_size, size=(2, 19))
    nxt = dec.prefill(torch.from_numpy(ids)).cpu().numpy()
    assert rel_err(dec.logits.cpu().numpy(), ora.forward(ids, 0)[:, -1, :]) < LOGIT_TOL
    dec.decode_step()
    assert rel_err(dec.logits.cpu().numpy(), ora.forward(nxt[:, None], 19)[:, -1, :]) < LOGIT_TOL


@pytest.mark.parametrize("kv", [None, "Q4_0"])
def test_sampled_generation(kv):
    cfg = LlamaConfig(num_layers=1, vocab_size=2048)
    full = synth_llama_weights(cfg, seed=3, device="cuda")
    dec = LlamaDecoder(LlamaWeights.from_full(cfg, full), batch=3, max_ctx=64, kv_type=kv)
    prompt = np.random.default_rng(4).integers(0, cfg.vocab_size, size=(3, 12))
    greedy = dec.generate(prompt, 6)
    dec.set_sampling(top_k=1)
    assert np.array_equal(dec.generate(prompt, 6), greedy)
    runs = []
    for seed, graph in ((1, True), (1, False), (2, True)):
        dec.set_sampling(temperature=1.5, top_p=0.95, min_p=1e-4, seed=seed)
        runs.append(dec.generate(prompt, 8, use_graph=graph))
    assert np.array_equal(runs[0], runs[1]) and not np.array_equal(runs[0], runs[2])
    assert ((0 <= runs[0]) & (runs[0] < cfg.vocab_size)).all()
    # the last step's token is the oracle's choice from the step's logits and numbers
    for b in range(3):
        tok, _ = KO.sample_row(dec.logits[b].cpu().numpy(), dec.u[b].item(), np.float32(1.5), 0, np.float32(0.95),
                               np.float32(1e-4))
        assert tok == runs[2][b, -1]
    dec.set_sampling(temperature=None)
    assert np.array_equal(dec.generate(prompt, 6), greedy)


def test_normalised_heads_need_a_paged_cache():
    cfg = LlamaConfig(num_layers=1, vocab_size=256, qk_norm=True)
    full = synth_llama_weights(cfg, seed=1, device="cuda")
    with pytest.raises(NotImplementedError, match="paged"):
        LlamaDecoder(LlamaWeights.from_full(cfg, full), batch=1, max_ctx=16)
