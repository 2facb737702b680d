"""CPU: shards of models whose blocks are not summed into the stream as they are."""

import pytest

from xanosmerks_b200.llama import LlamaConfig, LlamaWeights

SIZES = dict(num_layers=2, hidden_size=512, num_heads=4, num_kv_heads=2, intermediate_size=768, vocab_size=1000)


@pytest.mark.parametrize("kw", [dict(num_experts=4), dict(post_norms=True), dict(residual_scale=0.5)])
def test_shards_are_refused_however_they_are_made(kw):
    cfg = LlamaConfig(**SIZES, **kw)
    with pytest.raises(NotImplementedError):
        LlamaWeights(cfg, None, [], None, None, rank=1, world=2)
    with pytest.raises(NotImplementedError):
        LlamaWeights.from_full(cfg, {}, rank=0, world=2)
    assert LlamaWeights(cfg, None, [], None, None).world == 1


def test_plain_shards_are_not():
    assert LlamaWeights(LlamaConfig(**SIZES), None, [], None, None, rank=1, world=2).rank == 1
