"""GPU: scoring sequences changes nothing that later tokens depend on."""

import numpy as np
import pytest
import torch

from tests.test_llama_moe_gpu import decoder

pytestmark = pytest.mark.gpu
CASE = (dict(post_norms=True), 2, 12, None, 1)


def test_sampled_tokens_go_on_as_without_a_score():
    cfg, dec, _, ids = decoder(CASE)
    prompt, seen = torch.from_numpy(ids), []
    for between in (False, True):
        dec.set_sampling(temperature=3.0, seed=5)
        first = dec.generate(prompt, 6)
        if between:
            dec.score(prompt, top=2)
            dec.score(prompt[:, :5])
        seen.append((first, dec.generate(prompt, 6)))
    assert np.array_equal(seen[0][0], seen[1][0]) and np.array_equal(seen[0][1], seen[1][1])
    assert not np.array_equal(seen[0][0], seen[0][1])          # (other numbers in the second: the test tells them apart)


def test_a_refused_score_leaves_the_decoder_as_it_was():
    cfg, dec, _, ids = decoder(CASE)
    prompt = torch.from_numpy(ids)
    want = dec.generate(prompt, 6)
    dec.reset()
    got = [dec.prefill(prompt).cpu().numpy()]
    dec.decode_step()
    dec.length += 1
    got.append(dec.next_ids.cpu().numpy())
    dec.capture()
    bad = prompt.clone()
    bad[1, 3] = cfg.vocab_size
    for args in ((prompt[:, :1],), (prompt[:1],), (prompt.repeat(1, 6),), (bad,), (-bad,), (prompt, 1.0, 65), (prompt, 1.0, -1)):
        with pytest.raises(ValueError):
            dec.score(*args)
    assert dec.length == 13 and dec.graph is not None
    for _ in range(4):
        dec.replay(1)
        got.append(dec.next_ids.cpu().numpy())
    assert np.array_equal(np.stack(got, 1), want)
