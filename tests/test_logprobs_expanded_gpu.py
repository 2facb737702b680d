"""GPU: several tokens scored under one row of logits, or under rows that overlap."""

import pytest
import torch

from tests.test_logprobs_gpu import compare, make
from xanosmerks_b200.sampling import logprobs

pytestmark = pytest.mark.gpu


def test_many_tokens_under_one_row():
    x, _ = make(1, 5003, seed=1)
    t = torch.arange(0, 5000, 500, device="cuda")
    compare(x.expand(10, -1), t, top=3)
    got = logprobs(x.expand(10, -1), t)
    assert torch.equal(got.logprob, logprobs(x.repeat(10, 1), t).logprob)


def test_rows_that_overlap():
    x, _ = make(1, 4096, seed=2, dtype=torch.bfloat16)
    compare(x[0].as_strided((5, 1000), (37, 1)), torch.arange(5, device="cuda"), top=5)
