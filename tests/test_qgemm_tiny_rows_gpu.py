"""GPU: the tensor-core GEMM on rows near fp32's smallest numbers (the reference's product, ops.py:62-67, has no range
of its own: a row is scaled by a power of two, and that power has to exist)."""

import numpy as np
import pytest
import torch

from oracle import gguf_dequant_oracle as O
from tests.helpers import GEMM_TOL
from xanosmerks_b200.ops import GGUFTensor, qlinear
from xanosmerks_b200.synth import make_weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["Q4_K", "Q6_K"])
def test_rows_near_the_smallest_numbers(name):
    m, n, k = 96, 256, 512
    raw = make_weight(name, n, k, seed=61)
    w = O.dequantize(raw, name, (n, k)).astype(np.float64)
    x = np.random.default_rng(62).standard_normal((m, k))
    x[:, ::7] = 0.0
    for r, s in enumerate((1e-33, 1e-34, 1e-35, 1e-36, 1e30)):
        x[r] *= s
    x = x.astype(np.float32)
    y = qlinear(GGUFTensor(raw, name, (n, k)), torch.from_numpy(x).cuda()).cpu().numpy().astype(np.float64)
    ref = x.astype(np.float64) @ w.T
    assert np.isfinite(y).all()
    for r in range(6):
        # (an output below 2^-126 is rounded to a multiple of 2^-149)
        assert np.abs(y[r] - ref[r]).max() <= GEMM_TOL * np.abs(ref[r]).max() + 2.0 ** -149, r
