"""GPU: the norm between blocks on a part of each sequence of a longer buffer, in place too.  Tolerances: those derived in
tests/test_residual_norm_gpu.py."""

import pytest
import torch

from tests.test_residual_norm_gpu import compare, make
from xanosmerks_b200.ops import residual_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_part_of_each_sequence_in_place(dtype):
    s, y, post, pre = make((3, 7, 512), seed=1, stream=dtype, y=dtype)
    long = torch.full((3, 12, 512), 5.0, dtype=dtype, device="cuda")
    part = long[:, 2:9]
    part.copy_(s)
    want = compare(s, y, post=post, pre=pre, scale=0.5)
    got = residual_norm(part, y, post_weight=post, pre_weight=pre, scale=0.5, out=part)
    assert got[0] is part and torch.equal(part, want[0]) and torch.equal(got[1], want[1])
    assert bool((long[:, :2] == 5).all()) and bool((long[:, 9:] == 5).all())


def test_another_tensor_s_part_and_rows_that_lie_on_one_another():
    s, y, post, pre = make((2, 4, 3, 256), seed=2)
    out = torch.zeros(2, 5, 6, 256, device="cuda")
    got = residual_norm(s, y, pre_weight=pre, out=out[:, 1:, ::2])
    want = residual_norm(s, y, pre_weight=pre)
    assert torch.equal(out[:, 1:, ::2], want[0]) and torch.equal(got[1], want[1])
    assert bool((out[:, 0] == 0).all()) and bool((out[:, :, 1::2] == 0).all())
    flat = torch.zeros(1, 1, 256, device="cuda").expand(3, 7, 256)
    with pytest.raises((ValueError, RuntimeError)):
        residual_norm(torch.zeros(3, 7, 256, device="cuda"), torch.zeros(3, 7, 256, device="cuda"), out=flat)
    empty = torch.zeros(3, 7, 256, device="cuda")[:, :0]
    assert residual_norm(empty, empty, pre_weight=pre, out=empty)[0] is empty
