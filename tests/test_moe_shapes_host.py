"""CPU: experts whose shapes or devices do not go together are refused before anything of the layer is on a device."""

import pytest
import torch

from xanosmerks_b200 import qtypes
from xanosmerks_b200._lib import XMError
from xanosmerks_b200.moe import MoELayer
from xanosmerks_b200.ops import GGUFTensor

E, H, F = 3, 512, 256


def weight(n, k, device="cpu"):
    w = object.__new__(GGUFTensor)                    # (its constructor takes CUDA tensors alone)
    w.qtype, w.shape = qtypes.normalize("Q4_K"), (n, k)
    w.data = torch.empty(qtypes.row_bytes(w.qtype, k) * n, dtype=torch.uint8, device=device)
    return w


def layer(gate=(E, H), **other):
    """A layer with the weights `other` ("w1_2": of expert 2) in the place of the right ones."""
    shape = {"w1": (F, H), "w2": (H, F), "w3": (F, H)}
    return MoELayer({"num_experts": E, "num_experts_per_tok": 2}, {
        "gate": {"weight": torch.zeros(gate)},
        "experts": {str(i): {n: {"weight": other.get(f"{n}_{i}") or weight(*s)} for n, s in shape.items()} for i in range(E)}})


@pytest.mark.parametrize("name,shape", [
    ("w1_1", (F - 128, H)), ("w3_0", (F - 128, H)), ("w3_2", (F, H - 256)), ("w2_1", (H - 256, F)), ("w2_0", (F, H)),
    ("w1_2", (H, F)), ("w1_0", (2 * F, H)),            # (the first expert's w1 says what F is: then the others are wrong)
])
def test_shapes(name, shape):
    with pytest.raises(ValueError, match="of expert"):
        layer(**{name: weight(*shape)})


def test_gate():
    for gate in ((E - 1, H), (E + 1, H)):
        with pytest.raises(ValueError, match="gate.weight has"):
            layer(gate=gate)
    with pytest.raises(ValueError, match="of expert"):
        layer(gate=(E, H + 256))


def test_device():
    with pytest.raises(ValueError, match="of expert 2"):
        layer(w3_2=weight(F, H, device="meta"))


def test_a_layer_without_steps_table(monkeypatch):
    """Where the table of the step cannot be made, the layer is there for the block of many tokens."""
    def fails(self):
        raise XMError("moe step: tensor map")
    monkeypatch.setattr(MoELayer, "_step_table", fails)
    made = layer()
    assert made._table is None and made.hidden == H
    with pytest.raises(XMError):
        made.step(torch.zeros(1, H))
