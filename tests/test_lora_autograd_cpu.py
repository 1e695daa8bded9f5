"""ops.lora and ops.router_balance refuse tensors whose gradient autograd would lose in silence."""

from __future__ import annotations

import pytest
import torch

from prismyra_b200 import ops

BF = torch.bfloat16


def arguments():
    return dict(x=torch.zeros(4, 64, dtype=BF), a=torch.zeros(2, 8, 64, dtype=BF), b=torch.zeros(2, 128, 8, dtype=BF),
                adapter=torch.zeros(4, dtype=torch.int32), scale=torch.ones(2), base=torch.zeros(4, 128, dtype=BF),
                out=torch.zeros(4, 128, dtype=BF))


@pytest.mark.parametrize("name", ["x", "a", "b", "scale", "base", "out"])
def test_adapters(name):
    args = arguments()
    args[name].requires_grad_()
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        ops.lora(**args)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check, which host tensors do not pass
        ops.lora(**args)


def test_balance():
    logits, ids = torch.zeros(4, 8, requires_grad=True), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="logits requires a gradient"):
        ops.router_balance(logits, ids)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        ops.router_balance(logits, ids)
