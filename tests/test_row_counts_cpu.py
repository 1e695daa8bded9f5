"""Row counts and widths that the C ABI's 32-bit int would wrap (2^32 + 5 rows as 5) are refused.  On tensors without memory, past the
checks of device and layout, which they cannot pass."""

from __future__ import annotations

import pytest
import torch

from prismyra_b200 import ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.fixture(autouse=True)
def layouts_pass(monkeypatch):
    def never(*a):
        raise AssertionError("the library was called")

    monkeypatch.setattr(ops, "_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_fits", lambda *a: 256)
    monkeypatch.setattr(ops, "_rows", lambda t, name, width, dev, rows=None, written=False: (256, t.shape[0], width))
    monkeypatch.setattr(ops, "_call_on", never)


@pytest.mark.parametrize("T", [(1 << 24) + 1, 2 ** 31, 2 ** 32 + 5])
def test_adapters(T):
    x, dy, ids = meta(T, 64), meta(T, 8), meta(T, dtype=torch.int32)
    a, b = meta(2, 8, 64), meta(2, 8, 8)
    with pytest.raises(ValueError, match="rows"):
        ops.lora(x, a, b, ids)
    with pytest.raises(ValueError, match="rows"):
        ops.lora_grad(dy, x, a, b, ids)


@pytest.mark.parametrize("K,O", [(2 ** 32 + 64, 8), (64, 2 ** 32 + 8)])
def test_adapter_widths(K, O):
    x, dy, ids = meta(4, K), meta(4, O), meta(4, dtype=torch.int32)
    a, b = meta(2, 8, K), meta(2, O, 8)
    with pytest.raises(ValueError, match="unsupported adapters"):
        ops.lora(x, a, b, ids)
    with pytest.raises(ValueError, match="unsupported adapters"):
        ops.lora_grad(dy, x, a, b, ids)


@pytest.mark.parametrize("T", [2 ** 31, 2 ** 32 + 5])
def test_router(T):
    logits, ids = meta(T, 1), meta(T, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        ops.router_balance(logits, ids)
    with pytest.raises(ValueError, match="rows"):
        ops.router_grad(logits, ids)
