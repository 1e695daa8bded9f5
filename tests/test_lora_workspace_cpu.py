"""ops.lora_workspace: as many bytes as the C ABI asks for, and always room for the status word."""

from __future__ import annotations

import pytest

from prismyra_b200 import _lib, ops


@pytest.mark.parametrize("sizes", [(1, 64, 64, 8, 1), (200, 64, 128, 8, 2), (5120, 2048, 4096, 64, 4), (0, 64, 64, 128, 3)])
@pytest.mark.parametrize("grad", [False, True])
def test_bytes(sizes, grad):
    n = _lib.load().pm_lora_workspace_bytes(*sizes, int(grad))
    assert ops.lora_workspace(*sizes, grad=grad, device="cpu").numel() == max(n, 16)
