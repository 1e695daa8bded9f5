"""Which kernels a call takes, seen from the scratch it asks for: the tiled kernels keep the hidden rows there, 4 bytes for each rank
(of multiples of 16) of 128 rows of up to T / 128 + min(T, N) blocks; the kernel on groups of 16 rows does not."""

from __future__ import annotations

import pytest

from prismyra_b200 import _lib


def tiled(T, R, N):
    hidden = (T // 128 + min(T, N)) * 128 * 4 * (-(-R // 16) * 16)
    return _lib.load().pm_lora_workspace_bytes(T, 2048, 2048, R, N, 0) >= hidden


@pytest.mark.parametrize("T,R,N", [(5120, 64, 512), (16384, 64, 1024), (8192, 64, 512), (1100, 64, 4), (16384, 32, 16)])
def test_long_batches_are_tiled_however_many_adapters_are_loaded(T, R, N):
    assert tiled(T, R, N)


@pytest.mark.parametrize("T,R,N", [(512, 16, 512), (4096, 16, 1024), (1000, 64, 4), (731, 8, 12), (4096, 64, 1024)])
def test_few_rows_in_all_or_for_each_loaded_adapter_go_in_groups(T, R, N):
    assert not tiled(T, R, N)
