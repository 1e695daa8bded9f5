"""The C ABI refuses a result on top of base with another row distance (rows would be overwritten before they are read), and one on
top of an input, as the Python calls do.  Before any kernel: no device is needed."""

from __future__ import annotations

import ctypes

import pytest

from prismyra_b200 import _lib


def at(i):
    return ctypes.c_void_p(4096 * i)  # aligned addresses that no refused call reads


def lora(T, x=1, base=5, ldbase=128, out=6, ldout=128):
    return _lib.load().pm_lora(at(x), 64, at(2), at(3), at(4), None, at(base), ldbase, at(out), ldout, T, 64, 128, 8, 2, at(7),
                               1 << 30, None)


def lora_grad(T, dy=1, x=2, base=6, ldbase=64, dx=7, lddx=64):
    return _lib.load().pm_lora_grad(at(dy), 128, at(x), 64, at(3), at(4), at(5), None, at(base), ldbase, at(dx), lddx, at(8), at(9),
                                    T, 64, 128, 8, 2, at(10), 1 << 30, None)


@pytest.mark.parametrize("T", [2, 60, 300, 2000])
def test_results_on_top_of_inputs(T):
    assert lora(T, out=5, ldbase=136) == 1 and lora(T, out=5, ldout=256) == 1 and lora(T, out=1) == 1
    assert lora_grad(T, dx=6, ldbase=72) == 1 and lora_grad(T, dx=1, lddx=128) == 1 and lora_grad(T, dx=2) == 1
