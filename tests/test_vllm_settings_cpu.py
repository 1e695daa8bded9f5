"""A test that sets one of vLLM's environment variables gets that setting, whatever tests before it asked vLLM (which keeps its
first answer for the life of the process).  With a stand-in for the module, so it needs neither vLLM nor a GPU."""

from __future__ import annotations

import functools
import os
import sys
import types

import pytest

NAME = "vllm.utils.deep_gemm"


@pytest.fixture(scope="module")
def stand_in():
    module = types.ModuleType(NAME)
    module.is_deep_gemm_e8m0_used = functools.cache(lambda: os.environ["VLLM_USE_DEEP_GEMM_E8M0"] == "1")
    before = sys.modules.get(NAME)
    sys.modules[NAME] = module
    yield module
    if before is None:
        del sys.modules[NAME]
    else:
        sys.modules[NAME] = before


@pytest.mark.parametrize("value", ["0", "1", "0"])
def test_each_test_has_its_own_setting(stand_in, monkeypatch, value):
    monkeypatch.setenv("VLLM_USE_DEEP_GEMM_E8M0", value)
    assert stand_in.is_deep_gemm_e8m0_used() == (value == "1")
