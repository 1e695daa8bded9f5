"""The adapter and router-training calls beside autograd: results written in place count as changes of their tensor, the calls
work within a torch.autograd.Function, and the serving module takes activations that require a gradient."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import cuda_ok
from tests.test_gpu_lora import make

pytestmark = pytest.mark.gpu

if cuda_ok():
    from prismyra_b200 import ops, synth

DEV = "cuda:0"


@pytest.mark.parametrize("T", [7, 300])
def test_results_in_place_are_changes(T):
    c = make(T, 264, 136, 16, 3, "mixed")
    w = torch.ones(136, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = c["base"] * w  # keeps base for its backward
    ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"], out=c["base"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    before = c["gbase"]._version
    ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], base=c["gbase"], out=c["gbase"])
    assert c["gbase"]._version > before
    logits = torch.randn(T, 8, device=DEV)
    ids = torch.zeros(T, 1, dtype=torch.int32, device=DEV)
    before = logits._version
    ops.router_grad(logits, ids, torch.ones(T, 1, device=DEV), torch.ones(T, 1, device=DEV), out=logits)
    assert logits._version > before
    with torch.inference_mode():  # whose tensors count no versions
        held = torch.zeros(T, 136, device=DEV, dtype=torch.bfloat16)
        ops.lora(c["x"], c["a"], c["b"], c["adapter"], out=held)


class Adapted(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, base, adapter, scale):
        ctx.save_for_backward(x, a, b, adapter, scale)
        return ops.lora(x, a, b, adapter, scale, base=base)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, b, adapter, scale = ctx.saved_tensors
        dx, da, db = ops.lora_grad(dy.contiguous(), x, a, b, adapter, scale)
        return dx, da, db, dy, None, None


@pytest.mark.parametrize("T,R,N", [(24, 16, 2), (300, 16, 5), (1101, 64, 4)])
def test_within_an_autograd_function(T, R, N):
    c = make(T, 264, 136, R, N, "mixed")
    x, a, b, base = (c[n].clone().requires_grad_() for n in ("x", "a", "b", "base"))
    out = Adapted.apply(x, a, b, base, c["adapter"], c["scale"])
    assert torch.equal(out, ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"]))
    out.backward(c["dy"])
    for got, want in zip((x.grad, a.grad, b.grad), ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"])):
        assert torch.equal(got, want)
    assert torch.equal(base.grad, c["dy"])


def test_the_serving_module_takes_activations_that_require_a_gradient():
    from transformers.integrations.finegrained_fp8 import FP8Linear

    from prismyra_b200.kernels.qwen3_moe import AdaptedProjection, Fp8Linear

    c = make(40, 256, 512, 16, 4, "mixed")
    w, s = synth.quantize_fp8_blocks(torch.randn(512, 256, device=DEV) * 0.02)
    p = FP8Linear(256, 512, block_size=(128, 128))
    p.weight = torch.nn.Parameter(w, requires_grad=False)
    p.weight_scale_inv = torch.nn.Parameter(s, requires_grad=False)
    m = AdaptedProjection(Fp8Linear(p.to(DEV)), (c["a"], torch.nn.Parameter(c["b"]), c["scale"]))
    out = m(c["x"].clone().requires_grad_(), c["adapter"])
    assert not out.requires_grad and torch.equal(out, m(c["x"], c["adapter"]))
