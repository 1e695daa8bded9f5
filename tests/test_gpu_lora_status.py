"""Whether a kernel of ops.lora or ops.lora_grad gave up on a bounded wait can be asked with ops.read_status, through a
workspace of the caller's.  No wait is made to run out here: the word is set from the host."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import cuda_ok
from tests.test_gpu_lora import make

pytestmark = pytest.mark.gpu

if cuda_ok():
    from prismyra_b200 import _lib, ops, synth

DEV = "cuda:0"


def status(ws):
    return ws[:4].view(torch.int32)


# one launch, groups of 16 rows, tiles; no rows
SHAPES = [(40, 264, 136, 16, 3), (300, 264, 136, 16, 5), (1101, 264, 136, 64, 4), (0, 64, 128, 16, 2), (0, 64, 128, 128, 2)]


@pytest.mark.parametrize("T,K,O,R,N", SHAPES)
def test_every_call_leaves_its_status(T, K, O, R, N):
    c = make(max(T, 1), K, O, R, N, "mixed")
    c = {k: v[:T] if k in ("x", "dy", "adapter", "base", "gbase") else v for k, v in c.items()}

    def forward(ws=None):
        return (ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"], workspace=ws),)

    def back(ws=None):
        return ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["gbase"], workspace=ws)

    for call, grad in ((forward, False), (back, True)):
        ws = ops.lora_workspace(T, K, O, R, N, grad=grad, device=DEV)
        want = call()
        for _ in range(2):
            status(ws).fill_(1)  # as a call that gave up would leave it: the next one starts at 0
            for u, v in zip(call(ws), want):
                assert torch.equal(u, v)
            ops.read_status(ws)
        status(ws).fill_(1)
        with pytest.raises(_lib.MoEKernelError) as e:
            ops.read_status(ws)
        assert e.value.status == _lib.PM_ERR_TIMEOUT


def test_workspaces_that_do_not_fit():
    c = make(300, 64, 128, 16, 2, "mixed")
    good = ops.lora_workspace(300, 64, 128, 16, 2, device=DEV)
    wide = torch.zeros(good.numel() + 16, dtype=torch.uint8, device=DEV)
    for bad in (good[:-16], good.cpu(), good.view(torch.int32), wide[8:8 + good.numel()], good[None], torch.zeros(0, dtype=torch.uint8, device=DEV)):
        with pytest.raises(ValueError):
            ops.lora(c["x"], c["a"], c["b"], c["adapter"], workspace=bad)
        with pytest.raises(ValueError):
            ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], workspace=bad)


def test_adapted_projections_take_workspaces():
    from transformers.integrations.finegrained_fp8 import FP8Linear

    from prismyra_b200.kernels.qwen3_moe import AdaptedProjection, Fp8Linear, FusedDenseProjection

    def projection(n, k):
        w, s = synth.quantize_fp8_blocks(torch.randn(n, k, device=DEV) * 0.02)
        m = FP8Linear(k, n, block_size=(128, 128))
        m.weight = torch.nn.Parameter(w, requires_grad=False)
        m.weight_scale_inv = torch.nn.Parameter(s, requires_grad=False)
        return Fp8Linear(m.to(DEV))

    T = 300
    c, d = make(T, 256, 512, 16, 4, "mixed"), make(T, 256, 256, 128, 4, "mixed")
    m = AdaptedProjection(FusedDenseProjection([projection(512, 256), projection(256, 256), projection(256, 256)]),
                          [(c["a"], c["b"], c["scale"]), None, (d["a"], d["b"])])
    ws = m.workspaces(T)
    assert ws[1] is None
    for u, v in zip(m(c["x"], c["adapter"], ws), m(c["x"], c["adapter"])):
        assert torch.equal(u, v)
    for w in (ws[0], ws[2]):
        ops.read_status(w)
