"""Infinite weights, activations and gradients of live rows in ops.lora and ops.lora_grad: the results are infinite (with their
sign) or NaN exactly where the definition in 64 bits is, and elsewhere as near to it as ever (the bound of
tests/test_gpu_lora.py).  The values between the two products travel as two halves; each half alone times an infinity would be
NaN or the other infinity.

Every path: one launch, groups of 16 rows and 128-row tiles, forward and gradient."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import cuda_ok
from tests.test_gpu_lora import definition, definition_grad, make

pytestmark = pytest.mark.gpu

if cuda_ok():
    from prismyra_b200 import ops

INF = float("inf")


def same(got, want, size, terms, what):
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want)), (what, "NaN")
    inf = torch.isinf(want)
    assert torch.equal(g[inf], want[inf]), (what, "infinite")
    ok = torch.isfinite(want)
    bound = 2.0 ** -8 * want[ok].abs() + (2.0 ** -16 + (terms + 8) * 2.0 ** -23) * size[ok] * (1 + 2.0 ** -8) + 1e-37
    worst = ((g[ok] - want[ok]).abs() / bound).max().item()
    assert worst <= 1.0, (what, worst)


# one launch at every tile of ranks; groups of 16 rows (gradients: with and without warps that share a block); tiles
SHAPES = [(40, 264, 136, 8, 3), (40, 264, 136, 16, 3), (40, 136, 264, 32, 3), (31, 264, 136, 64, 2), (40, 264, 136, 128, 3),
          (300, 264, 136, 8, 5), (300, 264, 520, 16, 5), (300, 264, 520, 16, 100), (400, 136, 264, 32, 5),
          (200, 264, 136, 128, 3), (700, 264, 136, 24, 4), (1101, 264, 520, 64, 4), (1101, 136, 264, 128, 3),
          (4200, 264, 520, 40, 2)]


@pytest.mark.parametrize("where", ["a", "b", "x", "dy", "several"])
@pytest.mark.parametrize("T,K,O,R,N", SHAPES)
def test_infinite_operands(T, K, O, R, N, where):
    c = make(T, K, O, R, N, "mixed")
    row = T // 2
    c["adapter"][row] = n = N - 1
    if where == "a":
        c["a"][n, 3, 17] = INF
    elif where == "b":
        c["b"][n, 21, 5] = -INF
    elif where == "x":
        c["x"][row, 9] = INF
    elif where == "dy":
        c["dy"][row, 33] = -INF
    else:  # of one sign and of both, in the first and last columns
        c["b"][n, 0, 0] = c["b"][n, 0, 1] = c["b"][n, O - 1, R - 1] = INF
        c["a"][n, 0, K - 1], c["x"][row, K - 2], c["dy"][row, O - 1] = -INF, -INF, INF
    mags = {k: v.abs() if v.is_floating_point() else v for k, v in c.items()}

    def forward(c):
        return definition(c["x"], c["a"], c["b"], c["adapter"], c["scale"], c["base"])

    def grads(c):
        return definition_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"], c["gbase"])

    want = forward(c)
    assert not torch.isfinite(want).all() or where == "dy"
    same(ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"]), want, forward(mags), K + R, "out")
    got = ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["gbase"])
    want = grads(c)
    assert not all(torch.isfinite(w).all() for w in want)
    for name, g, w, s, terms in zip(("dx", "da", "db"), got, want, grads(mags), (O + R, O + T, K + T)):
        same(g, w, s, terms, name)
