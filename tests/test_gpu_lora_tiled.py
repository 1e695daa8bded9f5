"""The tiled adapter kernels (tcgen05, 128 rows a block) beyond their values: in place and on strided and broadcast rows, without the
optional arguments, with values that are not finite, repeated and with the rows in another order, captured and replayed on new
inputs, and from two threads at once.  Every size is asserted to be one that goes to them in both directions."""

from __future__ import annotations

import threading

import pytest
import torch

from tests.conftest import cuda_ok
from tests.test_gpu_lora import _captured, check, check_grad, make

pytestmark = pytest.mark.gpu

if cuda_ok():
    from prismyra_b200 import _lib, ops

DEV = "cuda:0"
BF = torch.bfloat16
# odd numbers of rows; ranks of one and of two 64-column boxes, and one that is no multiple of 16; widths that fill no last tile
SIZES = [(1101, 264, 520, 64, 4), (3001, 136, 264, 24, 5), (1025, 520, 136, 128, 3)]
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def tiled(request):
    """Sizes are of the tiled kernels: their scratch holds the hidden rows, 4 bytes a rank, for the gradients twice."""
    T, K, O, R, N = request.getfixturevalue("size")
    hidden = (T // 128 + min(T, N)) * 128 * 4 * (-(-R // 16) * 16)
    f = _lib.load().pm_lora_workspace_bytes
    assert f(T, K, O, R, N, 0) >= hidden and f(T, K, O, R, N, 1) >= 2 * hidden


def both(c, base=True):
    return (ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"] if base else None),
            *ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["gbase"] if base else None))


def same(got, want):
    return all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("size", SIZES)
def test_in_place_and_strided_rows(size):
    T, K, O, R, N = size
    c = make(*size, "mixed")
    want = both(c)
    wide = {n: torch.randn(T + 3, c[n].shape[1] + 72, device=DEV).to(BF) for n in ("x", "base", "dy", "gbase")}
    part = {n: w[:T, 24:24 + c[n].shape[1]] for n, w in wide.items()}
    for n, p in part.items():
        p.copy_(c[n])
    before = {n: w.clone() for n, w in wide.items()}
    y, g = part["base"], part["gbase"]
    got = ops.lora(part["x"], c["a"], c["b"], c["adapter"], c["scale"], base=y, out=y)
    assert got.data_ptr() == y.data_ptr() and torch.equal(y, want[0])
    assert same(ops.lora_grad(part["dy"], part["x"], c["a"], c["b"], c["adapter"], c["scale"], base=g, out=g), want[1:])
    before["base"][:T, 24:24 + O], before["gbase"][:T, 24:24 + K] = want[0], want[1]
    for n, w in wide.items():
        assert torch.equal(w, before[n]), n
    # results elsewhere than base, with rows further apart
    out, dx = (torch.zeros(T + 1, w + 16, device=DEV, dtype=BF) for w in (O, K))
    ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"], out=out[:T, 8:8 + O])
    ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["gbase"], out=dx[:T, 8:8 + K])
    for wide_out, w, r in ((out, O, want[0]), (dx, K, want[1])):
        assert torch.equal(wide_out[:T, 8:8 + w], r)
        assert not wide_out[T:].any() and not wide_out[:, :8].any() and not wide_out[:, 8 + w:].any()


@pytest.mark.parametrize("size", SIZES)
def test_broadcast_rows(size):
    c = make(*size, "mixed")
    one = {n: c[n][:1].expand_as(c[n]) for n in ("x", "dy", "base", "gbase")}
    assert same(both(c | one), both(c | {n: t.contiguous() for n, t in one.items()}))


@pytest.mark.parametrize("size", SIZES)
def test_optional_arguments(size):
    c = make(*size, "mixed")
    plain = c | {"base": torch.zeros_like(c["base"]), "gbase": torch.zeros_like(c["gbase"]), "scale": torch.ones_like(c["scale"])}
    out = ops.lora(c["x"], c["a"], c["b"], c["adapter"])
    check(plain, out)
    got = ops.lora_grad(c["dy"], c["x"], c["a"], c["b"], c["adapter"])
    check_grad(plain, got)
    none = c["adapter"] < 0
    assert none.any() and not out[none].any() and not got[0][none].any()
    T, K, O = size[:3]
    if T % 5 == 0:
        assert torch.equal(ops.lora(c["x"].view(5, T // 5, K), c["a"], c["b"], c["adapter"], c["scale"],
                                    base=c["base"].view(5, T // 5, O)).view(T, O), both(c)[0])


@pytest.mark.parametrize("size", SIZES)
def test_values_that_are_not_finite_stay_in_their_rows(size):
    c = make(*size, "mixed")
    N = size[4]
    c["adapter"][0], c["adapter"][1], c["adapter"][2] = -1, 0, 1
    c["adapter"][3:] = torch.where(c["adapter"][3:] == 0, 1, c["adapter"][3:])  # row 1 is the only one of adapter 0,
    c["adapter"][3:] = torch.where(c["adapter"][3:] == N - 1, -1, c["adapter"][3:])  # no row has the last
    clean = both(c)
    d = {n: t.clone() for n, t in c.items()}
    d["x"][0], d["x"][1], d["dy"][0], d["dy"][1] = NAN, INF, INF, NAN
    d["base"][0, :4] = torch.tensor([INF, NAN, -0.0, 3.0e38], device=DEV)
    d["gbase"][0, :2] = torch.tensor([NAN, -INF], device=DEV)
    d["a"][N - 1], d["b"][N - 1] = NAN, INF
    out, dx, da, db = both(d)
    assert torch.equal(out[0].view(torch.int16), d["base"][0].view(torch.int16)) and not torch.isfinite(out[1]).any()
    assert torch.equal(dx[0].view(torch.int16), d["gbase"][0].view(torch.int16)) and not torch.isfinite(dx[1]).any()
    assert torch.equal(out[2:], clean[0][2:]) and torch.equal(dx[2:], clean[1][2:])
    for got, want in ((da, clean[2]), (db, clean[3])):
        assert not torch.isfinite(got[0]).any() and torch.equal(got[1:], want[1:]) and not got[N - 1].any()


@pytest.mark.parametrize("size", SIZES)
def test_repeats_and_row_order(size):
    T = size[0]
    c = make(*size, "runs")
    want = both(c)
    for _ in range(4):
        assert same(both(c), want)
    perm = torch.randperm(T, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    got = both({n: t[perm] if n in ("x", "dy", "adapter", "base", "gbase") else t for n, t in c.items()})
    assert torch.equal(want[0][perm], got[0]) and torch.equal(want[1][perm], got[1])


@pytest.mark.parametrize("size", SIZES)
def test_captured_calls_replay_on_new_inputs(size):
    """Two captured graphs, replayed at the same time on two streams, and then with the inputs of both exchanged: other values,
    another order of the adapters, other rows without one."""
    c, d = make(*size, "mixed"), make(*size, "runs", seed=9)
    want = {True: both(c), False: both(d)}
    held = [{n: t.clone() for n, t in c.items()} for _ in range(2)]
    graphs = [_captured(lambda h=h: both(h)) for h in held]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for first in (True, False, True):
        for h, mine in zip(held, (first, not first)):
            for n in h:
                h[n].copy_((c if mine else d)[n])
        torch.cuda.synchronize()
        for _ in range(3):
            for (graph, _out), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (_g, out), mine in zip(graphs, (first, not first)):
            assert same(out, want[mine])


@pytest.mark.parametrize("size", SIZES[:2])
def test_one_call_after_another_without_a_pause(size):
    """Forward and gradient calls back to back on one stream, each on the last one's results: a launch that started too early
    would read what its predecessor is still writing."""
    T, K, O, R, N = size
    c = make(*size, "mixed")
    b2, a2 = (c["b"].transpose(1, 2).contiguous(), c["a"].transpose(1, 2).contiguous())  # O -> K adapters

    def chain(pause):
        y = ops.lora(c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=c["base"])
        pause()
        z = ops.lora(y, b2, a2, c["adapter"], c["scale"], base=c["x"])
        pause()
        dy, db2, da2 = ops.lora_grad(c["gbase"], y, b2, a2, c["adapter"], c["scale"])
        pause()
        dx, da, db = ops.lora_grad(dy, c["x"], c["a"], c["b"], c["adapter"], c["scale"], base=z)
        pause()
        return y, z, dy, db2, da2, dx, da, db, ops.lora(dx, da, db, c["adapter"], c["scale"])

    want = chain(torch.cuda.synchronize)
    for _ in range(10):
        got = chain(lambda: None)
        for u, v in zip(got, want):
            assert torch.equal(u.view(torch.int16), v.view(torch.int16))


@pytest.mark.parametrize("size", SIZES[:2])
def test_two_threads_on_two_streams(size):
    cs = [make(*size, "runs", seed=i) for i in range(2)]
    want = [both(c) for c in cs]
    torch.cuda.synchronize()
    wrong = []

    def lane(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got = [both(cs[i]) for _ in range(10)]
                s.synchronize()
            wrong.extend(i for g in got if not same(g, want[i]))
        except Exception as e:  # pragma: no cover - reported below
            wrong.append(e)

    threads = [threading.Thread(target=lane, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    assert not wrong, wrong
