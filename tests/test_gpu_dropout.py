"""Dropout's kernels against the 64-bit oracle.

The mask is compared exactly. A value has three fp32 roundings at most (the scale, its product, the sum) of 2^-24 of their
results, whose magnitudes |residual| + |scaled update| bounds, and the output's own of half a step.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from foldforge_amd import kernels
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _inputs(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (0.3 * torch.randn(*shape, generator=g)).to(dtype), torch.randn(*shape, generator=g).to(dtype)


def _check(got, x, res, shared, p, seed, offset):
    want = oracle.dropout_add(x, res, shared, p, seed, offset)
    drop = round(65536 * p)
    size = x.double().abs() * 65536 / max(65536 - drop, 1) + (0 if res is None else res.double().abs())
    tol = 3 * 2.0**-24 * size + torch.finfo(x.dtype).eps / 2 * want.abs()
    got = got.cpu()
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.double() - want).abs()
    assert not (off > tol).any(), (float(off.max()), int((off > tol).sum()))
    keep = oracle.dropout_mask(x.shape, shared, p, seed, offset).expand(x.shape)
    if res is None:
        assert torch.equal(got != 0, keep & (x != 0))


SHAPES = [((1,), None), ((7,), None), ((8,), None), ((384,), None), ((5, 451), None), ((33, 40, 64), None),
          ((2, 5, 7, 128), 1), ((2, 5, 7, 128), 2), ((1, 1, 9, 64), 1), ((1, 9, 1, 64), 2), ((3, 50, 11, 13), 1),
          ((3, 50, 11, 13), 2), ((3, 50, 11, 13), 0), ((3, 50, 11, 13), 3), ((2, 3, 301, 7), 2), ((1, 300, 70, 256), 1),
          ((40, 17, 8), -2), ((257, 3, 4099), 0), ((1, 37, 2, 2056), 1), ((600, 3), -1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape,shared", SHAPES)
def test_dropout_is_the_definition(shape, shared, dtype):
    x, res = _inputs(shape, dtype)
    how = dict(p=0.3, seed=123456789012345, offset=77, shared=shared)
    xg, rg = x.to(DEV), res.to(DEV)
    _check(kernels.dropout_add(xg, rg, **how), x, res, shared, 0.3, how["seed"], 77)
    back = kernels.dropout_backward(xg, **how)
    _check(back, x, None, shared, 0.3, how["seed"], 77)
    # in place
    assert torch.equal(kernels.dropout_add(xg.clone(), rg, **how), kernels.dropout_add(xg, rg, **how, out=rg))
    assert torch.equal(kernels.dropout_backward(xg, **how, out=xg), back)


@pytest.mark.parametrize("p", [0.0, 2.0**-18, 2.0**-16, 0.05, 0.5, 0.999, 1 - 2.0**-16, 1.0])
@pytest.mark.parametrize("shared", [None, 0])
def test_rates(p, shared):
    x, res = _inputs((9, 2049), F32)
    _check(kernels.dropout_add(x.to(DEV), res.to(DEV), p=p, seed=3, offset=4, shared=shared), x, res, shared, p, 3, 4)
    _check(kernels.dropout_backward(x.to(DEV), p=p, seed=3, offset=4, shared=shared), x, None, shared, p, 3, 4)


@pytest.mark.parametrize("seed,offset", [(0, 0), (2**63 - 1, 2**63 - 1), (2**32, 1), (1, 2**32), (2**32 - 1, 2**32 - 1)])
def test_seeds_and_offsets_use_all_their_bits(seed, offset):
    x, _ = _inputs((6, 777), BF16)
    for shared in (None, 0):
        _check(kernels.dropout_backward(x.to(DEV), p=0.5, seed=seed, offset=offset, shared=shared), x, None, shared, 0.5,
               seed, offset)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("skip", [1, 3, 8])
def test_rows_off_the_wide_alignment(dtype, skip):
    """Contiguous views whose storage begins between 16-byte places."""
    x, res = _inputs((4 * 6 * 64 + 16,), dtype)
    xg, rg = x.to(DEV), res.to(DEV)
    for shared in (None, 1):
        a, b = (t[skip:skip + 4 * 6 * 64].view(4, 6, 64) for t in (x, res))
        ag, bg = (t[skip:skip + 4 * 6 * 64].view(4, 6, 64) for t in (xg, rg))
        _check(kernels.dropout_add(ag, bg, p=0.4, seed=8, offset=1, shared=shared), a, b, shared, 0.4, 8, 1)


@pytest.mark.parametrize("shared", [None, 0])
def test_a_dropped_value_does_not_reach_the_result(shared):
    x = torch.full((16, 512), float("nan"))
    x[:, ::2] = float("inf")
    res = torch.randn(16, 512, generator=torch.Generator().manual_seed(1))
    keep = oracle.dropout_mask(x.shape, shared, 0.5, 21, 0).expand(x.shape)
    for dtype in (BF16, F32):
        got = kernels.dropout_add(x.to(DEV, dtype), res.to(DEV, dtype), p=0.5, seed=21, shared=shared).cpu()
        assert torch.equal(got[~keep], res.to(dtype)[~keep])
        assert not torch.isfinite(got[keep]).any()


def test_values_far_apart_stay_apart():
    """The largest values: no step between overflows that the result does not."""
    big = torch.finfo(F32).max
    x = torch.full((64,), big / 4)
    _check(kernels.dropout_add(x.to(DEV), -x.to(DEV), p=0.5, seed=2), x, -x, None, 0.5, 2, 0)


def test_an_empty_tensor_and_one_row():
    for shape in ((0, 64), (4, 0, 64)):
        x = torch.empty(shape, dtype=BF16, device=DEV)
        assert kernels.dropout_add(x, x, p=0.5, seed=1, shared=0).shape == shape


def test_captured_calls_draw_anew_at_each_replay():
    """A seed on the device is read at each replay; other work goes on between them."""
    x, res = _inputs((3, 40, 64), BF16)
    xg, rg = x.to(DEV), res.to(DEV)
    state = torch.tensor([99, 0], dtype=torch.int64, device=DEV)
    y, dx = torch.empty_like(xg), torch.empty_like(xg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.dropout_add(xg, rg, p=0.25, seed=state, offset=5, shared=1, out=y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.dropout_add(xg, rg, p=0.25, seed=state, offset=5, shared=1, out=y)
        kernels.dropout_backward(rg, p=0.25, seed=state, offset=6, out=dx)
        state[1:].add_(16)
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        _check(y, x, res, 1, 0.25, 99, 5 + 16 * step)
        _check(dx, res, None, None, 0.25, 99, 6 + 16 * step)
        assert torch.equal(y, kernels.dropout_add(xg, rg, p=0.25, seed=99, offset=5 + 16 * step, shared=1))


def test_a_seed_on_the_device_is_the_same_draw():
    x, res = _inputs((5, 451), F32)
    state = torch.tensor([31, 2**40], dtype=torch.int64, device=DEV)
    for shared in (None, 0):
        assert torch.equal(kernels.dropout_add(x.to(DEV), res.to(DEV), p=0.1, seed=state, offset=3, shared=shared),
                           kernels.dropout_add(x.to(DEV), res.to(DEV), p=0.1, seed=31, offset=2**40 + 3, shared=shared))


def test_two_streams_at_once():
    x, res = _inputs((64, 64, 128), BF16)
    xg, rg = x.to(DEV), res.to(DEV)
    want = [kernels.dropout_add(xg, rg, p=0.25, seed=4, offset=i, shared=1) for i in range(2)]
    torch.cuda.synchronize()
    got, streams = [None, None], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = kernels.dropout_add(xg, rg, p=0.25, seed=4, offset=i, shared=1)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shape, shared", [((2**31 + 4099,), None), ((1, 2, 2**31 + 1001), 1), ((2, 3, 2**30 + 8), 1)])
def test_more_values_than_32_bits_count(shape, shared):
    """Places and mask numbers behind 2^31, in place, at both ends and around the powers of two."""
    x = torch.ones(shape, dtype=BF16, device=DEV)
    assert kernels.dropout_backward(x, p=0.5, seed=2**40 + 3, offset=9, shared=shared, out=x) is x
    flat, n = x.view(-1), x.numel()
    inner = shape[-1] if shared is not None else n
    for begin in (0, 2**30 - 50, 2**31 - 50, 2**32 - 50, inner - 60, inner * shape[0] - 60, n - 100):
        if not 0 <= begin < n - 1:
            continue
        place = torch.arange(begin, min(begin + 100, n))
        row, col = place // inner, place % inner
        number = col if shared is None else row // shape[1] * inner + col  # of the mask
        block = (number >> 3).numpy().astype("uint64")
        counter = np.stack([block % 2**32, block // 2**32, np.full_like(block, 9), np.zeros_like(block)], 1)
        words = oracle.philox(counter, 2**40 + 3)
        halves = np.stack([words % 2**16, words // 2**16], 2).reshape(-1, 8)
        keep = torch.from_numpy(halves[np.arange(len(place)), (number & 7).numpy()] >= 32768)
        assert torch.equal(flat[begin:begin + len(place)].cpu(), 2.0 * keep.to(BF16)), begin
