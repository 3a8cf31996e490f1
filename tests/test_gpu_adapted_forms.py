"""Projections with low-rank adapters: every instantiation of every form, each case with the form that it is meant for.

The form of a call shows in its workspace: one pass over the rows needs none forward and a slot of sums for each workgroup and
request backward; few rows keep their adapter's number and the fp32 row ``A x``; tiles keep more. A border that moves fails
here and does not take a kernel out of the tests. Tolerances: ``test_gpu_adapted``.
"""

from __future__ import annotations

import pytest
import torch

from foldforge_amd import _native, kernels
from oracle import training as oracle
from tests.test_gpu_adapted import (BF16, DEV, F32, HALF, backward, check_backward, check_forward, forward, gpu, make, near,
                                    rows_of)

pytestmark = pytest.mark.gpu


def _up(n: int) -> int:
    return (n + 255) // 256 * 256


def form(t: dict, direction: str) -> str:
    """The form of the call on ``t``."""
    q = kernels._adapted(*(t[k] for k in ("x", "weight", "bias", "down", "up", "scale", "offsets", "adapter")))
    size = getattr(_native.calls(), "ffk_adapted_linear" + ("_backward" if direction == "backward" else "") + "_workspace")(*q)
    if direction == "backward":
        slots = min((q.rows + 31) // 32, torch.cuda.get_device_properties(0).multi_processor_count) + q.requests
        return "rows" if size == _up(slots * 16 * (q.d_in + q.d_out) * 4) else "tiles"
    return "rows" if size == 0 else "few" if size == _up(4 * q.rows) + _up(4 * q.rows * q.rank) else "tiles"


def _lengths(rows: int, each: int) -> list[int]:
    """Requests of ``each`` rows and of none, one and a tile's rows, with padding behind them."""
    lengths = [0, 31, 33, 0, 1, 1, 64, 63, 2]
    left = rows - sum(lengths) - 11
    return lengths + [each] * (left // each) + [left % each]


#: channels in, outputs (a slice's width, or several slices of it); rank 16 and below, and above
ONE_PASS = [(64, 64), (64, 192), (64, 128), (64, 384), (64, 256), (64, 512), (128, 64), (128, 128), (128, 384), (128, 256),
            (128, 512), (128, 1024), (256, 64), (256, 128), (256, 256), (256, 512), (384, 128), (384, 256), (384, 1536),
            (512, 128), (512, 256)]
#: rows from which on one pass serves so many channels in: the last tile is not full
LEAST = {64: 1003, 128: 1003, 256: 12289, 384: 6151, 512: 12297}


@pytest.mark.parametrize("rank", [5, 16, 17, 32])
@pytest.mark.parametrize("d_in, d_out", ONE_PASS)
def test_one_pass(d_in, d_out, rank):
    rows = LEAST[d_in]
    for weight, adapter in ((BF16, BF16), (F32, F32)):
        t = make(rows, d_in, d_out, rank, 3, _lengths(rows, 1 + rows // 3), weight=weight, adapter=adapter, seed=d_out, bias=True)
        g = gpu(t)
        assert form(g, "forward") == "rows"
        check_forward(t, forward(g))


@pytest.mark.parametrize("adapter", [BF16, F32])
@pytest.mark.parametrize("d_in, d_out", [(64, 64), (64, 128), (128, 64), (64, 256), (256, 64), (128, 128), (128, 256), (256, 128),
                                         (128, 512), (512, 128), (256, 256)])
def test_one_pass_backward(d_in, d_out, adapter):
    rows = 8199 if d_in + d_out > 320 else 4103
    t = make(rows, d_in, d_out, 13, 3, _lengths(rows, 1 + rows // 3), adapter=adapter, seed=d_out)
    g = gpu(t)
    assert form(g, "backward") == "rows"
    check_backward(t, backward(g))


#: rows, d_in, d_out, rank: 16, 32, 64 and 128 channels of the rank, widths that are and are not multiples of 8 and of 64, few
#: and many output tiles
TILES = [(390, 449, 100, 9), (390, 72, 449, 16), (700, 384, 100, 30), (390, 449, 100, 20), (390, 449, 72, 50), (300, 101, 99, 65),
         (390, 72, 72, 50), (300, 192, 384, 128), (2100, 1000, 1024, 7), (4130, 449, 512, 31), (4130, 512, 449, 48),
         (4130, 512, 512, 100), (4130, 320, 512, 40)]


@pytest.mark.parametrize("weight, adapter", [(BF16, BF16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("rows, d_in, d_out, rank", TILES)
def test_tiles(rows, d_in, d_out, rank, weight, adapter):
    t = make(rows, d_in, d_out, rank, 4, _lengths(rows, 1 + rows // 5), weight=weight, adapter=adapter, seed=rank, bias=True)
    g = gpu(t)
    assert form(g, "forward") == "tiles" and form(g, "backward") == "tiles"
    check_forward(t, forward(g))
    check_backward(t, backward(g))


@pytest.mark.parametrize("weight, adapter", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows, d_in, d_out, rank", [(1, 384, 100, 8), (3, 449, 64, 128), (16, 101, 99, 3), (17, 384, 384, 33),
                                                     (40, 449, 100, 20), (256, 100, 72, 128), (257, 384, 384, 32),
                                                     (300, 449, 384, 5), (384, 768, 100, 16), (384, 72, 449, 31)])
def test_few_rows(rows, d_in, d_out, rank, weight, adapter):
    """``A x`` and the adapters in fp32 throughout: no rounding but W's (fp32 ones) and the result's."""
    lengths = [rows // 3, 0, rows // 3, 1] if rows > 3 else [1] * rows
    t = make(rows, d_in, d_out, rank, 3, lengths, weight=weight, adapter=adapter, seed=rank, bias=True)
    g = gpu(t)
    assert form(g, "forward") == "few"
    of, args = rows_of(t), [t[k] for k in ("x", "weight", "bias", "down", "up", "scale")]
    sizes = [a.abs() for a in args]
    want, mag = oracle.adapted_linear(*args, of), oracle.adapted_linear(*sizes, of)
    tol = (d_in + rank + 8) * 2.0**-24 * mag + HALF * want.abs()
    if weight == F32:
        tol = tol + HALF * (1 + HALF) * oracle.adapted_linear(*sizes, torch.full_like(of, -1))
    near(forward(g), want, tol, 1e-2, "y")


@pytest.mark.parametrize("rows, d_in, d_out, rank, served", [
    (385, 384, 384, 32, "tiles"), (257, 384, 384, 33, "tiles"), (257, 128, 512, 32, "rows"), (256, 128, 512, 32, "few"),
    (6143, 384, 384, 16, "tiles"), (6144, 384, 384, 16, "rows"), (12287, 512, 128, 16, "tiles"), (12288, 256, 256, 16, "rows")])
def test_borders(rows, d_in, d_out, rank, served):
    t = make(rows, d_in, d_out, rank, 2, [rows // 2, rows // 2 - 1])
    g = gpu(t)
    assert form(g, "forward") == served
    check_forward(t, forward(g))


def test_more_requests_than_one_pass_joins():
    """600 requests of pair rows: by tiles, and 512 of the same in one pass."""
    for requests, served in ((600, "tiles"), (512, "rows")):
        t = make(65536, 128, 256, 8, 5, [65536 // requests - 1] * requests, adapter=F32)
        g = gpu(t)
        assert form(g, "backward") == served
        check_backward(t, backward(g))


@pytest.mark.parametrize("rank, served", [(16, "rows"), (40, "tiles")])
def test_more_values_than_32_bits_count(rank, served):
    """Rows whose offsets pass 2^31 values (and 2^32 bytes): outputs and dx at the first rows, around 2^31 values and at the
    last; the gradients are sums of those rows, the others' inputs are zeros."""
    d_in, d_out, rows = 512, 128, 2**22 + 77
    windows = [range(0, 40), range(2**21 - 20, 2**21 + 20), range(2**22 - 33, 2**22 + 33), range(rows - 40, rows)]
    at = torch.tensor(sorted({r for w in windows for r in w}))
    t = make(len(at), d_in, d_out, rank, 2, [])
    g = gpu(t)
    for name, width in (("x", d_in), ("dy", d_out)):
        whole = torch.zeros(rows, width, dtype=BF16, device=DEV)
        whole[at.to(DEV)] = g[name]
        g[name] = whole
    ends = [0, 2**21 + 3, rows - 7]
    g["offsets"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
    g["adapter"] = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    assert form(g, "forward") == form(g, "backward") == served
    # the same rows alone, each request's in order
    t["offsets"] = torch.tensor([int((at < e).sum()) for e in ends], dtype=torch.int32)
    t["adapter"] = torch.tensor([1, 0], dtype=torch.int32)
    # (186 rows are looked at, which check_forward would take for a call that keeps A x in fp32; the call of 2^22 rows rounds it
    # to bf16: 2^-8 of each product of the adapter's part, beside the sums' and the result's own roundings)
    of, args = rows_of(t), [t[k] for k in ("x", "weight", "bias", "down", "up", "scale")]
    sizes = [None if a is None else a.abs() for a in args]
    want, mag = oracle.adapted_linear(*args, of), oracle.adapted_linear(*sizes, of)
    base = oracle.adapted_linear(*sizes, torch.full_like(of, -1))
    tol = (d_in + rank + 8) * 2.0**-24 * mag + HALF * want.abs() + HALF * (1 + 2 * HALF) * (mag - base)
    near(forward(g)[at.to(DEV)], want, tol, 1e-2, "y")
    got = backward(g)
    check_backward(t, kernels.AdaptedGradients(got.x[at.to(DEV)], got.down, got.up))
    assert int((got.x != 0).any(1).sum()) <= len(at)


@pytest.mark.parametrize("rows, d_in, d_out, each, served", [(16000, 64, 256, 32, "rows"), (16000, 128, 128, 32, "rows"),
                                                             (16031, 256, 192, 32, "rows"), (16016, 512, 128, 33, "rows"),
                                                             (15990, 128, 128, 63, "tiles"), (16000, 128, 512, 31, "tiles"),
                                                             (16000, 384, 384, 63, "tiles"), (6400, 384, 128, 64, "rows")])
def test_short_requests(rows, d_in, d_out, each, served):
    """Several requests to a tile, forward."""
    t = make(rows, d_in, d_out, 9, 5, [each] * (rows // each), adapter=F32)
    g = gpu(t)
    assert form(g, "forward") == served
    check_forward(t, forward(g))


@pytest.mark.parametrize("rows, d_in, d_out, each, served", [(4100, 64, 64, 48, "rows"), (8200, 128, 512, 48, "rows"),
                                                             (4100, 128, 128, 47, "tiles"), (8200, 512, 128, 50, "rows"),
                                                             (24600, 256, 256, 48, "rows")])
def test_short_requests_backward(rows, d_in, d_out, each, served):
    t = make(rows, d_in, d_out, 9, 5, [each] * (rows // each), adapter=F32)
    g = gpu(t)
    assert form(g, "backward") == served
    check_backward(t, backward(g))
