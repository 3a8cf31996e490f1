"""Dropout on the CPU: the oracle's generator against published answers, the mask's statistics, the refusals of the
kernels' entry points."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from foldforge_amd import kernels
from oracle import training as oracle


def test_generator_gives_the_published_answers():
    """The known answers of Philox4x32-10 that its authors publish: all zeros, all ones, and digits of pi."""
    counter = np.array([[0] * 4, [0xFFFFFFFF] * 4, [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], dtype=np.uint64)
    want = [[0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8], [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD],
            [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]]
    for i, key in enumerate((0, 2**64 - 1, 0x299F31D0A4093822)):
        assert oracle.philox(counter[i:i + 1], key)[0].tolist() == want[i]


@pytest.mark.parametrize("p", [0.0, 0.1, 0.25, 0.5, 0.9, 1.0])
def test_mask_drops_its_rate(p):
    n = 1 << 17
    kept = oracle.dropout_mask((n,), None, p, 5, 9).double().mean().item()
    rate = round(65536 * p) / 65536
    assert abs(1 - kept - rate) <= 5 * math.sqrt(rate * (1 - rate) / n)


def test_masks_of_other_seeds_and_offsets_are_others():
    one = oracle.dropout_mask((4096,), None, 0.5, 1, 1)
    for seed, offset in ((2, 1), (1, 2), (1 + 2**32, 1), (1, 1 + 2**32)):
        same = (oracle.dropout_mask((4096,), None, 0.5, seed, offset) == one).double().mean().item()
        assert abs(same - 0.5) <= 5 * 0.5 / 64


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(kernels, "DEVICE_TYPE", "cpu")


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,how,message", [
    ((_x(4, 8, dtype=torch.float16),), {}, "bf16 or fp32"),
    ((_x(8, 4).T,), {}, "contiguous"),
    ((_x(4, 8), _x(4, 8, dtype=torch.float32)), {}, "residual"),
    ((_x(4, 8), _x(8, 4)), {}, "residual"),
    ((_x(4, 8), _x(8, 4).T), {}, "residual"),
    ((_x(4, 8),), {"p": -0.1}, "p must be"),
    ((_x(4, 8),), {"p": 1.5}, "p must be"),
    ((_x(4, 8),), {"p": math.nan}, "p must be"),
    ((_x(4, 8),), {"seed": -1}, "seed"),
    ((_x(4, 8),), {"seed": 2**63}, "seed"),
    ((_x(4, 8),), {"offset": -1}, "offset"),
    ((_x(4, 8),), {"offset": 2**63}, "offset"),
    ((_x(4, 8),), {"seed": torch.zeros(2)}, "seed"),
    ((_x(4, 8),), {"seed": torch.zeros(3, dtype=torch.int64)}, "seed"),
    ((_x(4, 8),), {"seed": torch.zeros(4, dtype=torch.int64)[::2]}, "seed"),
    ((_x(4, 8),), {"shared": 2}, "axis"),
    ((_x(4, 8),), {"shared": -3}, "axis"),
    ((_x(4, 8),), {"out": _x(4, 7)}, "out"),
    ((_x(4, 8),), {"out": _x(4, 8, dtype=torch.float32)}, "out"),
])
def test_refusals(on_cpu, args, how, message):
    with pytest.raises(ValueError, match=message):
        kernels.dropout_add(*args, **{"p": 0.1, "seed": 1, **how})


@pytest.mark.parametrize("which", ["update", "residual"])
def test_an_output_over_a_part_of_an_input_is_refused(on_cpu, which):
    memory = torch.zeros(100)
    args = {"update": torch.zeros(4, 8), "residual": torch.zeros(4, 8), which: memory[:32].view(4, 8)}
    for at in (1, 31):
        with pytest.raises(ValueError, match="overlaps " + which):
            kernels.dropout_add(**args, p=0.1, seed=1, out=memory[at:at + 32].view(4, 8))


def test_axes_of_the_mask():
    assert kernels.mask_axes((2, 3, 4, 5), None) == (1, 1, 120)
    assert kernels.mask_axes((2, 3, 4, 5), 1) == (2, 3, 20)
    assert kernels.mask_axes((2, 3, 4, 5), -2) == (6, 4, 5)
    assert kernels.mask_axes((2, 3, 4, 5), 3) == (24, 5, 1)
