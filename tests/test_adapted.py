"""Projections with low-rank adapters on the CPU: the oracle against autograd, the refusals of the entry points, the
workspace's sizes."""

from __future__ import annotations

import pytest
import torch

from foldforge_amd import _native, kernels
from oracle import training as oracle


def _call(rows=6, d_in=16, d_out=24, rank=4, n=3, requests=2, dtype=torch.bfloat16):
    return dict(x=torch.zeros(rows, d_in, dtype=torch.bfloat16), weight=torch.zeros(d_out, d_in, dtype=dtype),
                bias=None, down=torch.zeros(n, rank, d_in, dtype=dtype), up=torch.zeros(n, d_out, rank, dtype=dtype),
                scale=torch.ones(n), offsets=torch.zeros(requests + 1, dtype=torch.int32),
                adapter=torch.zeros(requests, dtype=torch.int32))


def test_oracle_against_autograd():
    g = torch.Generator().manual_seed(0)
    x, w, down, up = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((9, 5), (7, 5), (3, 2, 5), (3, 7, 2)))
    bias, scale, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((7,), (3,), (9, 7)))
    offsets, adapter = torch.tensor([1, 4, 4, 8]), torch.tensor([2, 0, 1])
    of = oracle.adapter_of_rows(9, offsets, adapter, 3)
    assert of.tolist() == [-1, 2, 2, 2, 1, 1, 1, 1, -1]
    leaves = [t.clone().requires_grad_(True) for t in (x, down, up)]
    rows = []
    for i, a in enumerate(of.tolist()):
        y = w @ leaves[0][i] + bias
        rows.append(y if a < 0 else y + scale[a] * leaves[2][a] @ (leaves[1][a] @ leaves[0][i]))
    y = torch.stack(rows)
    assert torch.allclose(oracle.adapted_linear(x, w, bias, down, up, scale, of), y.detach(), rtol=1e-12, atol=1e-12)
    y.backward(dy)
    for got, leaf in zip(oracle.adapted_linear_backward(dy, x, w, down, up, scale, of), leaves):
        assert torch.allclose(got, leaf.grad, rtol=1e-12, atol=1e-12)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(kernels, "DEVICE_TYPE", "cpu")


BAD = [
    ({"x": torch.zeros(6, 16)}, "bf16"),
    ({"x": torch.zeros(16, 6, dtype=torch.bfloat16).T}, "contiguous"),
    ({"x": torch.zeros(6, 12, dtype=torch.bfloat16)}, "d_in"),
    ({"x": torch.zeros(6 * 16 + 1, dtype=torch.bfloat16)[1:].view(6, 16)}, "aligned"),
    ({"weight": torch.zeros(24, 16, dtype=torch.float16)}, "bf16 or fp32"),
    ({"weight": torch.zeros(16, 24, dtype=torch.bfloat16).T}, "contiguous"),
    ({"weight": torch.zeros(24 * 16)}, "2 axes"),
    ({"down": torch.zeros(3, 4, 12, dtype=torch.bfloat16)}, "d_in"),
    ({"down": torch.zeros(3, 4, 16)}, "one type"),
    ({"up": torch.zeros(3, 24, 5, dtype=torch.bfloat16)}, "rank"),
    ({"up": torch.zeros(2, 24, 4, dtype=torch.bfloat16)}, "adapters"),
    ({"down": torch.zeros(3, 129, 16, dtype=torch.bfloat16), "up": torch.zeros(3, 24, 129, dtype=torch.bfloat16)}, "rank"),
    ({"down": torch.zeros(0, 4, 16, dtype=torch.bfloat16), "up": torch.zeros(0, 24, 4, dtype=torch.bfloat16),
      "scale": None}, "adapters"),
    ({"scale": torch.ones(2)}, "scale"),
    ({"scale": torch.ones(6)[::2]}, "scale"),
    ({"scale": torch.ones(3, dtype=torch.float64)}, "scale"),
    ({"offsets": torch.zeros(2, dtype=torch.int32)}, "offsets"),
    ({"offsets": torch.zeros(3, dtype=torch.int64)}, "offsets"),
    ({"offsets": torch.zeros(6, dtype=torch.int32)[::2]}, "offsets"),
    ({"adapter": torch.zeros(2, 1, dtype=torch.int32)}, "adapter"),
    ({"adapter": torch.zeros(2, dtype=torch.int64)}, "adapter"),
]


@pytest.mark.parametrize("change,message", BAD + [({"bias": torch.zeros(23)}, "bias"),
                                                  ({"bias": torch.zeros(48)[::2]}, "bias"),
                                                  ({"out": torch.zeros(6, 24)}, "out"),
                                                  ({"out": torch.zeros(24, 6, dtype=torch.bfloat16).T}, "out")])
def test_forward_refusals(on_cpu, change, message):
    args = {**_call(), **change}
    with pytest.raises(ValueError, match=message):
        kernels.adapted_linear(args.pop("x"), args.pop("weight"), args.pop("bias"), **args)


@pytest.mark.parametrize("change,message", BAD + [({"dy": torch.zeros(6, 24)}, "dy"),
                                                  ({"dy": torch.zeros(6, 16, dtype=torch.bfloat16)}, "dy"),
                                                  ({"dy": torch.zeros(24, 6, dtype=torch.bfloat16).T}, "dy"),
                                                  ({"grad_dtype": torch.float16}, "grad_dtype")])
def test_backward_refusals(on_cpu, change, message):
    args = {"dy": torch.zeros(6, 24, dtype=torch.bfloat16), **_call(), **change}
    args.pop("bias")
    if tuple(args["x"].shape) != (6, 16) or args["x"].dtype != torch.bfloat16:
        args["dy"] = torch.zeros(*args["x"].shape[:-1], 24, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=message):
        kernels.adapted_linear_backward(args.pop("dy"), args.pop("x"), args.pop("weight"), **args)


def test_an_output_over_the_input_is_refused(on_cpu, monkeypatch):
    memory = torch.zeros(400, dtype=torch.bfloat16)
    args = {**_call(d_in=24), "x": memory[:144].view(6, 24)}
    with pytest.raises(ValueError, match="overlap"):
        kernels.adapted_linear(args.pop("x"), args.pop("weight"), out=memory[8:152].view(6, 24), **{**args, "bias": None})


def test_sizes_that_are_served():
    assert kernels.adapted_linear_supported(1, 1, 1) and kernels.adapted_linear_supported(449, 384, 64, 65535)
    for d_in, d_out, rank, n in ((0, 8, 4, 1), (8, 65537, 4, 1), (8, 8, 0, 1), (8, 8, 129, 1), (8, 8, 4, 65536),
                                 (65536, 8, 128, 4096)):
        assert not kernels.adapted_linear_supported(d_in, d_out, rank, n)


def test_calls_of_more_workgroups_than_a_launch_has():
    """2^24 workgroups of 256 threads are more than a launch takes: such a call is refused (its workspace is 0) before
    anything runs, the largest below it is not."""
    lib = _native.lib()
    forward, backward = lib.ffk_adapted_linear_workspace, lib.ffk_adapted_linear_backward_workspace
    bf16 = (0, 0)
    # 16 rows a workgroup for the thin products (four of them where requests are short), forward and of both matrices backward
    assert forward(2**27, 64, 64, 1, 48, 1, *bf16) > 0 and forward(2**28, 64, 64, 1, 48, 1, *bf16) == 0
    assert forward(2**25, 64, 64, 1, 48, 2**25, *bf16) > 0 and forward(2**26, 64, 64, 1, 48, 2**26, *bf16) == 0
    assert backward(2**26, 64, 64, 1, 48, 1, *bf16) > 0 and backward(2**27, 64, 64, 1, 48, 1, *bf16) == 0
    # a sum of every adapter in each 16384 rows
    assert backward(2**19, 72, 72, 65535, 1, 16, *bf16) > 0 and backward(2**20, 72, 72, 65535, 1, 16, *bf16) == 0
    # and the join of those sums
    assert backward(2**15, 8192, 8192, 1000, 64, 16, *bf16) > 0 and backward(2**15, 8192, 8192, 1000, 128, 16, *bf16) == 0


def test_as_many_requests_as_are_counted_in_32_bits():
    """The passes over the offsets go on in steps of 256: a count next to 2^31 would run over and never end."""
    lib = _native.lib()
    for size in (lib.ffk_adapted_linear_workspace, lib.ffk_adapted_linear_backward_workspace):
        assert size(1000, 72, 72, 1, 4, 2**31 - 2000, 0, 0) > 0
        assert size(1000, 72, 72, 1, 4, 2**31 - 1, 0, 0) == 0
