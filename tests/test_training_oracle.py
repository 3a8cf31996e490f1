"""The 64-bit training oracle on the CPU: against autograd, differences and torch's own e4m3."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle import training as oracle


def test_e4m3_is_torchs():
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randn(4000, generator=g) * 2.0 ** torch.randint(-12, 7, (4000,), generator=g),
                   torch.arange(0, 449, 0.5), torch.arange(0, 64) * 2.0**-10]).clamp(-448, 448)
    assert torch.equal(oracle.nearest_e4m3(v).float(), v.to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("cols", [1, 31, 32, 33, 100])
def test_held_values_are_within_half_a_step(cols):
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(50, cols, generator=g) * torch.exp(torch.randn(50, cols, generator=g))
    values, exps = oracle.held(x)
    s = exps.repeat_interleave(32, -1)[:, :cols]
    assert ((values - x.double()).abs() <= torch.maximum(2.0**-4 * x.double().abs(), torch.exp2(s - 10))).all()
    top = F.pad(x.abs(), (0, -cols % 32)).reshape(50, -1, 32).amax(-1).double()
    assert (top <= 448 * torch.exp2(exps)).all() and (top > 224 * torch.exp2(exps)).all()


def test_held_values_at_the_end_of_the_range():
    """From 1.9375 * 2^127 on (half way from e4m3's 240 to 256, times 2^120) a value is nearest to 2^128, which neither
    type has; below it the bound holds."""
    last = torch.finfo(torch.float32).max
    x = torch.tensor([[1.9375 * 2.0**127, last, torch.finfo(torch.bfloat16).max, (1.9375 - 2.0**-23) * 2.0**127]])
    values, _ = oracle.held(x)
    assert values.tolist() == [[2.0**128, 2.0**128, 2.0**128, 240 * 2.0**120]]
    assert values.float().isinf().tolist() == [[True, True, True, False]]


def _case(rows=7, d=10, h=14):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return n(rows, d), n(rows, d), dict(ln_weight=1 + 0.1 * n(d), ln_bias=n(d), expand_a=n(h, d), expand_b=n(h, d),
                                        squeeze=n(d, h))


def _forward(x, p, residual):
    h = F.layer_norm(x, x.shape[-1:], p["ln_weight"], p["ln_bias"], 1e-5)
    y = F.linear(F.silu(F.linear(h, p["expand_a"])) * F.linear(h, p["expand_b"]), p["squeeze"])
    return x + y if residual else y


@pytest.mark.parametrize("residual", [True, False])
def test_transition_backward_is_autograds_and_differences(residual):
    dy, x, p = _case()
    leaves = {"x": x.clone().requires_grad_(), **{k: v.clone().requires_grad_() for k, v in p.items()}}
    params = {k: v for k, v in leaves.items() if k != "x"}
    _forward(leaves["x"], params, residual).backward(dy)
    got = oracle.transition_backward(dy, x, **p, residual=residual)
    for k, leaf in leaves.items():
        torch.testing.assert_close(got[k], leaf.grad, rtol=1e-10, atol=1e-10)
    step = 1e-6
    for k in got:
        move = torch.randn(got[k].shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            at = {"x": x, **p}
            at[k] = at[k] + sign * step * move
            ends.append((_forward(at["x"], {n: v for n, v in at.items() if n != "x"}, residual) * dy).sum())
        torch.testing.assert_close((got[k] * move).sum(), (ends[0] - ends[1]) / (2 * step), rtol=1e-6, atol=1e-6)


def test_layer_norm_backward_is_autograds():
    dy, x, p = _case(5, 33)
    leaf, w, b = x.clone().requires_grad_(), p["ln_weight"].clone().requires_grad_(), p["ln_bias"].clone().requires_grad_()
    F.layer_norm(leaf, (33,), w, b, 1e-5).backward(dy)
    for got, want in zip(oracle.layer_norm_backward(dy, x, p["ln_weight"]), (leaf.grad, w.grad, b.grad)):
        torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-10)
