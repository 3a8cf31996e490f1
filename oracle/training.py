"""The training operators at 64 bits, from their definitions: the 8-bit activation, LayerNorm's backward
pass and the SwiGLU transition's (the gradients of ``legacy/reference/transition.py:28-59`` of the
reference and of the LayerNorm in front of it)."""

from __future__ import annotations

import torch

Tensor = torch.Tensor

BLOCK = 32  # channels that share a scale
LARGEST = 448.0  # e4m3's largest number


def _e4m3_numbers() -> Tensor:
    """Every non-negative e4m3 number in order: 7 subnormal steps of 2^-9 above 0, then eight to each
    power of two from 2^-6 on, up to 448 (the place of 480 is NaN's)."""
    small = [i * 2.0**-9 for i in range(8)]
    return torch.tensor(small + [(1 + i / 8) * 2.0**e for e in range(-6, 9) for i in range(8)][:-1],
                        dtype=torch.float64)


def nearest_e4m3(v: Tensor) -> Tensor:
    """The e4m3 number nearest to each ``|v| <= 448``, halves to the one with the even code."""
    numbers = _e4m3_numbers()
    m = v.abs().double().contiguous()
    up = torch.searchsorted(numbers, m).clamp_max(len(numbers) - 1)
    down = (up - 1).clamp_min(0)
    low, high = m - numbers[down], numbers[up] - m
    take_up = (high < low) | ((high == low) & (up % 2 == 0))
    return torch.copysign(numbers[torch.where(take_up, up, down)], v.double())


def held(x: Tensor) -> tuple[Tensor, Tensor]:
    """``(values, s)`` of the 8-bit activation of ``x [..., c]`` on the CPU: the values as fp64 and each
    block's exponent."""
    rows = x.double().reshape(-1, x.shape[-1])
    values, exps = torch.empty_like(rows), []
    for c in range(0, rows.shape[1], BLOCK):
        v = rows[:, c:c + BLOCK]
        finite = torch.where(torch.isfinite(v), v.abs(), 0.0)
        top = finite.amax(1)
        s = torch.full_like(top, -126)
        while True:  # the least power of two that holds the block
            more = top > LARGEST * torch.exp2(s)
            if not more.any():
                break
            s = s + more
        unit = torch.exp2(s)[:, None]
        code = nearest_e4m3(torch.where(torch.isfinite(v), v / unit, 0.0))
        values[:, c:c + BLOCK] = torch.where(torch.isfinite(v), code * unit, torch.nan)
        exps.append(s)
    return values.reshape(x.shape), torch.stack(exps, 1).reshape(*x.shape[:-1], -1)


def normalised(x: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    c = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    return c * rstd, rstd


def layer_norm_backward(dy: Tensor, x: Tensor, weight: Tensor | None, eps: float = 1e-5) -> tuple[Tensor, Tensor, Tensor]:
    """``(dx, dweight, dbias)``."""
    dy, x = dy.double(), x.double()
    xh, rstd = normalised(x, eps)
    g = dy if weight is None else dy * weight.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    axes = tuple(range(x.dim() - 1))
    return dx, (dy * xh).sum(axes), dy.sum(axes)


def transition_backward(dy: Tensor, x: Tensor, *, ln_weight: Tensor, ln_bias: Tensor, expand_a: Tensor,
                        expand_b: Tensor, squeeze: Tensor, residual: bool = True, eps: float = 1e-5) -> dict[str, Tensor]:
    """Gradients by name, ``x`` the input's."""
    shape = x.shape
    dy, x = (t.double().reshape(-1, shape[-1]) for t in (dy, x))
    w, wa, wb, wo = (t.double() for t in (ln_weight, expand_a, expand_b, squeeze))
    n = normalised(x, eps)[0] * w + ln_bias.double()
    a, b = n @ wa.T, n @ wb.T
    s = torch.sigmoid(a)
    du = dy @ wo
    da = du * b * s * (1 + a * (1 - s))
    db = du * a * s
    dx, dw, dbias = layer_norm_backward(da @ wa + db @ wb, x, ln_weight, eps)
    return dict(x=((dy if residual else 0) + dx).reshape(shape), ln_weight=dw, ln_bias=dbias, expand_a=da.T @ n,
                expand_b=db.T @ n, squeeze=dy.T @ (a * s * b))
