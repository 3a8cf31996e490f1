"""Training with the hip kernels: LayerNorm and the SwiGLU transition under autograd.

The hip kernels of the other ops are forward-only. :func:`install` makes a model of engine-op modules ready for a
fine-tuning step: Transitions, and LayerNorms that are modules of their own, keep their inputs (as they are, or in 8
bits) and run their backward kernels; every other op, the norms inside it included, takes its ``pytorch`` backend, whose
equations autograd differentiates (the reference's fine-tuning runs its modules the same way,
``src/foldforge/train/step.py:320-338``).

:func:`layer_norm` and :func:`transition` are the differentiable functions on their own, the autograd side of
:func:`foldforge_amd.kernels.layer_norm_backward` and :func:`foldforge_amd.kernels.transition_backward`. Nothing
but the input is kept between the passes (the backward kernels take the statistics and the hidden rows from it
again); with ``keep="8bit"`` the gradient is taken at the values that the 8 bits stand for. The gradients of fp32
parameters are fp32; the transition's come from products on bf16 and fp16 operands, as its forward pass, and are off by some
3e-3 of their norm (``pytorch``: fp32 throughout). They differentiate once.

Autograd does not reach into graph capture here: a backward pass whose leaves were used by an eager graph on
another stream ends the process when it is captured, so these functions refuse a capturing stream. A captured step
calls the kernels' functions themselves (``transition_checkpoint``, ``transition_backward``, ...).
"""

from __future__ import annotations

from collections.abc import Iterator

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from foldforge_amd import kernels

Tensor = torch.Tensor

#: what a forward pass keeps of its input
KEEPS = ("input", "8bit")

_TRANSITION = ("ln_weight", "ln_bias", "expand_a", "expand_b", "squeeze")


def _check(keep: str) -> None:
    if keep not in KEEPS:
        raise ValueError(f"keep must be one of {KEEPS} (got {keep!r})")
    _eager()


def _eager() -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("autograd under graph capture is not served: capture the calls of "
                           "foldforge_amd.kernels (forward and backward) instead")


def _keep(ctx, x: Tensor | kernels.Activation8, *others: Tensor | None) -> None:
    if isinstance(x, kernels.Activation8):
        ctx.dtype = x.dtype
        ctx.save_for_backward(x.codes, x.scales, *others)
    else:
        ctx.dtype = None
        ctx.save_for_backward(x, None, *others)


def _kept(ctx) -> tuple[Tensor | kernels.Activation8, tuple[Tensor | None, ...]]:
    x, scales, *others = ctx.saved_tensors
    return (x if ctx.dtype is None else kernels.Activation8(x, scales, ctx.dtype)), tuple(others)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        if keep == "8bit":
            y, kept = kernels.layer_norm_checkpoint(x, weight, bias, eps)
        else:
            y, kept = kernels.layer_norm(x, weight, bias, eps), x
        _keep(ctx, kept, weight)
        ctx.eps = eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        x, (weight,) = _kept(ctx)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dweight, dbias = kernels.layer_norm_backward(dy.contiguous(), x, weight, ctx.eps, with_bias=need_b)
        return dx if need_x else None, dweight if need_w else None, dbias, None, None


class _Transition(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ln_weight, ln_bias, expand_a, expand_b, squeeze, residual, eps, keep):
        params = (ln_weight, ln_bias, expand_a, expand_b, squeeze)
        args = dict(zip(_TRANSITION, params), residual=residual, eps=eps)
        if keep == "8bit":
            y, kept = kernels.transition_checkpoint(x, **args)
        else:
            y, kept = kernels.transition(x, **args), x
        _keep(ctx, kept, *params)
        ctx.residual, ctx.eps = residual, eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        x, params = _kept(ctx)
        dy = dy.contiguous()
        if dy.data_ptr() % 16:
            dy = dy.clone()
        grads = kernels.transition_backward(dy, x, **dict(zip(_TRANSITION, params)), residual=ctx.residual, eps=ctx.eps)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float = 1e-5, *,
               keep: str = "input") -> Tensor:
    """:func:`foldforge_amd.kernels.layer_norm`, differentiable; ``keep``: what is kept of ``x``."""
    _check(keep)
    return _LayerNorm.apply(x.contiguous(), weight, bias, float(eps), keep)


def transition(x: Tensor, *, ln_weight: Tensor, ln_bias: Tensor, expand_a: Tensor, expand_b: Tensor, squeeze: Tensor,
               residual: bool = True, eps: float = 1e-5, keep: str = "input") -> Tensor:
    """:func:`foldforge_amd.kernels.transition`, differentiable; ``keep``: what is kept of ``x``."""
    _check(keep)
    d = x.shape[-1]
    if not kernels.transition_backward_supported(d, expand_a.shape[0] // d):
        raise ValueError(f"width {d} x {expand_a.shape[0] // d} (the backward kernels take a multiple of 64 up to "
                         "768, factor up to 64)")
    return _Transition.apply(x.contiguous(), ln_weight, ln_bias, expand_a, expand_b, squeeze, residual, float(eps), keep)


def wanted(module: nn.Module, *inputs: Tensor) -> bool:
    """Whether a call of an engine-op module is to be differentiated by the hip kernels: the module keeps something
    (:func:`install`), autograd is on, and an input or a parameter asks for a gradient."""
    return (getattr(module, "keep", None) is not None and torch.is_grad_enabled()
            and (any(t.requires_grad for t in inputs) or any(p.requires_grad for p in module.parameters())))


def _ops(model: nn.Module) -> Iterator[tuple[str, nn.Module]]:
    """The engine ops of ``model``, without those inside another (an op reads its norms as parameters, it does not call
    them)."""
    from foldforge_amd.modules import EngineOp

    inside: set[nn.Module] = set()
    for name, module in model.named_modules():
        if isinstance(module, EngineOp) and module not in inside:
            inside.update(module.modules())
            yield name, module


def _has_backward(module: nn.Module) -> bool:
    """Whether the kernels differentiate an op of its kind and width (and it lists them)."""
    from foldforge_amd.modules import LayerNorm, Transition

    if "hip" not in module.backends:
        return False
    if isinstance(module, LayerNorm):
        return len(module.normalized_shape) == 1
    return isinstance(module, Transition) and kernels.transition_backward_supported(module.d, module.n)


#: a module's record of what :func:`install` changed
_BEFORE = "_before_training"


def _place(module: nn.Module, backend: str) -> None:
    """Give an op its backend for training and keep the one it had (a caller's own choice since the last time counts
    as such)."""
    before, given = module.__dict__.get(_BEFORE, (None, None))
    if module.backend != given:
        before = module.backend
    module.set_backend(backend)
    module.__dict__[_BEFORE] = (before, backend)


def _take_back(module: nn.Module) -> None:
    before, given = module.__dict__.pop(_BEFORE, (None, None))
    if before is not None and module.backend == given:
        module.set_backend(before)


#: a module's record of the parameters of its own whose gradients :func:`install` switched on
_FROZEN = "_frozen_before_training"


def _unfreeze(model: nn.Module) -> None:
    for module in model.modules():
        frozen = {n for n, p in module.named_parameters(recurse=False, remove_duplicate=False) if not p.requires_grad}
        if frozen:
            module.__dict__[_FROZEN] = module.__dict__.get(_FROZEN, set()) | frozen
    model.requires_grad_(True)


def _freeze_again(model: nn.Module) -> None:
    for module in model.modules():
        frozen = module.__dict__.pop(_FROZEN, ())
        for name, p in module.named_parameters(recurse=False, remove_duplicate=False):
            if name in frozen:
                p.requires_grad_(False)


def install(model: nn.Module, keep: str | None = "8bit", *, requires_grad: bool = True) -> dict[str, list[str]]:
    """Make ``model``'s engine ops trainable: every Transition, and every LayerNorm that is a module of its own (not a
    part of another op), keeps ``keep`` of its input and runs forward and backward on the hip kernels; every other op,
    and widths without backward kernels, go to ``pytorch``. ``requires_grad``: switch the parameters' gradients on
    (models are placed without). ``keep=None`` takes it all back: ops that still have the backend they were given here
    get the one they had before, parameters whose gradients were switched on here lose them. Returns the names of the
    ops by the backend they then have: ``{"hip": [...], "pytorch": [...]}``."""
    if keep is not None and keep not in KEEPS:
        raise ValueError(f"keep must be one of {KEEPS} or None (got {keep!r})")
    report: dict[str, list[str]] = {"hip": [], "pytorch": []}
    for name, module in _ops(model):
        served = _has_backward(module)
        if served:
            module.keep = keep
        if keep is None:
            _take_back(module)
        else:
            _place(module, "hip" if served else "pytorch")
        report.setdefault(module.backend, []).append(name)
    if keep is None:
        _freeze_again(model)
    elif requires_grad:
        _unfreeze(model)
    return report
