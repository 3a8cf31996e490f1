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

:func:`dropout_add` and :func:`adapted_linear` are the differentiable forms of the kernels of those names.
:func:`set_dropout` gives the ops that carry a rate (``p_drop``) their dropout, :func:`adapt` gives a model's Transitions
low-rank adapters, one for each of several requests, beside their frozen projections.

Autograd does not reach into graph capture here: a backward pass whose leaves were used by an eager graph on
another stream ends the process when it is captured, so these functions refuse a capturing stream. A captured step
calls the kernels' functions themselves (``transition_checkpoint``, ``transition_backward``, ...).
"""

from __future__ import annotations

import threading
from collections.abc import Iterator
from contextlib import AbstractContextManager, contextmanager, nullcontext
from contextvars import ContextVar

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


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, update, residual, p, seed, offset, shared):
        if isinstance(seed, Tensor):
            seed = seed.clone()  # (the backward pass draws this mask, whatever the caller's tensor holds by then)
        ctx.save_for_backward(seed if isinstance(seed, Tensor) else None)
        ctx.draw = dict(p=p, seed=seed if not isinstance(seed, Tensor) else 0, offset=offset, shared=shared)
        return kernels.dropout_add(update, residual, **{**ctx.draw, "seed": seed})

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        need_update, need_residual = ctx.needs_input_grad[:2]
        (seed,) = ctx.saved_tensors
        draw = ctx.draw if seed is None else {**ctx.draw, "seed": seed}
        update = kernels.dropout_backward(dy.contiguous(), **draw) if need_update else None
        return update, dy if need_residual else None, None, None, None, None


def dropout_add(update: Tensor, residual: Tensor | None = None, *, p: float, seed: int | Tensor, offset: int = 0,
                shared: int | None = None) -> Tensor:
    """:func:`foldforge_amd.kernels.dropout_add`, differentiable: nothing is kept for the backward pass, which draws the
    mask again."""
    _eager()
    return _DropoutAdd.apply(update.contiguous(), None if residual is None else residual.contiguous(), float(p), seed,
                             offset, shared)


class _AdaptedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, down, up, scale, offsets, adapter):
        y = kernels.adapted_linear(x, weight, bias, down=down, up=up, scale=scale, offsets=offsets, adapter=adapter)
        ctx.save_for_backward(x, weight, down, up, scale, offsets, adapter)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        x, weight, down, up, scale, offsets, adapter = ctx.saved_tensors
        dy = dy.contiguous()
        if dy.data_ptr() % 16:
            dy = dy.clone()
        grads = kernels.adapted_linear_backward(dy, x, weight, down=down, up=up, scale=scale, offsets=offsets,
                                                adapter=adapter, with_x=ctx.needs_input_grad[0], grad_dtype=down.dtype)
        need_down, need_up = ctx.needs_input_grad[3:5]
        return grads.x, None, None, grads.down if need_down else None, grads.up if need_up else None, None, None, None


def adapted_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, down: Tensor, up: Tensor,
                   scale: Tensor | None = None, offsets: Tensor, adapter: Tensor) -> Tensor:
    """:func:`foldforge_amd.kernels.adapted_linear`, differentiable in ``x``, ``down`` and ``up``. The projection and the
    scales are frozen: ones that ask for a gradient are refused."""
    _eager()
    for t, name in ((weight, "weight"), (bias, "bias"), (scale, "scale")):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} asks for a gradient: a projection with adapters is frozen (requires_grad_(False))")
    x = x.contiguous()
    return _AdaptedLinear.apply(x.clone() if x.data_ptr() % 16 else x, weight, bias, down, up, scale, offsets, adapter)


#: whether what runs now is to be captured and replayed
_REPLAYED: ContextVar[bool] = ContextVar("replayed", default=False)


@contextmanager
def replayed() -> Iterator[None]:
    """What runs inside is captured, or is the warm-up of a capture: a :class:`DropoutStream` refuses it."""
    token = _REPLAYED.set(True)
    try:
        yield
    finally:
        _REPLAYED.reset(token)


#: held while an offset is taken (threads of one process may share a stream; one lock for all keeps streams copyable)
_TAKING = threading.Lock()


class DropoutStream:
    """The draws of a run's dropouts: one seed, and an offset of its own for each call. ``offset`` is where the next call
    begins; with ``seed`` it is all that a checkpoint has to hold to go on with the same draws. A forward pass that is run
    again for its backward pass has to start from the offset that it had (set ``offset`` back for it, or run it under
    :meth:`at`; :meth:`recomputed` gives ``torch.utils.checkpoint`` both), else its gradients would be another mask's: a
    forward pass inside a backward pass that did not set the offset is refused. Ranks that see other data take other seeds.
    A captured graph would replay the offsets of its capture, one mask for ever: calls under capture
    are refused (:func:`foldforge_amd.kernels.dropout_add` takes a seed on the device there)."""

    def __init__(self, seed: int, offset: int = 0) -> None:
        for value, name in ((seed, "seed"), (offset, "offset")):
            if not isinstance(value, int) or not 0 <= value < 2**63:
                raise ValueError(f"{name} must be a whole number in [0, 2^63) (got {value!r})")
        self.seed, self.offset = seed, offset

    @property
    def offset(self) -> int:
        return self._offset

    @offset.setter
    def offset(self, value: int) -> None:
        self._offset = value
        self._placed = torch._C._current_graph_task_id()  # (the backward pass that set it, -1 for none)

    @contextmanager
    def at(self, offset: int) -> Iterator[None]:
        """The draws from ``offset`` on inside; afterwards the stream goes on where it was."""
        before = self._offset, self._placed
        self.offset = offset
        try:
            yield
        finally:
            self._offset, self._placed = before

    def recomputed(self) -> tuple[AbstractContextManager, AbstractContextManager]:
        """``torch.utils.checkpoint.checkpoint(..., use_reentrant=False, context_fn=stream.recomputed)``: the forward pass
        draws on, its second run draws what it drew."""
        return nullcontext(), self.at(self.offset)

    def take(self) -> int:
        """The offset of one call."""
        if _REPLAYED.get() or (torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()):
            raise RuntimeError("a captured graph would replay one dropout mask: capture the model in evaluation mode, or "
                               "call foldforge_amd.kernels.dropout_add with a seed on the device")
        task = torch._C._current_graph_task_id()
        if task != -1 and task != self._placed:
            raise RuntimeError("a forward pass run again inside a backward pass would draw other masks than it did: set the "
                               "DropoutStream's offset to where it began (checkpoint: context_fn=stream.recomputed)")
        with _TAKING:
            self._offset += 1
            return self._offset - 1


def set_dropout(model: nn.Module, stream: DropoutStream | None, p: float | None = None) -> list[str]:
    """Give every op of ``model`` that has a dropout (the triangle ops and the MSA pair-weighted averaging) its own, drawn
    from ``stream``, at the op's rate ``p_drop`` (the factories', the trunk's and the blocks' keyword; 0 by default) or, all
    of them, at ``p``; ops at rate 0 get none. The masks are AF3's: one for all rows
    of a pair or MSA tensor, for the ending node's attention one for all columns. They apply where the module is in training
    mode (``model.train()``), to the update before it is added, with or without gradients. ``stream=None`` takes them
    away. Returns the names of the ops that have one now."""
    from foldforge_amd.modules import Dropout, device_arch

    named = []
    for name, module in list(_ops(model)):
        if getattr(module, "dropout_axis", None) is None:
            continue
        module._modules.pop("dropout", None)
        rate = module.p_drop if p is None else p
        if stream is None or rate == 0.0:
            continue
        device = next(module.parameters()).device
        hip = device.type == "cuda" and device_arch(device) == "gfx950"
        module.dropout = Dropout(rate, module.dropout_axis, stream, backend="hip" if hip else "pytorch")
        module.dropout.train(module.training)
        named.append(name)
    return named


def adapt(model: nn.Module, rank: int, *, adapters: int = 1, scale: float = 1.0, seed: int = 0) -> list[str]:
    """Give every Transition of ``model`` ``adapters`` low-rank adapters of ``rank`` beside each of its three projections
    (``down`` normal of deviation ``d_in^-1/2``, ``up`` zeros: the model's results are as before at first, on ``hip`` but for
    the roundings of the projections' results, which the op without adapters does not make), fp32, and
    freeze the model's own parameters: the adapters alone ask for gradients (with :func:`install`, pass
    ``requires_grad=False`` there). A checkpoint of the model itself is loaded before. Returns the names of the
    Transitions."""
    from foldforge_amd.modules import Transition, TransitionAdapters

    generator = torch.Generator().manual_seed(seed)
    made = {name: (module, TransitionAdapters(module.d, module.n, rank, adapters, scale, generator))
            for name, module in _ops(model) if isinstance(module, Transition)}
    model.requires_grad_(False)
    for module, new in made.values():
        module.adapters = new.to(module.squeeze.weight.device)
    return list(made)


def select_adapters(model: nn.Module, adapter: Tensor | None) -> None:
    """Which adapter each element of a batch has: ``adapter [B]`` int32 on the device (-1: none), for all adapted ops of
    ``model``; None: the first for all."""
    from foldforge_amd.modules import TransitionAdapters

    for module in model.modules():
        if isinstance(module, TransitionAdapters):
            module.adapter = adapter


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
