"""Factories of the op classes, with the signatures FoldForge's graph builders call
(``src/foldforge/modules/engine/modules.py:133-226`` and ``pairformer.py:16-62`` of the
reference): family selector keys, fp32-master or plain-fp32 parameters, norm eps. Every
factory builds on ``pytorch``; :func:`foldforge_amd.dispatch.install` gives the modules
their backend afterwards.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Literal, TypeVar

import torch
from torch import nn

from foldforge_amd.modules import (
    LayerNorm,
    MasterWeights,
    MSABlock,
    MSAPairWeightedAveraging,
    OuterProductMean,
    PairformerBlock,
    PairformerConfig,
    Transition,
    TriangleAttention,
    TriangleMultiplication,
)

Precision = Literal["master", "fp32"]
PRECISIONS = ("master", "fp32")
M = TypeVar("M", bound=nn.Module)


@dataclass(frozen=True)
class ModelKeys:
    """Selector keys of one family: ``triangle`` is ``TriangleAttention(model=)``."""

    triangle: str | None
    confidence: str | None = None


#: ``DenseSpec.family`` -> keys, for the families whose pair stack this build serves
#: (``src/foldforge/modules/engine/modules.py:64-81`` of the reference).
MODEL_KEYS: dict[str, ModelKeys] = {
    "alphafold3": ModelKeys("af3"),
    "intellifold2": ModelKeys("intellifold2"),
    "openbind0": ModelKeys("openfold3"),
    "openfold3": ModelKeys("openfold3_preview2"),
    "protenix1": ModelKeys("protenix"),
    "protenix2": ModelKeys("protenix"),
    "opendde": ModelKeys("opendde"),
    "boltz2": ModelKeys("boltz2"),
}


def model_keys(family: str) -> ModelKeys:
    """The selector keys of ``family`` (``ValueError`` naming the known ones otherwise)."""
    keys = MODEL_KEYS.get(family)
    if keys is None:
        raise ValueError(f"no engine selector keys for family {family!r}; known: {', '.join(sorted(MODEL_KEYS))}")
    return keys


#: The LayerNorm eps a freshly built module carries; :func:`set_norm_eps` replaces only this.
DEFAULT_NORM_EPS = 1e-5


def set_norm_eps(module: nn.Module, eps: float) -> None:
    """Give ``eps`` to the LayerNorms of ``module`` still at :data:`DEFAULT_NORM_EPS` (a norm
    built with its own eps, e.g. a grouped outer product's ``product_norm``, keeps it)."""
    defaults = [m for m in module.modules() if isinstance(m, nn.LayerNorm) and m.eps == DEFAULT_NORM_EPS]
    for norm in defaults:
        norm.eps = eps


def finish(module: M, precision: Precision = "master", *, norm_eps: float | None = None) -> M:
    """Parameter dtype of a new module: ``master`` pins fp32 masters that survive a bulk cast
    (modules without the mixin become plain fp32), ``fp32`` is plain fp32."""
    if precision == "master":
        pin = module.set_master_weights if isinstance(module, MasterWeights) else module.float
        pin()
    elif precision == "fp32":
        module.float()
    else:
        raise ValueError(f"precision must be one of {PRECISIONS}, got {precision!r}")
    if norm_eps is not None:
        set_norm_eps(module, norm_eps)
    return module


def transition(d_hidden: int, n: int = 4, *, precision: Precision = "master",
               norm_eps: float | None = None) -> Transition:
    return finish(Transition(d_hidden, n), precision, norm_eps=norm_eps)


def triangle_multiplication(d_pair: int, *, outgoing: bool, d_hidden: int | None = None,
                            divide_by_length: bool = False, precision: Precision = "master",
                            norm_eps: float | None = None, p_drop: float = 0.0) -> TriangleMultiplication:
    module = TriangleMultiplication(d_pair, d_hidden=d_hidden, outgoing=outgoing, p_drop=p_drop,
                                    model="rf3" if divide_by_length else None)
    return finish(module, precision, norm_eps=norm_eps)


def triangle_attention(d_pair: int, n_head: int, *, starting: bool, model: str,
                       d_hidden: int | None = None, precision: Precision = "master",
                       norm_eps: float | None = None, p_drop: float = 0.0) -> TriangleAttention:
    module = TriangleAttention(d_pair, n_head, d_hidden=d_hidden, starting=starting, p_drop=p_drop,
                               model=model)
    return finish(module, precision, norm_eps=norm_eps)


def msa_pair_weighted_averaging(d_msa: int, d_pair: int, n_head: int = 8,
                                d_hidden: int | None = None, *, precision: Precision = "master",
                                norm_eps: float | None = None, p_drop: float = 0.0) -> MSAPairWeightedAveraging:
    """``MSAPairWeightedAveraging`` (residual included), as
    ``src/foldforge/modules/engine/modules.py:214-226`` builds it."""
    return finish(MSAPairWeightedAveraging(d_msa, d_pair, n_head, d_hidden, p_drop=p_drop),
                  precision, norm_eps=norm_eps)


#: AF3's divisor offset (``n + 1e-3``), FoldForge's default for ungrouped outer product means
#: (``src/foldforge/modules/engine/modules.py:42``).
OPM_COUNT_OFFSET: float | None = 1e-3


def outer_product_mean(d_msa: int, d_pair: int, d_hidden: int = 32, *, groups: int = 1,
                       projection_bias: bool = False, normalize_before_proj: bool = True,
                       product_norm_eps: float = 0.1, count_offset: float | None = None,
                       precision: Precision = "master",
                       norm_eps: float | None = None) -> OuterProductMean:
    """``OuterProductMean`` (the raw update, no residual), as
    ``src/foldforge/modules/engine/modules.py:184-210`` builds it: ``normalize_before_proj=False``
    is AF3's bias-before-divide form, ``count_offset`` AF3's ``n + 1e-3`` divisor (None: the
    clamp), ``projection_bias`` RoseTTAFold3's, ``groups`` Chai-1's."""
    return finish(OuterProductMean(d_msa, d_pair, d_hidden, normalize_before_proj=normalize_before_proj,
                                   projection_bias=projection_bias, groups=groups,
                                   product_norm_eps=product_norm_eps, count_offset=count_offset),
                  precision, norm_eps=norm_eps)


def layer_norm(d: int | tuple[int, ...], *, eps: float = 1e-5, bias: bool = True,
               elementwise_affine: bool = True) -> LayerNorm:
    return LayerNorm(d, eps=eps, bias=bias, elementwise_affine=elementwise_affine)


def pairformer_block(*, d_pair: int, triangle_model: str, d_single: int = 0,
                     d_hidden_tri_multi: int | None = None, d_hidden_tri_attention: int = 32,
                     n_head_tri_attention: int = 4, n_head_single: int = 16,
                     single_gate_bias: float = 0.0, pair_transition_n: int = 4,
                     single_transition_n: int = 4, use_triangle_attention: bool = True,
                     parallel: bool = False, divide_by_length: bool = False,
                     precision: Precision = "master", norm_eps: float | None = None,
                     p_drop: float = 0.0) -> PairformerBlock:
    """One block, residuals included (``src/foldforge/modules/engine/pairformer.py:16-62``). ``p_drop``: the rate that
    :func:`foldforge_amd.training.set_dropout` gives its triangle ops."""
    config = PairformerConfig(
        d_pair=d_pair,
        d_hidden_tri_multi=d_pair if d_hidden_tri_multi is None else d_hidden_tri_multi,
        d_hidden_tri_attention=d_hidden_tri_attention,
        n_head_tri_attention=n_head_tri_attention,
        p_drop=p_drop,
        use_triangle_attention=use_triangle_attention,
        model=triangle_model,
        d_single=d_single,
        n_head_single=n_head_single,
        single_gate_bias=single_gate_bias,
        pair_transition_n=pair_transition_n,
        single_transition_n=single_transition_n,
        parallel=parallel,
    )
    block = PairformerBlock(config)
    if divide_by_length:
        hidden = config.d_hidden_tri_multi
        block.tri_multi_outgoing = TriangleMultiplication(d_pair, hidden, outgoing=True, p_drop=p_drop, model="rf3")
        block.tri_multi_incoming = TriangleMultiplication(d_pair, hidden, outgoing=False, p_drop=p_drop, model="rf3")
    return finish(block, precision, norm_eps=norm_eps)


def msa_block(c_msa: int = 64, c_pair: int = 128, n_heads_pair: int = 4, *,
              precision: Precision = "master", norm_eps: float | None = None,
              **options) -> MSABlock:
    """An AF3 MSA-stack block (``src/foldforge/modules/engine/graph.py:240-276``); ``options``
    are :class:`foldforge_amd.modules.MSABlock`'s (Boltz order, Chai-1 parallel stages, the
    outer-product-mean form, the dropouts' rates)."""
    return finish(MSABlock(c_msa, c_pair, n_heads_pair, **options), precision, norm_eps=norm_eps)


def token_mask(pair_mask: torch.Tensor | None) -> torch.Tensor | None:
    """The token mask of an outer-product pair mask ``[..., L, L]``: its diagonal, as bool
    (read on the device, no host sync)."""
    if pair_mask is None:
        return None
    return torch.diagonal(pair_mask, dim1=-2, dim2=-1).gt(0).contiguous()


def residue_mask(pair_mask: torch.Tensor | None) -> torch.Tensor | None:
    """The key mask ``[1, L]`` (bool) the blocks take, from an unbatched pair mask ``[L, L]``."""
    tokens = token_mask(pair_mask)
    return tokens if tokens is None else tokens.unsqueeze(0)
