"""Dropout and adapters under autograd and in the op classes, on the GPU.

The ``hip`` and ``pytorch`` backends draw the same masks, so their results are compared under them. An adapted transition's
three projections round their inputs, weights and results to bf16, as the transition without adapters does: an op is held
to 1e-2 of its update in norm, a block to 3e-2. A gradient of the adapters comes back through the same products, each of
them with the rounding of its gradient beside those of the values: 2e-2 for an op, 6e-2 through a block.
"""

from __future__ import annotations

import pytest
import torch

from foldforge_amd import dispatch, execution, kernels, modules, training
from foldforge_amd.trunk import PairformerTrunk, randomise
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _norm(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("on_device", [False, True])
def test_dropout_under_autograd(dtype, on_device):
    g = torch.Generator().manual_seed(0)
    x, res, dy = (torch.randn(2, 6, 10, 64, generator=g).to(dtype) for _ in range(3))
    xg, rg = (t.to(DEV).requires_grad_(True) for t in (x, res))
    seed = torch.tensor([7, 100], dtype=torch.int64, device=DEV) if on_device else 7
    offset = 3 if on_device else 103
    y = training.dropout_add(xg, rg, p=0.25, seed=seed, offset=offset, shared=2)
    if on_device:
        seed.fill_(1)  # the draw was taken
    assert torch.equal(y, kernels.dropout_add(x.to(DEV), res.to(DEV), p=0.25, seed=7, offset=103, shared=2))
    y.backward(dy.to(DEV))
    assert torch.equal(rg.grad.cpu(), dy)
    keep = oracle.dropout_mask(x.shape, 2, 0.25, 7, 103)
    want = torch.where(keep, dy.double() * 65536 / (65536 - 16384), 0.0)
    assert ((xg.grad.cpu().double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0**-22) * want.abs()).all()
    alone = training.dropout_add(xg, p=0.25, seed=7, offset=103, shared=2)
    assert torch.equal(alone, kernels.dropout_add(x.to(DEV), p=0.25, seed=7, offset=103, shared=2))


def test_adapted_linear_under_autograd():
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(2, 9, 64, generator=g).to(DEV, BF16), torch.randn(2, 9, 96, generator=g).to(DEV, BF16)
    w = torch.randn(96, 64, generator=g).to(DEV)
    down, up = torch.randn(3, 4, 64, generator=g).to(DEV), torch.randn(3, 96, 4, generator=g).to(DEV)
    how = dict(offsets=torch.tensor([0, 9, 18], dtype=torch.int32, device=DEV),
               adapter=torch.tensor([2, 0], dtype=torch.int32, device=DEV))
    leaves = [t.clone().requires_grad_(True) for t in (x, down, up)]
    y = training.adapted_linear(leaves[0], w, down=leaves[1], up=leaves[2], **how)
    assert torch.equal(y, kernels.adapted_linear(x, w, down=down, up=up, **how))
    y.backward(dy)
    want = kernels.adapted_linear_backward(dy, x, w, down=down, up=up, **how)
    assert all(torch.equal(leaf.grad, v) for leaf, v in zip(leaves, want))
    # a gradient that is not contiguous, an input off its alignment
    wide = torch.zeros(2 * 9 * 64 + 1, dtype=BF16, device=DEV)[1:].view(2, 9, 64).copy_(x)
    for leaf in leaves:
        leaf.grad = None
    y = training.adapted_linear(wide, w, down=leaves[1], up=leaves[2], **how)
    y.backward(dy.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(leaves[1].grad, want.down) and torch.equal(leaves[2].grad, want.up)


def test_capture_is_refused_under_autograd():
    x = torch.zeros(4, 64, dtype=BF16, device=DEV, requires_grad=True)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="capture"):
                training.dropout_add(x, p=0.5, seed=1)
        finally:
            graph.capture_end()
    torch.cuda.synchronize()


def _block(p_drop=0.25):
    config = modules.PairformerConfig(p_drop=p_drop)
    block = randomise(modules.PairformerBlock(config), 3, out_scale=0.25)
    block.set_master_weights()
    return block.to(DEV)


def _inputs(n=40, batch=1):
    g = torch.Generator().manual_seed(1)
    mask = torch.ones(batch, n, dtype=torch.bool)
    mask[:, -3:] = False
    return torch.randn(batch, n, n, 128, generator=g).to(DEV, BF16), mask.to(DEV)


def test_block_with_dropout_at_inference():
    """Forward passes with dropout on the hip kernels: each op's update through its mask."""
    block, (z, mask) = _block(), _inputs()
    block.set_backend("hip")
    training.set_dropout(block, training.DropoutStream(11))
    assert block.tri_multi_outgoing.dropout.backend == "hip"
    dispatch.clear_ledgers(block)
    with torch.no_grad():
        got = block(z, mask)
        want = z
        for i, (op, axis) in enumerate([(block.tri_multi_outgoing, 1), (block.tri_multi_incoming, 1),
                                        (block.tri_atten_starting, 1), (block.tri_atten_ending, 2)]):
            update = op._forward_hip(want, mask, residual=False)
            want = kernels.dropout_add(update, want, p=0.25, seed=11, offset=i, shared=axis)
            keep = oracle.dropout_mask(update.shape, axis, 0.25, 11, i).expand(update.shape).to(DEV)
            assert torch.equal(kernels.dropout_add(update, p=0.25, seed=11, offset=i, shared=axis) != 0, keep & (update != 0))
        want = block.transition_pair(want)
    assert torch.equal(got, want)
    assert dispatch.ledger_of(block.tri_atten_ending.dropout).served["hip"] == 1
    block.eval()
    with torch.no_grad():
        plain = block(z, mask)
        training.set_dropout(block, None)
        assert torch.equal(block(z, mask), plain)


def _with_adapters(model, adapters, seed=5):
    training.adapt(model, 8, adapters=adapters, scale=0.5, seed=2)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, modules.TransitionAdapters):
                for n in m.NAMES:
                    up = m.matrices(n)[1]
                    up.copy_(0.05 * torch.randn(up.shape, generator=g).to(up.device))


@pytest.mark.parametrize("d,factor,n", [(128, 4, 40), (64, 2, 9), (384, 4, 5)])
def test_adapted_transition(d, factor, n):
    """Values and gradients of both backends, a batch whose elements have adapters of their own."""
    tr = randomise(modules.Transition(d, factor), 3)
    tr.set_master_weights()
    tr.to(DEV)
    _with_adapters(tr, 2)
    training.select_adapters(tr, torch.tensor([1, -1, 0], dtype=torch.int32, device=DEV))
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, n, n, d, generator=g).to(DEV, BF16).requires_grad_(True)
    dy = torch.randn(3, n, n, d, generator=g).to(DEV, BF16)
    results = {}
    for backend in ("pytorch", "hip"):
        tr.set_backend(backend)
        x.grad = None
        tr.zero_grad()
        update = tr.delta(x)
        update.backward(dy)
        results[backend] = dict(update=update.detach(), x=x.grad.clone(),
                                **{n: p.grad.clone() for n, p in tr.named_parameters() if p.requires_grad})
    with torch.no_grad():
        assert torch.equal(tr.delta(x.detach()), results["hip"]["update"])
    assert len(results["hip"]) == 8
    for k, want in results["pytorch"].items():
        assert _norm(results["hip"][k], want) <= (1e-2 if k == "update" else 2e-2), k


def test_a_fine_tuning_step():
    """Dropout, adapters and 8-bit activations together: a block's step on the kernels against the equations in plain torch
    under the same masks; and the next step's draws are others."""
    block, (z, mask) = _block(), _inputs(batch=2)
    _with_adapters(block, 2)
    training.select_adapters(block, torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    g = torch.Generator().manual_seed(9)
    dy = torch.randn(z.shape, generator=g).to(DEV, BF16)
    results = []
    for native in (False, True):
        if native:
            report = training.install(block, requires_grad=False)
            assert report["hip"] == ["transition_pair"]
            block.transition_pair.keep = "input"
        else:
            block.set_backend("pytorch")
        training.set_dropout(block, training.DropoutStream(21))
        for op in (block.tri_multi_outgoing, block.tri_atten_ending):
            op.dropout.set_backend("hip" if native else "pytorch")
        block.train()
        block.zero_grad()
        out = block(z, mask)
        out.backward(dy)
        results.append(dict(update=(out - z).detach(),
                            **{n: p.grad.clone() for n, p in block.named_parameters() if p.requires_grad}))
    assert len(results[0]) == 7
    for k, want in results[0].items():
        assert _norm(results[1][k], want) <= (3e-2 if k == "update" else 6e-2), k
    again = block(z, mask)
    assert not torch.equal(again, out)


def test_overlapped_trunk_with_dropout_and_adapters():
    """The single track on its second stream: adapters there as well, the same values as one stream gives."""
    model = randomise(PairformerTrunk(2, d_single=384), 3, out_scale=0.25)
    for block in model.blocks:
        block.set_master_weights()
        block.set_backend("hip")
    model.to(DEV)
    _with_adapters(model, 1)
    z, mask = _inputs(n=32)
    s = torch.randn(1, 32, 384, generator=torch.Generator().manual_seed(3)).to(DEV, BF16)
    results = []
    for overlap in (False, True, True):
        model.overlap_single = overlap
        training.set_dropout(model, training.DropoutStream(4), p=0.25)
        with torch.no_grad():
            results.append(model(z, mask, s, passes=2))
        torch.cuda.synchronize()
    for got in results[1:]:
        assert torch.equal(got[0], results[0][0]) and torch.equal(got[1], results[0][1])


def test_a_captured_model_with_dropout_is_refused():
    """Before the capture begins: the streams are as they were. In evaluation mode it is captured, with adapters of each
    element, and every replay gives the eager values."""
    model = randomise(PairformerTrunk(2, d_single=384), 3, out_scale=0.25)
    for block in model.blocks:
        block.set_master_weights()
        block.set_backend("hip")
    model.to(DEV)
    _with_adapters(model, 2)
    training.select_adapters(model, torch.tensor([1], dtype=torch.int32, device=DEV))
    z, mask = _inputs(n=32)
    s = torch.randn(1, 32, 384, generator=torch.Generator().manual_seed(3)).to(DEV, BF16)
    stream = training.DropoutStream(4, 10)
    training.set_dropout(model, stream, p=0.25)
    with pytest.raises(RuntimeError, match="dropout"):
        execution.capture_trunk(model, z, mask, s)
    assert stream.offset == 10
    with torch.no_grad():
        model(z, mask, s)
    assert stream.offset == 18
    model.eval()
    captured = execution.capture_trunk(model, z, mask, s)
    for step in range(3):
        zs = z + step
        got = [t.clone() for t in captured(zs, mask, s)]
        with torch.no_grad():
            want = model(zs, mask, s)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_adapters_of_a_model_that_keeps_8_bits():
    """``keep="8bit"`` after ``adapt``: the values and the adapters' gradients are those of ``"input"`` bit for bit (the
    projections keep their own inputs). The input's gradient passes the norm at the values that the 8 bits stand for, each off
    by at most 2^-4 of itself: of dx = rstd (g - mean g - n mean(g n)), rstd and both n by as much at most."""
    tr = randomise(modules.Transition(128, 4), 3)
    tr.set_master_weights()
    tr.to(DEV)
    _with_adapters(tr, 2)
    training.select_adapters(tr, torch.tensor([1, 0], dtype=torch.int32, device=DEV))
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(2, 24, 24, 128, generator=g).to(DEV, BF16) for _ in range(2))
    results = []
    for keep in ("input", "8bit"):
        assert training.install(tr, keep, requires_grad=False)["hip"] == [""]
        leaf = x.clone().requires_grad_(True)
        tr.zero_grad()
        update = tr.delta(leaf)
        update.backward(dy)
        results.append((update.detach(), leaf.grad, *(p.grad.clone() for p in tr.parameters() if p.requires_grad)))
    assert len(results[0]) == 8
    for i, (a, b) in enumerate(zip(*results)):
        if i == 1:
            assert 0 < _norm(b, a) <= 3 * 2.0**-4
        else:
            assert torch.equal(a, b), i


def test_new_adapters_on_the_kernels():
    """``up`` of zeros: the op runs as its three projections, whose results it rounds, and stays as near to the equations as the
    op without adapters does."""
    tr = randomise(modules.Transition(128, 4), 3)
    tr.set_master_weights()
    tr.to(DEV)
    x = torch.randn(2, 24, 24, 128, generator=torch.Generator().manual_seed(2)).to(DEV, BF16)
    with torch.no_grad():
        want = tr.delta(x.float())
        training.adapt(tr, 8, adapters=2)
        tr.set_backend("hip")
        for selected in (None, torch.tensor([1, -1], dtype=torch.int32, device=DEV)):
            training.select_adapters(tr, selected)
            assert _norm(tr.delta(x), want) <= 1e-2
            assert torch.equal(tr(x), x + tr.delta(x))
