"""LayerNorm and Transition modules under autograd on the hip kernels, and a fine-tuning step of a block.

Tolerances: a module's gradients are those of ``tests/test_gpu_training.py``'s operators (1e-2 of the norm for the
transition; the LayerNorm's bf16 gradients half a step, 2^-8), against the ``pytorch`` backend at fp32 on the values
that were kept. In a block every op's gradient passes through bf16 activations between the ops (autograd rounds to the
activation's type: 2^-8 / sqrt(3) = 2.3e-3 of it in root mean square) on both sides alike, and the transition's 5e-3 join
them; two sides that differ by up to 5e-3 in one of eight ops' gradients stay within 2e-2.
"""

from __future__ import annotations

import copy
import dataclasses

import pytest
import torch

from foldforge_amd import dispatch, factories, kernels, modules, training
from foldforge_amd.trunk import PairformerTrunk, randomise

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _grads(module, x, dy, *args):
    x = x.detach().clone().requires_grad_()
    for p in module.parameters():
        p.grad = None
    y = module(x, *args)
    y.backward(dy)
    return y, x.grad, {n: p.grad for n, p in module.named_parameters()}


@pytest.mark.parametrize("keep", ["input", "8bit"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_module(dtype, keep):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 50, 100, generator=g).to(DEV, dtype)
    dy = torch.randn(3, 50, 100, generator=g).to(DEV, dtype)
    m = randomise(modules.LayerNorm(100), 1).to(DEV)
    plain = copy.deepcopy(m)
    training.install(m, keep)
    before = dispatch.ledger_of(m).served["hip"]
    y, dx, grads = _grads(m, x, dy)
    assert dispatch.ledger_of(m).served["hip"] == before + 1
    with torch.no_grad():
        # (the norm that keeps 8 bits adds its rows in another order at this width)
        torch.testing.assert_close(y, m(x), rtol=2**-7 if dtype == BF16 else 1e-6, atol=1e-6)
    at = kernels.quantize_activation(x).restore() if keep == "8bit" else x
    _, want, wants = _grads(plain, at.float(), dy.float())
    assert dx.dtype == dtype and _rel(dx, want) <= (2**-8 if dtype == BF16 else 1e-6)
    for n, t in wants.items():
        assert grads[n].dtype == F32 and _rel(grads[n], t) <= 1e-5, n


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("keep", ["input", "8bit"])
@pytest.mark.parametrize("d,n,shape", [(128, 4, (1, 20, 20)), (64, 4, (2, 3, 33)), (384, 4, (70,)), (256, 2, (1, 9, 11))])
def test_transition_module(d, n, shape, keep, residual):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(*shape, d, generator=g).to(DEV, BF16)
    dy = torch.randn(*shape, d, generator=g).to(DEV, BF16)
    m = randomise(modules.Transition(d, n), 2).to(DEV)
    plain = copy.deepcopy(m)
    training.install(m, keep)
    call = m if residual else m.delta
    leaf = x.clone().requires_grad_()
    y = call(leaf)
    with torch.no_grad():
        assert torch.equal(y, call(x))  # the same forward kernels
    y.backward(dy)
    at = (kernels.quantize_activation(x).restore() if keep == "8bit" else x).float().requires_grad_()
    (plain if residual else plain.delta)(at).backward(dy.float())
    assert _rel(leaf.grad, at.grad) <= 1e-2
    for (name, p), q in zip(m.named_parameters(), plain.parameters()):
        assert p.grad.dtype == F32 and _rel(p.grad, q.grad) <= 1e-2, name


def test_only_what_asks_gets_a_gradient():
    m = randomise(modules.Transition(128, 4), 3).to(DEV)
    training.install(m, "8bit")
    m.squeeze.weight.requires_grad_(False)
    x = torch.randn(7, 128, device=DEV, dtype=BF16)
    m(x).float().sum().backward()  # (an expanded gradient: made whole on the way)
    assert m.squeeze.weight.grad is None and m.expand_a.weight.grad is not None
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(m(leaf).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()  # differentiates once


def test_without_install_hip_still_cuts_the_graph():
    m = randomise(modules.Transition(128, 4), 3).to(DEV)
    m.set_backend("hip")
    assert not m(torch.randn(7, 128, device=DEV, dtype=BF16, requires_grad=True)).requires_grad


def _at_kept_values(transition):
    """``transition`` on ``pytorch`` with the gradient that a kept 8-bit input has: the value at the input, the
    derivative at what the 8 bits stand for."""
    plain = transition.forward

    def forward(x):
        kept = kernels.quantize_activation(x.detach().contiguous()).restore()
        y = plain(kept.float() + (x.float() - x.float().detach())).to(x.dtype)
        return y + (plain(x) - y).detach()

    transition.forward = forward


@pytest.mark.parametrize("keep", ["input", "8bit"])
def test_block_step(keep):
    """One step of a block: forward, gradients of everything, against the block on ``pytorch`` (with 8 bits: its
    transitions differentiated at the values that those stand for)."""
    g = torch.Generator().manual_seed(4)
    n = 24
    z = torch.randn(1, n, n, 128, generator=g).to(DEV, BF16)
    s = torch.randn(1, n, 384, generator=g).to(DEV, BF16)
    mask = torch.ones(1, n, dtype=torch.bool, device=DEV)
    mask[0, -3:] = False
    block = randomise(factories.pairformer_block(d_pair=128, triangle_model="af3", d_single=384), 5).to(DEV)
    plain = copy.deepcopy(block)
    plain.set_backend("pytorch")
    if keep == "8bit":
        _at_kept_values(plain.transition_pair)
        _at_kept_values(plain.single_transition)
    block.set_backend("hip")
    training.install(block, keep)
    weights = torch.randn(1, n, n, 128, generator=g).to(DEV), torch.randn(1, n, 384, generator=g).to(DEV)

    def step(b):
        for p in b.parameters():
            p.grad = None
        zz, ss = z.clone().requires_grad_(), s.clone().requires_grad_()
        pair, single = b(zz, mask, ss)
        ((pair.float() * weights[0]).mean() + (single.float() * weights[1]).mean()).backward()
        return zz.grad, ss.grad, {k: p.grad for k, p in b.named_parameters()}

    got, want = step(block), step(plain)
    assert dispatch.ledger_of(block.transition_pair).served["hip"] == 1
    assert dispatch.ledger_of(block.single_transition).served["hip"] == 1
    assert _rel(got[0], want[0]) <= 2e-2 and _rel(got[1], want[1]) <= 2e-2
    for k, t in want[2].items():
        if t is not None and float(t.norm()) > 0:
            assert _rel(got[2][k], t) <= 2e-2, k
    # and it steps: the parameters move and stay finite
    opt = torch.optim.SGD(block.parameters(), lr=1e-2)
    opt.step()
    assert all(p.isfinite().all() for p in block.parameters())
    with torch.no_grad():
        assert block(z, mask, s)[0].isfinite().all()


@pytest.mark.parametrize("parallel", [False, True])
@pytest.mark.parametrize("keep", ["input", "8bit"])
def test_trunk_step(keep, parallel):
    """Two blocks whose single tracks run on a second stream (the trunk's default): the gradients are those of the blocks
    one after the other. The caller drops the inputs before the backward pass, and the memory that comes free in it is
    written over on the first stream."""
    g = torch.Generator().manual_seed(6)
    n = 40
    trunk = randomise(PairformerTrunk(2, d_single=128, n_head_single=4), 5, out_scale=0.3).to(DEV)
    for block in trunk.blocks:
        block.config = dataclasses.replace(block.config, parallel=parallel)
    training.install(trunk, keep)
    z, s = torch.randn(1, n, n, 128, generator=g).to(DEV, BF16), torch.randn(1, n, 128, generator=g).to(DEV, BF16)
    mask = torch.ones(1, n, dtype=torch.bool, device=DEV)
    mask[0, -3:] = False
    weights = torch.randn(1, n, n, 128, generator=g).to(DEV), torch.randn(1, n, 128, generator=g).to(DEV)

    def write_over(_):
        torch.full((n, 128), float("nan"), device=DEV, dtype=BF16)

    def step(overlap):
        trunk.overlap_single = overlap
        for p in trunk.parameters():
            p.grad = None
        pair, single = trunk(z.clone(), mask, s.clone())
        loss = (pair.float() * weights[0]).mean() + (single.float() * weights[1]).mean()
        del pair, single
        hooks = [p.register_post_accumulate_grad_hook(write_over) for p in trunk.parameters()]
        loss.backward()
        for h in hooks:
            h.remove()
        return {k: p.grad for k, p in trunk.named_parameters()}

    want = step(False)
    for _ in range(3):
        got = step(True)
        for k, t in want.items():
            if t is not None and float(t.norm()) > 0:
                assert _rel(got[k], t) <= 2e-2, k


@pytest.mark.parametrize("keep", ["input", "8bit"])
def test_what_install_names_is_what_runs(keep):
    """A step of a block and of a norm beside it: every module named under ``hip`` ran there once, forward and backward,
    every other op on ``pytorch``."""
    n = 12
    block = factories.pairformer_block(d_pair=128, triangle_model="af3", d_single=384)
    model = randomise(torch.nn.ModuleDict({"norm": factories.layer_norm(128), "block": block}), 7).to(DEV)
    report = training.install(model, keep)
    z = torch.randn(1, n, n, 128, device=DEV, dtype=BF16)
    s = torch.randn(1, n, 384, device=DEV, dtype=BF16)
    pair, single = model["block"](model["norm"](z), torch.ones(1, n, dtype=torch.bool, device=DEV), s)
    (pair.float().square().mean() + single.float().square().mean()).backward()
    assert report["hip"] == ["norm", "block.transition_pair", "block.single_transition"]
    for backend, names in report.items():
        for name in names:
            module = model.get_submodule(name)
            assert dispatch.ledger_of(module).served == {backend: 1}, name
    for name in report["hip"]:
        assert all(p.grad is not None for p in model.get_submodule(name).parameters()), name
