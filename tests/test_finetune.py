"""Dropout and adapters in the op classes, on the CPU: the ``pytorch`` backend's masks are the oracle's, rates and axes per op,
batches with an adapter each against merged weights."""

from __future__ import annotations

import copy
import time
from concurrent.futures import ThreadPoolExecutor
from contextlib import nullcontext

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import foldforge_amd
from foldforge_amd import dispatch, factories, modules, torch_ops, training
from foldforge_amd.trunk import PairformerTrunk, randomise
from oracle import training as oracle


def _block(p_drop=0.25, **how):
    block = modules.PairformerBlock(modules.PairformerConfig(d_pair=64, d_hidden_tri_multi=64, d_hidden_tri_attention=16,
                                                             p_drop=p_drop, **how))
    return randomise(block, 3)


def _inputs(n=9, batch=1, d=64):
    g = torch.Generator().manual_seed(1)
    mask = torch.ones(batch, n, dtype=torch.bool)
    mask[:, -1] = False
    return torch.randn(batch, n, n, d, generator=g), mask


@pytest.mark.parametrize("shape,shared", [((5, 451), None), ((2, 5, 7, 12), 1), ((2, 5, 7, 12), 2), ((3, 1, 8), 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plain_dropout_is_the_oracles(shape, shared, dtype):
    g = torch.Generator().manual_seed(0)
    x, res = torch.randn(*shape, generator=g).to(dtype), torch.randn(*shape, generator=g).to(dtype)
    seed, offset = 2**62 + 12345, 2**40 + 7
    got = torch_ops.dropout_add(x, res, shared=shared, dropped=round(65536 * 0.3), seed=seed, offset=offset)
    want = oracle.dropout_add(x, res, shared, 0.3, seed, offset)
    size = x.double().abs() * 65536 / (65536 - round(65536 * 0.3)) + res.double().abs()
    assert ((got.double() - want).abs() <= 3 * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * want.abs()).all()
    alone = torch_ops.dropout_add(x, None, shared=shared, dropped=round(65536 * 0.3), seed=seed, offset=offset)
    assert torch.equal(alone != 0, oracle.dropout_mask(shape, shared, 0.3, seed, offset).expand(shape) & (x != 0))


def test_ops_get_their_rate_and_axis():
    block = _block()
    names = training.set_dropout(block, training.DropoutStream(5))
    assert names == ["tri_multi_outgoing", "tri_multi_incoming", "tri_atten_starting", "tri_atten_ending"]
    assert [getattr(block, n).dropout.axis for n in names] == [1, 1, 1, 2]
    assert all(getattr(block, n).dropout.p == 0.25 for n in names)
    assert not any("dropout" in k for k in block.state_dict())
    assert training.set_dropout(block, training.DropoutStream(5), p=0.0) == []
    assert block.tri_atten_ending.active_dropout() is None
    assert training.set_dropout(_block(p_drop=0.0), training.DropoutStream(5)) == []
    msa = factories.msa_pair_weighted_averaging(64, 128)
    assert training.set_dropout(msa, training.DropoutStream(5), p=0.15) == [""] and msa.dropout.axis == 1
    with pytest.raises(ValueError, match="p must"):
        training.set_dropout(block, training.DropoutStream(5), p=1.5)


@pytest.mark.parametrize("parallel", [False, True])
def test_block_drops_each_update(parallel):
    """Every op's own update through the mask of its draw, in order; none in evaluation mode."""
    block, (z, mask) = _block(parallel=parallel), _inputs()
    plain = block(z, mask)
    training.set_dropout(block, training.DropoutStream(11))
    block.eval()
    assert torch.equal(block(z, mask), plain)
    block.train()
    got = block(z, mask)
    ops = [(block.tri_multi_outgoing, 1), (block.tri_multi_incoming, 1), (block.tri_atten_starting, 1),
           (block.tri_atten_ending, 2)]
    want, updates = z, []
    for i, (op, axis) in enumerate(ops):
        update = op._forward_pytorch(z if parallel else want, mask, residual=False)
        dropped = oracle.dropout_add(update, None, axis, 0.25, 11, i).float()
        updates.append(dropped)
        want = want + dropped
    want = z + sum(updates) + block.transition_pair.delta(z) if parallel else block.transition_pair(want)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    assert not torch.equal(block(z, mask), got)  # the next draws
    training.set_dropout(block, None)
    assert torch.equal(block(z, mask), plain)


def test_stream_goes_on_from_a_checkpoint():
    block, (z, mask) = _block(), _inputs()
    stream = training.DropoutStream(11)
    training.set_dropout(block, stream)
    block(z, mask)
    seed, offset = stream.seed, stream.offset
    want = block(z, mask)
    training.set_dropout(block, training.DropoutStream(seed, offset))
    assert torch.equal(block(z, mask), want)


@pytest.mark.parametrize("seed, offset", [(-1, 0), (2**63, 0), (1, -1), (torch.tensor([1, 0]), 0), (0.5, 0)])
def test_a_stream_is_of_whole_numbers(seed, offset):
    with pytest.raises(ValueError, match="whole number"):
        training.DropoutStream(seed, offset)


def test_calls_are_counted_where_they_run():
    block, (z, mask) = _block(), _inputs()
    training.set_dropout(block, training.DropoutStream(1))
    dispatch.clear_ledgers(block)
    block(z, mask)
    assert dispatch.served_count(block, "pytorch") == 5
    assert dispatch.ledger_of(block.tri_multi_outgoing.dropout).served["pytorch"] == 1


def _adapted(batch=3, adapters=2, rank=4):
    block = _block(p_drop=0.0)
    names = training.adapt(block, rank, adapters=adapters, scale=0.5, seed=2)
    assert names == ["transition_pair"]
    g = torch.Generator().manual_seed(4)
    ad = block.transition_pair.adapters
    with torch.no_grad():
        for n in ad.NAMES:
            ad.matrices(n)[1].copy_(0.1 * torch.randn(ad.matrices(n)[1].shape, generator=g))
    return block.transition_pair, _inputs(batch=batch)[0]


def test_new_adapters_change_nothing():
    block, (z, mask) = _block(p_drop=0.0), _inputs()
    want = block(z, mask)
    training.adapt(block, 8)
    assert torch.equal(block(z, mask), want)
    asks = {n for n, p in block.named_parameters() if p.requires_grad}
    assert asks == {f"transition_pair.adapters.{m}_{k}" for m in ("expand_a", "expand_b", "squeeze") for k in ("down", "up")}
    assert all(p.dtype == torch.float32 for p in block.transition_pair.adapters.parameters())


def test_each_batch_element_runs_its_own_adapter():
    """Against the transition with W + s B A for its weights."""
    tr, z = _adapted()
    training.select_adapters(tr, torch.tensor([1, -1, 0], dtype=torch.int32))
    got = tr(z)
    for b, a in enumerate((1, -1, 0)):
        merged = modules.Transition(tr.d, tr.n)
        merged.load_state_dict({k: v for k, v in tr.state_dict().items() if not k.startswith("adapters")})
        if a >= 0:
            with torch.no_grad():
                for n in tr.adapters.NAMES:
                    down, up = tr.adapters.matrices(n)
                    getattr(merged, n).weight += 0.5 * up[a] @ down[a]
        assert torch.allclose(got[b:b + 1], merged(z[b:b + 1]), rtol=1e-4, atol=1e-5)
    with pytest.raises(ValueError, match="batch"):
        tr(z[:2])
    training.select_adapters(tr, None)
    assert not torch.equal(tr(z)[1], got[1])


def test_gradients_reach_the_adapters_alone():
    tr, z = _adapted()
    training.select_adapters(tr, torch.tensor([1, 1, -1], dtype=torch.int32))
    tr(z).square().sum().backward()
    for n, p in tr.named_parameters():
        assert (p.grad is not None) == n.startswith("adapters"), n
    assert not tr.adapters.squeeze_up.grad[0].any() and tr.adapters.squeeze_up.grad[1].any()


def test_refusals():
    block = _block()
    with pytest.raises(ValueError, match="rank"):
        training.adapt(block, 129)
    assert block.transition_pair.adapters is None and block.transition_pair.squeeze.weight.requires_grad
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    w = torch.zeros(8, 8, requires_grad=True)
    with pytest.raises(ValueError, match="frozen"):
        training.adapted_linear(x, w, down=torch.zeros(1, 2, 8), up=torch.zeros(1, 8, 2),
                                offsets=torch.zeros(2, dtype=torch.int32), adapter=torch.zeros(1, dtype=torch.int32))


def test_calls_by_name_and_without_the_residual_under_dropout():
    """Every form of a call that an op takes without a dropout, it takes with one."""
    block, (z, mask) = _block(), _inputs()
    g = torch.Generator().manual_seed(6)
    msa, msa_op = torch.randn(1, 3, 9, 64, generator=g), randomise(modules.MSAPairWeightedAveraging(64, 64), 3)
    for op, axis, first, args in ((block.tri_multi_outgoing, 1, "x", (z, mask)), (block.tri_atten_ending, 2, "x", (z, mask)),
                                  (msa_op, 1, "m", (msa, z, mask))):
        names = (first, "mask") if len(args) == 2 else (first, "z", "mask")
        by_name = dict(zip(reversed(names), reversed(args)))  # (the input is not the first of them)
        for dropped in (False, True):
            update = op._forward_pytorch(*args, residual=False)
            whole = op._forward_pytorch(*args)
            training.set_dropout(op, training.DropoutStream(9) if dropped else None, p=0.25)
            if dropped:
                keep = [oracle.dropout_mask(update.shape, axis, 0.25, 9, i) for i in range(4)]
            for i, (got, added) in enumerate(((op(*args), True), (op(**by_name), True), (op(*args, residual=False), False),
                                              (op(**by_name, residual=False), False))):
                want = whole if added else update
                if dropped:
                    want = torch.where(keep[i], update * (4 / 3), 0.0) + (args[0] if added else 0.0)
                # (a scale, its product and a sum in fp32: 3 roundings of 2^-24 of values below 2^6)
                assert ((got - want).abs() <= 3 * 2.0**-18).all(), (type(op).__name__, dropped, i)


def test_a_stream_refuses_a_capture(monkeypatch):
    """A graph would replay the offsets that its capture saw."""
    block, (z, mask) = _block(), _inputs()
    stream = training.DropoutStream(11, 40)
    training.set_dropout(block, stream)
    with training.replayed(), pytest.raises(RuntimeError, match="capture"):
        block(z, mask)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        block(z, mask)
    assert stream.offset == 40
    block.eval()
    with training.replayed():
        block(z, mask)
    monkeypatch.undo()
    block.train()
    block(z, mask)
    assert stream.offset == 44


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_forward_draws_its_masks_again(reentrant):
    """Under torch.utils.checkpoint without the stream's context the gradients would be another mask's: an error."""
    block, (z, mask) = _block(), _inputs()
    stream = training.DropoutStream(11)
    training.set_dropout(block, stream)
    z.requires_grad_(True)
    dy = torch.randn(z.shape, generator=torch.Generator().manual_seed(7))

    def gradients(run):
        z.grad, stream.offset = None, 5
        block.zero_grad()
        y = run()
        y.backward(dy)
        return [z.grad.clone()] + [p.grad.clone() for p in block.parameters()] + [y.detach()]

    want = gradients(lambda: block(z, mask))
    assert stream.offset == 9
    with pytest.raises(RuntimeError, match="offset"):
        gradients(lambda: checkpoint(block, z, mask, use_reentrant=reentrant))
    if reentrant:  # by hand: the offset set back where the second run begins
        calls = []

        def run(*args):
            with stream.at(5) if calls else nullcontext():
                calls.append(1)
                return block(*args)

        got = gradients(lambda: checkpoint(run, z, mask, use_reentrant=True))
    else:
        got = gradients(lambda: checkpoint(block, z, mask, use_reentrant=False, context_fn=stream.recomputed))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert stream.offset == 9  # the next forward pass goes on behind the first
    # one call with the context (the one that is run again first), one without
    with pytest.raises(RuntimeError, match="offset"):
        gradients(lambda: checkpoint(block, checkpoint(block, z, mask, use_reentrant=reentrant), mask, use_reentrant=False,
                                     context_fn=stream.recomputed))


def test_a_stream_set_back_inside_a_backward_pass():
    """The offset set by hand, as a recomputing autograd function does."""
    stream = training.DropoutStream(3)
    taken = []

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.offset = stream.offset
            taken.append(stream.take())
            return x.clone()

        @staticmethod
        def backward(ctx, dy):
            stream.offset = ctx.offset
            taken.append(stream.take())
            return dy

    x = torch.ones(1, requires_grad=True)
    Again.apply(x).backward()
    assert taken == [0, 0] and stream.take() == 1


def test_draws_of_two_threads_are_their_own():
    """A thread that is held between reading the offset and counting it up does not share it."""
    class Slow(int):
        def __add__(self, other):
            time.sleep(0.005)
            return Slow(int(self) + other)

    stream = training.DropoutStream(1, Slow(0))
    with ThreadPoolExecutor(4) as pool:
        taken = [int(t) for t in pool.map(lambda _: stream.take(), range(24))]
    assert sorted(taken) == list(range(24))
    assert copy.deepcopy(stream).take() == 24


def test_models_are_built_with_their_rates():
    """AF3's two rates through every way to build a model; without them no op has a dropout."""
    stream, tri = training.DropoutStream(1), dict(d_pair=64, n_head=4, starting=True, model="af3")
    made = [(factories.triangle_multiplication(64, outgoing=True, p_drop=0.25), 1, {0.25}),
            (factories.triangle_attention(**tri, p_drop=0.25), 1, {0.25}),
            (factories.msa_pair_weighted_averaging(64, 64, p_drop=0.15), 1, {0.15}),
            (factories.pairformer_block(d_pair=64, triangle_model="af3", p_drop=0.25), 4, {0.25}),
            (factories.pairformer_block(d_pair=64, triangle_model="af3", divide_by_length=True, p_drop=0.25), 4, {0.25}),
            (factories.msa_block(64, 64, p_drop=0.25, p_drop_msa=0.15), 5, {0.25, 0.15}),
            (PairformerTrunk(2, d_pair=64, d_single=0, p_drop=0.25), 8, {0.25}),
            (foldforge_amd.load(backend="pytorch", device="cpu", blocks=1, d_single=0, p_drop=0.25), 4, {0.25})]
    for model, ops, rates in made:
        names = training.set_dropout(model, stream)
        assert len(names) == ops
        assert {m.p for m in model.modules() if isinstance(m, modules.Dropout)} == rates
        assert all("msa_attention" not in n or model.get_submodule(n).dropout.p == 0.15 for n in names)
    assert training.set_dropout(factories.msa_block(64, 64), stream) == []
    assert training.set_dropout(PairformerTrunk(1, d_pair=64, d_single=0), stream) == []


def test_a_dropout_refuses_as_its_op_does():
    """What the kernel does not take falls back, or raises, by the policy of the op, also one that is set later."""
    block, (z, mask) = _block(), _inputs()
    op = block.tri_multi_outgoing
    training.set_dropout(block, training.DropoutStream(3, 20))
    op.dropout.set_backend("hip")  # (the tensors are on the CPU)
    with pytest.raises(modules.BackendUnsupported):
        op(z, mask)
    dispatch.set_refusal(block, "fallback")
    op.dropout.stream.offset = 20
    got = op(z, mask)
    assert dispatch.ledger_of(op.dropout).served["pytorch"] == 1
    op.dropout.set_backend("pytorch")
    op.dropout.stream.offset = 20
    assert torch.equal(op(z, mask), got)
    op.dropout.set_backend("hip")
    dispatch.set_refusal(block, "error")
    with pytest.raises(dispatch.BackendUnsupportedError):
        op.delta(z, mask)
