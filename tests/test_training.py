"""The training operators on the host: what :mod:`foldforge_amd.kernels` and :mod:`foldforge_amd.training` refuse, the
sizes the library asks for, and what ``install`` makes of a model. Nothing here reaches a device."""

from __future__ import annotations

import contextlib
import copy

import pytest
import torch

from foldforge_amd import _native, build, factories, kernels, modules, training, trunk
from foldforge_amd.trunk import randomise

BF16 = torch.bfloat16


@pytest.fixture
def cpu_checks(monkeypatch):
    monkeypatch.setattr(kernels, "DEVICE_TYPE", "cpu")

    def refuse_native():
        raise AssertionError("an argument check let a bad call reach the library")

    monkeypatch.setattr(kernels._native, "lib", refuse_native)
    monkeypatch.setattr(kernels._native, "calls", refuse_native)


def _activation(rows=4, cols=40, dtype=BF16, **change):
    parts = dict(codes=torch.zeros(rows, cols, dtype=torch.float8_e4m3fn),
                 scales=torch.zeros(rows, -(-cols // 32), dtype=torch.uint8), dtype=dtype)
    return kernels.Activation8(**{**parts, **change})


@pytest.mark.parametrize("x,match", [
    (torch.zeros(4, 8, dtype=torch.float16), "bf16 or fp32"),
    (torch.zeros(4, 8).t(), "contiguous"),
    (torch.tensor(1.0), "last axis"),
    (torch.zeros(4, 0), "last axis"),
    (None, "contiguous device tensor"),
])
def test_quantize_refuses(cpu_checks, x, match):
    with pytest.raises(ValueError, match=match):
        kernels.quantize_activation(x)
    with pytest.raises(ValueError, match=match):
        kernels.layer_norm_checkpoint(x, None, None)


@pytest.mark.parametrize("change,match", [
    (dict(codes=torch.zeros(4, 40, dtype=torch.uint8)), "codes"),
    (dict(scales=torch.zeros(4, 1, dtype=torch.uint8)), "scales"),
    (dict(scales=torch.zeros(4, 2)), "scales"),
    (dict(scales=torch.zeros(2, 4, dtype=torch.uint8).t()), "scales"),
    (dict(dtype=torch.float16), "dtype"),
])
def test_a_bad_activation_is_refused(cpu_checks, change, match):
    a = _activation(**change)
    with pytest.raises(ValueError, match=match):
        kernels.restore_activation(a)
    with pytest.raises(ValueError, match=match):
        kernels.layer_norm_backward(torch.zeros(4, 40, dtype=BF16), a)


def test_restore_refuses_a_bad_out(cpu_checks):
    for out, match in ((torch.zeros(4, 41, dtype=BF16), "shape"), (torch.zeros(4, 40), "must be"),
                       (torch.zeros(40, 4, dtype=BF16).t(), "contiguous")):
        with pytest.raises(ValueError, match=match):
            kernels.restore_activation(_activation(), out=out)


def test_layer_norm_backward_refuses(cpu_checks):
    dy = torch.zeros(4, 40, dtype=BF16)
    for x in (torch.zeros(4, 41, dtype=BF16), torch.zeros(4, 40), torch.zeros(5, 40, dtype=BF16),
              _activation(cols=41), _activation(dtype=torch.float32)):
        with pytest.raises(ValueError, match="not like x"):
            kernels.layer_norm_backward(dy, x)
    with pytest.raises(ValueError, match="weight"):
        kernels.layer_norm_backward(dy, dy, torch.ones(41))
    with pytest.raises(ValueError, match="fp32"):
        kernels.layer_norm_backward(dy, dy, torch.ones(40, dtype=BF16))
    with pytest.raises(ValueError, match="grad_dtype"):
        kernels.layer_norm_backward(dy, dy, torch.ones(40), grad_dtype=torch.float16)


@pytest.mark.parametrize("cols,narrower", [(2**31 - 1023, True), (2**31 - 1, True), (2**26 - 15, False), (2**30, False)])
def test_more_channels_than_the_kernels_count(cpu_checks, monkeypatch, cols, narrower):
    """A row's channels are counted in 32 bits, with a workgroup's step beyond them; the sums of the backward pass
    take 64 threads a channel, and a launch has less than 2^32."""
    monkeypatch.setattr(kernels, "DEVICE_TYPE", "meta")
    x = torch.empty(1, cols, dtype=BF16, device="meta")
    with pytest.raises(ValueError, match="channels"):
        kernels.layer_norm_backward(x, x)
    if narrower:
        a = kernels.Activation8(x.to(torch.float8_e4m3fn), torch.empty(1, -(-cols // 32), dtype=torch.uint8, device="meta"),
                                BF16)
        for call in (lambda: kernels.quantize_activation(x), lambda: kernels.layer_norm_checkpoint(x, None, None),
                     lambda: kernels.restore_activation(a)):
            with pytest.raises(ValueError, match="channels"):
                call()


def _params(d=64, h=128, **change):
    return {**dict(ln_weight=torch.ones(d), ln_bias=torch.zeros(d), expand_a=torch.zeros(h, d),
                   expand_b=torch.zeros(h, d), squeeze=torch.zeros(d, h)), **change}


def test_transition_backward_refuses(cpu_checks):
    x = torch.zeros(4, 64, dtype=BF16)
    for change, match in ((dict(squeeze=torch.zeros(128, 64)), "squeeze"), (dict(ln_weight=torch.ones(65)), "ln_weight"),
                          (dict(expand_b=torch.zeros(64, 64)), "expand_b"), (dict(ln_bias=None), "ln_bias"),
                          (dict(expand_a=torch.zeros(128, 64, dtype=BF16)), "expand_a"),
                          (dict(expand_a=torch.zeros(32, 64)), "width")):
        with pytest.raises(ValueError, match=match):
            kernels.transition_backward(x, x, **_params(**change))
    for d in (32, 96, 832):
        t = torch.zeros(4, d, dtype=BF16)
        with pytest.raises(ValueError, match="width"):
            kernels.transition_backward(t, t, **_params(d, 4 * d))
    with pytest.raises(ValueError, match="bf16"):
        kernels.transition_backward(x.float(), x.float(), **_params())
    with pytest.raises(ValueError, match="not like x"):
        kernels.transition_backward(x, torch.zeros(5, 64, dtype=BF16), **_params())
    with pytest.raises(ValueError, match="grad_dtype"):
        kernels.transition_backward(x, x, **_params(), grad_dtype=torch.float64)
    odd = torch.zeros(1 + 4 * 64, dtype=BF16)[1:].view(4, 64)
    with pytest.raises(ValueError, match="aligned"):
        kernels.transition_backward(x, odd, **_params())


def test_transition_checkpoint_keeps_the_input_of_an_in_place_call(monkeypatch):
    """The transition may write over its input: the 8 bits are those of the input all the same."""
    x = torch.arange(8.0)
    monkeypatch.setattr(kernels, "transition", lambda x, *, out=None, **_: (out if out is not None else x.clone()).mul_(-1))
    monkeypatch.setattr(kernels, "quantize_activation", lambda x: x.clone())
    for out in (None, x):
        y, kept = kernels.transition_checkpoint(x, **({} if out is None else {"out": out}))
        assert torch.equal(kept, torch.arange(8.0)) and torch.equal(y, -torch.arange(8.0))
        assert out is None or y is x


def test_functions_refuse_a_bad_keep_and_a_capturing_stream(monkeypatch):
    x = torch.zeros(4, 64, dtype=BF16)
    with pytest.raises(ValueError, match="keep"):
        training.layer_norm(x, None, None, keep="4bit")
    with pytest.raises(ValueError, match="keep"):
        training.install(factories.layer_norm(64), "4bit")
    with pytest.raises(ValueError, match="width"):
        training.transition(torch.zeros(4, 96, dtype=BF16), **_params(96, 192))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: training.layer_norm(x, None, None), lambda: training.transition(x, **_params())):
        with pytest.raises(RuntimeError, match="capture"):
            call()


def test_workspaces():
    if not build.LIBRARY.exists():
        build.build()
    lib = _native.lib()
    assert lib.ffk_layer_norm_backward_workspace(-1, 64) == lib.ffk_layer_norm_backward_workspace(4, 0) == 0
    assert lib.ffk_layer_norm_backward_workspace(4, 64) == 0  # one workgroup
    # a workgroup's sums of two gradients for every 4 rows, up to 4 workgroups a CU (256 without a device)
    assert lib.ffk_layer_norm_backward_workspace(400, 96) == 100 * 2 * 96 * 4
    assert lib.ffk_layer_norm_backward_workspace(1 << 30, 96) == 1024 * 2 * 96 * 4
    assert lib.ffk_layer_norm_backward_workspace(1000, 1500) >= (64 * 2 * 1500 + 2000) * 4
    for bad in ((-1, 64, 4), (10, 32, 4), (10, 832, 4), (10, 64, 0), (10, 64, 65)):
        assert lib.ffk_transition_backward_workspace(*bad) == 0
    # rows are taken in chunks: the workspace stops growing
    assert lib.ffk_transition_backward_workspace(1 << 30, 128, 4) == lib.ffk_transition_backward_workspace(1 << 26, 128, 4)
    assert lib.ffk_transition_backward_workspace(1 << 30, 256, 4) == lib.ffk_transition_backward_workspace(1 << 26, 256, 4)


@pytest.mark.parametrize("cols", [1024, 1025, 1536, 1600, 2048])
@pytest.mark.parametrize("rows", [1, 4, 256, 257, 300, 1000, 1 << 20])
def test_layer_norm_backward_workspace_holds_every_form(rows, cols):
    """Whichever form a call takes, by its type and its tensors' alignment: rows of up to 1024 channels, and bf16 rows
    of 1536 in 16-byte pieces, lie in registers, up to 4 workgroups a CU (256 without a device) of 4 rows at least,
    each with a row of sums of two gradients; others have 64 such rows and every row's mean and rstd."""
    if not build.LIBRARY.exists():
        build.build()
    floats = 0
    if cols <= 1024 or cols == 1536:
        parts = min(-(-rows // 4), 1024)
        floats = parts * 2 * cols if parts > 1 else 0
    if cols > 1024:
        floats = max(floats, 64 * 2 * cols + 2 * rows)
    assert _native.lib().ffk_layer_norm_backward_workspace(rows, cols) >= 4 * floats


def test_install_and_take_back():
    block = randomise(factories.pairformer_block(d_pair=64, triangle_model="af3", d_single=128), 0)
    block.set_backend("hip")
    block.requires_grad_(False)
    report = training.install(block, "8bit")
    assert {"transition_pair", "single_transition"} <= set(report["hip"])
    assert {"tri_multi_outgoing", "tri_atten_ending", "single_attention"} <= set(report["pytorch"])
    assert all(p.requires_grad for p in block.parameters())
    assert block.transition_pair.keep == "8bit" and block.transition_pair.backend == "hip"
    assert block.tri_atten_starting.backend == "pytorch"
    x = torch.zeros(1, 4, 4, 64, dtype=BF16)
    assert training.wanted(block.transition_pair, x)
    with torch.no_grad():
        assert not training.wanted(block.transition_pair, x)
    training.install(block, None)
    assert block.transition_pair.keep is None and not training.wanted(block.transition_pair, x)


def test_install_names_the_modules_that_run_on_the_kernels():
    """The norms inside an op are parameters of it: they are neither called nor named. Ops without backward kernels of
    their kind or width take ``pytorch``."""
    block = randomise(factories.pairformer_block(d_pair=64, triangle_model="af3", d_single=128), 0)
    report = training.install(block, "8bit")
    assert sorted(report["hip"]) == ["single_transition", "transition_pair"]
    assert sorted(report["pytorch"]) == ["single_attention", "tri_atten_ending", "tri_atten_starting",
                                         "tri_multi_incoming", "tri_multi_outgoing"]
    assert all(m.keep is None and m.backend == "pytorch" for m in block.modules() if isinstance(m, modules.LayerNorm))
    model = torch.nn.ModuleDict({
        "norm": factories.layer_norm(100), "wide": modules.Transition(832, 1), "odd": modules.Transition(96, 2),
        "grid": modules.LayerNorm((4, 8)), "inner": torch.nn.Sequential(modules.Transition(64, 4))})
    report = training.install(model, "input")
    assert sorted(report["hip"]) == ["inner.0", "norm"] and sorted(report["pytorch"]) == ["grid", "odd", "wide"]
    for name, module in (("norm", model["norm"]), ("inner.0", model["inner"][0])):
        assert (module.backend, module.keep) == ("hip", "input"), name
    for name in ("grid", "odd", "wide"):
        assert (model[name].backend, model[name].keep) == ("pytorch", None), name
    assert training.install(factories.layer_norm(64))["hip"] == [""]


def test_install_leaves_an_op_that_lists_no_hip_on_pytorch():
    class Plain(modules.Transition):
        backends = ("pytorch",)

    model = torch.nn.Sequential(Plain(64, 4), modules.Transition(64, 4))
    assert training.install(model, "8bit") == {"hip": ["1"], "pytorch": ["0"]}
    assert model[0].keep is None


def test_taking_back_restores_backends_and_gradients():
    block = randomise(factories.pairformer_block(d_pair=64, triangle_model="af3", d_single=128), 0)
    block.set_backend("hip")
    block.requires_grad_(False)
    block.tri_multi_incoming.set_backend("pytorch")
    block.single_attention.requires_grad_(True)
    ops = {n: m for n, m in block.named_children()}
    backends = {n: m.backend for n, m in ops.items()}
    asked = {n: p.requires_grad for n, p in block.named_parameters()}
    training.install(block, "8bit")
    training.install(block, "input")  # (another kind: what there was before the first is still known)
    block.single_transition.set_backend("pytorch")  # a later choice of the caller's stays
    report = training.install(block, None)
    backends["single_transition"] = "pytorch"
    assert {n: m.backend for n, m in ops.items()} == backends
    assert {n: p.requires_grad for n, p in block.named_parameters()} == asked
    assert sorted(report["hip"] + report["pytorch"]) == sorted(ops) and set(report["hip"]) == {
        n for n, b in backends.items() if b == "hip"}
    block.requires_grad_(True)
    block.set_backend("pytorch")
    training.install(block, None)  # nothing to take back: nothing changes
    assert all(p.requires_grad for p in block.parameters()) and all(m.backend == "pytorch" for m in ops.values())
    training.install(block, "8bit", requires_grad=False)
    training.install(block, None)
    assert all(p.requires_grad for p in block.parameters())


def test_taking_back_a_part_and_a_copy():
    block = randomise(factories.pairformer_block(d_pair=64, triangle_model="af3", d_single=128), 0)
    block.set_backend("hip")
    block.requires_grad_(False)
    training.install(block, "8bit")
    other = copy.deepcopy(block)
    training.install(block.single_attention, None)
    assert block.single_attention.backend == "hip" and not any(p.requires_grad for p in block.single_attention.parameters())
    assert block.tri_multi_outgoing.backend == "pytorch" and all(p.requires_grad for p in block.transition_pair.parameters())
    for model in (block, other):
        training.install(model, None)
        assert all(m.backend == "hip" for m in model.children()) and not any(p.requires_grad for p in model.parameters())


def test_a_width_without_backward_kernels_is_refused_when_it_is_to_be_differentiated(monkeypatch):
    m = modules.Transition(832, 1)
    m.set_backend("hip")
    monkeypatch.setattr(modules, "hip_reason", lambda *t: None)
    x = torch.zeros(2, 832, dtype=BF16)
    assert m.unsupported(x) is None
    m.keep = "8bit"
    assert "backward" in m.unsupported(x)
    with torch.no_grad():
        assert m.unsupported(x) is None


def test_overlapped_trunk_records_what_its_second_stream_keeps(monkeypatch):
    """A step keeps tensors of the main stream for the second one's backward pass: each is recorded there, so that its
    memory is not handed out while that still reads it, whoever drops it first."""
    class Stream:
        wait_stream = wait_event = lambda self, other: None

    class Event:
        record = lambda self, stream: None  # noqa: E731

    recorded, side = [], Stream()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: stream is side and recorded.append(t))
    monkeypatch.setattr(trunk, "_side_stream", lambda device: side)
    model = randomise(trunk.PairformerTrunk(1, d_pair=64, d_single=64, n_head_single=4), 0)
    pair, single, mask = torch.randn(1, 3, 3, 64), torch.randn(1, 3, 64), torch.ones(1, 3, dtype=torch.bool)
    out, _ = model._forward_overlapped(pair, mask, single, 1)
    for t in (pair, out, single, mask):
        assert any(r is t for r in recorded)
