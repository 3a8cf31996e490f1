"""The training operators' kernels on the GPU against the 64-bit oracle.

Tolerances. An 8-bit activation is compared exactly. LayerNorm's gradients are fp32 computations: each of
the operations between the inputs and an output is off by at most 2^-24 of its result, and
``_norm_bounds`` multiplies the magnitudes of those results by the count of the operations; a bf16 output
adds half a step, 2^-8 of the value. The transition's products take rounded operands: one rounded to bf16 is off by
r = 2^-8 / sqrt(3) of itself in root mean square at most, to fp16 by r / 8. On the way to a gradient lie the
rounding of S under dy, of a hidden gradient or u, of xh or a weight beside it, and of the result, in bf16, and
an eighth of two more in a and b; they add in quadrature: r sqrt(4 + 2 / 64) = 4.6e-3 of the result's norm at most
(2 r for an ordinary r of 1.7e-3: 3.3e-3), held to 1e-2 as every op of the stack. A single value is held to 6 of
its own standard deviations, which ``_deviations`` follows through the formulas.
"""

from __future__ import annotations

import pytest
import torch

from foldforge_amd import kernels
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _stream_rows(g, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))
    return (x + 0.5 * torch.randn(cols, generator=g)).to(dtype)


def _close(got, want, tol, name):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    over = off > tol
    assert not over.any(), (name, int(over.sum()), float(off.max()), float(want.abs().max()))


# ------------------------------------------------------------------------------------ 8-bit activations
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 64), (1030, 64), (257, 128), (9, 100),
                                       (63, 384), (17, 451), (3, 1000), (5, 1500)])
def test_activation_is_the_definition(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = _stream_rows(g, rows, cols, dtype)
    a = kernels.quantize_activation(x.to(DEV))
    values, exps = oracle.held(x)
    assert torch.equal(a.scales.cpu().double(), exps + 127)
    assert torch.equal(a.codes.cpu().double(), values / torch.exp2(exps.repeat_interleave(32, -1)[..., :cols]))
    assert torch.equal(kernels.restore_activation(a).cpu().double(), values)
    assert a.restore().dtype == dtype and a.shape == x.shape


@pytest.mark.parametrize("cols", [64, 50])
def test_activation_of_extreme_values(cols):
    big = torch.finfo(F32).max
    rows = [
        [0.0], [-0.0], [448.0], [449.0, 1.0], [big, -big, 1e30], [2.0**-149], [2.0**-126, 2.0**-130], [1e-38, 3e-39],
        [float("inf"), 1.0], [float("-inf")], [float("nan"), -2.0, 0.1], [1.75], [1.7500001], [17.0, 448.0],
        [0.0009765625 * 7, 448.0], [0.0029296875, 448.0], [1.0625 * 2.0**-6, 448.0],
    ]
    x = torch.zeros(len(rows), cols)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
        x[i, 40:40 + len(r)] = torch.tensor(r)  # the short block, where there is one
    a = kernels.quantize_activation(x.to(DEV))
    values, exps = oracle.held(x)
    assert torch.equal(a.scales.cpu().double(), exps + 127)
    got = a.restore().cpu().double()
    # (fp32 has no value below 2^-149; the restored ones here are multiples of 2^-126 * 2^-9 at least)
    want = values.float().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_activation_of_views_off_alignment_and_empty():
    g = torch.Generator().manual_seed(5)
    flat = torch.randn(1 + 40 * 64, generator=g).to(DEV)
    x = flat[1:].view(40, 64)  # 4 bytes past alignment
    assert torch.equal(kernels.quantize_activation(x).restore(), kernels.quantize_activation(x.clone()).restore())
    a = kernels.quantize_activation(torch.empty(0, 64, device=DEV, dtype=BF16))
    assert a.restore().shape == (0, 64) and a.scales.shape == (0, 2)


# ------------------------------------------------------------------------------------ LayerNorm
def _norm_bounds(dy, x, w, eps, dtype, grad_dtype, want):
    """Elementwise bounds of (dx, dw, db): 32 fp32 operations (two sums' trees, the products between them) at
    the largest magnitudes they reach: rstd max|g| for a term of dx, times 1 + max|x| rstd for each of the two
    factors xh it can carry; for the sums over rows, their terms' magnitudes, and one more operation for every
    64 rows that a lane adds one after the other."""
    u = 2.0**-24
    dy, x = dy.double(), x.double()
    xh, rstd = oracle.normalised(x, eps)
    g = (dy if w is None else dy * w.double()).abs()
    grow = 1 + x.abs().amax(-1, keepdim=True) * rstd
    rows = max(1, x.numel() // x.shape[-1])
    half = 2.0**-8
    dx = 32 * u * rstd * g.amax(-1, keepdim=True) * grow**2 + (half if dtype == BF16 else u) * want[0].abs()
    axes = tuple(range(x.dim() - 1))
    count = (32 + rows / 64) * u
    last = half if grad_dtype == BF16 else u
    return (dx, count * (dy.abs() * grow).sum(axes) + last * want[1].abs(),
            count * dy.abs().sum(axes) + last * want[2].abs())


def _check_norm(x, dy, w, kept, eps=1e-5, grad_dtype=F32):
    """``x`` and ``dy`` on the CPU; ``kept``: what the kernel is given."""
    values = x if isinstance(kept, torch.Tensor) else oracle.held(x)[0]
    want = oracle.layer_norm_backward(dy, values, w, eps)
    got = kernels.layer_norm_backward(dy.to(DEV), kept, None if w is None else w.to(DEV), eps, grad_dtype=grad_dtype)
    bounds = _norm_bounds(dy, values, w, eps, dy.dtype, grad_dtype, want)
    assert got[0].dtype == dy.dtype
    for t, r, b, name in zip(got, want, bounds, ("dx", "dweight", "dbias")):
        if t is None:
            assert name == "dweight" and w is None
            continue
        if name != "dx":
            assert t.dtype == grad_dtype
        _close(t, r, b, name)
    return got


WIDTHS = [1, 2, 3, 31, 64, 65, 100, 128, 192, 256, 257, 384, 451, 512, 768, 777, 1000, 1024, 1025, 1500, 2050]


@pytest.mark.parametrize("keep", ["input", "8bit"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", WIDTHS)
def test_layer_norm_backward_widths(cols, dtype, keep):
    g = torch.Generator().manual_seed(cols)
    for rows in (1, 37):
        x, dy = _stream_rows(g, rows, cols, dtype), torch.randn(rows, cols, generator=g).to(dtype)
        w, b = 1 + 0.1 * torch.randn(cols, generator=g), torch.randn(cols, generator=g)
        if keep == "8bit":
            y, kept = kernels.layer_norm_checkpoint(x.to(DEV), w.to(DEV), b.to(DEV))
            xh, rstd = oracle.normalised(x.double(), 1e-5)
            grow = 1 + x.double().abs().amax(-1, keepdim=True) * rstd
            ref = xh * w.double() + b.double()
            _close(y, ref, 16 * 2.0**-24 * grow * (w.abs().double() + b.abs().double() + 1)
                   + (2.0**-8 if dtype == BF16 else 2.0**-24) * ref.abs(), "y")
            assert torch.equal(kept.restore(), kernels.quantize_activation(x.to(DEV)).restore())
        else:
            kept = x.to(DEV)
        _check_norm(x, dy, w, kept)


@pytest.mark.parametrize("rows,cols,dtype", [(5000, 128, BF16), (3001, 64, F32), (40009, 33, BF16), (4099, 384, BF16),
                                             (2100, 451, F32), (700, 1025, F32), (1, 768, BF16), (66000, 64, BF16)])
def test_layer_norm_backward_many_rows(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows)
    x, dy = _stream_rows(g, rows, cols, dtype), (0.02 * torch.randn(rows, cols, generator=g)).to(dtype)
    w = 1 + 0.1 * torch.randn(cols, generator=g)
    first = _check_norm(x, dy, w, x.to(DEV))
    again = kernels.layer_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # the same bits on every run
    _check_norm(x, dy, w, kernels.quantize_activation(x.to(DEV)))


@pytest.mark.parametrize("rows,dtype,off", [(3, BF16, 0), (257, BF16, 0), (300, BF16, 0), (5003, BF16, 0), (300, BF16, 1),
                                           (300, F32, 0)])
def test_layer_norm_backward_1536_channels(rows, dtype, off):
    """The widest rows that lie in registers (bf16, aligned): each of up to 1024 workgroups has a part of the affine's
    sums. Off alignment and in fp32 the same width takes the wide form."""
    cols = 1536
    g = torch.Generator().manual_seed(rows)
    x, dy = _stream_rows(g, rows, cols, dtype), torch.randn(rows, cols, generator=g).to(dtype)
    w = 1 + 0.1 * torch.randn(cols, generator=g)
    moved = torch.empty(off + x.numel(), dtype=dtype, device=DEV)[off:].view(rows, cols)
    moved.copy_(x)
    first = _check_norm(x, dy, w, moved)
    again = kernels.layer_norm_backward(dy.to(DEV), moved, w.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    _check_norm(x, dy, w, kernels.layer_norm_checkpoint(x.to(DEV), w.to(DEV), None)[1], grad_dtype=BF16)


def test_layer_norm_backward_forms():
    g = torch.Generator().manual_seed(3)
    x, dy = _stream_rows(g, 6 * 5, 128, BF16).view(2, 3, 5, 128), torch.randn(2, 3, 5, 128, generator=g).to(BF16)
    w = 1 + 0.1 * torch.randn(128, generator=g)
    _check_norm(x, dy, None, x.to(DEV))
    _check_norm(x, dy, w, x.to(DEV), grad_dtype=BF16)
    _check_norm(x, dy, w, x.to(DEV), eps=0.1)
    dx, dw, db = kernels.layer_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), with_bias=False)
    assert db is None and dw is not None
    dx, dw, db = kernels.layer_norm_backward(dy.to(DEV), x.to(DEV), None, with_bias=False)
    assert db is None and dw is None
    assert torch.equal(dx, kernels.layer_norm_backward(dy.to(DEV), x.to(DEV), None)[0])
    # no rows: empty dx, sums over nothing
    e = torch.empty(0, 128, device=DEV)
    dx, dw, db = kernels.layer_norm_backward(e, e, w.to(DEV))
    assert dx.shape == (0, 128) and not dw.any() and not db.any()


@pytest.mark.parametrize("cols", [64, 50, 1100])
def test_layer_norm_backward_eps_zero_rows_past_the_end(cols):
    """eps = 0 on finite rows: the lanes past the last row must not put 0 / 0 into the sums."""
    g = torch.Generator().manual_seed(cols)
    x, dy = _stream_rows(g, 3, cols, F32), torch.randn(3, cols, generator=g)
    _check_norm(x, dy, torch.ones(cols), x.to(DEV), eps=0.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_backward_off_alignment(dtype):
    g = torch.Generator().manual_seed(8)
    n = 33 * 128
    base = [torch.randn(1 + n, generator=g).to(dtype) for _ in range(2)]
    x, dy = (t[1:].view(33, 128) for t in base)
    xd, dyd = (t.to(DEV)[1:].view(33, 128) for t in base)
    w = torch.ones(129)[1:]
    want = oracle.layer_norm_backward(dy, x, w)
    got = kernels.layer_norm_backward(dyd, xd, torch.ones(129, device=DEV)[1:])
    for t, r, b, name in zip(got, want, _norm_bounds(dy, x, w, 1e-5, dtype, F32, want), ("dx", "dw", "db")):
        _close(t, r, b, name)


def test_layer_norm_backward_keeps_non_finite_rows_apart():
    g = torch.Generator().manual_seed(9)
    x, dy = torch.randn(40, 128, generator=g), torch.randn(40, 128, generator=g)
    clean = kernels.layer_norm_backward(dy.to(DEV), x.to(DEV))[0]
    x[7, 5], dy[21, 3] = float("nan"), float("inf")
    dx = kernels.layer_norm_backward(dy.to(DEV), x.to(DEV))[0]
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[7, 21]] = True
    assert torch.equal(dx.cpu()[~bad], clean.cpu()[~bad]) and dx[7].isnan().all() and not dx[21].isfinite().any()


def test_layer_norm_backward_past_32_bits():
    """A tensor of more than 2^31 values: the last rows, and the sums, are those of the whole tensor."""
    rows, cols = (1 << 24) + 5, 128
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.empty(rows, cols, dtype=BF16, device=DEV).normal_(generator=g)
    dy = torch.empty(rows, cols, dtype=BF16, device=DEV).normal_(generator=g)
    dx, dw, db = kernels.layer_norm_backward(dy, x)[0], *kernels.layer_norm_backward(dy, x, torch.ones(cols, device=DEV))[1:]
    tail = slice(rows - 300, rows)
    want = oracle.layer_norm_backward(dy[tail].cpu(), x[tail].cpu(), None)
    _close(dx[tail], want[0], _norm_bounds(dy[tail].cpu(), x[tail].cpu(), None, 1e-5, BF16, F32, want)[0], "dx")
    s, t = torch.zeros(cols, dtype=torch.float64, device=DEV), torch.zeros(cols, dtype=torch.float64, device=DEV)
    big = torch.zeros(cols, dtype=torch.float64, device=DEV)
    for r in range(0, rows, 1 << 20):
        d, v = dy[r:r + (1 << 20)].double(), x[r:r + (1 << 20)].double()
        xh = oracle.normalised(v, 1e-5)[0]
        s += (d * xh).sum(0)
        t += d.sum(0)
        big += d.abs().sum(0)
    # a lane adds rows / (1024 workgroups * 16) of them one after the other
    bound = 2.0**-24 * (64 + rows / 16384) * big.cpu() * 6
    _close(dw, s.cpu(), bound, "dweight")
    _close(db, t.cpu(), bound, "dbias")
    a = kernels.quantize_activation(x)
    assert torch.equal(a.restore()[tail].cpu().double(), oracle.held(x[tail].cpu())[0])


# ------------------------------------------------------------------------------------ transition
def _transition_case(rows, d, factor, seed):
    g = torch.Generator().manual_seed(seed)
    h = factor * d
    x, dy = _stream_rows(g, rows, d, BF16), (0.02 * torch.randn(rows, d, generator=g)).to(BF16)
    params = dict(ln_weight=1 + 0.1 * torch.randn(d, generator=g), ln_bias=0.1 * torch.randn(d, generator=g),
                  expand_a=torch.randn(h, d, generator=g) * d**-0.5, expand_b=torch.randn(h, d, generator=g) * d**-0.5,
                  squeeze=torch.randn(d, h, generator=g) * h**-0.5)
    return x, dy, params


def _deviations(dy, x, p, eps):
    """The standard deviation of each gradient's values under the roundings of the operands (bf16: r of each at
    most; fp16, under a and b: r / 8). (A value of a product's sum over channels: the terms' deviations in
    quadrature, since every term has roundings of its own. A sum over rows: the magnitudes added, since a weight's
    rounding is the same in every row, and one of xh the same for every hidden channel. A function of a and b: its
    derivatives' magnitudes times theirs. The rows' operand is xh, and the norm's affine comes after it: where
    xh w and the offset cancel in n, the error is that of xh w.)"""
    r = 2.0**-8 / 3**0.5
    dy, x = dy.double(), x.double()
    w, v, wa, wb, wo = (p[k].double() for k in ("ln_weight", "ln_bias", "expand_a", "expand_b", "squeeze"))
    xh, rstd = oracle.normalised(x, eps)
    scaled = xh * w
    n = scaled + v

    def quad(u, v):  # sqrt(sum over k of (u v)^2)
        return ((u * u) @ (v * v)).sqrt()

    a, b, du = n @ wa.T, n @ wb.T, dy @ wo
    sa, sb, sdu = 2**0.5 * r / 8 * quad(scaled, wa.T), 2**0.5 * r / 8 * quad(scaled, wb.T), r * quad(dy, wo)
    s = torch.sigmoid(a)
    silu, slope = a * s, s * (1 + a * (1 - s))
    bend = s * (1 - s) * (2 + a * (1 - 2 * s))  # slope's derivative
    u, db, da = silu * b, du * silu, du * b * slope
    su = (b * slope).abs() * sa + silu.abs() * sb + r * u.abs()
    sdb = silu.abs() * sdu + (du * slope).abs() * sa + r * db.abs()
    sda = (b * slope).abs() * sdu + (du * slope).abs() * sb + (du * b * bend).abs() * sa + r * da.abs()
    dn = da @ wa + db @ wb
    sdn = (quad(sda, wa) ** 2 + quad(sdb, wb) ** 2 + r * r * (quad(da, wa) ** 2 + quad(db, wb) ** 2)).sqrt()
    g = sdn * w.abs()
    dx = rstd * (g + g.mean(-1, keepdim=True) + xh.abs() * (g * xh.abs()).mean(-1, keepdim=True))
    return dict(x=dx, ln_weight=(sdn * xh.abs() + r * (dn * xh).abs()).sum(0), ln_bias=sdn.sum(0),
                expand_a=sda.T @ n.abs() + r * da.abs().T @ scaled.abs(),
                expand_b=sdb.T @ n.abs() + r * db.abs().T @ scaled.abs(), squeeze=dy.abs().T @ su)


def _near(got, want, deviation, name, dtype, norm):
    got, want, deviation = got.double().cpu(), want.double().cpu(), deviation.cpu()
    assert got.shape == want.shape
    off, size = got - want, want.norm()
    assert not norm or off.norm() <= 1e-2 * size, (name, float(off.norm() / size))
    over = off.abs() > 6 * deviation + (2.0**-8 if dtype == BF16 else 2.0**-20) * want.abs()
    assert not over.any(), (name, int(over.sum()), float(off.abs().max()))


def _check_transition(x, dy, params, kept, *, residual, grad_dtype=F32, eps=1e-5, norm=True):
    values = x if isinstance(kept, torch.Tensor) else oracle.held(x)[0]
    dev = {k: v.to(DEV) for k, v in params.items()}
    got = kernels.transition_backward(dy.to(DEV), kept, **dev, residual=residual, grad_dtype=grad_dtype, eps=eps)
    # (the oracle's arithmetic on the device: 64-bit products of these sizes are slow on the host)
    want = oracle.transition_backward(dy.to(DEV), values.to(DEV), **dev, residual=residual, eps=eps)
    deviations = _deviations(dy.to(DEV), values.to(DEV), dev, eps)
    for name, t in got._asdict().items():
        assert t.dtype == (BF16 if name == "x" else grad_dtype), name
        _near(t, want[name], deviations[name], name, t.dtype, norm)
    return got


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("keep", ["input", "8bit"])
@pytest.mark.parametrize("rows,d,factor", [(1, 64, 2), (1, 128, 4), (2, 384, 4), (31, 64, 1), (33, 128, 4), (65, 128, 2),
                                           (100, 384, 4), (129, 64, 4), (130, 256, 2), (257, 128, 4), (300, 192, 3),
                                           (64, 768, 3), (1000, 128, 4), (1025, 64, 4)])
def test_transition_backward(rows, d, factor, keep, residual):
    x, dy, params = _transition_case(rows, d, factor, rows + d)
    kept = kernels.quantize_activation(x.to(DEV)) if keep == "8bit" else x.to(DEV)
    _check_transition(x, dy, params, kept, residual=residual)


@pytest.mark.parametrize("rows,d,factor", [
    (5000, 128, 4), (20001, 64, 4), (9999, 64, 2), (23000, 256, 4), (45000, 128, 4),
    # the fused kernels from where they begin, one row past a tile, hidden widths that fill no workgroup
    (4096, 64, 4), (4097, 64, 1), (4223, 64, 3), (16384, 128, 4), (16385, 128, 1), (16641, 128, 3), (17000, 128, 16),
    (16400, 128, 17), (4500, 64, 33),
    # two chunks of rows, the second a short one
    (262144 + 33, 128, 4), (262144 + 65, 64, 2), (33001, 256, 4), (66001, 256, 2),
    # 128 x 128 and 64 x 64 tiles
    (4095, 256, 2), (4097, 256, 1), (5001, 384, 4), (6000, 192, 3), (4100, 320, 2), (9000, 512, 1), (4200, 768, 2)])
def test_transition_backward_many_rows(rows, d, factor):
    x, dy, params = _transition_case(rows, d, factor, rows)
    first = _check_transition(x, dy, params, x.to(DEV), residual=True, grad_dtype=BF16)
    dev = {k: v.to(DEV) for k, v in params.items()}
    again = kernels.transition_backward(dy.to(DEV), x.to(DEV), **dev, grad_dtype=BF16)
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # the same bits on every run
    _check_transition(x, dy, params, kernels.quantize_activation(x.to(DEV)), residual=False)


@pytest.mark.parametrize("rows,d,factor", [
    # both sides of the rule for the fused kernels
    (16384, 128, 1), (16448, 128, 2), (8191, 64, 8), (8192, 64, 5), (8193, 64, 32), (4096, 64, 2),
    # and of the one for rows that stream by
    (9728, 256, 2), (9729, 256, 2), (4100, 256, 8), (19600, 256, 1)])
def test_transition_backward_at_the_rules(rows, d, factor):
    x, dy, params = _transition_case(rows, d, factor, rows + factor)
    _check_transition(x, dy, params, x.to(DEV), residual=True)


def test_transition_backward_past_32_bits():
    """More than 2^31 values: the last rows' gradients are those of the rows alone."""
    rows, d = (1 << 24) + 77, 128
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.empty(rows, d, dtype=BF16, device=DEV).normal_(generator=g)
    dy = torch.empty(rows, d, dtype=BF16, device=DEV).normal_(generator=g)
    params = {k: v.to(DEV) for k, v in _transition_case(1, d, 1, 5)[2].items()}
    got = kernels.transition_backward(dy, x, **params)
    tail = slice(rows - 400, rows)
    want = oracle.transition_backward(dy[tail], x[tail], **params)
    _near(got.x[tail], want["x"], _deviations(dy[tail], x[tail], params, 1e-5)["x"], "x", BF16, True)
    # the sums over all rows are those of two halves
    half = [kernels.transition_backward(dy[s], x[s], **params) for s in (slice(0, 1 << 23), slice(1 << 23, rows))]
    for name in ("ln_weight", "ln_bias", "expand_a", "expand_b", "squeeze"):
        a, b, c = (getattr(t, name) for t in (got, *half))
        # (fp32 sums of the same products in another order: 2^-24 of their magnitudes for each of some 2^10 additions)
        assert float((a - b - c).norm()) <= 2.0**-14 * float(b.norm() + c.norm()) + 1e-30, name


def test_transition_backward_no_rows():
    _, _, params = _transition_case(1, 128, 4, 0)
    e = torch.empty(0, 128, dtype=BF16, device=DEV)
    got = kernels.transition_backward(e, e, **{k: v.to(DEV) for k, v in params.items()})
    assert got.x.shape == (0, 128)
    assert all(not t.any() for t in got[1:])


def test_transition_backward_large_gates():
    """Gates far to both sides: the logistic function at 0 and 1, no NaN. Values of a of about 60 are off by
    60 * 2^(1/2) * 2^-8 / 3^(1/2) / 8 = 0.024 where the slope goes from 0 to 1 within a few units, so the norms' bound,
    which is for gates of order one, says nothing here; each value's own deviations (bend times that of a) do."""
    x, dy, params = _transition_case(96, 128, 4, 1)
    params["expand_a"] *= 60
    _check_transition(x, dy, params, x.to(DEV), residual=True, norm=False)


@pytest.mark.parametrize("rows,d", [(3, 64), (300, 128), (20000, 128)])
def test_transition_backward_with_zero_weights_of_the_norm(rows, d):
    """Channels whose LayerNorm weight is 0 (or all of them): their gradient is still the sum over the rows."""
    x, dy, params = _transition_case(rows, d, 4, 11)
    params["ln_weight"][::3] = 0
    _check_transition(x, dy, params, x.to(DEV), residual=False)
    params["ln_weight"].zero_()
    _check_transition(x, dy, params, x.to(DEV), residual=True)


def test_transition_backward_scales():
    """Weights and gradients far from 1 (fp16 holds neither as they are): the results scale with them exactly."""
    x, dy, params = _transition_case(130, 128, 4, 12)
    want = kernels.transition_backward(dy.to(DEV), x.to(DEV), **{k: v.to(DEV) for k, v in params.items()}, residual=False)
    # expand_b and dy times powers of two: u and db scale, so every gradient does
    for kb, ky in ((-40, 0), (30, -60), (0, 40)):
        p = {**params, "expand_b": params["expand_b"] * 2.0**kb}
        got = kernels.transition_backward((dy.float() * 2.0**ky).to(BF16).to(DEV), x.to(DEV),
                                          **{k: v.to(DEV) for k, v in p.items()}, residual=False)
        for name, e in (("x", kb + ky), ("ln_weight", kb + ky), ("ln_bias", kb + ky), ("expand_a", kb + ky),
                        ("expand_b", ky), ("squeeze", kb + ky)):
            assert torch.equal(getattr(got, name).float(), getattr(want, name).float() * 2.0**e), (name, kb, ky)


@pytest.mark.parametrize("rows", [130, 16400])
def test_transition_backward_scales_of_the_affine(rows):
    """The norm's weight or bias or a weight matrix powers of two away from the rest. A weight or a matrix scaled by
    powers whose product is 1 leaves the hidden values, so every gradient scales exactly; a weight far below its bias
    still gives the formula's gradients."""
    x, dy, params = _transition_case(rows, 128, 4, 12)
    x, dy = x.to(DEV), dy.to(DEV)
    dev = {k: v.to(DEV) for k, v in params.items()}
    want = kernels.transition_backward(dy, x, **dev, residual=False)
    for k in (-90, -40, 60):  # weight and bias by 2^k, the matrices by 2^-k
        p = {**dev, **{n: dev[n] * 2.0**k for n in ("ln_weight", "ln_bias")},
             **{n: dev[n] * 2.0**-k for n in ("expand_a", "expand_b")}}
        got = kernels.transition_backward(dy, x, **p, residual=False)
        for name, e in (("x", 0), ("ln_weight", -k), ("ln_bias", -k), ("expand_a", k), ("expand_b", k), ("squeeze", 0)):
            assert torch.equal(getattr(got, name).float(), getattr(want, name).float() * 2.0**e), (name, k)
    for k in (-100, -30):
        p = {**params, "ln_weight": params["ln_weight"] * 2.0**k}
        _check_transition(x.cpu(), dy.cpu(), p, x, residual=False)
    # both matrices tiny: u and dS (2^-160) end below fp32, the other gradients scale
    p = {**dev, **{n: dev[n] * 2.0**-80 for n in ("expand_a", "expand_b")}}
    got = kernels.transition_backward(dy, x, **p, residual=False)
    assert all(torch.isfinite(t.float()).all() for t in got) and not got.squeeze.any()


@pytest.mark.parametrize("rows,d,factor", [(130, 128, 4), (4100, 64, 4), (24600, 128, 2), (4500, 256, 1)])
def test_transition_backward_hidden_channels_of_unlike_size(rows, d, factor):
    """Hidden channels up to 2^20 apart, neighbours among them: the fused kernels scale 32 of them by one power of two
    for fp16, whose range leaves the small ones their bits (their entries' last bit is 2^-25, 2^-17 of the entries of
    the smallest channel, far below r / 8). Every channel's gradients are held to its own deviations."""
    x, dy, params = _transition_case(rows, d, factor, 13)
    g = torch.Generator().manual_seed(14)
    for name in ("expand_a", "expand_b"):
        params[name] *= torch.exp2(-torch.randint(0, 21, (factor * d, 1), generator=g).float())
    _check_transition(x, dy, params, x.to(DEV), residual=False)


@pytest.mark.parametrize("keep", ["input", "8bit"])
@pytest.mark.parametrize("rows,d,factor", [
    (33, 128, 4), (100, 384, 4),  # few rows
    (2001, 128, 4), (6001, 192, 3),  # 64 x 64 tiles
    (9801, 256, 2), (5001, 384, 2),  # streamed hidden gradients, 128 x 128 tiles
    (4129, 64, 4), (24641, 128, 1)])  # the fused kernels
def test_transition_backward_keeps_non_finite_rows_apart(rows, d, factor, keep):
    """Rows share tiles, and the last one stands in for those behind the end: one that is not finite leaves the others'
    dx as they are, bit for bit, and reaches every gradient of the parameters."""
    x, dy, params = _transition_case(rows, d, factor, 15)
    dev = {k: v.to(DEV) for k, v in params.items()}

    def run(x, dy):
        kept = x.to(DEV) if keep == "input" else kernels.quantize_activation(x.to(DEV))
        return kernels.transition_backward(dy.to(DEV), kept, **dev)

    clean = run(x, dy).x
    bad_x, bad_dy = x.clone(), dy.clone()
    bad_x[7, 5] = bad_x[-1, 0] = float("nan")
    bad_dy[21, 3] = float("inf")
    for got, bad in ((run(bad_x, dy), [7, rows - 1]), (run(x, bad_dy), [21])):
        kept = torch.ones(rows, dtype=torch.bool, device=DEV)
        kept[bad] = False
        assert torch.equal(got.x[kept], clean[kept]) and not got.x[~kept].isfinite().any()
        for name, t in list(got._asdict().items())[1:]:
            if name == "squeeze" and bad == [21]:  # dS = dy^T u: the one channel's
                assert t[torch.arange(d, device=DEV) != 3].isfinite().all()
                t = t[3]
            assert not t.isfinite().any(), name


def test_transition_checkpoint_is_the_forward():
    x, _, params = _transition_case(333, 128, 4, 2)
    dev = {k: v.to(DEV) for k, v in params.items()}
    y, a = kernels.transition_checkpoint(x.to(DEV), **dev)
    assert torch.equal(y, kernels.transition(x.to(DEV), **dev))
    assert torch.equal(a.restore().cpu().double(), oracle.held(x)[0])


@pytest.mark.parametrize("rows,d,factor", [(333, 128, 4), (70, 384, 4)])
def test_transition_checkpoint_in_place(rows, d, factor):
    """Written over its input (or into another tensor) it keeps the 8 bits of the input."""
    x, dy, params = _transition_case(rows, d, factor, 3)
    dev = {k: v.to(DEV) for k, v in params.items()}
    y, a = kernels.transition_checkpoint(x.to(DEV), **dev)
    other = torch.empty(rows, d, dtype=BF16, device=DEV)
    for given, out in ((x.to(DEV), other), (x.to(DEV), None)):
        out = given if out is None else out
        got, kept = kernels.transition_checkpoint(given, out=out, **dev)
        assert got is out and torch.equal(got, y)
        assert torch.equal(kept.restore(), a.restore()) and torch.equal(kept.scales, a.scales)
        for t, want in zip(kernels.transition_backward(dy.to(DEV), kept, **dev),
                           kernels.transition_backward(dy.to(DEV), a, **dev)):
            assert torch.equal(t, want)


# ------------------------------------------------------------------------------------ streams and graphs
def test_on_another_stream():
    x, dy, params = _transition_case(400, 128, 4, 6)
    dev = {k: v.to(DEV) for k, v in params.items()}
    x, dy = x.to(DEV), dy.to(DEV)
    want = kernels.transition_backward(dy, x, **dev)
    norm = kernels.layer_norm_backward(dy, kernels.quantize_activation(x), dev["ln_weight"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = kernels.transition_backward(dy, x, **dev)
        got_norm = kernels.layer_norm_backward(dy, kernels.quantize_activation(x), dev["ln_weight"])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*want, *norm), (*got, *got_norm)))


@pytest.mark.parametrize("rows,d,factor", [(100, 384, 4), (1, 64, 2), (2000, 128, 4), (4200, 64, 4), (16500, 128, 4),
                                           (4500, 256, 2)])
def test_every_form_captured(rows, d, factor):
    """Each form's call in a graph, replayed on new inputs and parameters."""
    x, dy, params = _transition_case(rows, d, factor, rows)
    x, dy, dev = x.to(DEV), dy.to(DEV), {k: v.to(DEV) for k, v in params.items()}
    kernels.transition_backward(dy, x, **dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.transition_backward(dy, x, **dev)
    for turn in range(3):
        x.copy_(torch.randn_like(x))
        dev["expand_a"].mul_(0.75)
        want = kernels.transition_backward(dy, x, **dev)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_streamed_form_captured():
    test_every_form_captured(9800, 256, 2)


def test_two_graphs_replayed():
    """Two captured steps, replayed in turn with eager work between them, on new inputs each time."""
    cases = []
    for rows, d in ((700, 128), (333, 64)):
        x, dy, params = _transition_case(rows, d, 4, rows)
        cases.append((x.to(DEV), dy.to(DEV), {k: v.to(DEV) for k, v in params.items()}))

    def step(x, dy, params):
        y, a = kernels.transition_checkpoint(x, **params)
        g = kernels.transition_backward(dy, a, **params)
        z, b = kernels.layer_norm_checkpoint(x, params["ln_weight"], params["ln_bias"])
        return (y, z, *g, *kernels.layer_norm_backward(dy, b, params["ln_weight"]))

    graphs = []
    for case in cases:
        step(*case)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*case)
        graphs.append((graph, out))
    for turn in range(3):
        for (graph, out), case in zip(graphs, cases):
            case[0].copy_(torch.randn_like(case[0]))
            case[1].mul_(0.5)
            want = step(*case)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
