"""Projections with low-rank adapters: the kernels against the 64-bit oracle.

Tolerances. A value is a sum of products whose magnitudes ``mag`` the oracle gives at the absolute values of everything.
Each fp32 operation is off by at most 2^-24 of its result, and no sum is longer than its terms' count: ``n 2^-24 mag``.
An operand rounded to bf16 is off by at most 2^-8 of itself, and with it every product that it enters: fp32 weights and the
rows ``A x`` (above 256 rows) in the outputs. For the adapters' gradients the rows and the fp32 adapters are kept as three
bf16: each leaves 2^-8 of what it rounds, 2^-24 after the third, as fp32 itself. A bf16 result adds 2^-8 of itself. These
bound every value. In norm, roundings of many terms add in quadrature: r = 2^-8 / sqrt(3) of the result for each operand
rounded, so sqrt(4) r = 4.5e-3 for the outputs (weight, rows, adapters and result), held to 1e-2 as every op of the stack,
and sqrt(n) 2^-24 for fp32 gradients, 1.2e-5 for the longest sum here (n = 40000 rows and a width), held to 1.5e-5.
"""

from __future__ import annotations

import pytest
import torch

from foldforge_amd import kernels
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
HALF = 2.0**-8  # bf16's half step


def make(rows, d_in, d_out, rank, adapters, lengths, *, weight=BF16, adapter=BF16, seed=0, bias=False, scale=True, ids=None):
    """The call's tensors on the CPU; ``lengths``: of the requests, in order (rows behind them have none)."""
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    ids = [i % adapters for i in range(len(lengths))] if ids is None else ids
    offsets = torch.tensor([0, *torch.tensor(lengths, dtype=torch.long).cumsum(0).tolist()], dtype=torch.int32)
    return dict(
        x=normal(rows, d_in).to(BF16), dy=(0.1 * normal(rows, d_out)).to(BF16),
        weight=(normal(d_out, d_in) * d_in**-0.5).to(weight), bias=normal(d_out) if bias else None,
        down=(normal(adapters, rank, d_in) * d_in**-0.5).to(adapter),
        up=(normal(adapters, d_out, rank) * rank**-0.5).to(adapter),
        scale=0.5 + torch.rand(adapters, generator=g) if scale else None,
        offsets=offsets, adapter=torch.tensor(ids, dtype=torch.int32))


def gpu(t):
    return {k: None if v is None else v.to(DEV) for k, v in t.items()}


def forward(t, **how):
    return kernels.adapted_linear(t["x"], t["weight"], t["bias"], down=t["down"], up=t["up"], scale=t["scale"],
                                  offsets=t["offsets"], adapter=t["adapter"], **how)


def backward(t, **how):
    return kernels.adapted_linear_backward(t["dy"], t["x"], t["weight"], down=t["down"], up=t["up"], scale=t["scale"],
                                           offsets=t["offsets"], adapter=t["adapter"], **how)


def near(got, want, tol, rel, name):
    got = got.double().cpu()
    assert got.shape == want.shape, name
    off = (got - want).abs()
    assert not (off > tol).any(), (name, int((off > tol).sum()), float(off.max()))
    assert not torch.isnan(got).any(), name
    if want.norm() > 0:
        assert float((got - want).norm() / want.norm()) <= rel, (name, float((got - want).norm() / want.norm()))


def rows_of(t):
    return oracle.adapter_of_rows(t["x"].shape[0], t["offsets"], t["adapter"], t["down"].shape[0])


def check_forward(t, got):
    of, d_in, rank = rows_of(t), t["x"].shape[1], t["down"].shape[1]
    args = [t[k] for k in ("x", "weight", "bias", "down", "up", "scale")]
    want = oracle.adapted_linear(*args, of)
    mag = oracle.adapted_linear(*(None if a is None else a.abs() for a in args), of)
    base = oracle.adapted_linear(*(None if a is None else a.abs() for a in args), torch.full_like(of, -1))
    few = t["x"].shape[0] <= 256
    tol = (d_in + rank + 8) * 2.0**-24 * mag + HALF * want.abs()
    if t["weight"].dtype == F32:
        tol += HALF * base
    # (two operands' roundings at once: their sum and product)
    tol += ((0 if few else 1) + (0 if few or t["down"].dtype == BF16 else 2)) * HALF * (1 + 2 * HALF) * (mag - base)
    near(got, want, tol, 1e-2, "y")


def check_backward(t, got, grad_dtype=F32):
    of, (rows, d_in), d_out, rank = rows_of(t), t["x"].shape, t["weight"].shape[0], t["down"].shape[1]
    args = [t[k] for k in ("dy", "x", "weight", "down", "up", "scale")]
    want = oracle.adapted_linear_backward(*args, of)
    mag = oracle.adapted_linear_backward(*(None if a is None else a.abs() for a in args), of)
    if got.x is not None:
        base = oracle.adapted_linear_backward(*(None if a is None else a.abs() for a in args), torch.full_like(of, -1))[0]
        tol = (d_out + rank + 8) * 2.0**-24 * mag[0] + HALF * want[0].abs()
        if t["weight"].dtype == F32:
            tol += HALF * base
        tol += (1 if t["down"].dtype == BF16 else 2) * HALF * (1 + 2 * HALF) * (mag[0] - base)
        near(got.x, want[0], tol, 1e-2, "dx")
    for g, w, m, width, name in ((got.down, want[1], mag[1], d_out, "down"), (got.up, want[2], mag[2], d_in, "up")):
        assert g.dtype == grad_dtype
        tol = (width + rows + 10) * 2.0**-24 * m
        if grad_dtype == BF16:
            tol += HALF * w.abs()
        near(g, w, tol, 1e-2 if grad_dtype == BF16 else 1.5e-5, name)


#: rows, d_in, d_out, rank, adapters, lengths of the requests
CASES = [
    (1, 64, 64, 4, 1, [1]),
    (1, 384, 1536, 8, 3, [0, 1, 0]),
    (7, 128, 128, 16, 7, [1] * 7),
    (33, 449, 384, 5, 4, [1] * 30),
    (64, 768, 768, 16, 64, [1] * 64),
    (100, 100, 36, 7, 2, [40, 0, 60]),
    (256, 384, 384, 33, 9, [1] * 256),
    (257, 384, 384, 16, 9, [1] * 257),
    (300, 128, 512, 16, 1, [300]),
    (301, 128, 512, 16, 3, [64, 64, 63, 1, 0, 109]),
    (1021, 449, 384, 5, 2, [500, 21, 500]),
    (1000, 72, 100, 64, 5, [10] * 90),
    (700, 17, 13, 1, 3, [100, 200, 400]),
    (600, 512, 128, 128, 2, [300, 299]),
    (513, 64, 256, 48, 64, [8] * 64),
    (2000, 384, 1536, 32, 4, [1000, 0, 0, 999]),
    (5000, 1536, 384, 16, 3, [123, 4000, 877]),
    (16500, 64, 192, 100, 2, [16384, 100]),
    (40000, 128, 256, 16, 2, [20000, 20000]),
    # the widths that are served in one pass, with one, few and many requests, shared adapters, short ones and padding
    (300, 64, 64, 16, 2, [299, 1]),
    (1000, 64, 128, 12, 3, [31, 33, 0, 500, 1, 1, 300]),
    (999, 128, 64, 3, 1, [999]),
    (5000, 64, 256, 16, 4, [1000, 63, 65, 2000, 1872]),
    (4097, 256, 64, 15, 2, [4096]),
    (2222, 128, 128, 16, 5, [7, 400, 9, 800, 1000]),
    (9001, 128, 512, 8, 3, [3000, 1, 2999, 3000]),
    (3001, 512, 128, 16, 7, [100] * 29),
    (700, 256, 128, 9, 2, [350, 350]),
    (1500, 256, 256, 16, 3, [20] * 20),
    (20000, 128, 512, 16, 2, [19968, 32]),
    (1300, 128, 512, 27, 2, [600, 650]),
    (900, 512, 128, 32, 3, [300, 300, 300]),
    (640, 256, 256, 20, 1, [640]),
]


@pytest.mark.parametrize("weight,adapter", [(BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_forward_is_the_definition(case, weight, adapter):
    t = make(*case, weight=weight, adapter=adapter, seed=len(str(case)), bias=case[0] % 2 == 1)
    check_forward(t, forward(gpu(t)))


@pytest.mark.parametrize("weight,adapter", [(BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_backward_is_the_definition(case, weight, adapter):
    t = make(*case, weight=weight, adapter=adapter, seed=len(str(case)))
    check_backward(t, backward(gpu(t)))


#: rows from which on the backward pass (and the forward of wide rows) is one pass: a tile more or less, short requests, long
#: ones, rows before, between and behind them
MANY = [
    (4096, 64, 64, 16, 2, [4000, 96]),
    (4129, 64, 128, 12, 3, [31, 33, 0, 500, 1, 1, 3500]),
    (5000, 128, 64, 3, 1, [5000]),
    (4100, 64, 256, 16, 4, [1000, 63, 65, 2000, 872]),
    (4097, 256, 64, 15, 2, [4096]),
    (6000, 128, 128, 16, 5, [7, 400, 9, 800, 1000] + [64] * 40),
    (8200, 128, 256, 16, 2, [4100, 4100]),
    (8193, 256, 128, 9, 2, [350, 350]),
    (8192, 256, 256, 5, 3, [17] * 100),
    (8999, 512, 128, 16, 7, [100] * 89),
    (8400, 128, 512, 11, 8, [64] * 131),
    (32768, 64, 64, 16, 9, [64] * 512),
    (12300, 256, 256, 20, 2, [6000, 6300]),
    (12289, 512, 256, 32, 3, [300, 300, 11000]),
    (6145, 384, 384, 16, 9, [96] * 64),
    (6200, 384, 256, 31, 1, [6177]),
]


@pytest.mark.parametrize("weight,adapter", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("case", MANY, ids=lambda c: "x".join(map(str, c[:5])))
def test_many_rows(case, weight, adapter):
    t = make(*case, weight=weight, adapter=adapter, seed=case[0], bias=case[0] % 2 == 1)
    check_forward(t, forward(gpu(t)))
    check_backward(t, backward(gpu(t)))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_many_rows_keep_infinities_to_their_request(value):
    n = 1399
    t = make(3 * n, 128, 128, 13, 3, [n, n, n], adapter=F32)
    sick = {k: None if v is None else v.clone() for k, v in t.items()}
    for row in (n, 2 * n - 1):  # the request's ends, in tiles that it shares
        sick["x"][row] = value
        sick["dy"][row] = value
    sick["up"][1, 3] = value
    sick["down"][1, :, 5] = value
    other = torch.ones(3 * n, dtype=torch.bool)
    other[n:2 * n] = False
    assert torch.equal(forward(gpu(sick)).cpu()[other], forward(gpu(t)).cpu()[other])
    a, b = backward(gpu(sick)), backward(gpu(t))
    assert torch.equal(a.x.cpu()[other], b.x.cpu()[other])
    for i in (0, 2):
        assert torch.equal(a.down[i], b.down[i]) and torch.equal(a.up[i], b.up[i])


def test_many_rows_and_an_infinite_gradient():
    rows, d = 4500, 64
    t = make(rows, d, d, 5, 2, [rows // 2, rows - rows // 2])
    for name, at in (("weight", 3), ("down", ...), ("up", (slice(None), 3))):
        t[name][at] = t[name][at].abs() + 0.125
    t["dy"][rows // 2 + 1, 3] = float("inf")
    dx = backward(gpu(t)).x.cpu()
    assert (dx[rows // 2 + 1] == float("inf")).all()
    assert dx.isfinite().sum() == (rows - 1) * d


def test_backward_forms_of_many_rows():
    t = make(4200, 128, 128, 8, 3, [2000, 2], adapter=F32, scale=False)
    g = gpu(t)
    whole = backward(g)
    short = backward(g, with_x=False)
    assert short.x is None and torch.equal(short.down, whole.down) and torch.equal(short.up, whole.up)
    check_backward(t, backward(g, grad_dtype=BF16), BF16)
    assert not whole.down[2].any() and not whole.up[2].any()  # an adapter without rows


@pytest.mark.parametrize("rows", [5, 300])
def test_backward_forms(rows):
    t = make(rows, 128, 192, 8, 3, [rows // 2, 2], adapter=F32, scale=False)
    g = gpu(t)
    whole = backward(g)
    check_backward(t, whole)
    short = backward(g, with_x=False)
    assert short.x is None and torch.equal(short.down, whole.down) and torch.equal(short.up, whole.up)
    check_backward(t, backward(g, grad_dtype=BF16), BF16)
    assert not whole.down[2].any() and not whole.up[2].any()  # an adapter without rows


@pytest.mark.parametrize("rows", [40, 400, 4500])
def test_requests_without_an_adapter(rows):
    """Ids that are none of the adapters, rows before the first and behind the last request: the projection alone."""
    n = rows // 5
    t = make(rows, 128, 128, 16, 2, [n] * 5, ids=[-1, 0, 2, 2**31 - 1, -2**31])
    t["offsets"] = (t["offsets"] // 2 + 3).to(torch.int32)
    got = forward(gpu(t))
    check_forward(t, got)
    check_backward(t, backward(gpu(t)))
    plain = make(rows, 128, 128, 16, 2, [])
    assert torch.equal(forward(gpu({**t, "offsets": plain["offsets"], "adapter": plain["adapter"]}))[:3], got[:3])


@pytest.mark.parametrize("offsets", [[5, 3, 9, 2], [-7, -3, 1000, 4], [2**31 - 1, -2**31, 0, 50], [0, 2**31 - 1, 2**31 - 1, 7]])
@pytest.mark.parametrize("rows", [50, 500, 5000])
def test_offsets_out_of_order_stay_within_the_rows(rows, offsets):
    """Offsets that decrease are not refused (they lie on the device): the adapters' values are unspecified then, but each row
    has some adapter or none and no access is out of range."""
    t = gpu(make(rows, 64, 64, 8, 3, [10, 10, 10]))
    t["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    assert torch.isfinite(forward(t).float()).all()
    assert torch.isfinite(backward(t).x.float()).all()


@pytest.mark.parametrize("rows", [48, 320])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_request_keeps_its_infinities_to_itself(rows, value):
    n = rows // 3
    t = make(rows, 128, 192, 16, 3, [n, n, n], adapter=F32)
    sick = {k: None if v is None else v.clone() for k, v in t.items()}
    sick["x"][n + 1] = value  # a row of the second request
    sick["dy"][n + 2] = value
    sick["up"][1, 3] = value  # and its adapter
    sick["down"][1, :, 5] = value
    other = torch.ones(rows, dtype=torch.bool)
    other[n:2 * n] = False
    assert torch.equal(forward(gpu(sick)).cpu()[other], forward(gpu(t)).cpu()[other])
    a, b = backward(gpu(sick)), backward(gpu(t))
    assert torch.equal(a.x.cpu()[other], b.x.cpu()[other])
    for i in (0, 2):
        assert torch.equal(a.down[i], b.down[i]) and torch.equal(a.up[i], b.up[i])
    assert not torch.isfinite(a.up[1]).all() and not torch.isfinite(a.down[1]).all()


@pytest.mark.parametrize("rows, d_in, d_out", [(20, 64, 64), (400, 64, 64), (400, 128, 192), (400, 72, 64)])
def test_an_infinite_input_stays_infinite(rows, d_in, d_out):
    """Weights above zero at the infinite channel: the row's every output is the infinity that the sums give, at a rank that
    fills no block of the products."""
    t = make(rows, d_in, d_out, 5, 2, [rows // 2, rows - rows // 2])
    for name, at in (("weight", (slice(None), 3)), ("down", (..., 3)), ("up", ...)):
        t[name][at] = t[name][at].abs() + 0.125
    t["x"][rows // 2 + 1, 3] = float("inf")
    y = forward(gpu(t)).cpu()
    assert (y[rows // 2 + 1] == float("inf")).all()
    assert y.isfinite().sum() == (rows - 1) * d_out
    t = make(rows, d_in, d_out, 5, 2, [rows // 2, rows - rows // 2])
    for name, at in (("weight", 3), ("down", ...), ("up", (slice(None), 3))):
        t[name][at] = t[name][at].abs() + 0.125
    t["dy"][rows // 2 + 1, 3] = float("inf")
    dx = backward(gpu(t)).x.cpu()
    assert (dx[rows // 2 + 1] == float("inf")).all()
    assert dx.isfinite().sum() == (rows - 1) * d_in


def test_requests_that_share_an_adapter():
    t = make(900, 128, 128, 16, 2, [100, 200, 300, 250], ids=[1, 0, 1, 1])
    check_forward(t, forward(gpu(t)))
    check_backward(t, backward(gpu(t)))


def test_gradients_against_differences():
    """The loss's change along a random direction of the adapters, at 64 bits, is the gradient's product with it."""
    t = make(500, 96, 80, 6, 2, [200, 300], adapter=F32)
    got = backward(gpu(t))
    of = rows_of(t)

    def loss(down, up):
        return (oracle.adapted_linear(t["x"], t["weight"], None, down, up, t["scale"], of) * t["dy"].double()).sum()

    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(("down", "up")):
        d = torch.randn(t[name].shape, generator=g, dtype=torch.float64)
        d = d / d.norm()
        h = 1e-4
        p = [t["down"].double(), t["up"].double()]
        plus, minus = list(p), list(p)
        plus[i], minus[i] = p[i] + h * d, p[i] - h * d
        slope = (loss(*plus) - loss(*minus)) / (2 * h)  # (the loss is quadratic in neither alone: exact but for rounding)
        grad = getattr(got, name).double().cpu()
        assert abs(float(slope - (grad * d).sum())) <= 1.5e-5 * float(grad.norm()) + 1e-8 * float(slope.abs())


def test_leading_axes_and_an_output():
    t = make(2 * 12 * 12, 64, 128, 8, 2, [144, 144])
    g = gpu(t)
    flat = forward(g)
    g["x"] = g["x"].view(2, 12, 12, 64)
    out = torch.empty(2, 12, 12, 128, dtype=BF16, device=DEV)
    assert forward(g, out=out) is out and torch.equal(out.view(-1, 128), flat)
    g["dy"] = g["dy"].view(2, 12, 12, 128)
    assert backward(g).x.shape == (2, 12, 12, 64)


def test_entries_refuse_an_output_over_an_input():
    t = gpu(make(40, 64, 64, 8, 1, [40]))
    q = kernels._adapted(*(t[k] for k in ("x", "weight", "bias", "down", "up", "scale", "offsets", "adapter")))
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    args = [t[k] for k in ("weight", "bias", "down", "up", "scale", "offsets", "adapter")]
    with pytest.raises(RuntimeError, match="null or x"):
        kernels._call(t["x"].device, "adapted_linear", t["x"], *args, t["x"], ws, ws.numel(), *q)
    grads = [torch.empty_like(t[k], dtype=F32) for k in ("down", "up")]
    args.pop(1)
    for dx in (t["x"], t["dy"]):
        with pytest.raises(RuntimeError, match="dx may not be"):
            kernels._call(dx.device, "adapted_linear_backward", t["dy"], t["x"], *args, dx, *grads, ws, ws.numel(), *q, 1)


def test_no_rows():
    t = gpu(make(0, 64, 64, 8, 2, [0, 0]))
    assert forward(t).shape == (0, 64)
    got = backward(t)
    assert got.x.shape == (0, 64) and not got.down.any() and not got.up.any()


@pytest.mark.parametrize("rows", [3, 700, 8200])
def test_captured_calls(rows):
    """A forward and a backward pass in a graph, replayed on new values between other work."""
    a, b = (make(rows, 128, 256, 8, 2, [rows // 3, rows // 2], adapter=F32, seed=s) for s in (1, 2))
    g = gpu(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward(g), backward(g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads = forward(g), backward(g)
    for t in (a, b, a):
        for k, v in g.items():
            if v is not None:
                v.copy_(t[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_forward(t, y)
        check_backward(t, grads)
        assert torch.equal(y, forward(g)) and all(torch.equal(p, q) for p, q in zip(grads, backward(g)))


def test_two_streams_at_once():
    sets = [gpu(make(900, 256, 128, 16, 3, [300, 200, 400], seed=s)) for s in (1, 2)]
    want = [(forward(t), *backward(t)) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for t, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append((forward(t), *backward(t)))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(p, q))


#: rows, d_in, d_out, rank: one pass at narrow and wide widths; tiles of each block of ranks
INFINITE = [(4500, 128, 512, 7), (4500, 64, 64, 16), (8300, 256, 256, 5), (130, 72, 100, 5), (130, 64, 128, 32), (700, 384, 192, 40),
            (300, 128, 64, 100)]


@pytest.mark.parametrize("where", ["x", "dy", "down", "up"])
@pytest.mark.parametrize("adapter", [BF16, F32])
@pytest.mark.parametrize("rows, d_in, d_out, rank", INFINITE)
def test_infinite_gradients_are_the_definitions(rows, d_in, d_out, rank, adapter, where):
    """An infinity in the rows or in an adapter: each gradient is infinite, of its sign, or NaN, where the sums at 64 bits
    are, and near them everywhere else. (u, v and fp32 adapters are kept in parts, whose own sums would be NaN.)"""
    t = make(rows, d_in, d_out, rank, 3, [rows // 3] * 3, adapter=adapter)
    row = rows // 3 + 1  # the second request's
    at = {"x": (row, 3), "dy": (row, 3), "down": (1, rank - 1, 3), "up": (1, 3, rank - 1)}[where]
    t[where][at] = float("-inf")
    got = backward(gpu(t))
    args, of = [t[k] for k in ("dy", "x", "weight", "down", "up", "scale")], rows_of(t)
    want = oracle.adapted_linear_backward(*args, of)
    mag = oracle.adapted_linear_backward(*(a.abs() for a in args), of)
    unlike = 0
    for g, w, m, width in zip(got, want, mag, (d_out, d_out, d_in)):
        g = g.double().cpu()
        assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g.isposinf(), w.isposinf())
        assert torch.equal(g.isneginf(), w.isneginf())
        unlike += int((~w.isfinite()).sum())
        tol = (width + rows + 10) * 2.0**-24 * m
        if w.shape == t["x"].shape:  # dx: bf16, from bf16 adapters and rounded v
            tol = tol + HALF * w.abs() + (1 if adapter == BF16 else 2) * HALF * (1 + 2 * HALF) * m
        fine = w.isfinite()
        assert ((g - w).abs()[fine] <= tol[fine]).all()
    assert unlike > rank


@pytest.mark.parametrize("rows, lengths", [(30011, [1] * 30000), (2000, [0] * 700 + [1000] + [0] * 9000 + [3, 0, 0, 900]),
                                           (300, [0] * 300 + [150, 0, 149] + [0] * 5000), (700, [2] * 300 + [0] * 257 + [99])])
def test_requests_by_the_thousand(rows, lengths):
    """One-row requests, and runs of empty ones, that no workgroup can walk from the first."""
    t = make(rows, 64, 72, 8, 5, lengths, adapter=F32)
    check_forward(t, forward(gpu(t)))
    check_backward(t, backward(gpu(t)))


def test_offsets_of_many_requests_out_of_order():
    """Any values: some adapter or none, no access out of range."""
    g = torch.Generator().manual_seed(3)
    for rows in (300, 3000):
        t = gpu(make(rows, 64, 64, 8, 3, [1] * 5000))
        for low, high in ((0, rows), (-2**31, 2**31 - 1), (rows - 1, rows + 1)):
            t["offsets"] = torch.randint(low, high, (5001,), generator=g, dtype=torch.int64).to(DEV, torch.int32)
            assert torch.isfinite(forward(t).float()).all()
            assert torch.isfinite(backward(t).x.float()).all()


def test_time_grows_with_the_rows_of_short_requests():
    """Ten times the one-row requests take some ten times as long, not a hundred times: no workgroup passes over all of
    them. (Both calls in the form for short requests; 30 leaves three times the rows' share to noise.)"""
    def time(n):
        t = gpu(make(n, 64, 64, 8, 4, [1] * n))
        times = []
        for _ in range(4):
            start, end = torch.cuda.Event(True), torch.cuda.Event(True)
            start.record()
            for _ in range(3):
                backward(t)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert time(200_000) <= 30 * time(20_000)
