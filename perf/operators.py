"""The training operators of the pair stack: LayerNorm and SwiGLU transition with their backward passes, and the
8-bit activations that a forward pass keeps for them.

Shapes are those of the stacks: pair rows (N x N tokens of 64, 128 or 256 channels), single rows (N tokens of
384), MSA rows (S x N of 64), and widths off all of these, from one row to a 512-token crop. Activations are a
residual stream's: channels of unlike size about means of their own, rows of unlike size; gradients are small.
"""

from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda"
#: channels that share a scale in an 8-bit activation
BLOCK = 32


def listed() -> list[dict]:
    return [
        # one token's single features: a call's latency
        dict(name="layer_norm_token", op="layer_norm", direction="backward", keep="input", rows=1, cols=384,
             dtype="bf16"),
        # a small crop's single rows with everything a step does: forward, 8-bit activation, backward
        dict(name="layer_norm_single_step", op="layer_norm", direction="step", keep="8bit", rows=384, cols=384,
             dtype="bf16"),
        # the pair norm of a 512-token crop from the kept input
        dict(name="layer_norm_pair", op="layer_norm", direction="backward", keep="input", rows=512 * 512, cols=128,
             dtype="bf16"),
        # the same as a step on an 8-bit activation
        dict(name="layer_norm_pair_step", op="layer_norm", direction="step", keep="8bit", rows=512 * 512, cols=128,
             dtype="bf16"),
        # fp32 features of a width and a count that are multiples of nothing
        dict(name="layer_norm_odd_f32", op="layer_norm", direction="step", keep="input", rows=40009, cols=451,
             dtype="f32"),
        # MSA rows kept in 8 bits and read back
        dict(name="activation_msa", op="activation", rows=512 * 384, cols=64, dtype="bf16"),
        # fp32 rows whose last block of channels is short
        dict(name="activation_odd_f32", op="activation", rows=10007, cols=333, dtype="f32"),
        # the single track's transition of a small crop
        dict(name="transition_single", op="transition", direction="backward", keep="input", rows=100, width=384,
             factor=4),
        # the MSA track's transition: many short rows
        dict(name="transition_msa_step", op="transition", direction="step", keep="8bit", rows=128 * 384, width=64,
             factor=4),
        # a pair transition of 256 channels
        dict(name="transition_wide", op="transition", direction="backward", keep="input", rows=200 * 200, width=256,
             factor=2),
        # the trunk's pair transition at a length that is a multiple of nothing
        dict(name="transition_pair_odd", op="transition", direction="backward", keep="input", rows=201 * 201, width=128,
             factor=4),
        # the trunk's pair transition of a 512-token crop: the step that bounds a training pass
        dict(name="transition_pair_step", op="transition", direction="step", keep="8bit", rows=512 * 512, width=128,
             factor=4),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["layer_norm", "layer_norm", "activation", "transition", "transition"])
    if op == "transition":
        width, factor = rng.choice([(64, 2), (64, 4), (128, 4), (128, 4), (128, 2), (256, 2), (256, 4), (384, 4)])
        rows = _spread(rng, 1, 2048 if width == 384 else 512 * 512 * 128 * 512 // (width * width * factor * 4))
        direction = rng.choice(["backward", "step"])
        keep = "input" if direction == "backward" else rng.choice(["input", "8bit"])
        return dict(op=op, direction=direction, keep=keep, rows=rows, width=width, factor=factor)
    cols = rng.choice([64, 128, 256, 384, 768, _spread(rng, 16, 1000), _spread(rng, 16, 1000)])
    rows = _spread(rng, 1, min(512 * 512, 512 * 512 * 128 // cols))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "activation":
        return dict(op=op, rows=rows, cols=cols, dtype=dtype)
    direction = rng.choice(["backward", "step"])
    keep = "input" if direction == "backward" else rng.choice(["input", "8bit"])
    return dict(op=op, direction=direction, keep=keep, rows=rows, cols=cols, dtype=dtype)


# ------------------------------------------------------------------------------------ inputs
def _stream(g: torch.Generator, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """Rows of a residual stream."""
    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    x = normal(rows, cols) * torch.exp(0.5 * normal(cols)) + 0.5 * normal(cols)
    return (x * torch.exp(0.3 * normal(rows, 1))).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    state = dict(case)
    d = case["width"] if case["op"] == "transition" else case["cols"]
    dtype = torch.float32 if case.get("dtype") == "f32" else torch.bfloat16
    state["x"] = _stream(g, case["rows"], d, dtype)
    if case["op"] == "activation":
        return state
    state["dy"] = (0.02 * normal(case["rows"], d)).to(dtype)
    state["ln_weight"] = 1 + 0.1 * normal(d)
    state["ln_bias"] = 0.1 * normal(d)
    if case["op"] == "transition":
        hidden = case["factor"] * d
        state["expand_a"] = normal(hidden, d) * d**-0.5
        state["expand_b"] = normal(hidden, d) * d**-0.5
        state["squeeze"] = normal(d, hidden) * hidden**-0.5
    return state


# ------------------------------------------------------------------------------------ plain forms
def _two_to(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for whole e in [-126, 127], by its bits."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _held(x: torch.Tensor) -> torch.Tensor:
    """The fp32 values that an 8-bit activation of ``x [rows, cols]`` stands for: each block of 32 channels as
    e4m3 numbers times the least power of two that holds its largest finite value within 448."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    top = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    s = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
    code = (v * _two_to(-s)).to(torch.float8_e4m3fn).float()
    return (code * _two_to(s)).reshape(rows, -1)[:, :cols]


def _norm(x: torch.Tensor, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """The normalised rows and 1 / deviation."""
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + eps)
    return c * rstd, rstd


def _norm_back(dn: torch.Tensor, xh: torch.Tensor, rstd: torch.Tensor, w: torch.Tensor):
    g = dn * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dn * xh).sum(0), dn.sum(0)


def _plain(s: dict):
    x = s["x"]
    if s["op"] == "activation":
        return _held(x).to(x.dtype)
    dy, w, b = s["dy"].float(), s["ln_weight"], s["ln_bias"]
    kept = _held(x) if s["keep"] == "8bit" else x.float()
    out = {}
    if s["op"] == "layer_norm":
        if s["direction"] == "step":
            out["y"] = (_norm(x.float())[0] * w + b).to(x.dtype)
        dx, dw, db = _norm_back(dy, *_norm(kept), w)
        return dict(out, dx=dx.to(x.dtype), dweight=dw, dbias=db)
    wa, wb, wo = s["expand_a"], s["expand_b"], s["squeeze"]
    if s["direction"] == "step":
        n = _norm(x.float())[0] * w + b
        a = n @ wa.T
        out["y"] = (x.float() + (a * torch.sigmoid(a) * (n @ wb.T)) @ wo.T).to(x.dtype)
    xh, rstd = _norm(kept)
    n = xh * w + b
    a, b_ = n @ wa.T, n @ wb.T
    sig = torch.sigmoid(a)
    du = dy @ wo
    dwo = dy.T @ (a * sig * b_)
    db = du * a * sig
    da = du * b_ * (sig + a * sig * (1 - sig))
    dx, dlw, dlb = _norm_back(da @ wa + db @ wb, xh, rstd, w)
    bf16 = torch.bfloat16
    return dict(out, dx=(dy + dx).to(bf16), ln_weight=dlw.to(bf16), ln_bias=dlb.to(bf16), expand_a=(da.T @ n).to(bf16),
                expand_b=(db.T @ n).to(bf16), squeeze=dwo.to(bf16))


# ------------------------------------------------------------------------------------ the framework's calls
def _own(s: dict):
    from foldforge_amd import kernels

    x = s["x"]
    if s["op"] == "activation":
        return kernels.restore_activation(kernels.quantize_activation(x))
    out, kept = {}, x
    step, packed = s["direction"] == "step", s["keep"] == "8bit"
    if s["op"] == "layer_norm":
        if step and packed:
            out["y"], kept = kernels.layer_norm_checkpoint(x, s["ln_weight"], s["ln_bias"])
        elif step:
            out["y"] = kernels.layer_norm(x, s["ln_weight"], s["ln_bias"])
        dx, dw, db = kernels.layer_norm_backward(s["dy"], kept, s["ln_weight"])
        return dict(out, dx=dx, dweight=dw, dbias=db)
    params = {k: s[k] for k in ("ln_weight", "ln_bias", "expand_a", "expand_b", "squeeze")}
    if step and packed:
        out["y"], kept = kernels.transition_checkpoint(x, **params)
    elif step:
        out["y"] = kernels.transition(x, **params)
    # gradients in the type that a bf16 gradient reduction sends
    g = kernels.transition_backward(s["dy"], kept, **params, grad_dtype=torch.bfloat16)
    return dict(out, dx=g.x, ln_weight=g.ln_weight, ln_bias=g.ln_bias, expand_a=g.expand_a, expand_b=g.expand_b,
                squeeze=g.squeeze)


def run(state: dict):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ floors
def work(case: dict) -> dict:
    rows = case["rows"]
    if case["op"] == "activation":
        return dict(bytes=2 * rows * case["cols"] * (4 if case["dtype"] == "f32" else 2), flops=0)
    step = case["direction"] == "step"
    if case["op"] == "layer_norm":
        size = 4 if case["dtype"] == "f32" else 2
        return dict(bytes=(4 if step else 3) * rows * case["cols"] * size + 16 * case["cols"], flops=0)
    d, hidden = case["width"], case["width"] * case["factor"]
    # x, dy, dx (and y); the parameters and their gradients
    moved = (4 if step else 3) * rows * d * 2 + (4 + 2) * (3 * d * hidden + 2 * d)
    # a, b and du again from the kept input, then the five products of the gradients (and the forward's three)
    return dict(bytes=moved, flops=(22 if step else 16) * rows * d * hidden)


# ------------------------------------------------------------------------------------ 64 bits
def _held64(x: torch.Tensor) -> torch.Tensor:
    """The definition of the 8-bit activation, by arithmetic: within a block, steps of 2^-3 of a value's own power
    of two (2^-9 at least) in units of the block's scale, halves to the even step."""
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    for c in range(0, cols, BLOCK):
        v = x[:, c:c + BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp_min(-126))
        # the logarithm decides within its rounding: the least power of two that holds the block, by trial
        scale = torch.where(top <= 448 * (scale / 2).clamp_min(2.0**-126), (scale / 2).clamp_min(2.0**-126), scale)
        scale = torch.where(top > 448 * scale, 2 * scale, scale)
        u = v / scale
        power = torch.frexp(u.abs()).exponent - 1
        step = torch.exp2((power.clamp_min(-6) - 3).double())
        out[:, c:c + BLOCK] = torch.round(u / step) * step * scale
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "activation":
        return _held64(s["x"])
    rows, d = s["x"].shape
    w, b = s["ln_weight"].double(), s["ln_bias"].double()
    step = case["direction"] == "step"
    names = ["ln_weight", "ln_bias"] + (["expand_a", "expand_b", "squeeze"] if case["op"] == "transition" else [])
    grads = {k: torch.zeros_like(s[k], dtype=torch.float64) for k in names}
    y, dx = (torch.empty(rows, d, dtype=torch.float64, device=DEVICE) for _ in range(2))

    def norm(x):
        mean = x.sum(1, keepdim=True) / d
        var = ((x - mean) ** 2).sum(1, keepdim=True) / d
        return (x - mean) / torch.sqrt(var + 1e-5), torch.sqrt(var + 1e-5)

    for r in range(0, rows, 32768):
        at = slice(r, r + 32768)
        x, dy = s["x"][at].double(), s["dy"][at].double()
        kept = _held64(s["x"][at]) if case["keep"] == "8bit" else x
        xh, dev = norm(kept)
        if case["op"] == "layer_norm":
            if step:
                y[at] = norm(x)[0] * w + b
            dn, dy = dy, 0
        else:
            wa, wb, wo = (s[k].double() for k in ("expand_a", "expand_b", "squeeze"))
            if step:
                n = norm(x)[0] * w + b
                a = n @ wa.T
                y[at] = x + (a / (1 + torch.exp(-a)) * (n @ wb.T)) @ wo.T
            n = xh * w + b
            a, v = n @ wa.T, n @ wb.T
            gate = 1 / (1 + torch.exp(-a))
            du = dy @ wo
            grads["squeeze"] += dy.T @ (a * gate * v)
            dv = du * a * gate
            da = du * v * gate * (1 + a - a * gate)
            grads["expand_a"] += da.T @ n
            grads["expand_b"] += dv.T @ n
            dn = da @ wa + dv @ wb
        g = dn * w
        along = (g * xh).sum(1, keepdim=True) / d
        dx[at] = dy + (g - g.sum(1, keepdim=True) / d - xh * along) / dev
        grads["ln_weight"] += (dn * xh).sum(0)
        grads["ln_bias"] += dn.sum(0)
    out = {"y": y} if step else {}
    if case["op"] == "layer_norm":
        return dict(out, dx=dx, dweight=grads["ln_weight"], dbias=grads["ln_bias"])
    return dict(out, dx=dx, **grads)
