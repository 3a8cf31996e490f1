"""Operators of fine-tuning and of serving fine-tuned models: dropout whose mask is drawn again where it is needed, and a
projection with low-rank adapters of many requests beside it.

Shapes are those of the stacks: pair tensors (N x N tokens of 64, 128 or 256 channels), single rows (N tokens of 384), MSA rows,
the transitions' projections (d to 2 d and 4 d and back), AF3's 449 input features, from one token to a 512-token crop's pairs.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
#: a mask's random numbers have 16 bits, eight of them to a block of the generator
LEVELS, PER_BLOCK = 65536, 8


def listed() -> list[dict]:
    return [
        # one token's single features: a call's latency
        dict(name="dropout_token", op="dropout", direction="forward", batch=1, rows=1, cols=1, width=384, shared="none",
             rate=0.1, dtype="bf16"),
        # a crop's pair update under AF3's row-wise dropout (one mask for all rows), added to the residual stream
        dict(name="dropout_pair_rows", op="dropout", direction="forward", batch=1, rows=512, cols=512, width=128,
             shared="rows", rate=0.25, dtype="bf16"),
        # the ending node's column-wise dropout, both directions of a training step, two crops of an odd length
        dict(name="dropout_pair_columns_step", op="dropout", direction="step", batch=2, rows=201, cols=201, width=128,
             shared="columns", rate=0.25, dtype="bf16"),
        # fp32 features of an odd width, every value with a mask of its own
        dict(name="dropout_odd_f32", op="dropout", direction="step", batch=1, rows=1, cols=40009, width=451, shared="none",
             rate=0.1, dtype="f32"),
        # one token through the single transition's expansion with its request's adapter: a call's latency
        dict(name="adapted_token", op="adapted", direction="forward", rows=1, tail=0, requests=1, adapters=1, rank=8,
             d_in=384, d_out=1536, dtype="bf16", bias=False),
        # 64 requests of one row each with adapters of their own
        dict(name="adapted_rows_of_64", op="adapted", direction="forward", rows=64, tail=0, requests=64, adapters=64, rank=16,
             d_in=768, d_out=768, dtype="bf16", bias=True),
        # single rows of 40 requests of unlike lengths, padding behind the last
        dict(name="adapted_ragged", op="adapted", direction="forward", rows=8000, tail=77, requests=40, adapters=8, rank=16,
             d_in=384, d_out=1536, dtype="bf16", bias=False),
        # the input features' projection, whose width is a multiple of nothing, under training
        dict(name="adapted_features_odd", op="adapted", direction="step", rows=1021, tail=0, requests=3, adapters=2, rank=5,
             d_in=449, d_out=384, dtype="f32", bias=True),
        # single rows of a training batch back through the transition's contraction
        dict(name="adapted_single_backward", op="adapted", direction="backward", rows=2900, tail=0, requests=8, adapters=8,
             rank=32, d_in=1536, d_out=384, dtype="bf16", bias=False),
        # two crops' pairs, each with its request's adapter, through the pair transition's contraction
        dict(name="adapted_pair_contract", op="adapted", direction="forward", rows=2 * 256 * 256, tail=0, requests=2,
             adapters=2, rank=16, d_in=512, d_out=128, dtype="bf16", bias=False),
        # a 512-token crop's pairs through the expansion: the step that bounds a fine-tuning pass
        dict(name="adapted_pair_step", op="adapted", direction="step", rows=512 * 512, tail=0, requests=1, adapters=1, rank=16,
             d_in=128, d_out=512, dtype="f32", bias=False),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    if rng.random() < 0.4:
        width = rng.choice([64, 128, 128, 256, 384, _spread(rng, 16, 1000)])
        most = 512 * 512 * 128 // width
        rate = rng.choice([0.0, 0.05, 0.1, 0.15, 0.25, 0.5, round(rng.uniform(0.01, 0.99), 3)])
        case = dict(op="dropout", direction=rng.choice(["forward", "backward", "step"]), rate=rate,
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
        shared = rng.choice(["none", "rows", "columns"])
        if shared == "none":
            return dict(case, batch=1, rows=1, cols=_spread(rng, 1, most // 2), width=width, shared=shared)
        n = _spread(rng, 1, min(512, math.isqrt(most // 2)))
        rows = n if rng.random() < 0.5 else _spread(rng, 1, 512)
        return dict(case, batch=rng.choice([1, 1, 2]), rows=rows, cols=n, width=width, shared=shared)
    direction = rng.choice(["forward", "forward", "backward", "step"])
    d_in, d_out = rng.choice([(64, 256), (256, 64), (128, 512), (512, 128), (128, 128), (256, 512), (384, 1536), (1536, 384),
                              (384, 384), (768, 768), (449, 384), (_spread(rng, 16, 1000), _spread(rng, 16, 1000))])
    rank = rng.choice([4, 8, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    adapters = _spread(rng, 1, 64)
    most = min(512 * 512, 512 * 512 * 640 // (d_in + d_out), 512 * 512 * 128 * 512 // (2 * d_in * d_out),
               512 * 512 * 128 // (adapters * rank))
    rows = _spread(rng, 1, most)
    requests = rows if rows <= 256 and rng.random() < 0.4 else _spread(rng, 1, min(rows, 128))
    tail = rng.randint(0, rows // 8) if requests < rows and rng.random() < 0.3 else 0
    return dict(op="adapted", direction=direction, rows=rows, tail=tail, requests=requests, adapters=adapters, rank=rank,
                d_in=d_in, d_out=d_out, dtype=rng.choice(["bf16", "f32"]), bias=rng.random() < 0.3)


# ------------------------------------------------------------------------------------ inputs
def _shape(case: dict) -> tuple[int, ...]:
    return case["batch"], case["rows"], case["cols"], case["width"]


_AXIS = {"none": None, "rows": 1, "columns": 2}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    h = np.random.RandomState(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    s = dict(case)
    if case["op"] == "dropout":
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        shape = _shape(case)
        if case["direction"] != "backward":
            # an update beside a residual stream of larger values
            s["update"] = (0.3 * normal(*shape) * torch.exp(0.5 * normal(shape[-1]))).to(dtype)
            s["residual"] = (normal(*shape) * torch.exp(0.5 * normal(shape[-1]))).to(dtype)
        if case["direction"] != "forward":
            s["dy"] = (0.02 * normal(*shape)).to(dtype)
        s["seed"], s["offset"] = int(h.randint(0, 2**62, dtype=np.int64)), int(h.randint(0, 2**40, dtype=np.int64))
        return s
    rows, n, rank, d_in, d_out = (case[k] for k in ("rows", "adapters", "rank", "d_in", "d_out"))
    # rows of a normalised stream, channels of unlike size
    s["x"] = (normal(rows, d_in) * torch.exp(0.3 * normal(d_in))).bfloat16()
    weights = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    s["weight"] = (normal(d_out, d_in) * d_in**-0.5).to(weights)
    s["bias"] = 0.1 * normal(d_out) if case["bias"] else None
    s["down"] = (normal(n, rank, d_in) * d_in**-0.5).to(weights)
    s["up"] = (0.3 * normal(n, d_out, rank) * rank**-0.5).to(weights)
    s["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device=DEVICE)
    # where each request's rows end: one row each, or anywhere (lengths of zero among them); requests that have an adapter
    # nearly all
    inside, r = rows - case["tail"], case["requests"]
    ends = np.arange(1, rows + 1) if r == rows else np.append(np.sort(h.randint(0, inside + 1, r - 1)), inside)
    adapter = h.permutation(np.arange(r) % n)
    if r > 4:
        adapter[h.rand(r) < 0.06] = -1
    s["offsets"] = torch.tensor(np.append(0, ends), dtype=torch.int32, device=DEVICE)
    s["adapter"] = torch.tensor(adapter, dtype=torch.int32, device=DEVICE)
    if case["direction"] != "forward":
        s["dy"] = (0.02 * normal(rows, d_out)).bfloat16()
    return s


# ------------------------------------------------------------------------------------ plain forms
def _round(c0, c1, c2, c3, k0, k1):
    """One round of Philox4x32 on words held in int64 (a product's upper word: of the 64 bits that wrap, the upper half)."""
    low = 0xFFFFFFFF
    p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low


def _numbers(blocks: torch.Tensor, seed: int, offset: int) -> torch.Tensor:
    """The eight 16-bit numbers of each block, [blocks, 8]."""
    low = 0xFFFFFFFF
    zero = torch.zeros_like(blocks)
    words = blocks & low, blocks >> 32, zero + (offset & low), zero + ((offset >> 32) & low)
    for i in range(10):
        words = _round(*words, ((seed & low) + i * 0x9E3779B9) & low, (((seed >> 32) & low) + i * 0xBB67AE85) & low)
    words = torch.stack(words, -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).flatten(-2)


def _kept(s: dict) -> torch.Tensor:
    """The mask of a call, of size 1 along the shared axis."""
    shape = list(_shape(s))
    if _AXIS[s["shared"]] is not None:
        shape[_AXIS[s["shared"]]] = 1
    n = math.prod(shape)
    numbers = _numbers(torch.arange(-(-n // PER_BLOCK), device=DEVICE), s["seed"], s["offset"])
    return (numbers.flatten()[:n] >= round(LEVELS * s["rate"])).view(shape)


def _dropped(x: torch.Tensor, kept: torch.Tensor, rate: float) -> torch.Tensor:
    return torch.where(kept, x.float() * (LEVELS / (LEVELS - round(LEVELS * rate))), 0.0)


def _adapter_of_rows(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Each row's adapter (0 where it has none) and its scale (0 there)."""
    rows = torch.arange(s["rows"], device=DEVICE, dtype=torch.int32)
    request = torch.searchsorted(s["offsets"], rows, right=True) - 1
    has = request < s["requests"]
    a = s["adapter"][request.clamp_max(s["requests"] - 1)].long()
    has &= a >= 0
    a = torch.where(has, a, 0)
    return a, torch.where(has, s["scale"][a], 0.0)


def _plain(s: dict):
    if s["op"] == "dropout":
        kept, out = _kept(s), {}
        if "update" in s:
            out["y"] = (s["residual"].float() + _dropped(s["update"], kept, s["rate"])).to(s["update"].dtype)
        if "dy" in s:
            out["update"] = _dropped(s["dy"], kept, s["rate"]).to(s["dy"].dtype)
        return out
    x, w, down, up = (s[k].float() for k in ("x", "weight", "down", "up"))
    n, rank, d_in, d_out = (s[k] for k in ("adapters", "rank", "d_in", "d_out"))
    a, scale = _adapter_of_rows(s)
    # all adapters side by side, and for each row the channels of its own
    mine = torch.zeros(s["rows"], n, 1, device=DEVICE).scatter_(1, a[:, None, None], scale[:, None, None])
    down, up = down.reshape(n * rank, d_in), up.permute(1, 0, 2).reshape(d_out, n * rank)
    u = ((x @ down.T).view(-1, n, rank) * mine).flatten(1)
    out = {}
    if s["direction"] != "backward":
        y = x @ w.T + u @ up.T
        out["y"] = (y if s["bias"] is None else y + s["bias"]).bfloat16()
    if s["direction"] != "forward":
        dy = s["dy"].float()
        v = ((dy @ up).view(-1, n, rank) * mine).flatten(1)
        out["x"] = (dy @ w + v @ down).bfloat16()
        out["down"] = (v.T @ x).view(n, rank, d_in)
        out["up"] = (dy.T @ u).view(d_out, n, rank).permute(1, 0, 2).contiguous()
    return out


# ------------------------------------------------------------------------------------ the framework's calls
def _own(s: dict):
    from foldforge_amd import kernels

    out = {}
    if s["op"] == "dropout":
        how = dict(p=s["rate"], seed=s["seed"], offset=s["offset"], shared=_AXIS[s["shared"]])
        if "update" in s:
            out["y"] = kernels.dropout_add(s["update"], s["residual"], **how)
        if "dy" in s:
            out["update"] = kernels.dropout_backward(s["dy"], **how)
        return out
    adapters = {k: s[k] for k in ("down", "up", "scale", "offsets", "adapter")}
    if s["direction"] != "backward":
        out["y"] = kernels.adapted_linear(s["x"], s["weight"], s["bias"], **adapters)
    if s["direction"] != "forward":
        g = kernels.adapted_linear_backward(s["dy"], s["x"], s["weight"], **adapters)
        out.update(x=g.x, down=g.down, up=g.up)
    return out


def run(state: dict):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ floors
def work(case: dict) -> dict:
    if case["op"] == "dropout":
        tensors = {"forward": 3, "backward": 2, "step": 5}[case["direction"]]
        return dict(bytes=tensors * math.prod(_shape(case)) * (4 if case["dtype"] == "f32" else 2), flops=0)
    rows, rank, d_in, d_out = (case[k] for k in ("rows", "rank", "d_in", "d_out"))
    size = 4 if case["dtype"] == "f32" else 2
    n, used = case["adapters"], min(case["adapters"], case["requests"])
    ends = rows * (d_in + d_out) * 2
    params = d_in * d_out * size + used * rank * (d_in + d_out) * size
    product, thin = 2 * rows * d_in * d_out, 2 * rows * rank * (d_in + d_out)
    moved = flops = 0
    if case["direction"] != "backward":
        moved, flops = ends + params, product + thin
    if case["direction"] != "forward":
        # dy, x and dx; the adapters' gradients in fp32
        moved += ends + rows * d_in * 2 + params + n * rank * (d_in + d_out) * 4
        flops += product + 2 * thin + 2 * rows * rank * d_in
    return dict(bytes=moved, flops=flops)


# ------------------------------------------------------------------------------------ 64 bits
def _mask64(case: dict, seed: int, offset: int) -> np.ndarray:
    """The definition of the mask: Philox4x32-10 of counters (block, offset) under the key, in unsigned 64-bit words."""
    shape = [case["batch"], case["rows"], case["cols"], case["width"]]
    if case["shared"] != "none":
        shape[1 if case["shared"] == "rows" else 2] = 1
    n = int(np.prod(shape))
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    m32, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [block & m32, block >> s32, np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & m32, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    number = np.empty((block.size, 8), dtype=np.uint32)
    for i in range(8):
        number[:, i] = (c[i // 2] >> np.uint64(16 * (i % 2))) & np.uint64(0xFFFF)
    return (number.ravel()[:n] >= round(65536 * case["rate"])).reshape(shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    out = {}
    if case["op"] == "dropout":
        kept = torch.from_numpy(_mask64(case, s["seed"], s["offset"])).to(DEVICE)
        share = 1 - round(65536 * case["rate"]) / 65536

        def drop(x):
            return torch.where(kept, x.double() / share, torch.zeros((), dtype=torch.float64, device=DEVICE))

        if "update" in s:
            out["y"] = s["residual"].double() + drop(s["update"])
        if "dy" in s:
            out["update"] = drop(s["dy"])
        return out
    w = s["weight"].double()
    ends, adapter = s["offsets"].tolist(), s["adapter"].tolist()
    if case["direction"] != "backward":
        out["y"] = s["x"].double() @ w.T + (0 if s["bias"] is None else s["bias"].double())
    if case["direction"] != "forward":
        out["x"] = s["dy"].double() @ w
        for k in ("down", "up"):
            out[k] = torch.zeros(s[k].shape, dtype=torch.float64, device=DEVICE)
    for lo, hi, a in zip(ends, ends[1:], adapter):
        if hi == lo or a < 0:
            continue
        x, down, up, scale = s["x"][lo:hi].double(), s["down"][a].double(), s["up"][a].double(), s["scale"][a].double()
        u = x @ down.T
        if "y" in out:
            out["y"][lo:hi] += scale * (u @ up.T)
        if "x" in out:
            dy = s["dy"][lo:hi].double()
            v = scale * (dy @ up)
            out["x"][lo:hi] += v @ down
            out["down"][a] += v.T @ x
            out["up"][a] += scale * (dy.T @ u)
    return out
