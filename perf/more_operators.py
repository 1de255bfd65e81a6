"""The measured workloads around a feature field's decoder.

Before the gated feed-forward block come the features themselves: a row of a table
for each Gaussian, pixel or token that names one (``embedding``), then the layer
norm that takes out what the pixel's alpha dimmed (``layer_norm``); behind it, in
training, channels are dropped (``dropout``), alone or on top of a residual.
``listed()`` are the fixed cases, ``draw(rng)`` another one of the same ranges,
``prepare`` what a user's program holds before the call, ``run`` one pass, ``work``
the bytes and operations that it cannot do without, ``exact`` what ``run`` returns,
in 64 bits.

A row is a pixel, a Gaussian or a token.  ``embed`` cases look ``count`` indices up
in a (rows, width) table; ``norm`` and ``drop`` cases have (rows, width) inputs.
"""

import math

import torch

own = False  # False: the plain form below; True: the framework's operators

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
DEVICE = "cuda"
EPS = 1e-5


def listed():
    return [
        # the label under a viewer's cursor: one Gaussian's code, looked up
        dict(name="embed_pick_one", op="embed", kind="decode", count=1, rows=4096, width=64,
             scaled=False, absent=0.0, index="int64", dtype="float32"),
        # a training step of a scene whose Gaussians share a codebook, some without a code;
        # few codes are popular
        dict(name="embed_codes_1m", op="embed", kind="train", count=1_000_003, rows=4096, width=32,
             scaled=False, absent=0.05, index="int32", dtype="float32"),
        # every pixel of a 720p batch takes its view's appearance: a few very popular rows
        dict(name="embed_views_720p", op="embed", kind="train", count=1280 * 720, rows=201, width=48,
             scaled=False, absent=0.0, index="int64", dtype="bfloat16"),
        # the tokens of a few texts in a long vocabulary, most of whose rows get no gradient
        dict(name="embed_tokens_wide", op="embed", kind="train", count=8205, rows=50_000, width=512,
             scaled=True, absent=0.0, index="int64", dtype="float16"),
        # one picked pixel before the decoder
        dict(name="norm_pick_one", op="norm", kind="decode", rows=1, width=32, affine=True,
             dtype="float32"),
        # every pixel of a 1080p feature render, in half the bytes
        dict(name="norm_view_1080p_half", op="norm", kind="decode", rows=1920 * 1080, width=96,
             affine=True, dtype="bfloat16"),
        # a training step on an odd crop: rows that no vector load fits
        dict(name="norm_crop_odd", op="norm", kind="train", rows=273 * 87, width=27, affine=True,
             dtype="float32"),
        # a training step over a whole 720p feature render
        dict(name="norm_train_720p", op="norm", kind="train", rows=1280 * 720, width=32, affine=True,
             dtype="float32"),
        # the hidden channels of a wide decoder's tokens, ragged, without weights
        dict(name="norm_tokens_wide", op="norm", kind="train", rows=8205, width=1365, affine=False,
             dtype="float16"),
        # a patch of pixels in an interactive correction, on top of the block's input
        dict(name="drop_patch", op="drop", rows=64, width=64, p=0.1, residual=True, counter="device",
             dtype="float32"),
        # the decoder's hidden channels of a whole 720p view
        dict(name="drop_hidden_720p", op="drop", rows=1280 * 720, width=128, p=0.1, residual=False,
             counter="host", dtype="bfloat16"),
        # decoded classes of an odd view on top of a residual
        dict(name="drop_residual_odd", op="drop", rows=641 * 479, width=21, p=0.5, residual=True,
             counter="device", dtype="float16"),
    ]


def _most(op):
    """The largest listed case's bytes of an operator, to stay below."""
    return max(work(c)["bytes"] for c in listed() if c["op"] == op)


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("embed", "norm", "drop"))
    most = _most(op)
    while True:
        dtype = rng.choice(tuple(TYPES))
        if op == "embed":
            case = dict(op=op, kind=rng.choice(("decode", "train")), count=_spread(rng, 1, 1_000_003),
                        rows=_spread(rng, 16, 50_000), width=_spread(rng, 1, 512),
                        scaled=rng.random() < 0.5, absent=rng.choice((0.0, 0.05, 0.5)),
                        index=rng.choice(("int32", "int64")), dtype=dtype)
        elif op == "norm":
            case = dict(op=op, kind=rng.choice(("decode", "train")), rows=_spread(rng, 1, 1920 * 1080),
                        width=_spread(rng, 4, 4096), affine=rng.random() < 0.7, dtype=dtype)
        else:
            case = dict(op=op, rows=_spread(rng, 1, 1280 * 720), width=_spread(rng, 1, 1365),
                        p=rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)), residual=rng.random() < 0.5,
                        counter=rng.choice(("host", "device")), dtype=dtype)
        if work(case)["bytes"] <= most:
            return case


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    dtype = TYPES[case["dtype"]]
    state = dict(case=dict(case))
    if case["op"] == "embed":
        count, rows, width = case["count"], case["rows"], case["width"]
        # popular rows: the k-th most popular one's share falls as k^(-2/3)
        popular = (rows * torch.rand((count,), generator=g, device=DEVICE).pow(3)).long()
        index = torch.randperm(rows, generator=g, device=DEVICE)[popular.clamp_(max=rows - 1)]
        gone = torch.rand((count,), generator=g, device=DEVICE) < case["absent"]
        kind = torch.int32 if case["index"] == "int32" else torch.int64
        state["index"] = index.masked_fill_(gone, -1).to(kind)
        train = case["kind"] == "train"
        size = 1.0 / math.sqrt(width) if case["scaled"] else 1.0
        state["table"] = (normal(rows, width) * size).to(dtype).requires_grad_(train)
        state["scale"] = math.sqrt(width) if case["scaled"] else 1.0
        if train:
            state["dy"] = (normal(count, width) * 0.1).to(dtype)
        return state
    rows, width = case["rows"], case["width"]
    if case["op"] == "norm":
        train = case["kind"] == "train"
        # composited features dimmed by the pixel's alpha, around a common offset
        alpha = 0.02 + 0.98 * torch.rand((rows, 1), generator=g, device=DEVICE)
        state["x"] = ((normal(rows, width) + 0.5) * alpha).to(dtype).requires_grad_(train)
        if case["affine"]:
            state["weight"] = (1.0 + 0.2 * normal(width)).to(dtype).requires_grad_(train)
            state["bias"] = (0.2 * normal(width)).to(dtype).requires_grad_(train)
        if train:
            state["dy"] = (normal(rows, width) * 0.1).to(dtype)
        return state
    state["x"] = normal(rows, width).to(dtype).requires_grad_(True)
    if case["residual"]:
        state["residual"] = normal(rows, width).to(dtype).requires_grad_(True)
    state["dy"] = (normal(rows, width) * 0.1).to(dtype)
    state["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 64)
    # the training loop's step: a number, or what a captured loop counts up on the device
    step = seed % 100_000
    state["step"] = (torch.full((1,), step, dtype=torch.int64, device=DEVICE)
                     if case["counter"] == "device" else step)
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "norm": _own_norm, "drop": _own_drop}[op](state)
    with torch.no_grad():
        return {"embed": _plain_embed, "norm": _plain_norm, "drop": _plain_drop}[op](state)


# ---- the framework's operators, as a user calls them ----

def _own_embed(state):
    from mlx3d_amd.nn import embedding

    y = embedding(state["index"], state["table"], scale=state["scale"])
    if state["case"]["kind"] == "decode":
        return {"y": y}
    return {"y": y.detach(), "d_table": torch.autograd.grad(y, state["table"], state["dy"])[0]}


def _own_norm(state):
    from mlx3d_amd.nn import layer_norm

    y = layer_norm(state["x"], state.get("weight"), state.get("bias"), eps=EPS)
    if state["case"]["kind"] == "decode":
        return {"y": y}
    names = [k for k in ("x", "weight", "bias") if k in state]
    grads = torch.autograd.grad(y, [state[k] for k in names], state["dy"])
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(names, grads)}}


def _own_drop(state):
    from mlx3d_amd.nn import dropout

    names = [k for k in ("x", "residual") if k in state]
    y = dropout(state["x"], state["case"]["p"], state["seed"], offset=state["step"],
                residual=state.get("residual"))
    grads = torch.autograd.grad(y, [state[k] for k in names], state["dy"])
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(names, grads)}}


# ---- the plain forms: elementary operations in 32 bits, rounded at the end ----

def _plain_embed(state):
    case = state["case"]
    table, index, scale = state["table"], state["index"].long(), state["scale"]
    here = (index >= 0) & (index < case["rows"])
    safe = torch.where(here, index, 0)
    y = torch.where(here[:, None], table[safe].float() * scale, 0.0).to(table.dtype)
    if case["kind"] == "decode":
        return {"y": y}
    told = torch.where(here[:, None], state["dy"].float(), 0.0)
    grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    return {"y": y, "d_table": (grad.index_add_(0, safe, told) * scale).to(table.dtype)}


def _plain_norm(state):
    dtype = state["x"].dtype
    x = state["x"].float()
    x = x - x.mean(dim=1, keepdim=True)
    inverse = torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS)
    x = x * inverse
    affine = "weight" in state
    y = x * state["weight"].float() + state["bias"].float() if affine else x
    out = {"y": y.to(dtype)}
    if state["case"]["kind"] == "decode":
        return out
    dy = state["dy"].float()
    if affine:
        out["d_weight"] = (dy * x).sum(dim=0).to(dtype)
        out["d_bias"] = dy.sum(dim=0).to(dtype)
        dy = dy * state["weight"].float()
    dx = dy - dy.mean(dim=1, keepdim=True) - x * (dy * x).mean(dim=1, keepdim=True)
    out["d_x"] = (dx * inverse).to(dtype)
    return out


def _philox(counter, key):
    """Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011): four 32-bit
    words of each 128-bit counter, all held in int64."""
    low = 0xFFFFFFFF
    a, b, c, d = counter
    k, m = key
    for _ in range(10):
        # a product of 64 bits wraps in int64; its halves are right all the same
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((q >> 32) & low) ^ b ^ k, q & low, ((p >> 32) & low) ^ d ^ m, p & low
        k, m = (k + 0x9E3779B9) & low, (m + 0xBB67AE85) & low
    return a, b, c, d


def _numbers(count, seed, step):
    """A 32-bit number for each element: element i's upper half is the half-word i % 8
    of the block i / 8, its lower half that of the block 2^63 + i / 8."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, device=DEVICE)
    key = (seed & low, seed >> 32)
    late = (torch.zeros_like(block) + (step & low), torch.zeros_like(block) + (step >> 32))
    halves = []
    for stream in (0, 0x80000000):
        words = torch.stack(_philox((block & low, (block >> 32) + stream, *late), key), dim=1)
        halves.append(torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:count])
    return (halves[0] << 16) | halves[1]


def _plain_drop(state):
    case = state["case"]
    x, p = state["x"], case["p"]
    kept = _numbers(x.numel(), state["seed"], state["step"]).view(x.shape) >= round(p * (1 << 32))
    y = torch.where(kept, x.float() * (1.0 / (1.0 - p)), 0.0)
    out = {"d_x": torch.where(kept, state["dy"].float() * (1.0 / (1.0 - p)), 0.0).to(x.dtype)}
    if case["residual"]:
        y = y + state["residual"].float()
        out["d_residual"] = state["dy"]
    out["y"] = y.to(x.dtype)
    return out


# ---- what a pass cannot do without ----

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "embed":
        count, rows, width = case["count"], case["rows"], case["width"]
        there = count * (1.0 - case["absent"])
        looked = int(rows * (1.0 - math.exp(-there / rows)))  # rows that are read, about
        index = count * (4 if case["index"] == "int32" else 8)
        if case["kind"] == "decode":
            return {"bytes": index + (count + looked) * width * size, "flops": count * width}
        return {"bytes": index + (2 * count + looked + rows) * width * size,
                "flops": 2 * count * width}
    rows, width = case["rows"], case["width"]
    if case["op"] == "norm":
        affine = 2 * width * size if case["affine"] else 0
        if case["kind"] == "decode":
            return {"bytes": 2 * rows * width * size + affine, "flops": 8 * rows * width}
        return {"bytes": 4 * rows * width * size + 2 * affine, "flops": 20 * rows * width}
    # the gradient of a residual is the incoming one itself
    return {"bytes": (5 if case["residual"] else 4) * rows * width * size, "flops": 4 * rows * width}


# ---- the definition in 64 bits, gradients by differentiation ----

def exact(case, seed):
    state = prepare(case, seed)
    leaf = {k: v.detach().double() for k, v in state.items()
            if k in ("table", "x", "weight", "bias", "residual")}
    train = case.get("kind") != "decode"
    if train:
        leaf = {k: v.requires_grad_(True) for k, v in leaf.items()}
    if case["op"] == "embed":
        # one more row, of zeros, stands for what lies outside the table
        padded = torch.cat([leaf["table"], torch.zeros_like(leaf["table"][:1])])
        index = state["index"].long()
        outside = index.lt(0) | index.ge(case["rows"])
        y = padded.index_select(0, index.masked_fill(outside, case["rows"])) * state["scale"]
    elif case["op"] == "norm":
        var, mean = torch.var_mean(leaf["x"], 1, unbiased=False, keepdim=True)
        y = (leaf["x"] - mean) / (var + EPS).sqrt()
        if case["affine"]:
            y = torch.addcmul(leaf["bias"], y, leaf["weight"])
    else:
        keep = _kept(case, state["seed"], int(state["step"]))
        y = leaf["x"] / (1.0 - case["p"]) * keep
        if case["residual"]:
            y = y + leaf["residual"]
    if not train:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaf.values()), state["dy"].double())
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(leaf, grads)}}


def _product(a, b):
    """High and low 32 bits of a (a tensor below 2^32) times b, by 16-bit limbs."""
    a1, a0, b1, b0 = a.div(65536, rounding_mode="floor"), a.remainder(65536), b // 65536, b % 65536
    low = a0 * b0
    middle = a1 * b0 + low.div(65536, rounding_mode="floor")
    cross = a0 * b1 + middle.remainder(65536)
    high = a1 * b1 + middle.div(65536, rounding_mode="floor") + cross.div(65536, rounding_mode="floor")
    return high, cross.remainder(65536) * 65536 + low.remainder(65536)


def _kept(case, seed, step):
    """1.0 where an element is kept: its number, block by block, is at least p 2^32."""
    shape = (case["rows"], case["width"])
    count = shape[0] * shape[1]
    at = torch.arange(-(-count // 8), device=DEVICE)
    number = 0
    for weight, stream in ((65536, 0), (1, 2 ** 31)):
        x = [at.remainder(2 ** 32), at.div(2 ** 32, rounding_mode="floor") + stream,
             torch.full_like(at, step % 2 ** 32), torch.full_like(at, step // 2 ** 32)]
        for r in range(10):
            key = [(seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
            h0, l0 = _product(x[0], 0xD2511F53)
            h1, l1 = _product(x[2], 0xCD9E8D57)
            x = [h1.bitwise_xor(x[1]).bitwise_xor(key[0]), l1,
                 h0.bitwise_xor(x[3]).bitwise_xor(key[1]), l0]
        half = torch.stack([h for w in x for h in (w.remainder(65536),
                                                   w.div(65536, rounding_mode="floor"))], dim=1)
        number = number + half.reshape(-1)[:count] * weight
    return (number >= round(case["p"] * 2 ** 32)).view(shape).double()
