"""Measured operators: matrices in microscaled 4-bit floating point (quantization; the linear layer
for few tokens, for a prompt and in training), and layer norm (training; quantized as it is made).

Format. A code is e2m1: a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. Each 32 values of a row share
a scale, a power of two. Rounded to nearest (ties to the even code), the scale is the smallest
power of two that brings the block's largest magnitude to at most 7, and what is above 6 becomes 6.
Rounded stochastically, it is the smallest that brings it to at most 6, and the scaled magnitude
(below 1 first rounded to a multiple of 2^-23) goes up to the next value with the probability of its
place between the two: when that place plus N / 2^22 reaches 1, N being 22 bits of
``h = mix(low32(p) ^ mix(key + high32(p)))``, ``p = row * ceil(columns / 2) + column // 2``: the top
22 of h for an even column, its low 16 followed by six zeros for an odd one. The key is
``mix(low32(seed) + 0x9E3779B1 * (high32(seed) + 1))``.

Linear layer. x is quantized with a scale for each row's 32 columns (for dW, each column's 32 rows),
W with one for each 32 x 32 tile, dy like x but stochastically, with the noise of dy's element for both
of its forms::

    y = x W^T + b      dx = dy W      dW = dy^T x      db = sum of dy over the rows

Layer norm of a row (mean m, biased variance v) and its gradients, ``u = (x - m) / sqrt(v + eps)``::

    y = u g + b      dx = (w - mean(w) - u mean(w u)) / sqrt(v + eps), w = dy g
    dg = sum of dy u over the rows      db = sum of dy over the rows

Quantized as it is made, y is not rounded to a type of its own first.
"""

import math

import torch

own = False

BLOCK = 32  # columns (and rows) that share a scale
STAGE = 256  # a kept matrix's rows are padded with zeros to a multiple of this
EPS = 1e-5
M32 = 0xFFFFFFFF


# ---- cases -------------------------------------------------------------------


def _quantize(name, rows, cols, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(name, op, tokens, inputs, outputs, dtype, bias):
    return {"name": name, "op": op, "tokens": tokens, "in": inputs, "out": outputs, "dtype": dtype,
            "bias": bias}


def _norm(name, rows, cols, dtype):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # A small matrix of no round size, quantized and read back: launches and ragged blocks.
        _quantize("quantize 333x1000", 333, 1000, "float16"),
        # The activations between an MLP's projections in an 8-billion-parameter model.
        _quantize("quantize 8192x14336", 8192, 14336, "bfloat16"),
        # Decoding one token: the key projection of a model of width 4096, the smallest weight.
        _linear("decode 1 4096-1024", "kept", 1, 4096, 1024, "bfloat16", False),
        # The head over the vocabulary for one token: a quarter of a gigabyte of weights.
        _linear("head 1 4096-128256", "kept", 1, 4096, 128256, "bfloat16", False),
        # A prompt through an up projection of an 8-billion-parameter model.
        _linear("prompt 4096 4096-14336", "kept", 4096, 4096, 14336, "bfloat16", False),
        # A short prompt of no round length: the norm before a block's first projection, and that.
        _linear("norm+linear 100 4096-6144", "norm kept", 100, 4096, 6144, "bfloat16", True),
        # The same for a batch of prompts in a model of width 768.
        _linear("norm+linear 8192 768-2304", "norm kept", 8192, 768, 2304, "float32", True),
        # Training a small layer of odd sizes in float32: launches, ragged blocks.
        _linear("train 130 200-99", "train", 130, 200, 99, "float32", True),
        # Training an expert's projection on the ragged number of tokens routed to it.
        _linear("train 3001 2048-1408", "train", 3001, 2048, 1408, "float16", True),
        # Training an up projection of an 8-billion-parameter model: the largest products.
        _linear("train 8192 4096-14336", "train", 8192, 4096, 14336, "bfloat16", False),
        # Training a small model's norm on a small batch, in float32: launches.
        _norm("norm train 512x768", 512, 768, "float32"),
        # Training a norm of an 8-billion-parameter model's width.
        _norm("norm train 8192x4096", 8192, 4096, "bfloat16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["quantize", "kept", "norm kept", "train", "train", "norm"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op in ("quantize", "norm"):
        # Norms of a few columns have no gradient worth the name: what is left of it cancels.
        cols = _log(rng, 1 if op == "quantize" else 16, 20000)
        return {"op": op, "rows": min(_log(rng, 1, 32768), 8192 * 14336 // cols), "cols": cols, "dtype": dtype}
    inputs, outputs = _log(rng, 64, 16384), _log(rng, 64, 16384)
    tokens = _log(rng, 1, 4096) if op == "kept" else _log(rng, 16, 8192)
    tokens = min(tokens, 8192 * 4096 * 14336 // (inputs * outputs))
    return {"op": op, "tokens": max(1, tokens), "in": inputs, "out": outputs, "dtype": dtype,
            "bias": rng.random() < 0.5}


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        # x read, codes and scales written and read, their values written.
        return {"bytes": n * (size + 4) + n + n / 16, "flops": 2 * n}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        # x read and y written; x and dy read and dx written; the parameters and their gradients.
        return {"bytes": 5 * n * size + 16 * case["cols"], "flops": 20 * n}
    m, k, n = case["tokens"], case["in"], case["out"]
    bias = 4 * n if case["bias"] else 0
    if case["op"] == "train":
        return {"bytes": size * m * (2 * k + 2 * n) + 2 * 4 * n * k + 2 * bias, "flops": 6 * m * n * k}
    weight, out = n * k / 2 + n * k / BLOCK, 2 if case["op"] == "norm kept" else size
    return {"bytes": weight + m * (size * k + out * n) + bias, "flops": 2 * m * n * k}


# ---- inputs --------------------------------------------------------------------


def _normal(gen, *sizes):
    return torch.randn(*sizes, device="cuda", generator=gen)


def _activations(gen, m, k):
    """A few channels are an order of magnitude larger than the others."""
    channel = torch.rand(k, device="cuda", generator=gen).pow_(8).mul_(10).add_(0.5)
    return _normal(gen, m, k).mul_(channel)


def _gradients(gen, m, n):
    """The rows' sizes differ by an order of magnitude."""
    return _normal(gen, m, n).mul_(_normal(gen, m, 1).exp_().mul_(1e-3))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = getattr(torch, case["dtype"]), case["op"]
    if op == "quantize":
        return {"op": op, "x": _activations(gen, case["rows"], case["cols"]).to(dtype)}
    if op == "norm":
        m, n = case["rows"], case["cols"]
        state = {"op": op, "x": _activations(gen, m, n).add_(0.3).to(dtype),
                 "g": 1 + 0.2 * _normal(gen, n), "b": 0.2 * _normal(gen, n),
                 "dy": _gradients(gen, m, n).to(dtype)}
        for name in ("x", "g", "b"):
            state[name].requires_grad_(own)
        return state
    m, k, n = case["tokens"], case["in"], case["out"]
    state = {"op": op, "x": _activations(gen, m, k).to(dtype)}
    w = _normal(gen, n, k).mul_(k ** -0.5)
    state["bias"] = _normal(gen, n).mul_(0.1) if case["bias"] else None
    if op == "train":
        state |= {"w": w, "dy": _gradients(gen, m, n).to(dtype), "seed": seed}
        for name in ("x", "w", "bias"):
            if state[name] is not None:
                state[name].requires_grad_(own)
        return state
    if op == "norm kept":
        state |= {"g": 1 + 0.2 * _normal(gen, k), "b": 0.2 * _normal(gen, k)}
    # A server keeps the weight in 4 bits only.
    state["data"], state["scale"], state["in"] = *_stored(w), k
    if own:
        from dionw_amd import Float4Matrix

        state["weight"] = Float4Matrix(state["data"], state["scale"], k)
    return state


def _stored(w):
    """A weight quantized by tiles as it is kept: two codes a byte, the first in the low half,
    ``[rows, depth / 2]`` (depth: columns rounded up to 256), and the rows' exponent bytes by column
    block, ``[depth / 32, rows rounded up to 16]``."""
    n, k = w.shape
    w = _padded(w, BLOCK, STAGE)
    tiles = w.view(w.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    byte = _exponent_byte(tiles.abs().amax((1, 3)), _NEAREST)
    u = (tiles * _power(254 - byte)[:, None, :, None]).view_as(w)[:n]
    values = torch.tensor(_VALUES, device="cuda")
    # The codes' borders: halfway between neighbours, ties to the even code.
    code = sum(((u.abs() > b) if i % 2 == 0 else (u.abs() >= b)).to(torch.uint8)
               for i, b in enumerate(((values[1:] + values[:-1]) / 2).tolist()))
    code |= (u < 0).to(torch.uint8) << 3
    scale = torch.zeros(byte.shape[1], -(-n // 16) * 16, dtype=torch.uint8, device="cuda")
    scale[:, :n] = byte.repeat_interleave(BLOCK, 0)[:n].t().to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, scale


# ---- one pass -------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _own_quantize(state):
    from dionw_amd import float4_quantize

    return float4_quantize(state["x"]).values()


def _own_kept(state):
    from dionw_amd import float4_linear

    return float4_linear(state["x"], state["weight"], state["bias"])


def _own_norm_kept(state):
    from dionw_amd import float4_layer_norm, float4_matmul

    x = float4_layer_norm(state["x"], state["g"], state["b"], EPS)
    return float4_matmul(x, state["weight"], state["bias"], dtype=torch.bfloat16)


def _own_train(state):
    from dionw_amd import float4_linear

    x, w, b = state["x"], state["w"], state["bias"]
    y = float4_linear(x, w, b, seed=state["seed"])
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], state["dy"])
    return {"y": y, **dict(zip(("dx", "dw", "db"), grads))}


def _own_norm(state):
    from dionw_amd import layer_norm

    x, g, b = state["x"], state["g"], state["b"]
    y = layer_norm(x, g, b, EPS)
    return dict(zip(("y", "dx", "dg", "db"), (y, *torch.autograd.grad(y, [x, g, b], state["dy"]))))


_own = {"quantize": _own_quantize, "kept": _own_kept, "norm kept": _own_norm_kept, "train": _own_train,
        "norm": _own_norm}


# ---- plain forms ------------------------------------------------------------------

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_NEAREST, _STOCHASTIC = 0x1FFFFF, 0x3FFFFF  # bits that carry a maximum past 7 or 6 into the next power


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _exponent_byte(largest, carry):
    """The scale's exponent byte for blocks' largest magnitudes."""
    return (((largest.view(torch.int32) + carry) >> 23) - 2).clamp_(min=1)


def _power(byte):
    return (byte << 23).view(torch.float32)


def _nearest(u):
    """Scaled values rounded to e2m1."""
    unit = torch.where(u.abs() < 2, 0.5, torch.where(u.abs() < 4, 1.0, 2.0))
    return ((u / unit).round() * unit).clamp(-6, 6)


def _row_values(x, noise=None):
    """x rounded in blocks of a row's 32 columns, as values."""
    full = _padded(x.to(torch.float32), 1, BLOCK).view(x.shape[0], -1, BLOCK)
    byte = _exponent_byte(full.abs().amax(2), _NEAREST if noise is None else _STOCHASTIC)[..., None]
    u = full * _power(254 - byte)
    u = _nearest(u) if noise is None else _by_noise(u, _padded(noise, 1, BLOCK).view_as(full))
    return (u * _power(byte)).view(x.shape[0], -1)[:, :x.shape[1]]


def _tile_values(w):
    """w rounded in blocks of 32 x 32, as values."""
    full = _padded(w, BLOCK, BLOCK)
    tiles = full.view(full.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    byte = _exponent_byte(tiles.abs().amax((1, 3), keepdim=True), _NEAREST)
    return (_nearest(tiles * _power(254 - byte)) * _power(byte)).view_as(full)[:w.shape[0], :w.shape[1]]


def _by_noise(u, noise):
    """Scaled values rounded to e2m1, up by ``noise`` of 2^22."""
    one = (u.abs() < 1).to(torch.float32)
    bits = ((u.abs() + one).view(torch.int32) + noise) & ~0x3FFFFF
    return (bits.view(torch.float32) - one).copysign(u)


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & M32
    x = x ^ (x >> 15)
    x = (x * 0x85EBCA77) & M32
    return x ^ (x >> 16)


def _noise(seed, rows, cols):
    """22 bits for every element, [rows, cols] int32."""
    pairs = (cols + 1) // 2
    p = torch.arange(rows * pairs, device="cuda")
    key = _mix(((seed & M32) + 0x9E3779B1 * ((seed >> 32 & M32) + 1)) & M32)
    h = _mix((p & M32) ^ _mix((key + (p >> 32)) & M32))
    both = torch.stack([h >> 10, (h & 0xFFFF) << 6], 1).to(torch.int32)
    return both.view(rows, 2 * pairs)[:, :cols]


def _kept_values(state):
    """The values of the weight that is kept."""
    data, n = state["data"], state["data"].shape[0]
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device="cuda")
    code = torch.stack([data & 15, data >> 4], 2).view(n, -1).to(torch.int32)
    w = table[code].view(n, -1, BLOCK) * _power(state["scale"][:, :n].t().to(torch.int32))[..., None]
    return w.view(n, -1)[:, :state["in"]]


def _plain_quantize(state):
    return _row_values(state["x"])


def _plain_kept(state):
    x, b = state["x"], state["bias"]
    y = _row_values(x) @ _kept_values(state).t()
    return (y if b is None else y + b).to(x.dtype)


def _plain_norm_kept(state):
    # In 64 bits up to the rounding: a value may lie next to a border between two codes.
    x = state["x"].double()
    x = x - x.mean(1, keepdim=True)
    x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt()
    y = _row_values((x * state["g"] + state["b"]).float()) @ _kept_values(state).t()
    return (y if state["bias"] is None else y + state["bias"]).to(torch.bfloat16)


def _plain_train(state):
    x, w, b, dy = state["x"], state["w"], state["bias"], state["dy"]
    noise = _noise(state["seed"], *dy.shape)
    wq = _tile_values(w)
    y = _row_values(x) @ wq.t()
    dx = _row_values(dy, noise) @ wq
    dw = _row_values(dy.t(), noise.t()) @ _row_values(x.t()).t()
    found = {"y": (y if b is None else y + b).to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}
    if b is not None:
        found["db"] = dy.to(torch.float32).sum(0)
    return found


def _plain_norm(state):
    x, g, dy = state["x"].to(torch.float32), state["g"], state["dy"].to(torch.float32)
    x = x - x.mean(1, keepdim=True)
    rstd = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
    u = x * rstd
    w = dy * g
    dx = (w - w.mean(1, keepdim=True) - u * (w * u).mean(1, keepdim=True)) * rstd
    y = u * g + state["b"]
    return {"y": y.to(state["x"].dtype), "dx": dx.to(state["x"].dtype), "dg": (dy * u).sum(0), "db": dy.sum(0)}


_plain = {"quantize": _plain_quantize, "kept": _plain_kept, "norm kept": _plain_norm_kept, "train": _plain_train,
          "norm": _plain_norm}


# ---- in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return _exact(prepare(case, seed))


def _exact(state):
    x, op = state["x"].double(), state["op"]
    if op == "quantize":
        return _rounded(x, 1)
    if op == "norm":
        return _exact_norm(x, state["g"].double(), state["b"].double(), state["dy"].double())
    b = 0.0 if state["bias"] is None else state["bias"].double()
    if op == "train":
        w, dy = _rounded(state["w"].double(), BLOCK), state["dy"].double()
        rows, cols = dy.shape
        noise = _noise(state["seed"], rows, cols).double()
        found = {"y": _rounded(x, 1) @ w.t() + b, "dx": _rounded(dy, 1, noise) @ w,
                 "dw": _rounded(dy.t(), 1, noise.t()) @ _rounded(x.t(), 1).t()}
        return found if state["bias"] is None else found | {"db": dy.sum(0)}
    if op == "norm kept":
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        x = (x - mean) / (var + EPS).sqrt() * state["g"].double() + state["b"].double()
    n, data = state["data"].shape[0], state["data"].to(torch.int64)
    code = torch.stack([data % 16, data // 16], 2).view(n, -1)
    # A code's value: its low bit is a half below the exponent's first step, a fraction bit above.
    field, half = (code % 8) // 2, (code % 2).double() / 2
    v = torch.where(field == 0, half, (1 + half) * _two_to(field - 1)) * (1 - code // 8 * 2)
    v = v.view(n, -1, BLOCK) * _two_to(state["scale"][:, :n].t().to(torch.int64) - 127)[..., None]
    return _rounded(x, 1) @ v.view(n, -1)[:, :x.shape[1]].t() + b


def _exact_norm(x, g, b, dy):
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    deviation = (var + EPS).sqrt()
    u, w = (x - mean) / deviation, dy * g
    along = (w * u).sum(1, keepdim=True) / x.shape[1]
    return {"y": u * g + b, "dx": (w - w.sum(1, keepdim=True) / x.shape[1] - u * along) / deviation,
            "dg": (dy * u).sum(0), "db": dy.sum(0)}


def _two_to(exponent):
    """2 to whole powers, exactly (a 64-bit power function may be off in the last place)."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded(x, rows, noise=None):
    """x rounded to e2m1 with one scale for each ``rows`` x 32 block, as values."""
    full = _padded(x, rows, BLOCK)
    v = full.view(full.shape[0] // rows, rows, -1, BLOCK)
    top = v.abs().amax((1, 3), keepdim=True) / (7.0 if noise is None else 6.0)
    mantissa, exponent = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))
    scale = _two_to(exponent - (mantissa == 0.5).to(exponent.dtype))
    u = v.abs() / scale
    unit = _two_to((torch.frexp(u)[1] - 1).clamp(min=0) - 1)
    if noise is None:
        u = ((u / unit).round() * unit).clamp(max=6.0)
    else:
        u = torch.where(u < 1, (u * 2.0 ** 23).round() / 2.0 ** 23, u)
        u = (u / unit + _padded(noise, rows, BLOCK).view_as(v) / 2.0 ** 22).floor() * unit
    return (u * scale).copysign(v).view_as(full)[:x.shape[0], :x.shape[1]]
