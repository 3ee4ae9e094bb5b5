"""Measured operators: the AdamW step with 8-bit states, and the 8-bit linear layer (few tokens; training).

Formats. ``e4m3`` is the 8-bit float with 4 exponent and 3 fraction bits (largest 448). ``u44`` is
an unsigned 8-bit float with 4 exponent bits (bias 8) and 4 fraction bits (largest 248). Every block
has a scale that is a power of two, the smallest that brings the block's largest magnitude to at
most the format's largest value; it is kept as the exponent byte of the float32 that it is.

AdamW, per element (r is the root of the second moment; m and r are held in e4m3 and u44, one scale
for 256 elements of a tensor each)::

    m = b1 m0 + (1 - b1) g      r = sqrt(b2 r0^2 + (1 - b2) g^2)
    p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (r / sqrt(1 - b2^t) + eps)

m and r are stored rounded up where the part that is dropped, in units of the last place kept, is at
least ``1 - R / 2^16``, down otherwise; R is 16 bits of a hash of the step, the tensor's position and
the element's index (low half for m, high half for r). An r above zero is never stored as zero.

Linear layer, on operands rounded to nearest in e4m3: x and dy with a scale for each row's 128
columns (for dW, each column's 128 rows), W with a scale for each 128 x 128 tile::

    y = x W^T + b      dx = dy W      dW = dy^T x      db = sum of dy over the rows
"""

import math

import torch

own = False

BETA1, BETA2, LR, EPS, DECAY = 0.9, 0.95, 1e-3, 1e-8, 0.05
BLOCK = 256  # elements of a tensor that share a scale of the AdamW state
TILE = 128  # columns (and rows) that share a scale of a product's operand
M32 = 0xFFFFFFFF


# ---- cases -------------------------------------------------------------------


def _adamw(name, sizes, step):
    """``sizes``: the tensors' element counts, ``AxB`` for A tensors of B elements."""
    return {"name": name, "op": "adamw", "sizes": sizes, "step": step}


def _linear(name, op, tokens, inputs, outputs, dtype, bias):
    return {"name": name, "op": op, "tokens": tokens, "in": inputs, "out": outputs, "dtype": dtype,
            "bias": bias}


def listed():
    return [
        # The norm weights of a 32-layer model of width 4096: one small launch, latency.
        _adamw("adamw 65 norms", "65x4096", 100),
        # Biases, norms and small embeddings of odd sizes, from one element to a few hundred thousand.
        _adamw("adamw ragged", "1x1,3x255,2x257,5x1001,4x7777,2x31415,1x250001,1x777777", 7),
        # A token embedding of a small model.
        _adamw("adamw embedding 50257x768", "1x38597376", 2000),
        # The embedding and the head of an 8-billion-parameter model are this size each.
        _adamw("adamw embedding 128256x4096", "1x525336576", 5),
        # Decoding one token: the key projection of a model of width 4096, the smallest weight.
        _linear("decode 1 4096-1024", "few", 1, 4096, 1024, "bfloat16", False),
        # Decoding for eight users: an up projection.
        _linear("decode 8 4096-14336", "few", 8, 4096, 14336, "bfloat16", False),
        # A short prompt of no round length through a down projection.
        _linear("prompt 100 14336-4096", "few", 100, 14336, 4096, "float16", True),
        # The head over the vocabulary for one token: half a gigabyte of weights.
        _linear("head 1 4096-128256", "few", 1, 4096, 128256, "bfloat16", False),
        # Training a small layer of odd sizes in float32: launches, ragged blocks.
        _linear("train 130 200-99", "train", 130, 200, 99, "float32", True),
        # Training the query/key/value projection of a model of width 768.
        _linear("train 8192 768-2304", "train", 8192, 768, 2304, "bfloat16", True),
        # Training an expert's projection on the ragged number of tokens routed to it.
        _linear("train 3001 2048-1408", "train", 3001, 2048, 1408, "float16", False),
        # Training an up projection of an 8-billion-parameter model: the largest products.
        _linear("train 8192 4096-14336", "train", 8192, 4096, 14336, "bfloat16", False),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["adamw", "few", "train"])
    if op == "adamw":
        groups, left = [], 1 << 27
        for _ in range(rng.randint(1, 6)):
            count, size = rng.randint(1, 12), _log(rng, 1, 1 << 27)
            count = max(1, min(count, left // size))
            if size <= left:
                groups.append("%dx%d" % (count, size))
                left -= count * size
        return {"op": op, "sizes": ",".join(groups), "step": _log(rng, 1, 5000)}
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    inputs, outputs = _log(rng, 64, 16384), _log(rng, 64, 16384)
    tokens = _log(rng, 1, 256) if op == "few" else _log(rng, 16, 8192)
    tokens = min(tokens, 8192 * 4096 * 14336 // (inputs * outputs))
    return {"op": op, "tokens": max(1, tokens), "in": inputs, "out": outputs, "dtype": dtype,
            "bias": rng.random() < 0.5}


def _tensor_sizes(case):
    """Element counts, in order."""
    found = []
    for part in case["sizes"].split(","):
        count, size = part.split("x")
        found += [int(size)] * int(count)
    return found


def work(case):
    if case["op"] == "adamw":
        n = sum(_tensor_sizes(case))
        # p and g read, p written; two code bytes read and written; both moments' values written.
        return {"bytes": n * (4 + 4 + 4 + 2 + 2 + 8) + n / BLOCK * 16, "flops": 20 * n}
    m, k, n = case["tokens"], case["in"], case["out"]
    size = 4 if case["dtype"] == "float32" else 2
    bias = 4 * n if case["bias"] else 0
    if case["op"] == "few":
        return {"bytes": n * k + n * k / TILE / TILE + size * m * (k + n) + bias, "flops": 2 * m * n * k}
    return {"bytes": size * m * (2 * k + 2 * n) + 2 * 4 * n * k + 2 * bias, "flops": 6 * m * n * k}


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    return _prepare_linear(case, gen)


def _prepare_adamw(case, gen):
    """A training run's tensors in the middle of it. They lie in one buffer each for parameters and
    gradients, every tensor at a multiple of 256 elements, as a flattened bucket holds them."""
    sizes = _tensor_sizes(case)
    starts, at = [], 0
    for size in sizes:
        starts.append(at)
        at += -(-size // BLOCK) * BLOCK
    blocks = [-(-size // BLOCK) for size in sizes]
    count = torch.tensor(blocks)
    first = torch.repeat_interleave(torch.tensor(starts), count).cuda()
    which = torch.repeat_interleave(torch.arange(len(sizes)), count).cuda()
    valid = None
    if at != sum(sizes):
        end = torch.repeat_interleave(torch.tensor([s + n for s, n in zip(starts, sizes)]), count).cuda()
        valid = torch.arange(at, device="cuda").view(-1, BLOCK) < end[:, None]
    params = torch.randn(at, device="cuda", generator=gen).mul_(0.02)
    grads = torch.randn(at, device="cuda", generator=gen)
    # Gradients of one block lie within a few binades of each other, blocks within many.
    grads.view(-1, BLOCK).mul_(torch.randn(at // BLOCK, 1, device="cuda", generator=gen).mul_(2).exp_().mul_(1e-4))
    r0 = torch.rand(at, device="cuda", generator=gen).add_(0.25).mul_(grads.abs().view(-1, BLOCK).mean(1).repeat_interleave(BLOCK))
    m0 = torch.randn(at, device="cuda", generator=gen).mul_(0.3).mul_(r0)
    if valid is not None:
        for t in (params, grads, r0, m0):
            t.mul_(valid.view(-1))
    m_byte = _exponent_byte(m0.view(-1, BLOCK).abs().amax(1), _E4M3)
    r_byte = _exponent_byte(r0.view(-1, BLOCK).amax(1), _U44)
    half = torch.full((1,), 1 << 15, dtype=torch.int32, device="cuda")  # to nearest
    m_codes = _encode(m0.view(-1, BLOCK), m_byte, half, _E4M3).to(torch.uint8)
    r_codes = _encode(r0.view(-1, BLOCK), r_byte, half, _U44).to(torch.uint8)
    state = {"op": "adamw", "params": params, "grads": grads, "step": case["step"] - 1,
             "sizes": sizes, "starts": starts, "first": first, "which": which, "valid": valid,
             "m": m_codes, "m_scale": _power(m_byte), "r": r_codes, "r_scale": _power(r_byte)}
    if own:
        state["optimizer"], state["parameters"] = _optimizer(state)
    return state


def _optimizer(state):
    """The framework's optimizer over the same tensors, its state set to the same codes."""
    from dionw_amd import AdamWState, Dion

    parameters = []
    for start, size in zip(state["starts"], state["sizes"]):
        p = torch.nn.Parameter(state["params"][start:start + size])
        p.grad = state["grads"][start:start + size]
        parameters.append(p)
    optimizer = Dion([{"params": parameters, "dion_route": "adamw"}], lr=LR, betas=(BETA1, BETA2),
                     weight_decay=DECAY, eps=EPS, adamw_state=AdamWState.EIGHT_BIT)
    for p, start, size in zip(parameters, state["starts"], state["sizes"]):
        entry, b0, b1 = optimizer.state[p], start // BLOCK, -(-(start + size) // BLOCK)
        entry["exp_avg"].copy_(state["m"].view(-1)[start:start + size].view(torch.float8_e4m3fn))
        entry["exp_avg_scale"].copy_(state["m_scale"][b0:b1])
        entry["exp_avg_rms"].copy_(state["r"].view(-1)[start:start + size])
        entry["exp_avg_rms_scale"].copy_(state["r_scale"][b0:b1])
        entry["adamw_step"].fill_(state["step"])
    return optimizer, parameters


def _prepare_linear(case, gen):
    m, k, n = case["tokens"], case["in"], case["out"]
    dtype = getattr(torch, case["dtype"])
    # Activations: a few channels are an order of magnitude larger than the others.
    channel = torch.rand(k, device="cuda", generator=gen).pow_(8).mul_(10).add_(0.5)
    x = (torch.randn(m, k, device="cuda", generator=gen) * channel).to(dtype)
    w = torch.randn(n, k, device="cuda", generator=gen).mul_(k ** -0.5)
    b = torch.randn(n, device="cuda", generator=gen).mul_(0.1) if case["bias"] else None
    state = {"op": case["op"], "x": x, "bias": b}
    if case["op"] == "few":
        # A server keeps the weight in 8 bits only.
        data, byte = _quantize_tiles(w)
        state["data"], state["scale"], state["in"] = _stored(data, byte.repeat_interleave(TILE, 0)[:n], n) + (k,)
        if own:
            from dionw_amd import Float8Matrix

            state["weight"] = Float8Matrix(state["data"], state["scale"], k)
        return state
    dy = torch.randn(m, n, device="cuda", generator=gen)
    dy.mul_(torch.randn(m, 1, device="cuda", generator=gen).exp_().mul_(1e-3))
    state |= {"w": w, "dy": dy.to(dtype)}
    if own:
        for name in ("x", "w", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


def _stored(data, byte, rows):
    """A quantized matrix as it is kept: codes ``[rows, depth]`` (depth: columns rounded up to 128)
    and the rows' exponent bytes by column block, ``[depth / 128, rows rounded up to 16]``."""
    scale = torch.zeros(byte.shape[1], -(-rows // 16) * 16, dtype=torch.uint8, device=data.device)
    scale[:, :rows] = byte.t().to(torch.uint8)
    return data.view(rows, -1), scale


# ---- one pass -------------------------------------------------------------------


def run(state):
    if state["op"] == "adamw":
        return _own_adamw(state) if own else _plain_adamw(state)
    if state["op"] == "few":
        return _own_few(state) if own else _plain_few(state)
    return _own_train(state) if own else _plain_train(state)


def _own_adamw(state):
    optimizer = state["optimizer"]
    optimizer.step()
    exp_avg, rms = optimizer.adamw_moments(state["parameters"])
    return {"params": state["params"], "exp_avg": exp_avg, "rms": rms}


def _own_few(state):
    from dionw_amd import float8_linear

    return float8_linear(state["x"], state["weight"], state["bias"])


def _own_train(state):
    from dionw_amd import float8_linear

    x, w, b = state["x"], state["w"], state["bias"]
    y = float8_linear(x, w, b)
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], state["dy"])
    return {"y": y, **dict(zip(("dx", "dw", "db"), grads))}


# ---- plain forms ------------------------------------------------------------------

# (fraction bits kept, bias, bits that carry a block's maximum into the next binade, binades from
# the scale to the maximum, unit of the subnormals as an exponent)
_E4M3 = (3, 7, 0x1FFFFF, 8, -9)
_U44 = (4, 8, 0x07FFFF, 7, -11)


def _exponent_byte(largest, form):
    """The scale's exponent byte for blocks' largest magnitudes."""
    return (((largest.view(torch.int32) + form[2]) >> 23) - form[3]).clamp_(min=1)


def _power(byte):
    return (byte << 23).view(torch.float32)


def _encode(x, byte, noise, form):
    """Codes (int32, without sign for u44) of blocks ``x`` [blocks, size], rounded up by ``noise`` of 2^16."""
    fraction, bias, _, _, unit = form
    u = x.abs() * _power(254 - byte)[:, None]
    normal = (u.view(torch.int32) - ((127 - bias) << 23) + (noise << (7 - fraction))) >> (23 - fraction)
    small = ((u * 2.0 ** (16 - unit)).to(torch.int32) + noise) >> 16
    code = torch.where(u < 2.0 ** (1 - bias), small, normal)
    return code | ((x.view(torch.int32) >> 24) & 0x80) if form is _E4M3 else code


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & M32
    x = x ^ (x >> 15)
    x = (x * 0x85EBCA77) & M32
    return x ^ (x >> 16)


def _noise(state, step):
    """32 bits for every element, [blocks, 256]."""
    at = torch.arange(state["m"].numel(), device="cuda").view(-1, BLOCK) - state["first"][:, None]
    key = _mix((state["which"] * 0x9E3779B1 + step) & M32)[:, None]
    return _mix((at & M32) ^ _mix((key + (at >> 32)) & M32))


def _u44_values(codes):
    c = codes.to(torch.int32)
    return torch.where(c < 16, c * 2.0 ** -11, ((c << 19) + (119 << 23)).view(torch.float32))


def _plain_adamw(state):
    state["step"] += 1
    t = state["step"]
    p, g = state["params"].view(-1, BLOCK), state["grads"].view(-1, BLOCK)
    m = state["m"].view(torch.float8_e4m3fn).to(torch.float32) * state["m_scale"][:, None]
    r = _u44_values(state["r"]) * state["r_scale"][:, None]
    m = m * BETA1 + g * (1 - BETA1)
    r = ((r * r) * BETA2 + (g * (1 - BETA2)) * g).sqrt()
    step_size, root = LR / (1 - BETA1 ** t), 1 / math.sqrt(1 - BETA2 ** t)
    p.copy_(p * (1 - LR * DECAY) - (m * step_size) / (r * root + EPS))
    noise = _noise(state, t)
    m_byte, r_byte = _exponent_byte(m.abs().amax(1), _E4M3), _exponent_byte(r.amax(1), _U44)
    state["m"].copy_(_encode(m, m_byte, (noise & 0xFFFF).to(torch.int32), _E4M3))
    codes = _encode(r, r_byte, (noise >> 16).to(torch.int32), _U44)
    state["r"].copy_(torch.maximum(codes, (r > 0).to(torch.int32)))
    state["m_scale"].copy_(_power(m_byte))
    state["r_scale"].copy_(_power(r_byte))
    exp_avg = state["m"].view(torch.float8_e4m3fn).to(torch.float32) * state["m_scale"][:, None]
    rms = _u44_values(state["r"]) * state["r_scale"][:, None]
    if state["valid"] is not None:
        exp_avg, rms = exp_avg[state["valid"]], rms[state["valid"]]
    return {"params": state["params"], "exp_avg": exp_avg.view(-1), "rms": rms.view(-1)}


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _quantize_rows(x):
    """e4m3 codes [rows, blocks, 128] and exponent bytes [rows, blocks]."""
    x = _padded(x.to(torch.float32), 1, TILE).view(x.shape[0], -1, TILE)
    byte = _exponent_byte(x.abs().amax(2), _E4M3)
    return (x * _power(254 - byte)[..., None]).to(torch.float8_e4m3fn), byte


def _quantize_tiles(w):
    """e4m3 codes [rows, blocks, 128] and exponent bytes [row blocks, blocks]."""
    n = w.shape[0]
    w = _padded(w.to(torch.float32), TILE, TILE)
    w = w.view(w.shape[0] // TILE, TILE, -1, TILE)
    byte = _exponent_byte(w.abs().amax((1, 3)), _E4M3)
    codes = (w * _power(254 - byte)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(-1, byte.shape[1], TILE)[:n], byte


def _row_values(x):
    data, byte = _quantize_rows(x)
    return (data.to(torch.float32) * _power(byte)[..., None]).view(x.shape[0], -1)[:, :x.shape[1]]


def _plain_few(state):
    x, data, scale = state["x"], state["data"], state["scale"]
    n, k = data.shape[0], state["in"]
    factor = _power(scale[:, :n].t().to(torch.int32))
    w = (data.to(torch.float32).view(n, -1, TILE) * factor[..., None]).view(n, -1)[:, :k]
    y = _row_values(x) @ w.t()
    return (y if state["bias"] is None else y + state["bias"]).to(x.dtype)


def _plain_train(state):
    x, w, b, dy = state["x"], state["w"], state["bias"], state["dy"]
    data, byte = _quantize_tiles(w)
    factor = _power(byte).repeat_interleave(TILE, 0)[:w.shape[0], :, None]
    wq = (data.to(torch.float32) * factor).view(w.shape[0], -1)[:, :w.shape[1]]
    y = _row_values(x) @ wq.t()
    dx = _row_values(dy) @ wq
    dw = _row_values(dy.t()) @ _row_values(x.t()).t()
    found = {"y": (y if b is None else y + b).to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}
    if b is not None:
        found["db"] = dy.to(torch.float32).sum(0)
    return found


# ---- in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(state)
    x = state["x"].double()
    b = None if state["bias"] is None else state["bias"].double()
    if case["op"] == "few":
        n, k = case["out"], case["in"]
        factor = _two_to(state["scale"][:, :n].t().to(torch.int64) - 127)
        w = (state["data"].double().view(n, -1, TILE) * factor[..., None]).view(n, -1)[:, :k]
        y = _nearest(x, 1) @ w.t()
        return y if b is None else y + b
    w, dy = _nearest(state["w"].double(), TILE), state["dy"].double()
    y = _nearest(x, 1) @ w.t()
    found = {"y": y if b is None else y + b, "dx": _nearest(dy, 1) @ w,
             "dw": _nearest(dy.t(), 1) @ _nearest(x.t(), 1).t()}
    if b is not None:
        found["db"] = dy.sum(0)
    return found


def _two_to(exponent):
    """2 to whole powers, exactly (a 64-bit power function may be off in the last place)."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _block_power(largest, top):
    """The smallest power of two that brings ``largest`` to at most ``top`` (1 for zero)."""
    mantissa, exponent = torch.frexp(torch.where(largest > 0, largest / top, torch.ones_like(largest)))
    return _two_to(exponent - (mantissa == 0.5).to(exponent.dtype))


def _unit(u, lowest, fraction):
    """The spacing of a format's values around ``u``."""
    exponent = torch.frexp(u)[1] - 1
    exponent = torch.where(u > 0, exponent, torch.full_like(exponent, lowest)).clamp(min=lowest)
    return _two_to(exponent - fraction)


def _nearest(x, rows):
    """x rounded to e4m3 with one scale for each ``rows`` x 128 block, as values."""
    full = _padded(x, rows, TILE)
    v = full.view(full.shape[0] // rows, rows, -1, TILE)
    scale = _block_power(v.abs().amax((1, 3), keepdim=True), 448.0)
    u = v / scale
    unit = _unit(u.abs(), -6, 3)
    return ((u / unit).round() * unit * scale).view_as(full)[:x.shape[0], :x.shape[1]]


def _noisy(x, noise, top, lowest, fraction):
    """Blocks ``x`` rounded by ``noise``, as values, and their scales."""
    scale = _block_power(x.abs().amax(1, keepdim=True), top)
    u = (x / scale).abs()
    unit = _unit(u, lowest, fraction)
    code = (u / unit + noise / 65536.0).floor()
    return code, unit, scale


def _exact_adamw(state):
    t, found = state["step"] + 1, ([], [], [])
    chunk = (1 << 26) // BLOCK
    for c in range(0, state["m"].shape[0], chunk):
        at = slice(c, c + chunk)
        p, g = (state[name].view(-1, BLOCK)[at].double() for name in ("params", "grads"))
        m = state["m"][at].view(torch.float8_e4m3fn).double() * state["m_scale"][at, None].double()
        code = state["r"][at].double()
        field = (code / 16).floor()
        r = torch.where(field == 0, code / 16 * 2.0 ** -7, (1 + code / 16 - field) * _two_to(field - 8))
        r = r * state["r_scale"][at, None].double()
        m = BETA1 * m + (1 - BETA1) * g
        r = (BETA2 * r ** 2 + (1 - BETA2) * g ** 2).sqrt()
        p = p * (1 - LR * DECAY) - LR / (1 - BETA1 ** t) * m / (r / math.sqrt(1 - BETA2 ** t) + EPS)
        i = torch.arange(c * BLOCK, c * BLOCK + m.numel(), device="cuda").view(-1, BLOCK)
        i = i - state["first"][at, None]
        key = _mix((state["which"][at, None] * 0x9E3779B1 + t) & M32)
        noise = _mix((i & M32) ^ _mix((key + (i >> 32)) & M32))
        count, unit, scale = _noisy(m, (noise & 0xFFFF).double(), 448.0, -6, 3)
        m = count * unit * scale * m.sign()
        count, unit, scale = _noisy(r, (noise >> 16).double(), 248.0, -7, 4)
        r = torch.maximum(count, (r > 0).double()) * unit * scale
        if state["valid"] is not None:
            m, r = m[state["valid"][at]], r[state["valid"][at]]
        for values, v in zip(found, (p, m, r)):
            values.append(v.reshape(-1))
    return dict(zip(("params", "exp_avg", "rms"), (torch.cat(v) for v in found)))
