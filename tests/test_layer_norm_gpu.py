"""Layer norm, its gradients, and the norm that is quantized as it is made, against float64 (GPU).

Bounds. u = 2^-24 is float32's rounding, L the additions that any value of a row's sum passes: 8
values of up to 4 chunks of a thread (16384 columns; 64 of longer rows), 6 levels of a wave and 16
waves, so ``L = 60`` up to 16384 columns, and with c columns more ``60 + c / 128`` past them. With
m the largest |x| of a row and s its deviation (with eps):

- the mean is off by ``(L + 2) u m``, which is ``r = (L + 2) u m / s`` deviations;
- the reciprocal deviation by a factor of ``1 +- ((L + 8) u + 2 r)`` (squares and their sum, a shift
  of the mean, the root and the division; the shift enters squared and as a cross term);
- so ``t = (x - mean) / s`` by ``e = r + |t| ((L + 10) u + 2 r)``;
- ``y = t g + b`` by ``e |g| + 2 u (|t g| + |b|)``;
- with w = dy g, A the mean of |w|, B that of |w t|: ``dx`` by
  ``((L + 8) u (|w| + A + |t| B) + e B + |t| A max(e)) / s + ((L + 8) u + 2 r) |dx|``;
- dg by ``sum |dy| e + (R + 4) u sum |dy t|`` and db by ``(R + 4) u sum |dy|``, R being the rows.

Each is rounded once more to its type.
"""

from __future__ import annotations

import pytest
import torch

from dionw_amd import LayerNorm, float4_layer_norm, float4_linear, float4_matmul, float4_quantize, layer_norm

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def _additions(cols):
    return 60 + (cols / 128 if cols > 16384 else 0)


def _within(got, want, bound):
    bound = bound + HALF[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    off = (got.detach().double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), float((off - bound).max())


class _Exact:
    """The formulas in float64, with their bounds."""

    def __init__(self, x, g, b, eps=1e-5):
        x = x.detach().double()
        self.n = x.shape[1]
        self.g = torch.ones(self.n, device="cuda", dtype=torch.float64) if g is None else g.detach().double()
        self.b = torch.zeros_like(self.g) if b is None else b.detach().double()
        mean = x.mean(1, keepdim=True)
        self.s = ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
        self.t = (x - mean) / self.s
        level = _additions(self.n)
        self.r = (level + 2) * U * x.abs().amax(1, keepdim=True) / self.s
        self.level = level
        self.e = self.r + self.t.abs() * ((level + 10) * U + 2 * self.r)

    def check_y(self, y):
        tg = self.t * self.g
        _within(y, tg + self.b, self.e * self.g.abs() + 2 * U * (tg.abs() + self.b.abs()))

    def check_gradients(self, dy, dx, dg, db):
        dy = dy.double()
        w = dy * self.g
        along = (w * self.t).mean(1, keepdim=True)
        if dx is not None:
            want = (w - w.mean(1, keepdim=True) - self.t * along) / self.s
            a, b = w.abs().mean(1, keepdim=True), (w * self.t).abs().mean(1, keepdim=True)
            bound = (self.level + 8) * U * (w.abs() + a + self.t.abs() * b)
            bound = bound + self.e * b + self.t.abs() * a * self.e.amax(1, keepdim=True)
            _within(dx, want, bound / self.s + ((self.level + 8) * U + 2 * self.r) * want.abs())
        rows = dy.shape[0] + 4
        if dg is not None:
            _within(dg, (dy * self.t).sum(0), (dy.abs() * self.e).sum(0) + rows * U * (dy * self.t).abs().sum(0))
        if db is not None:
            _within(db, dy.sum(0), rows * U * dy.abs().sum(0))


def _inputs(m, n, dtype, seed=1, held=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, n, generator=gen, device="cuda") * 2 + 0.5
    g = (1 + 0.3 * torch.randn(n, generator=gen, device="cuda")).to(held)
    b = (0.3 * torch.randn(n, generator=gen, device="cuda")).to(held)
    dy = torch.randn(m, n, generator=gen, device="cuda") * torch.rand(m, 1, generator=gen, device="cuda")
    return x.to(dtype), g, b, dy.to(dtype)


# One value, ragged, around every width at which the kernels change, many and few rows.
SIZES = [(1, 1), (7, 2), (3, 100), (5, 128), (9, 129), (1000, 300), (33, 512), (40, 513), (2500, 768), (17, 1024),
         (6, 1025), (70, 2048), (5, 2049), (600, 4096), (11, 4097), (4, 8192), (300, 8192), (3, 8193), (2, 16384),
         (3, 16385), (2, 40001), (70, 20000), (5000, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_the_norm_and_its_gradients(size, dtype) -> None:
    x, g, b, dy = _inputs(*size, dtype)
    args = [t.requires_grad_() for t in (x, g, b)]
    y = layer_norm(*args)
    grads = torch.autograd.grad(y, args, dy)
    assert [t.dtype for t in (y, *grads)] == [dtype, dtype, torch.float32, torch.float32]
    exact = _Exact(x, g, b)
    exact.check_y(y)
    exact.check_gradients(dy, *grads)


@pytest.mark.parametrize("held", DTYPES)
@pytest.mark.parametrize("which", ["both", "weight", "bias", "neither"])
def test_parameters_of_every_type_and_none(which, held) -> None:
    for dtype in (torch.bfloat16, torch.float32):
        x, g, b, dy = _inputs(100, 1000, dtype, 2, held)
        g, b = (g if which in ("both", "weight") else None), (b if which in ("both", "bias") else None)
        args = [t.requires_grad_() for t in (x, g, b) if t is not None]
        y = layer_norm(x, g, b)
        grads = list(torch.autograd.grad(y, args, dy))
        exact = _Exact(x, g, b)
        exact.check_y(y)
        dx = grads.pop(0)
        dg = grads.pop(0) if g is not None else None
        db = grads.pop(0) if b is not None else None
        assert all(t is None or t.dtype is held for t in (dg, db))
        exact.check_gradients(dy, dx, dg, db)


@pytest.mark.parametrize("size", [(50, 300), (50, 5000), (20, 20000)], ids=str)
def test_only_the_gradients_asked_for(size) -> None:
    x, g, b, dy = _inputs(*size, torch.bfloat16)
    full = [t.clone().requires_grad_() for t in (x, g, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for mask in range(1, 8):
        args = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, g, b))]
        asked = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(layer_norm(*args), asked, dy)
        for grad, t in zip(got, asked):
            assert torch.equal(grad, want[[t is a for a in args].index(True)])


def test_gradients_are_the_differences() -> None:
    """Along a step d the loss changes by the gradient's product with it, and by d^3 / 6 times its
    third derivative, which a step of 2^-6 of the values keeps below 2^-9 of the sum of |g d|."""
    x, g, b, dy = (t.double() for t in _inputs(20, 300, torch.float32))
    args = [t.float().requires_grad_() for t in (x, g, b)]
    grads = torch.autograd.grad(layer_norm(*args), args, dy.float())

    def loss(x, g, b):
        t = x - x.mean(1, keepdim=True)
        return ((t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * g + b) * dy).sum()

    gen = torch.Generator(device="cuda").manual_seed(5)
    for place, grad in enumerate(grads):
        step = torch.randn(grad.shape, generator=gen, device="cuda", dtype=torch.float64) * 2.0 ** -6
        moved = [[t + s * step if i == place else t for i, t in enumerate((x, g, b))] for s in (1, -1)]
        change = float(loss(*moved[0]) - loss(*moved[1])) / 2
        assert abs(change - float((grad.double() * step).sum())) <= 2.0 ** -9 * float((grad.double() * step).abs().sum())


@pytest.mark.parametrize("cols", [100, 3000, 20000])
def test_rows_far_from_zero_keep_their_digits(cols) -> None:
    """A row of 1000 +- 1: a variance from sums of squares would be off by 6%."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(50, cols, generator=gen, device="cuda") + 1000
    y = layer_norm(x)
    exact = _Exact(x, None, None)
    exact.check_y(y)
    assert float((y.double() - exact.t).norm() / exact.t.norm()) < 1e-3


@pytest.mark.parametrize("cols", [1, 100, 3000, 20000])
def test_constant_rows_and_large_and_small_values(cols) -> None:
    x = torch.zeros(6, cols, device="cuda")
    x[1], x[2], x[3] = 7.5, -3e38 if cols == 1 else 1e15, 1e-30
    x[4] = torch.linspace(-1, 1, cols, device="cuda") * 1e-20
    x[5] = torch.linspace(-1, 1, cols, device="cuda") * 1e15
    b = torch.linspace(0, 1, cols, device="cuda")
    x.requires_grad_()
    y = layer_norm(x, None, b)
    _Exact(x, None, b).check_y(y)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool(dx.isfinite().all())


@pytest.mark.parametrize("cols", [100, 3000, 20000])
def test_values_that_are_not_finite_stay_in_their_rows(cols) -> None:
    x, g, b, dy = _inputs(20, cols, torch.float32)
    clean = layer_norm(x, g, b)
    x[3, 5], x[4, 0], x[5, cols - 1] = float("nan"), float("inf"), -float("inf")
    x.requires_grad_()
    y = layer_norm(x, g, b)
    assert y[3:6].isnan().all()
    keep = [i for i in range(20) if i not in (3, 4, 5)]
    assert torch.equal(y[keep], clean[keep])
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx[3:6].isnan().all() and dx[keep].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_shapes_and_broadcast_gradients(dtype) -> None:
    base = _inputs(300, 700, dtype)[0]
    for x in (base[:, :333], base[:, 1:334], base[::2, 4:400], base.t(), base[5:6], base[0].expand(50, 700),
              base.view(3, 100, 700), base.view(3, 100, 700).transpose(0, 1), base[0], base[:, :1].expand(300, 200)):
        x = x.detach().requires_grad_()
        y = layer_norm(x)
        assert y.shape == x.shape
        flat = x.detach().reshape(-1, x.shape[-1])
        exact = _Exact(flat, None, None)
        exact.check_y(y.view(flat.shape))
        (dx,) = torch.autograd.grad(y.sum() * 2, x)
        exact.check_gradients(torch.full_like(flat, 2), dx.reshape(flat.shape), None, None)
    # A gradient whose rows lie apart, and parameters that do.
    x, g, b, dy = _inputs(40, 500, dtype)
    wide = torch.cat([dy, dy], 1)[:, 500:]
    spread = torch.stack([g, b], 1)
    args = [x.requires_grad_(), spread[:, 0].requires_grad_(), spread[:, 1].requires_grad_()]
    y = layer_norm(*args)
    exact = _Exact(x, g, b)
    exact.check_y(y)
    exact.check_gradients(dy, *torch.autograd.grad(y, args, wide))


def test_empty_batches() -> None:
    norm = LayerNorm(200).cuda()
    x = torch.zeros(0, 200, device="cuda", requires_grad=True)
    y = norm(x)
    y.sum().backward()
    assert y.shape == x.grad.shape == (0, 200)
    assert not norm.weight.grad.any() and not norm.bias.grad.any()
    assert float4_layer_norm(x.detach()).shape == (0, 200)


def test_the_module() -> None:
    x = _inputs(30, 60, torch.float32)[0]
    norm = LayerNorm(60).cuda()
    assert torch.equal(norm(x), layer_norm(x, norm.weight, norm.bias, norm.eps))
    both = LayerNorm((3, 20), eps=1e-3).cuda()
    with torch.no_grad():
        both.weight.normal_()
        both.bias.normal_()
    y = both(x.view(30, 3, 20))
    flat = layer_norm(x, both.weight.flatten(), both.bias.flatten(), 1e-3)
    assert torch.equal(y.view(30, 60), flat)
    y.sum().backward()
    assert both.weight.grad.shape == (3, 20)
    plain = torch.nn.LayerNorm(60).cuda()
    plain.load_state_dict(norm.state_dict())


def test_another_stream_a_graph_and_repeats() -> None:
    for size in ((50, 300), (50, 5000), (30, 20000)):
        x, g, b, dy = _inputs(*size, torch.bfloat16)
        args = [t.requires_grad_() for t in (x, g, b)]

        def train():
            y = layer_norm(*args)
            return [y.detach(), *torch.autograd.grad(y, args, dy)]

        want = train()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = train()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train()
        for k in range(3):
            with torch.no_grad():
                x.copy_(_inputs(*size, torch.bfloat16, 20 + k)[0])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, train()))


def test_more_rows_than_a_launch_has_workgroups_of_a_wave() -> None:
    """2^24 rows and more, forward and backward and in 4 bits: the last ones are as they are alone."""
    rows, last = (1 << 24) + 9, 25
    x, g, b, dy = _inputs(last, 8, torch.float16)
    big, up = torch.ones(rows, 8, dtype=torch.float16, device="cuda"), torch.zeros(rows, 8, dtype=torch.float16,
                                                                                  device="cuda")
    big[-last:], up[-last:] = x, dy
    args, alone = [t.requires_grad_() for t in (big, g, b)], x.requires_grad_()
    y, want = layer_norm(*args), layer_norm(alone, g, b)
    assert torch.equal(y[-last:], want)
    grads = torch.autograd.grad(y, args, up)
    assert torch.equal(grads[0][-last:], torch.autograd.grad(want, alone, dy)[0])
    _Exact(x, g, b).check_gradients(dy, None, grads[1], grads[2])  # the other rows add zeros
    with torch.no_grad():
        q, part = float4_layer_norm(big, g, b), float4_layer_norm(x, g, b)
    assert torch.equal(q.data[-last:], part.data)
    assert torch.equal(q.scale[:, rows - last:rows], part.scale[:, :last])


def test_two_threads_at_once() -> None:
    """Calls from two threads on streams of their own, forward and backward, give what they give in turn."""
    from threading import Thread

    def work(k):
        x, g, b, dy = _inputs(130 + k, 700, torch.bfloat16, 30 + k)
        w = _inputs(200, 700, torch.float32, 40 + k)[0]
        args = [t.requires_grad_() for t in (x, g, b, w)]
        kept = float4_quantize(w.detach(), tiles=True)
        up = _inputs(130 + k, 200, torch.bfloat16, 50 + k)[0]
        torch.cuda.current_stream().synchronize()
        results = []
        for _ in range(20):
            y = float4_linear(layer_norm(*args[:3]), w, seed=7)
            grads = torch.autograd.grad(y, args, up)
            with torch.no_grad():
                served = float4_matmul(float4_layer_norm(x, g, b), kept)
                one = float4_linear(x[:3], kept)
            results.append([y.detach(), *grads, served, one])
        torch.cuda.current_stream().synchronize()
        assert all(torch.equal(p, q) for r in results[1:] for p, q in zip(results[0], r))
        found[k] = results[0]

    def threaded(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            work(k)

    found = {}
    for k in range(2):
        work(k)
    want, found = found, {}
    threads = [Thread(target=threaded, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert found.keys() == want.keys()
    assert all(torch.equal(p, q) for k in want for p, q in zip(found[k], want[k]))


def test_serving_in_a_graph() -> None:
    """A prompt's norm in 4 bits, its product and single tokens' on kept weights, replayed on new rows."""
    x, g, b, _ = _inputs(100, 700, torch.bfloat16)
    kept = float4_quantize(_inputs(300, 700, torch.float32, 5)[0], tiles=True)

    def serve():
        with torch.no_grad():
            q = float4_layer_norm(x, g, b)
            return [float4_matmul(q, kept), q.values(), float4_linear(x, kept), float4_linear(x[:1], kept),
                    float4_quantize(x, seed=4).values()]

    serve()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serve()
    for k in range(4):
        x.copy_(_inputs(100, 700, torch.bfloat16, 60 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, serve()))


@pytest.mark.parametrize("held", DTYPES)
def test_parameters_at_odd_places(held) -> None:
    """Parts of longer vectors, which begin between the places that wide loads prefer, and strided ones."""
    for cols in (300, 1029, 8195):
        x, g, b, dy = _inputs(9, cols, torch.bfloat16, held=held)
        want = layer_norm(x, g, b)
        for step in (1, 2):
            places = slice(1, 1 + step * cols, step)
            far = [torch.zeros(2 * cols + 2, dtype=held, device="cuda") for _ in range(2)]
            far[0][places], far[1][places] = g, b
            args = [t[places].detach().requires_grad_() for t in far]
            y = layer_norm(x, *args)
            assert torch.equal(y, want)
            _Exact(x, g, b).check_gradients(dy, None, *torch.autograd.grad(y, args, dy))


def test_rows_behind_the_last_are_left_alone() -> None:
    """Nothing is written past a matrix, whichever way its rows are spread over the GPU."""
    from dionw_amd import _lib

    for rows, cols in ((5, 100), (5, 700), (9, 3000), (3, 20000)):
        x, g, b, dy = _inputs(rows, cols, torch.float32)
        y, dx = (torch.full((rows + 20, cols), 77.0, device="cuda") for _ in range(2))
        stats = torch.full((2, rows + 20), 77.0, device="cuda")
        stream = _lib.stream_handle(x.device)
        _lib.call("dionw_layer_norm_forward", 2, x.data_ptr(), cols, rows, cols, 2, g.data_ptr(), 2, b.data_ptr(),
                  1e-5, y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), stream)
        _lib.call("dionw_layer_norm_backward", 2, x.data_ptr(), cols, dy.data_ptr(), cols, rows, cols, 2,
                  g.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(), None, 2, None, None, 0,
                  stream)
        depth = -(-cols // 256) * 256
        data = torch.full((rows + 20, depth // 2), 77, dtype=torch.uint8, device="cuda")
        scale = torch.full((depth // 32 + 1, 32), 77, dtype=torch.uint8, device="cuda")
        _lib.call("dionw_layer_norm_float4", 2, x.data_ptr(), cols, rows, cols, 2, g.data_ptr(), 2, b.data_ptr(),
                  1e-5, data.data_ptr(), scale.data_ptr(), 32, stream)
        for t in (y[rows:], dx[rows:], stats[:, rows:], data[rows:], scale[-1], scale[:, rows:]):
            assert bool((t == 77).all())
        assert not (stats[:, :rows] == 77).any()


def test_nothing_is_written_past_the_scratch_and_the_parameters_gradients() -> None:
    from dionw_amd import _lib

    for rows, cols in ((1, 1), (9, 100), (2500, 300), (5, 700), (70, 2048), (9, 6001), (70, 20001)):
        x, g, b, dy = _inputs(rows, cols, torch.float32)
        stats = torch.zeros(2, rows, device="cuda")
        size = _lib.library().dionw_layer_norm_backward_scratch(rows, cols)
        scratch, dx, dg, db = (torch.full((n // 4 + 9999,), 77.0, device="cuda")
                               for n in (size, 4 * rows * cols, 4 * cols, 4 * cols))
        for at in ((dg, db), (dg, None), (None, db)):
            _lib.call("dionw_layer_norm_backward", 2, x.data_ptr(), cols, dy.data_ptr(), cols, rows, cols, 2, g.data_ptr(),
                      stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(),
                      None if at[0] is None else dg.data_ptr(), 2, None if at[1] is None else db.data_ptr(),
                      scratch.data_ptr(), size, _lib.stream_handle(x.device))
            for t in (scratch, dx, dg, db):
                assert bool((t[-9999:] == 77).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 1), (3, 200), (100, 768), (70, 1500), (5, 2048), (600, 4096), (9, 6000),
                                  (2, 16000), (3, 20000), (1000, 256)], ids=str)
def test_the_norm_quantized_as_it_is_made(size, dtype) -> None:
    """The codes are those of the float32 norm, which is one of the values that the bound allows: each
    code must be the one of a value within it."""
    x, g, b, _ = _inputs(*size, dtype)
    q = float4_layer_norm(x, g, b)
    y = layer_norm(x.float(), g, b)
    want = float4_quantize(y)
    assert q.shape == want.shape and q.cols == size[1]
    assert torch.equal(q.scale[:, :size[0]], want.scale[:, :size[0]])
    assert torch.equal(q.data, want.data)
    _Exact(x, g, b).check_y(y)


def test_the_operators_together() -> None:
    """A block of a model, trained and then served from kept weights: the same operators in a row."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g, b, dy = _inputs(130, 300, torch.bfloat16)
    w = (torch.randn(99, 300, generator=gen, device="cuda") * 300 ** -0.5).requires_grad_()
    bias = torch.randn(99, generator=gen, device="cuda").requires_grad_()
    args = [t.requires_grad_() for t in (x, g, b)]
    h = layer_norm(*args)
    y = float4_linear(h, w, bias, seed=3)
    up = torch.randn(130, 99, generator=gen, device="cuda").bfloat16()
    grads = torch.autograd.grad(y, [*args, w, bias], up)
    # The same chain, a link at a time.
    hd = h.detach().requires_grad_()
    z = float4_linear(hd, w, bias, seed=3)
    dh, dw, dbias = torch.autograd.grad(z, (hd, w, bias), up)
    assert torch.equal(y, z) and torch.equal(grads[3], dw) and torch.equal(grads[4], dbias)
    exact = _Exact(x, g, b)
    exact.check_y(h)
    exact.check_gradients(dh, *grads[:3])
    with torch.no_grad():
        kept = float4_quantize(w, tiles=True)
        served = float4_matmul(float4_layer_norm(x, g, b), kept, bias, dtype=torch.float32)
        assert torch.equal(served, float4_linear(layer_norm(x.float(), g, b), kept, bias)[:, :])
