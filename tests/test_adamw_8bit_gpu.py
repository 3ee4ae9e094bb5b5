"""AdamW with 8-bit moments against its definition in float64 (GPU).

Bounds. The kernel works in float32, each operation rounded once (relative error 2^-24 at
most): m is a sum of two products (its error is at most 3 x 2^-24 of the larger term's
magnitude), r the root of a sum of two products of three factors (at most 4 x 2^-24 relative),
the update adds at most 8 more roundings. So new parameters are held to
``2 x 2^-24 |p| + 16 x 2^-24 |update|``, with the update of the terms' magnitudes. A code is
at most 16 (e4m3) or 32 (u44) units of its last place, so those errors move an element by at
most 32 x 4 x 2^-24 = 2^-17 of a unit of the last place (and the cancellation of m's two terms
scales its error): codes must equal the oracle's wherever the rounding was further than that
from the neighbouring code, and be the neighbour's otherwise.
"""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import dionw_amd as dionw
from dionw_amd import AdamWState, Dion, EMAConfig, StepGraph
from tests import adamw_8bit_oracle as oracle

pytestmark = pytest.mark.gpu

HYPER = {"lr": 3e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}
EPS = 2.0 ** -24


def _optimizer(params, **more):
    return Dion([{"params": params, "dion_route": "adamw"}], **{**HYPER, **more},
                adamw_state=AdamWState.EIGHT_BIT)


def _tensors(sizes, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.05).cuda()) for s in sizes]


def _grads(params, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        spread = torch.exp(2 * torch.randn(p.shape, generator=gen))
        p.grad = (torch.randn(p.shape, generator=gen) * spread * 1e-3).cuda()


def _values(entry):
    """(m, r) of a tensor's state as float64, and its codes."""
    mc = entry["exp_avg"].contiguous().view(torch.uint8).cpu().numpy().reshape(-1)
    rc = entry["exp_avg_rms"].cpu().numpy().reshape(-1)
    ms = entry["exp_avg_scale"].cpu().numpy().astype(np.float64)
    rs = entry["exp_avg_rms_scale"].cpu().numpy().astype(np.float64)
    n = mc.size
    return (oracle.e4m3_values(mc) * np.repeat(ms, 256)[:n],
            oracle.u44_values(rc) * np.repeat(rs, 256)[:n], mc, rc, ms, rs)


def _flat(t):
    return t.detach().contiguous().cpu().numpy().reshape(-1).astype(np.float64)


def _before(opt, params):
    return [(_flat(p), None if p.grad is None else _flat(p.grad), *_values(opt.state[p])[:2],
             float(opt.state[p]["adamw_step"])) for p in params]


def _check(opt, params, before, hyper=HYPER):
    beta1, beta2 = hyper["betas"]
    for place, (param, (p0, g, m0, r0, t0)) in enumerate(zip(params, before)):
        m_now, r_now, mc, rc, ms, rs = _values(opt.state[param])
        if g is None:
            assert np.array_equal(_flat(param), p0) and np.array_equal(m_now, m0)
            assert float(opt.state[param]["adamw_step"]) == t0
            continue
        step = int(t0) + 1
        assert float(opt.state[param]["adamw_step"]) == step
        p, m, r, bits = oracle.update(p0, g, m0, r0, step, place, lr=hyper["lr"], beta1=beta1,
                                      beta2=beta2, eps=hyper["eps"],
                                      weight_decay=hyper["weight_decay"])
        terms = beta1 * np.abs(m0) + (1 - beta1) * np.abs(g)
        most = (hyper["lr"] / (1 - beta1 ** step) * terms
                / (r / np.sqrt(1 - beta2 ** step) + hyper["eps"]))
        assert np.all(np.abs(_flat(param) - p) <= 2 * EPS * np.abs(p0) + 16 * EPS * most + 1e-45)
        for now, x, scale_now, noise, form, size in (
                (np.abs(m_now), m, ms, bits[0], oracle.E4M3, terms), (r_now, r, rs, bits[1], oracle.U44, r)):
            xb = oracle.blocks_of(x)
            scale = oracle.block_scales(xb, form)
            assert np.array_equal(scale, scale_now)
            want, margin = oracle.rounded(xb, scale, oracle.blocks_of(noise), form)
            want, margin = want.reshape(-1)[:x.size], margin.reshape(-1)[:x.size]
            if form is oracle.U44:
                unit = np.repeat(scale, 256)[:x.size] * 2.0 ** -11
                want = np.where((x > 0) & (want == 0), unit, want)
            ratio = size / np.maximum(np.abs(x), 1e-300)
            clear = margin > 2.0 ** -17 * np.minimum(ratio, 1e6)
            assert np.array_equal(now[clear], want[clear])
            assert x.size < 1000 or clear.mean() > 0.99
            assert np.all(np.abs(now - np.abs(x)) <= np.abs(x) * 2.0 ** -form[0] * 1.001
                          + np.repeat(scale, 256)[:x.size] * 2.0 ** (form[1] - form[0]) * 1.001)
        assert np.all(np.sign(m_now) * np.sign(m) >= 0)


@pytest.mark.parametrize("sizes", [
    [1], [255, 256, 257], [(3, 85), (4096,), (16, 257)], [4095, 4097, 12345, 2], [(1000, 333)],
])
@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.0, 0.0), (0.95, 0.999)])
def test_steps_match_the_definition(sizes, betas) -> None:
    params = _tensors(sizes)
    opt = _optimizer(params, betas=betas)
    for k in range(4):
        _grads(params, 100 + k)
        before = _before(opt, params)
        opt.step()
        _check(opt, params, before, {**HYPER, "betas": betas})


def test_more_tensors_than_a_launch_holds() -> None:
    params = _tensors([1 + 7 * i % 600 for i in range(300)])
    opt = _optimizer(params)
    for k in range(2):
        _grads(params, k)
        for p in params[k::9]:
            p.grad = None
        before = _before(opt, params)
        opt.step()
        _check(opt, params, before)


def test_alignments_layouts_and_empty_tensors() -> None:
    base = torch.randn(5000, device="cuda")
    params = [torch.nn.Parameter(base[1:1002]), torch.nn.Parameter(base[2003:3000].view(-1)),
              torch.nn.Parameter(torch.randn(8, 16, 5, 5, device="cuda").to(memory_format=torch.channels_last)),
              torch.nn.Parameter(torch.randn(40, 30, device="cuda").t()),
              torch.nn.Parameter(torch.randn(0, 4, device="cuda"))]
    outside = base.clone()
    opt = _optimizer(params)
    for k in range(3):
        _grads(params, k)
        if k == 1:
            params[2].grad = params[2].grad.to(memory_format=torch.channels_last)
            params[0].grad = torch.cat([params[0].grad, params[0].grad])[::2].clone()
            params[0].grad = torch.stack([params[0].grad] * 2, 1)[:, 0]  # a stride of 2
        before = _before(opt, params)
        opt.step()
        _check(opt, params, before)
    for part in (slice(0, 1), slice(1002, 2003), slice(3000, 5000)):
        assert torch.equal(base[part], outside[part])


def test_zero_tiny_and_large_gradients() -> None:
    params = _tensors([1024])
    opt = _optimizer(params, weight_decay=0.0)
    start = params[0].detach().clone()
    params[0].grad = torch.zeros_like(params[0])
    opt.step()
    assert torch.equal(params[0], start) and not opt.state[params[0]]["exp_avg"].view(torch.uint8).any()
    grad = torch.full((1024,), 1e-30, device="cuda")
    grad[256:512] = 1e12
    grad[512:768] = torch.logspace(-12, 4, 256, device="cuda")
    params[0].grad = grad
    for _ in range(3):
        opt.step()
        m, r = _values(opt.state[params[0]])[:2]
        assert np.isfinite(m).all() and np.isfinite(r).all()
        assert torch.isfinite(params[0]).all()
    # No element's divisor is zero where its gradient's square is not.
    assert (r[256:768] > 0).all()
    assert (params[0].detach() - start).abs().max() < 4 * 3 * HYPER["lr"] * 1.5


def test_elements_that_are_not_finite_stay_alone() -> None:
    params, twins = _tensors([700]), _tensors([700])
    opt, twin = _optimizer(params), _optimizer(twins)
    bad = [3, 300, 301, 699]
    for k in range(3):
        _grads(params, k)
        twins[0].grad = params[0].grad.clone()
        twins[0].grad[bad] = 0.0
        if k == 1:
            params[0].grad[bad] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38],
                                               device="cuda")
        else:
            params[0].grad[bad] = 0.0
        opt.step()
        twin.step()
    good = torch.ones(700, dtype=torch.bool)
    good[bad] = False
    assert torch.equal(params[0].cpu()[good], twins[0].cpu()[good])
    for key in ("exp_avg", "exp_avg_rms"):
        a, b = (o.state[q]["%s" % key].view(torch.uint8).cpu() for o, q in ((opt, params[0]), (twin, twins[0])))
        assert torch.equal(a[good], b[good])
    assert torch.isnan(params[0].detach().cpu()[bad]).all()


def test_a_long_average_is_unbiased() -> None:
    """With b2 = 0.999 a step moves r by a thirtieth of a code: rounded to nearest it would stand
    still. From 4 times too large it has to reach the gradient's size; around it the codes' noise
    raises the mean square by 0.4% at most (a step adds unit x |change|, and decays by 0.001)."""
    param = torch.nn.Parameter(torch.zeros(16384, device="cuda"))
    opt = _optimizer([param], betas=(0.9, 0.999), weight_decay=0.0)
    size = torch.logspace(-6, 0, 16384, device="cuda")[torch.randperm(16384)]
    param.grad = 4 * size
    for _ in range(60):
        opt.step()
    for _ in range(9000):  # e^-9 of the excess is left
        param.grad = size
        opt.step()
    m, r = opt.adamw_moments([param])
    block = size.view(64, 256).amax(1).repeat_interleave(256)
    seen = size > block * 2.0 ** -16  # not among the block's subnormal values
    assert abs(float((r / size)[seen].double().mean()) - 1) < 0.01
    assert abs(float((m / size)[seen].double().mean()) - 1) < 0.01


def test_gpu_ema_rides_on_the_pass() -> None:
    params, twins = _tensors([1000, 257]), _tensors([1000, 257])
    opt = _optimizer(params, ema=EMAConfig(decay=0.9))
    twin = _optimizer(twins)
    shadows = None
    for k in range(4):
        _grads(params, k)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step()
        twin.step()
        if shadows is None:
            shadows = [q.detach().clone() for q in twins]
        else:
            torch._foreach_lerp_(shadows, [q.detach() for q in twins], 1 - 0.9)
        for p, q, s in zip(params, twins, shadows):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["ema_shadow"], s)


def test_cpu_ema_follows() -> None:
    params, twins = _tensors([1000]), _tensors([1000])
    opt = _optimizer(params, ema=EMAConfig(decay=0.9, device=dionw.EMADevice.CPU))
    twin = _optimizer(twins)
    shadow = None
    for k in range(3):
        _grads(params, k)
        twins[0].grad = params[0].grad.clone()
        opt.step()
        twin.step()
        now = twins[0].detach().cpu()
        shadow = now.clone() if shadow is None else shadow.lerp_(now, 1 - 0.9)
    assert torch.equal(params[0], twins[0])
    opt.ema.flush_pending_updates()
    assert torch.equal(opt.state[params[0]]["ema_shadow"], shadow)


def test_moments_are_the_codes_values() -> None:
    params = _tensors([(3, 100), 257, 5000, 1])
    opt = _optimizer(params)
    _grads(params, 1)
    opt.step()
    for chosen in (params, [params[2]], [params[3], params[0]]):
        m, r = opt.adamw_moments(chosen)
        want = [_values(opt.state[p])[:2] for p in chosen]
        assert np.array_equal(m.cpu().numpy(), np.concatenate([w[0] for w in want]).astype(np.float32))
        assert np.array_equal(r.cpu().numpy(), np.concatenate([w[1] for w in want]).astype(np.float32))


def test_a_saved_state_resumes_bit_for_bit(tmp_path) -> None:
    params = _tensors([(30, 40), 777])
    opt = _optimizer(params)
    for k in range(3):
        _grads(params, k)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    saved = torch.load(tmp_path / "opt.pt", weights_only=True)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin = _optimizer(twins)
    for q in twins:  # a state of its own, to be replaced
        q.grad = torch.ones_like(q)
    twin.step()
    with torch.no_grad():
        for p, q in zip(params, twins):
            q.copy_(p)
    twin.load_state_dict(saved)
    again = twin.state_dict()["state"]
    for index, entry in opt.state_dict()["state"].items():
        assert set(entry) == {"exp_avg", "exp_avg_scale", "exp_avg_rms", "exp_avg_rms_scale", "adamw_step"}
        for key, value in entry.items():
            other = again[index][key]
            assert other.dtype is value.dtype and other.shape == value.shape
            assert torch.equal(other.view(torch.uint8) if value.dim() else other,
                               value.view(torch.uint8) if value.dim() else value)
    for k in range(3, 6):
        _grads(params, k)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step()
        twin.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)


def test_a_saved_state_with_an_ema_resumes_bit_for_bit() -> None:
    params = _tensors([(30, 40), 777])
    opt = _optimizer(params, ema=EMAConfig(decay=0.9))
    for k in range(3):
        _grads(params, k)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin = _optimizer(twins, ema=EMAConfig(decay=0.9))
    twin.load_state_dict(saved)
    for k in range(3, 6):
        _grads(params, k)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step()
        twin.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
            assert torch.equal(opt.state[p]["ema_shadow"], twin.state[q]["ema_shadow"])
    # Two optimizers that share a loaded dict share no state.
    assert twin.state[twins[0]]["exp_avg"].data_ptr() != opt.state[params[0]]["exp_avg"].data_ptr()


def test_states_of_another_kind_are_refused() -> None:
    params = _tensors([100])
    eight = _optimizer(params)
    plain = Dion([{"params": params, "dion_route": "adamw"}], **HYPER)
    assert "adamw_state" not in plain.state_dict()["param_groups"][0]
    for target, source in ((eight, plain), (plain, eight)):
        with pytest.raises(ValueError, match="adamw_state"):
            target.load_state_dict(copy.deepcopy(source.state_dict()))
    with pytest.raises(ValueError):
        Dion([{"params": params, "dion_route": "adamw", "adamw_state": "4bit"}], **HYPER)
    with pytest.raises(ValueError, match="8-bit"):
        plain.adamw_moments(params)
    with pytest.raises(ValueError, match="8-bit"):
        eight.adamw_moments([])
    params[0].grad = torch.ones(100, device="cuda")
    broken = copy.deepcopy(eight.state_dict())
    broken["state"][0]["exp_avg_scale"] = torch.zeros(7, device="cuda")
    with pytest.raises(ValueError, match="exp_avg_scale"):
        eight.load_state_dict(broken)


def test_a_group_may_choose_for_itself() -> None:
    a, b = _tensors([300]), _tensors([300])
    opt = Dion([{"params": a, "dion_route": "adamw", "adamw_state": "8bit"},
                {"params": b, "dion_route": "adamw"}], **HYPER)
    assert "exp_avg_rms" in opt.state[a[0]] and "exp_avg_sq" in opt.state[b[0]]
    _grads(a, 0)
    b[0].grad = a[0].grad.clone()
    opt.step()
    # The first step's moments are unrounded when they are used: both kinds give the same update
    # but for rounding.
    assert torch.allclose(a[0], b[0], rtol=1e-6, atol=1e-9)


def test_another_stream_and_a_graph() -> None:
    matrix = torch.nn.Parameter(torch.randn(128, 128, device="cuda") * 0.02)
    params = [matrix] + _tensors([1000, 257])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]

    def build(ps):
        return Dion([{"params": ps[:1], "dion_route": "matrix"},
                     {"params": ps[1:], "dion_route": "adamw"}], **HYPER,
                    adamw_state=AdamWState.EIGHT_BIT)

    opt, twin = build(params), build(twins)
    for p, q in zip(params, twins):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    graph = StepGraph(opt)
    side = torch.cuda.Stream()
    for k in range(4):
        _grads(twins, k)
        for p, q in zip(params, twins):
            p.grad.copy_(q.grad)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            twin.step()
        torch.cuda.synchronize()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
            for key, value in twin.state[q].items():
                assert torch.equal(opt.state[p][key].float(), value.float()), key


def test_indexes_past_32_bits() -> None:
    size = 2 ** 32 + 777
    param = torch.nn.Parameter(torch.zeros(size, device="cuda"))
    param.grad = torch.zeros(size, device="cuda")
    ends = [slice(0, 1024), slice(size - 1801, size)]  # the last from a block's start on
    gen = torch.Generator().manual_seed(0)
    for part in ends:
        param.grad[part] = torch.randn(param.grad[part].shape, generator=gen).cuda()
    opt = _optimizer([param])
    opt.step()
    beta1, beta2 = HYPER["betas"]
    start = size - 1801
    assert start % 256 == 0
    g = param.grad[start:].cpu().numpy().astype(np.float64)
    m, r = (1 - beta1) * g, np.sqrt((1 - beta2) * g ** 2)
    bits = oracle.noise(1, 0, np.arange(start, size, dtype=np.uint64))
    entry = opt.state[param]
    now = oracle.e4m3_values(entry["exp_avg"][start:].view(torch.uint8).cpu().numpy())
    now = np.abs(now * np.repeat(entry["exp_avg_scale"][start // 256:].cpu().numpy(), 256)[:g.size])
    xb = oracle.blocks_of(m)
    want, margin = oracle.rounded(xb, oracle.block_scales(xb, oracle.E4M3),
                                  oracle.blocks_of(bits[0]), oracle.E4M3)
    clear = margin.reshape(-1)[:g.size] > 2.0 ** -17
    assert np.array_equal(now[clear], want.reshape(-1)[:g.size][clear])
    assert int((entry["exp_avg"].view(torch.uint8) & 127).ne(0).sum()) <= 1024 + 1801
    assert not param[1024:start].any() and param[start:].all()
