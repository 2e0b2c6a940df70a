"""Rotary positions on the GPU against the complex product in float64, within derived bounds (sequence_oracle),
and the run of rotary and linear_recurrence together behind the signature operators."""
import math

import numpy as np
import pytest
import torch

import pysiglib_b200 as psl
import sequence_oracle as so
from pysiglib_b200 import load_cusig, torch_api

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


def normal(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64).to(dtype)


def frequencies(r, **kw):
    return torch.from_numpy(psl.rotary_frequencies(r, **kw))


def cuda(t):
    return None if t is None else t.cuda()


def check_turn(x, f, positions, interleaved, scale=1.0, inverse=False, view=lambda t: t):
    how = {"interleaved": interleaved, "scale": scale, "inverse": inverse}
    before = load_cusig.launch_count()
    y = psl.rotary(view(x.cuda()), cuda(f), cuda(positions), **how)
    assert load_cusig.launch_count() > before and y.dtype == x.dtype
    so.check(y, so.rotary(view(x), f, positions, interleaved, scale, inverse), "y")
    dx = psl.rotary_backprop(view(x.cuda()), cuda(f), cuda(positions), **how)
    so.check(dx, so.rotary(view(x), f, positions, interleaved, scale, not inverse), "dx")
    part = 2 * f.shape[0]
    assert torch.equal(y[..., part:].cpu(), view(x)[..., part:])
    return y


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,part", [(2, 2), (3, 2), (5, 0), (6, 4), (16, 16), (32, 16), (48, 20), (64, 64), (80, 80), (96, 64), (128, 128), (257, 256), (34, 34)])
def test_widths(dtype, interleaved, dim, part):
    for shape in ((1, dim), (7, dim), (2, 33, dim), (2, 3, 9, dim)):
        check_turn(normal(dim + part, *shape, dtype=dtype), frequencies(part), None, interleaved, 0.5 if dim == 64 else 1.0)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, F32, F64])
@pytest.mark.parametrize("lead", [(1, 1, 20), (3, 1, 20), (1, 4, 20), (3, 4, 20), (20,), (4, 20), (3, 1, 1)])
def test_positions(kind, lead):
    g = torch.Generator().manual_seed(3)
    p = torch.rand(*lead, generator=g, dtype=F64) * 1e5 - 2e4
    p = p.to(kind) if kind.is_floating_point else p.round().to(kind)
    for dtype in (F32, BF16):
        check_turn(normal(4, 3, 4, 20, 32, dtype=dtype), frequencies(32), p, False)


def test_far_positions_keep_their_angles():
    p = torch.tensor([0, 1, 131071, 10 ** 6, 2 ** 31 + 5, 10 ** 12])
    check_turn(normal(5, 6, 64), frequencies(64), p, False)
    check_turn(normal(5, 6, 64, dtype=F64), frequencies(64), p, True)


def test_views_and_layouts():
    f = frequencies(32)
    p = torch.arange(19) * 3
    for dtype in (F32, BF16):
        x = normal(6, 2, 19, 4, 32, dtype=dtype)
        y = check_turn(x, f, p, False, view=lambda t: t.transpose(1, 2))
        assert y.stride() == x.transpose(1, 2).stride()
        check_turn(normal(7, 2, 19, 4, 3 * 32 + 8, dtype=dtype), f, p, True, view=lambda t: t[..., 32:64].transpose(1, 2))
        check_turn(normal(8, 2, 19, 4, 33, dtype=dtype), f, p, False, view=lambda t: t[..., 1:].transpose(1, 2))
        check_turn(normal(9, 2, 19, 32, dtype=dtype), f, p, False, view=lambda t: t.unsqueeze(1).expand(2, 5, 19, 32))
        check_turn(normal(10, 32, 19, dtype=dtype), f, p, False, view=lambda t: t.T)
        check_turn(normal(11, 2, 3, 2, 5, 19, 32, dtype=dtype), f, p, True, view=lambda t: t.transpose(0, 3))
        check_turn(normal(12, 2, 3, 2, 19, 32, dtype=dtype), f, torch.rand(2, 1, 2, 19, dtype=F64), True)
        check_turn(normal(13, 6, 38, 32, dtype=dtype), f, p, False, view=lambda t: t[::2, ::2])


def test_turning_back_and_the_adjoint():
    x, d = normal(14, 2, 50, 48, dtype=F64).cuda(), normal(15, 2, 50, 48, dtype=F64).cuda()
    f, p = frequencies(40).cuda(), torch.rand(2, 50, dtype=F64).cuda() * 100
    y = psl.rotary(x, f, p, scale=2.0)
    back = psl.rotary(y, f, p, scale=0.5, inverse=True)
    assert float((back[..., :40] - x[..., :40]).abs().max()) < 40 * 2.0 ** -53 * float(x.abs().max()) * 2
    lhs, rhs = (y * d).sum(), (x * psl.rotary_backprop(d, f, p, scale=2.0)).sum()
    assert abs(float(lhs - rhs)) < 1e-12 * float((y * d).abs().sum())
    X = x.clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda t: torch_api.rotary(t, f, p, interleaved=True, scale=1.5), (X,), eps=1e-6, atol=1e-6)


def test_nonfinite_values_stay_in_their_pair():
    x = normal(16, 10, 64)
    x[3, 5], x[4, 40] = float("nan"), float("inf")
    y = psl.rotary(x.cuda(), frequencies(64).cuda()).cpu()
    touched = torch.zeros(10, 64, dtype=torch.bool)
    touched[3, 5] = touched[3, 37] = touched[4, 40] = touched[4, 8] = True
    assert torch.isfinite(y[~touched]).all() and not torch.isfinite(y[3, [5, 37]]).any() and not torch.isfinite(y[4, [8, 40]]).any()
    p = torch.zeros(10, dtype=F32)
    p[2], p[6] = float("nan"), float("inf")
    y = psl.rotary(normal(16, 10, 64).cuda(), frequencies(64).cuda(), p.cuda()).cpu()
    assert torch.isnan(y[[2, 6]]).all() and torch.isfinite(y[[0, 1, 3, 4, 5, 7, 8, 9]]).all()


def test_more_than_32_bits_of_elements():
    rows = (1 << 31) // 4096 + 64
    x = torch.zeros(rows, 32, 128, dtype=BF16, device="cuda").transpose(0, 1)
    x[31, rows - 1] = 1.0
    y = psl.rotary(x, frequencies(128).cuda())
    so.check(y[31, rows - 1:], so.rotary(torch.ones(1, 128, dtype=BF16), frequencies(128), torch.tensor([rows - 1]), False, 1.0), "y")
    assert float(y[:, : rows - 1].abs().max()) == 0


def test_side_streams_and_graphs():
    f, p = frequencies(64).cuda(), torch.arange(100, device="cuda")
    xs = [normal(20 + k, 2, 4, 100, 64, dtype=BF16).cuda() for k in range(2)]
    expects = [so.rotary(x.cpu(), f.cpu(), p.cpu(), True, 1.0) for x in xs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = psl.rotary(xs[0], f, p, interleaved=True)
    stream.synchronize()
    so.check(y, expects[0], "y")
    graph = torch.cuda.CUDAGraph()
    static = xs[0].clone()
    with torch.cuda.graph(graph):
        out = psl.rotary(static, f, p, interleaved=True)
    for k in (0, 1, 0):
        static.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        so.check(out, expects[k], "y")


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
def test_host_arrays(dtype):
    x = normal(30, 2, 3, 11, 20, dtype={np.float32: F32, np.float64: F64, np.float16: F16}[dtype])
    f = psl.rotary_frequencies(12)
    for p in (None, np.arange(11) + 5, np.random.default_rng(0).uniform(0, 50, (2, 1, 11))):
        y = psl.rotary(x.numpy(), f, p, interleaved=True, scale=2.0)
        expect = so.rotary(x, torch.from_numpy(f), None if p is None else torch.from_numpy(p), True, 2.0)
        assert isinstance(y, np.ndarray) and y.dtype == dtype
        so.check(torch.from_numpy(y), expect, "y")
    y = psl.rotary(x.to(BF16), torch.from_numpy(f))
    so.check(y, so.rotary(x.to(BF16), torch.from_numpy(f), None, False, 1.0), "y")


def test_oscillators_of_a_sampled_path():
    """Turned, scanned and turned back, the recurrence has the complex factors a_t exp(i w (p_t - p_{t-1})):
    the gated scan of an irregularly sampled path, checked row by row in complex float64, and the gradient
    that reaches the path through log signatures of its windows."""
    torch.manual_seed(0)
    paths = (torch.randn(4, 30, 9, 3, dtype=F64).cumsum(2) * 0.3).cuda().requires_grad_()  # 30 windows of 9 points
    times = torch.rand(4, 30, dtype=F64, device="cuda").cumsum(1) * 3
    gate = torch.randn(4, 30, 14, dtype=F64, device="cuda").requires_grad_()
    f = torch.tensor([0.0, 0.1, 0.5, 1.0, 2.0, 5.0, 9.0], dtype=F64, device="cuda")

    def model(paths, gate):
        features = torch_api.log_sig(paths, 3)                      # (4, 30, 14)
        u = torch_api.rotary(features, f, times, inverse=True)
        h = torch_api.linear_recurrence(u, gate.repeat(1, 1, 1), gate_form="logit", complement=False)
        return features, torch_api.rotary(h, f, times)

    # one gate for both channels of a pair: the factor of a complex number
    shared = torch.cat([gate[..., :7], gate[..., :7]], -1)
    features, h = model(paths, shared)
    z = torch.complex(features[..., :7], features[..., 7:]).detach().cpu()
    a = torch.sigmoid(gate[..., :7]).detach().cpu()
    t, w = times.cpu(), f.cpu()
    now = torch.zeros(4, 7, dtype=torch.complex128)
    for k in range(30):
        gap = t[:, k] - t[:, k - 1] if k else torch.zeros(4, dtype=F64)
        now = a[:, k] * torch.polar(torch.ones(4, 7, dtype=F64), gap[:, None] * w) * now + z[:, k]
        got = torch.complex(h[:, k, :7], h[:, k, 7:]).detach().cpu()
        # angles up to 9 * 90 radians, each within 8 units of 2^-53 of itself, over a memory of at most 30 rows
        assert float((got - now).abs().max()) < 30 * 9 * 90 * 8 * 2.0 ** -53 * float(z.abs().max()) * 30
    loss = (h * torch.linspace(-1, 1, h.numel(), dtype=F64, device="cuda").view_as(h)).sum()
    gp, gg = torch.autograd.grad(loss, (paths, gate))
    step = 1e-5
    for leaf, grad in ((paths, gp), (gate, gg)):
        direction = torch.randn_like(leaf)
        with torch.no_grad():
            values = []
            for s in (step, -step):
                args = [leaf + s * direction if leaf is t else t for t in (paths, gate)]
                both = torch.cat([args[1][..., :7], args[1][..., :7]], -1)
                values.append(float((model(args[0], both)[1] * torch.linspace(-1, 1, h.numel(), dtype=F64, device="cuda").view_as(h)).sum()))
        slope = (values[0] - values[1]) / (2 * step)
        exact = float((grad * direction).sum())
        assert abs(slope - exact) < 1e-5 * max(1.0, abs(exact), float((grad * direction).abs().sum()) * 1e-2), (slope, exact)


def test_a_float32_chain_in_training():
    """The same layer in 16 bits with float32 gates, packed: gradients reach every leaf and are finite."""
    x = normal(40, 500, 64, dtype=BF16).cuda().requires_grad_()
    gate = normal(41, 500, 4).cuda().requires_grad_()
    offsets = torch.tensor([0, 100, 100, 380, 500], device="cuda")
    start = torch.zeros(4, 64, device="cuda", requires_grad=True)
    f = frequencies(64).cuda()
    u = torch_api.rotary(x, f, inverse=True)
    h, state = torch_api.linear_recurrence(u, gate, start, gate_form="logit", complement=True, offsets=offsets, return_state=True)
    y = torch_api.rotary(h, f)
    (y.float().square().sum() + state.sum()).backward()
    for leaf in (x, gate, start):
        assert leaf.grad is not None and torch.isfinite(leaf.grad).all() and float(leaf.grad.abs().max()) > 0
    assert float(state[1].abs().max()) == 0


def near_quarter_turns(odd):
    """Angles (the frequency is 1) 1e-4 to 1e-2 from odd or even quarter turns, whose cosine or sine is that small."""
    rng = np.random.default_rng(17)
    k = 2.0 * rng.integers(-1000, 1000, 4000) + odd
    return k * (np.pi / 2) + rng.choice([-1.0, 1.0], 4000) * 10.0 ** rng.uniform(-4, -2, 4000)


@pytest.mark.parametrize("odd", [0, 1])
def test_small_sines_and_cosines_keep_their_digits(odd):
    """float32 rows: what is left of the angle is rounded once, relative to itself (1 unit of 2^-24), its sine is
    within 2 units more (the series' product, a tenth of a unit, its sum, one, and its rest); the angle itself is
    within 4 units of 2^-53."""
    angle = near_quarter_turns(odd)
    x = torch.zeros(4000, 2)
    x[:, 0] = 1.0
    for interleaved in (False, True):
        y = psl.rotary(x.cuda(), torch.ones(1, dtype=F64).cuda(), torch.from_numpy(angle).cuda(), interleaved=interleaved).cpu().double().numpy()
        exact = (np.cos if odd else np.sin)(angle.astype(np.longdouble)).astype(np.float64)
        off = np.abs(y[:, 0 if odd else 1] - exact) - (4 * 2.0 ** -24 * np.abs(exact) + 4 * 2.0 ** -53 * np.abs(angle))
        assert off.max() <= 0, off.max()


@pytest.mark.parametrize("dtype", [F32, F64])
def test_turns_past_counting_keep_the_length(dtype):
    """Angles so large that 64 bits hold no fraction of a turn any more are some angle all the same."""
    angle = torch.tensor([2.0 ** 49 + 0.25, 2.0 ** 51 + 1, 2.0 ** 53 + 2, 1e17, 1e30, -1e40, 1e200, 1e300], dtype=F64)
    x = torch.zeros(8, 2, dtype=dtype)
    x[:, 0] = 1.0
    y = psl.rotary(x.cuda(), torch.ones(1, dtype=F64).cuda(), angle.cuda()).cpu().double()
    assert float((y.square().sum(1) - 1).abs().max()) < 16 * so.unit(dtype)  # twice 4 units each for sine and cosine


@pytest.mark.parametrize("odd", [0, 1])
def test_small_sines_and_cosines_keep_their_digits_in_float64(odd):
    """The series are within 2 units of 2^-53 each, the remainder within one, its low part adds one rounding."""
    if np.finfo(np.longdouble).nmant < 63:
        pytest.skip("needs an oracle of more than 64 bits")
    angle = near_quarter_turns(odd)
    x = torch.zeros(4000, 2, dtype=F64)
    x[:, 0] = 1.0
    y = psl.rotary(x.cuda(), torch.ones(1, dtype=F64).cuda(), torch.from_numpy(angle).cuda()).cpu().numpy()
    exact = (np.cos if odd else np.sin)(angle.astype(np.longdouble))
    off = np.abs(y[:, 0 if odd else 1].astype(np.longdouble) - exact) - 6 * 2.0 ** -53 * np.abs(exact)
    assert off.max() <= 0, off.max()
