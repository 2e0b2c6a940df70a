"""Row-by-row float64 definitions of the sequence operators, with bounds on what the roundings of a
correct implementation can add up to.

Unit roundoff of the arithmetic: u = eps / 2 of the state type.  One row of the recurrence costs at most ROUNDINGS
of them relative to |a| |h| + |b|: the gate factor (an exponential and a quotient, by CUDA's library or a Taylor series,
within 4 units, 1 - a within 2, its product with x 1), the product of a run's factors 1 and the multiply-add 1.  Errors already
made are handed on through |a|.  For gates of 16 bits e^v is taken by CUDA's __expf, whose documented error is
2 + floor(1.173 |v|) ulp (2 units each) where exp's is within the 4 units above: 2.4 |v| units more.  The
bounds below are that recursion, written out."""
import torch

ROUNDINGS = 10


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def state_type(dtype):
    return torch.float64 if dtype is torch.float64 else torch.float32


def factors(gate, form, dim):
    v = gate.double().repeat_interleave(dim // gate.shape[-1], -1)
    if form == "value":
        return v, 1 - v
    if form == "log":
        return torch.exp(v), -torch.expm1(v)
    return torch.sigmoid(v), torch.sigmoid(-v)


def spans_of(offsets, rows):
    if offsets is None:
        return [(0, rows)]
    o = [int(v) for v in offsets]
    return list(zip(o[:-1], o[1:]))


def recurrence(x, gate, initial, form, complement, offsets=None, derivs=None, state_derivs=None):
    """Values and error bounds, {name: (value, bound)}, for x (batch, rows, dim) or, packed, (rows, dim): h, state and,
    given derivs, dx, dgate, dinitial.  All on the CPU."""
    dtype, gate_dtype = x.dtype, gate.dtype
    roundings = ROUNDINGS
    if gate_dtype in (torch.float16, torch.bfloat16) and form != "value":
        roundings += 2.4 * float(gate.double().abs().max())
    u = unit(state_type(dtype)) * roundings
    packed = offsets is not None
    dim = x.shape[-1]
    a, rest = factors(gate, form, dim)
    v = x.double()
    b = rest * v if complement else v
    if packed:
        a, rest, b, v = (t[None] for t in (a, rest, b, v))
    batch, rows = b.shape[0], b.shape[1]
    spans = spans_of(offsets, rows)
    count = len(spans) if packed else batch
    start = torch.zeros(count, dim, dtype=torch.float64) if initial is None else initial.double()
    h, eh = torch.zeros_like(b), torch.zeros_like(b)
    before, eb = torch.zeros_like(b), torch.zeros_like(b)
    last, el = start.clone(), torch.zeros_like(start)
    for k, (lo, hi) in enumerate(spans):
        pick = slice(k, k + 1) if packed else slice(None)
        now, err, size = start[pick].clone(), torch.zeros_like(start[pick]), start[pick].abs()
        for t in range(lo, hi):
            before[:, t], eb[:, t] = now, err
            err = a[:, t].abs() * err + u * (a[:, t].abs() * size + b[:, t].abs())
            size = a[:, t].abs() * size + b[:, t].abs()
            now = a[:, t] * now + b[:, t]
            h[:, t], eh[:, t] = now, err
        last[pick], el[pick] = now, err
    tiny = torch.finfo(dtype).smallest_normal * unit(dtype) * 2

    def rounded(value, err, to):
        return value, err + unit(to) * (value.abs() + err) + torch.finfo(to).smallest_normal * torch.finfo(to).eps

    def shaped(t):
        return t[0] if packed else t

    result = {"h": rounded(shaped(h), shaped(eh), dtype), "state": (last, el + tiny * 0 + 1e-38)}
    if derivs is None:
        return result
    d = derivs.double()[None] if packed else derivs.double()
    g, eg = torch.zeros_like(b), torch.zeros_like(b)
    first, ef = torch.zeros_like(start), torch.zeros_like(start)
    for k, (lo, hi) in enumerate(spans):
        pick = slice(k, k + 1) if packed else slice(None)
        back = torch.zeros_like(start[pick]) if state_derivs is None else state_derivs.double()[pick].clone()
        err, size = torch.zeros_like(back), back.abs()
        for t in range(hi - 1, lo - 1, -1):
            g[:, t], eg[:, t] = d[:, t] + back, err + u * (size + d[:, t].abs())
            size = a[:, t].abs() * (size + d[:, t].abs())
            err = a[:, t].abs() * eg[:, t] + u * size
            back = a[:, t] * g[:, t]
        first[pick], ef[pick] = back, err
    inside = torch.zeros(rows, dtype=torch.bool)
    for lo, hi in spans:
        inside[lo:hi] = True
    inner = before - v if complement else before
    slope = {"value": torch.ones_like(a), "log": a, "logit": a * rest}[form]
    da = g * inner * slope
    eda = slope.abs() * (inner.abs() * eg + g.abs() * (eb + u * (before.abs() + (v.abs() if complement else 0)))
                         + u * (g * inner).abs())
    dx, edx = (rest * g, rest.abs() * eg + u * (rest * g).abs()) if complement else (g, eg)
    dx, edx, da, eda = (torch.where(inside[None, :, None], t, torch.zeros(())) for t in (dx, edx, da, eda))
    gates = gate.shape[-1]
    if gates != dim:
        group = dim // gates
        # a sum of `group` products in any order: at most `group` roundings on the sum of magnitudes
        eda = (eda + u / roundings * group * da.abs()).unflatten(-1, (gates, group)).sum(-1)
        da = da.unflatten(-1, (gates, group)).sum(-1)
    result["dx"] = rounded(shaped(dx), shaped(edx), dtype)
    result["dgate"] = rounded(shaped(da), shaped(eda), gate_dtype)
    result["dinitial"] = None if initial is None else (first, ef + 1e-38)
    return result


def rotary(x, frequencies, positions, interleaved, scale, inverse=False):
    """Value and bound of the turn, for x (.., rows, dim) and positions that broadcast to x.shape[:-1]."""
    half = frequencies.shape[0]
    if positions is None:
        positions = torch.arange(x.shape[-2])
    angle = positions.double()[..., None] * frequencies.double()
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle) * scale
    y = x.double().clone()
    p, q = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(y[..., p], y[..., q]) * turn
    size = torch.zeros_like(y)
    size[..., p] = size[..., q] = torch.complex(y[..., p], y[..., q]).abs() * abs(scale)
    y[..., p], y[..., q] = z.real, z.imag
    # relative to the pair's length: the angle (its product and quotient in 64 bits: 4 units of 2^-53 of it; its
    # remainder in the arithmetic's type: pi units), sine and cosine within 2 units each, scale, two products, a sum
    u = unit(state_type(x.dtype))
    turns = torch.zeros_like(y)
    turns[..., p] = turns[..., q] = (angle.abs() * 4 * 2.0 ** -53).expand(y[..., p].shape)
    err = size * (12 * u + turns) + unit(x.dtype) * (y.abs() + 12 * u * size)
    err = err + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    err[..., 2 * half:] = 0
    return y, err


def check(got, expected, what):
    value, bound = expected
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    if not got.numel():
        return
    over = (got - value).abs() - bound
    over = torch.where(torch.isfinite(over), over, torch.full_like(over, float("inf")))
    at = int(over.argmax())
    assert float(over.max()) <= 0, "%s: off by %.3e of %.3e, %.3e allowed, at %d" % (
        what, float((got - value).abs().flatten()[at]), float(value.flatten()[at]), float(bound.expand(value.shape).flatten()[at]), at)
