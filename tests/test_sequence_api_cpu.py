"""Argument contract of the sequence operators, checked without a GPU: every case fails or returns before any
native compute call; the frequencies against their formulas; the oracle against its own definition."""
import ctypes
import inspect
import math

import numpy as np
import pytest
import torch

import pysiglib_b200 as psl
import sequence_oracle as so
from pysiglib_b200 import load_cusig, torch_api

X, G, S = np.zeros((2, 5, 6), np.float32), np.zeros((2, 5, 3), np.float32), np.zeros((2, 6), np.float32)


def test_signatures():
    assert list(inspect.signature(psl.linear_recurrence).parameters) == [
        "x", "gate", "initial", "gate_form", "complement", "offsets", "return_state", "return_checkpoints"]
    assert list(inspect.signature(psl.linear_recurrence_backprop).parameters) == [
        "derivs", "x", "gate", "initial", "gate_form", "complement", "offsets", "state_derivs", "checkpoints"]
    assert list(inspect.signature(psl.linear_recurrence_step).parameters) == ["x", "gate", "state", "gate_form", "complement"]
    for name in ("rotary", "rotary_backprop"):
        assert list(inspect.signature(getattr(psl, name)).parameters)[1:] == ["frequencies", "positions", "interleaved", "scale", "inverse"]
    for name in ("linear_recurrence", "rotary"):
        assert list(inspect.signature(getattr(torch_api, name)).parameters) == list(inspect.signature(getattr(psl, name)).parameters)
        assert getattr(torch_api, name).__doc__ == getattr(psl, name).__doc__
        assert not hasattr(torch_api, name + "_backprop")


@pytest.mark.parametrize("error,message,args,kw", [
    (TypeError, "x must be of type", ([[0.0]], G), {}),
    (TypeError, "x.dtype", (X.astype(np.int32), G), {}),
    (TypeError, "gate.dtype", (X, G.astype(np.float64)), {}),
    (TypeError, "gate.dtype", (X.astype(np.float64), G), {}),
    (TypeError, "gate.dtype", (X.astype(np.float16), G.astype(np.float64)), {}),
    (ValueError, "rank 2", (np.zeros(6, np.float32), np.zeros(3, np.float32)), {}),
    (ValueError, "0 channels", (np.zeros((5, 0), np.float32), np.zeros((5, 1), np.float32)), {}),
    (ValueError, "gate must have shape", (X, np.zeros((2, 5, 4), np.float32)), {}),
    (ValueError, "gate must have shape", (X, np.zeros((2, 5, 0), np.float32)), {}),
    (ValueError, "gate must have shape", (X, np.zeros((2, 4, 3), np.float32)), {}),
    (ValueError, "gate must have shape", (X, np.zeros((5, 3), np.float32)), {}),
    (ValueError, "both be numpy", (X, torch.zeros(2, 5, 3)), {}),
    (ValueError, "initial must have shape", (X, G, S[:1]), {}),
    (TypeError, "initial.dtype", (X, G, S.astype(np.float64)), {}),
    (TypeError, "initial.dtype", (X.astype(np.float16), G, S.astype(np.float16)), {}),
    (ValueError, "gate_form must be", (X, G), {"gate_form": "sigmoid"}),
    (TypeError, "gate_form", (X, G), {"gate_form": 1}),
    (TypeError, "complement", (X, G), {"complement": 1}),
    (ValueError, "offsets", (X, G), {"offsets": np.array([0, 5])}),
    (ValueError, "at least 2 values", (X[0], G[0]), {"offsets": np.array([0])}),
    (TypeError, "offsets.dtype", (X[0], G[0]), {"offsets": np.array([0.0, 5.0])}),
    (ValueError, "must not decrease", (X[0], G[0]), {"offsets": np.array([0, 3, 2, 5])}),
    (ValueError, "must not decrease", (X[0], G[0]), {"offsets": np.array([0, 6])}),
    (ValueError, "must not decrease", (X[0], G[0]), {"offsets": np.array([-1, 5])}),
    (ValueError, "initial must have shape", (X[0], G[0], S), {"offsets": np.array([0, 2, 4, 5])}),
])
def test_recurrence_refusals(error, message, args, kw):
    with pytest.raises(error, match=message):
        psl.linear_recurrence(*args, **kw)
    x, gate, *rest = args
    with pytest.raises(error, match=message):
        psl.linear_recurrence_backprop(x, x, gate, *rest, **kw)


def test_backprop_and_step_refusals():
    with pytest.raises(ValueError, match="derivs must have the shape"):
        psl.linear_recurrence_backprop(X[:1], X, G)
    with pytest.raises(TypeError, match="derivs.dtype"):
        psl.linear_recurrence_backprop(X.astype(np.float64), X, G)
    with pytest.raises(ValueError, match="checkpoints must have shape"):
        psl.linear_recurrence_backprop(X, X, G, checkpoints=np.zeros((2, 2, 6), np.float32))
    with pytest.raises(ValueError, match="state_derivs must have shape"):
        psl.linear_recurrence_backprop(X, X, G, state_derivs=S[:1])
    for bad, error, message in ((S.astype(np.float64), TypeError, "state.dtype"), (S[:1], ValueError, "shape of x"),
                                (np.zeros((6, 2), np.float32).T, ValueError, "contiguous")):
        with pytest.raises(error, match=message):
            psl.linear_recurrence_step(X[:, 0], G[:, 0], bad)
    with pytest.raises(ValueError, match="require a gradient"):
        psl.linear_recurrence_step(torch.zeros(2, 6), torch.zeros(2, 3), torch.zeros(2, 6, requires_grad=True))
    with pytest.raises(ValueError, match="gate must have shape"):
        psl.linear_recurrence_step(X[:, 0], G, S)
    with pytest.raises(ValueError, match="checkpoints are kept"):
        torch_api.linear_recurrence(torch.zeros(2, 5, 6, requires_grad=True), torch.zeros(2, 5, 6), return_checkpoints=True)


def test_recurrence_without_rows():
    for shape, gates in (((0, 5, 6), (0, 5, 3)), ((2, 0, 6), (2, 0, 6))):
        x, g = np.zeros(shape, np.float32), np.zeros(gates, np.float32)
        start = np.arange(shape[0] * 6, dtype=np.float32).reshape(shape[0], 6)
        h, state, marks = psl.linear_recurrence(x, g, start, return_state=True, return_checkpoints=True)
        assert h.shape == shape and marks.shape == (shape[0], -(-shape[1] // 16), 6)
        np.testing.assert_array_equal(state, start)
        dx, dg, ds = psl.linear_recurrence_backprop(x, x, g, start, state_derivs=start + 1, checkpoints=marks)
        assert dx.shape == shape and dg.shape == gates
        np.testing.assert_array_equal(ds, start + 1)
    h, state = psl.linear_recurrence(np.zeros((0, 4)), np.zeros((0, 4)), offsets=np.array([0, 0, 0]), return_state=True)
    assert h.shape == (0, 4) and (state == np.zeros((2, 4))).all()
    assert psl.linear_recurrence_step(np.zeros((0, 4)), np.zeros((0, 4)), np.zeros((0, 4))).shape == (0, 4)


@pytest.mark.parametrize("error,message,args,kw", [
    (TypeError, "x must be of type", ([1.0], np.zeros(1)), {}),
    (ValueError, "rank 2", (np.zeros(4), np.zeros(1)), {}),
    (TypeError, "frequencies.dtype", (X, np.zeros(3, np.float32)), {}),
    (ValueError, "pairs of channels", (X, np.zeros(4)), {}),
    (ValueError, "pairs of channels", (X, np.zeros((1, 3))), {}),
    (ValueError, "both be numpy", (X, torch.zeros(3, dtype=torch.float64)), {}),
    (TypeError, "positions.dtype", (X, np.zeros(3), np.zeros(5, np.int16)), {}),
    (ValueError, "broadcast", (X, np.zeros(3), np.arange(4)), {}),
    (ValueError, "broadcast", (X, np.zeros(3), np.zeros((1, 2, 5))), {}),
    (TypeError, "scale", (X, np.zeros(3)), {"scale": 1}),
    (TypeError, "interleaved", (X, np.zeros(3)), {"interleaved": 1}),
    (TypeError, "inverse", (X, np.zeros(3)), {"inverse": 1}),
])
def test_rotary_refusals(error, message, args, kw):
    with pytest.raises(error, match=message):
        psl.rotary(*args, **kw)
    with pytest.raises(error, match=message.replace("x must", "derivs must")):
        psl.rotary_backprop(*args, **kw)


def test_rotary_has_gradients_for_x_only():
    x = torch.zeros(4, 6, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient with respect to frequencies"):
        torch_api.rotary(x, torch.zeros(3, dtype=torch.float64, requires_grad=True))
    with pytest.raises(ValueError, match="no gradient with respect to positions"):
        torch_api.rotary(x, torch.zeros(3, dtype=torch.float64), torch.zeros(4, requires_grad=True))
    assert psl.rotary(np.zeros((0, 5, 6)), np.zeros(3)).shape == (0, 5, 6)
    assert psl.rotary(np.zeros((2, 0, 6)), np.zeros(3), np.zeros((2, 0))).shape == (2, 0, 6)


def test_frequencies():
    f = psl.rotary_frequencies(8, base=100.0)
    np.testing.assert_allclose(f, [1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], rtol=1e-15)
    np.testing.assert_allclose(psl.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0), f / 4, rtol=1e-15)
    stretched = psl.rotary_frequencies(8, base=100.0, scaling="base", factor=4.0)
    np.testing.assert_allclose(stretched[[0, -1]], [f[0], f[-1] / 4], rtol=1e-14)
    parts = psl.rotary_frequencies(64, scaling="parts", factor=8.0, original_length=2048)
    plain = psl.rotary_frequencies(64)
    turns = 2048 * plain / (2 * math.pi)
    np.testing.assert_array_equal(parts[turns >= 32], plain[turns >= 32])
    np.testing.assert_allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    assert ((np.diff(parts) < 0).all() and (turns >= 32).any() and (turns <= 1).any())
    assert psl.rotary_frequencies(0).shape == (0,) and psl.rotary_frequencies(2, scaling="base", factor=2.0).tolist() == [1.0]
    for error, args, kw in ((ValueError, (7,), {}), (ValueError, (8,), {"scaling": "ntk"}), (TypeError, (8,), {"base": 10}),
                            (ValueError, (8,), {"factor": 0.0}), (ValueError, (8,), {"fast_turns": 1.0}), (TypeError, (8.0,), {}),
                            (ValueError, (8,), {"original_length": 0})):
        with pytest.raises(error):
            psl.rotary_frequencies(*args, **kw)


def test_native_entry_points_refuse_without_a_gpu():
    """Calls that the C entry points turn down before they look for a device."""
    lib = load_cusig.library()
    buffer = (ctypes.c_double * 64)()
    p = ctypes.addressof(buffer)

    def recurrence(type=0, gate_type=0, x=p, gate=p, offsets=None, out=p, batch=2, rows=4, dim=4, gates=4, sequences=0, form=0):
        return lib.sigb200_linear_recurrence(type, gate_type, x, gate, None, offsets, out, None, None, batch, rows, dim, gates,
                                             sequences, rows * dim, dim, rows * gates, gates, form, False, True, -1, None, 1)
    for kw in ({"type": 4}, {"type": -1}, {"gate_type": 1}, {"type": 1, "gate_type": 0}, {"gates": 3}, {"gates": 0}, {"dim": 0},
               {"form": 3}, {"x": None}, {"gate": None}, {"out": None}, {"sequences": 1}, {"sequences": 1, "offsets": p}):
        assert recurrence(**kw) == 2, (kw, load_cusig.last_error_message())
        assert "linear_recurrence" in load_cusig.last_error_message()
    assert recurrence(batch=1 << 40, rows=1 << 20) == 3 and recurrence(rows=1 << 30) == 3
    assert recurrence(batch=0) == 0 and recurrence(rows=0) == 0

    def rotary(type=0, kind=0, x=p, f=p, positions=None, out=p, rows=4, dim=4, part=4):
        freq = ctypes.cast(f, ctypes.POINTER(ctypes.c_double)) if f else None
        return lib.sigb200_rotary(type, kind, x, f, positions, out, 1, 1, rows, dim, part, 0, 0, dim, 0, 0, dim, 0, 0, 1,
                                  False, False, 1.0, -1, None, 1)
    for kw in ({"type": 9}, {"kind": 5}, {"part": 3}, {"part": 6}, {"x": None}, {"f": None}, {"out": None}, {"kind": 2}):
        assert rotary(**kw) == 2, (kw, load_cusig.last_error_message())
    assert rotary(rows=0) == 0


@pytest.mark.parametrize("form", ["value", "log", "logit"])
def test_the_oracle_is_the_definition(form):
    """The row-by-row oracle against torch's autograd of the written-out recurrence, in float64."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 6, generator=g, dtype=torch.float64, requires_grad=True)
    gate = (-torch.rand(7, 3, generator=g, dtype=torch.float64)).requires_grad_()
    start = torch.randn(3, 6, generator=g, dtype=torch.float64, requires_grad=True)
    d, tail = torch.randn(7, 6, generator=g, dtype=torch.float64), torch.randn(3, 6, generator=g, dtype=torch.float64)
    offsets = torch.tensor([1, 4, 4, 7])
    a = {"value": lambda v: v, "log": torch.exp, "logit": torch.sigmoid}[form](gate).repeat_interleave(2, -1)
    rows, states = [x[0] * 0], []
    for k, (lo, hi) in enumerate(so.spans_of(offsets, 7)):
        now = start[k]
        for t in range(lo, hi):
            now = a[t] * now + (1 - a[t]) * x[t]
            rows.append(now)
        states.append(now)
    h, state = torch.stack(rows), torch.stack(states)
    grads = torch.autograd.grad((h * d).sum() + (state * tail).sum(), (x, gate, start))
    got = so.recurrence(x.detach(), gate.detach(), start.detach(), form, True, offsets, d, tail)
    for name, want in zip(("h", "state", "dx", "dgate", "dinitial"), (h, state, *grads)):
        torch.testing.assert_close(got[name][0], want.detach(), rtol=1e-12, atol=1e-12)


def test_autograd_asks_for_what_somebody_reads(monkeypatch):
    """Checkpoints only where a gradient may be asked for, the state there or where the caller wants it."""
    import sys
    module = sys.modules[torch_api.linear_recurrence.__module__]
    asked = []

    def forward(x, gate, initial=None, *, return_state, return_checkpoints, **how):
        asked.append((return_state, return_checkpoints))
        parts = [x * 1.0] + [x[:, -1] * 1.0] * return_state + [x[:, :1] * 1.0] * return_checkpoints
        return tuple(parts) if len(parts) > 1 else parts[0]
    monkeypatch.setattr(module, "linear_recurrence_forward", forward)
    x, gate, leaf = torch.zeros(2, 5, 6), torch.zeros(2, 5, 6), torch.zeros(2, 5, 6, requires_grad=True)
    for return_state in (False, True):
        for args, keep in (((x, gate), False), ((leaf, gate), True), ((x, leaf), True), ((x, gate, leaf[:, 0]), True)):
            for grad_mode in (True, False):
                with torch.set_grad_enabled(grad_mode):
                    out = torch_api.linear_recurrence(*args, return_state=return_state)
                assert asked.pop() == (return_state, keep and grad_mode)
                h = out[0] if return_state else out
                assert h.requires_grad == (keep and grad_mode) and (not return_state or out[1].shape == (2, 6))


def test_a_step_does_not_drop_a_gradient_unseen():
    x, gate, state = torch.zeros(0, 6), torch.zeros(0, 3), torch.zeros(0, 6)
    for args in ((x.clone().requires_grad_(), gate), (x, gate.clone().requires_grad_())):
        with pytest.raises(ValueError, match="a step has no gradient"):
            psl.linear_recurrence_step(*args, state)
        with torch.no_grad():
            assert psl.linear_recurrence_step(*args, state).shape == (0, 6)
        assert psl.linear_recurrence_step(*(t.detach() for t in args), state).shape == (0, 6)
