"""Rotary positions: ``rotary``, its adjoint, and the frequencies it turns by.

``transform_path(time_aug=True)`` adds time to a path as one more channel; ``rotary`` works it into the
channels there are, by turning pairs of them at the angle ``position * frequency``.  Around
``linear_recurrence`` it makes a bank of damped oscillators: turned by ``-p_t w`` before the scan and by
``+p_t w`` after it, ``h_t = a_t R(w (p_t - p_{t-1})) h_{t-1} + x_t``, at the time stamps of the path.
No counterpart in the reference."""
import math
from math import prod
from typing import Union

import numpy as np
import torch

from .param_checks import check_type
from .sequence_inputs import TORCH_TYPES, call, check_like, contiguous, element_type, empty, pointer, raw_stream

POSITION_TYPES = {torch.int32: 1, torch.int64: 2, torch.float32: 3, torch.float64: 4, np.dtype(np.int32): 1,
                  np.dtype(np.int64): 2, np.dtype(np.float32): 3, np.dtype(np.float64): 4}


def rotary_frequencies(
        rotary_dimension: int,
        *,
        base: float = 10000.,
        scaling: str = "none",
        factor: float = 1.,
        original_length: int = 4096,
        slow_turns: float = 1.,
        fast_turns: float = 32.
) -> np.ndarray:
    """Frequencies ``base ** (-2 i / rotary_dimension)``, in radians for each unit of position, as a float64
    array of ``rotary_dimension / 2`` values; for contexts ``factor`` times as long as ``original_length``:

    * ``scaling="linear"`` divides all frequencies by ``factor`` (positions are interpolated);
    * ``scaling="base"`` raises the base to ``base * factor ** (r / (r - 2))``: the fastest pair keeps its
      frequency and the slowest one's is divided by ``factor``;
    * ``scaling="parts"`` keeps the pairs that turn at least ``fast_turns`` times in ``original_length``,
      divides by ``factor`` those that turn at most ``slow_turns`` times, and blends linearly in the
      number of turns between.

    Move it to the device once (``torch.from_numpy(f).cuda()``) and keep it with the model's weights.
    """
    check_type(rotary_dimension, "rotary_dimension", int)
    for value, name in ((base, "base"), (factor, "factor"), (slow_turns, "slow_turns"), (fast_turns, "fast_turns")):
        check_type(value, name, float)
    check_type(original_length, "original_length", int)
    check_type(scaling, "scaling", str)
    if rotary_dimension < 0 or rotary_dimension % 2:
        raise ValueError("rotary_dimension must be an even non-negative integer, got %d" % rotary_dimension)
    if scaling not in ("none", "linear", "base", "parts"):
        raise ValueError("scaling must be one of 'none', 'linear', 'base' or 'parts', got %r" % scaling)
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError("base and factor must be positive")
    if original_length <= 0 or not 0 <= slow_turns < fast_turns:
        raise ValueError("original_length must be positive and slow_turns below fast_turns")
    half = rotary_dimension // 2
    if scaling == "base" and half > 1:
        base = base * factor ** (rotary_dimension / (rotary_dimension - 2))
    f = base ** (-np.arange(half, dtype=np.float64) / max(half, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        turns = original_length * f / (2 * math.pi)
        kept = np.clip((turns - slow_turns) / (fast_turns - slow_turns), 0.0, 1.0)
        f = f * (kept + (1 - kept) / factor)
    return f


def _common_axes(shape, strides):
    """``(n0, n1)`` and, for each array, its strides ``(outer, inner, row)``, with the lead axes of ``shape`` (lead
    axes, rows, dimension) read as the same two axes of all arrays; None where that cannot be."""
    lead = len(shape) - 2
    if lead == 2:
        return shape[0], shape[1], strides
    if lead == 1:
        return 1, shape[0], [(0, *s) for s in strides]
    if lead == 0:
        return 1, 1, [(0, 0, *s) for s in strides]
    merged = []
    for i in range(lead):
        n = shape[i]
        if n == 1:
            continue
        now = [s[i] for s in strides]
        if merged and all(outer == n * inner for outer, inner in zip(merged[-1][1], now)):
            merged[-1] = (merged[-1][0] * n, now)
        else:
            merged.append((n, now))
    if len(merged) > 2:
        return None
    none = (1, [0] * len(strides))
    n0, outer = merged[0] if len(merged) == 2 else none
    n1, inner = merged[-1] if merged else none
    return n0, n1, [(o, i, s[lead]) for o, i, s in zip(outer, inner, strides)]


def _position_strides(positions, lead):
    """Strides along the axes ``lead`` of an array that broadcasts to them."""
    strides = positions.stride()
    if positions.shape == lead:
        return strides
    return (0,) * (len(lead) - len(strides)) + tuple([0 if n == 1 else s for n, s in zip(positions.shape, strides)])


def _rotate(x, frequencies, positions, interleaved, scale, inverse, name):
    on_device = isinstance(x, torch.Tensor) and x.is_cuda
    code = TORCH_TYPES.get(x.dtype) if on_device else None
    if code is None:
        code = element_type(x, name)
    if not (on_device and isinstance(frequencies, torch.Tensor) and frequencies.device == x.device):
        check_like(frequencies, "frequencies", x, name)
    if interleaved is not True and interleaved is not False:
        check_type(interleaved, "interleaved", bool)
    if inverse is not True and inverse is not False:
        check_type(inverse, "inverse", bool)
    if not isinstance(scale, float):
        check_type(scale, "scale", float)
    shape = x.shape
    if len(shape) < 2:
        raise ValueError("%s must have at least rank 2, got rank %d." % (name, len(shape)))
    if POSITION_TYPES.get(frequencies.dtype) != 4:
        raise TypeError("frequencies.dtype must be float64, got %s instead" % frequencies.dtype)
    if len(frequencies.shape) != 1 or 2 * frequencies.shape[0] > shape[-1]:
        raise ValueError("frequencies must be one value for each of at most %d pairs of channels, got shape %s"
                         % (shape[-1] // 2, tuple(frequencies.shape)))
    lead, kind = shape[:-1], 0
    if positions is not None:
        if not (on_device and isinstance(positions, torch.Tensor) and positions.device == x.device):
            check_like(positions, "positions", x, name)
        kind = POSITION_TYPES.get(positions.dtype)
        if kind is None:
            raise TypeError("positions.dtype must be int32, int64, float32 or float64, got %s instead" % positions.dtype)
        tail = positions.shape
        if tail != lead and (len(tail) < 1 or len(tail) > len(lead) or
                             any(p != 1 and p != n for p, n in zip(tail, lead[len(lead) - len(tail):]))):
            raise ValueError("positions must broadcast to %s, got %s" % (tuple(lead), tuple(tail)))
    frequencies = contiguous(frequencies)
    rows, dim = shape[-2], shape[-1]
    if on_device:
        if x.stride(-1) != 1 and dim != 1:
            x = x.contiguous()
        out = torch.empty_like(x)
        if out.stride(-1) != 1 and dim != 1:
            out = x.new_empty(shape)
        p = (0,) * len(lead) if positions is None else _position_strides(positions, lead)
        views = _common_axes(shape, [x.stride()[:-1], out.stride()[:-1], p])
        if views is None:  # lead axes that no two strides describe
            x = x.contiguous()
            out = x.new_empty(shape)
            if positions is not None:
                positions = positions.expand(lead).contiguous()
                p = positions.stride()
            views = _common_axes(shape, [x.stride()[:-1], out.stride()[:-1], p])
        n0, n1, ((x0, x1, x_row), (y0, y1, y_row), (p0, p1, p_row)) = views
        if out.numel():
            device = x.get_device()
            call("rotary", code, kind, x.data_ptr(), frequencies.data_ptr(), positions.data_ptr() if kind else None, out.data_ptr(),
                 n0, n1, rows, dim, 2 * frequencies.shape[0], x0, x1, x_row, y0, y1, y_row, p0, p1, p_row, interleaved, inverse, scale,
                 device, raw_stream(device), 0)
        return out
    x = contiguous(x)
    out = empty(x, shape, x.dtype)
    if positions is not None:
        positions = (positions.expand(lead).contiguous() if isinstance(positions, torch.Tensor) else
                     np.ascontiguousarray(np.broadcast_to(positions, lead)))
    if 0 not in shape:
        call("rotary", code, kind, pointer(x), pointer(frequencies), pointer(positions), pointer(out), 1, prod(shape[:-2]), rows,
             dim, 2 * frequencies.shape[0], 0, rows * dim, dim, 0, rows * dim, dim, 0, rows, 1, interleaved, inverse, scale, -1,
             None, 0)
    return out


def rotary(
        x: Union[np.ndarray, torch.Tensor],
        frequencies: Union[np.ndarray, torch.Tensor],
        positions: Union[np.ndarray, torch.Tensor, None] = None,
        *,
        interleaved: bool = False,
        scale: float = 1.,
        inverse: bool = False
) -> Union[np.ndarray, torch.Tensor]:
    """Turns pairs of channels of every row by ``position * frequency``.

    :param x: ``(..., length, dimension)`` of type float32, float64, float16 or bfloat16; heads are leading
        axes (``(batch, heads, length, dimension)``, where a view of ``(batch, length, heads, dimension)``
        serves as well: CUDA views with adjacent channels are read in place, and dense ones give a
        result of the same strides).  CUDA tensors are processed on the current stream of their device,
        without waiting for the result.
    :param frequencies: float64, one for each pair, in radians for each unit of position (see
        ``rotary_frequencies``), on the device of ``x``.  ``2 * len(frequencies)`` channels are turned, the
        others are copied.
    :param positions: int32, int64, float32 or float64 (time stamps) values that broadcast to
        ``x.shape[:-1]``; the row index if absent.  Angles are formed in 64 bits.
    :param interleaved: pair the channels ``(2i, 2i + 1)``; else ``(i, i + len(frequencies))``.
    :param scale: factor on the turned channels.
    :param inverse: turn the other way.
    :return: array of the kind, shape, type and device of ``x``.

    Example::

        f = torch.from_numpy(pysiglib_b200.rotary_frequencies(64)).cuda()
        q = pysiglib_b200.rotary(torch.randn(4, 8, 1000, 64, device="cuda"), f)
    """
    return _rotate(x, frequencies, positions, interleaved, scale, inverse, "x")


def rotary_backprop(
        derivs: Union[np.ndarray, torch.Tensor],
        frequencies: Union[np.ndarray, torch.Tensor],
        positions: Union[np.ndarray, torch.Tensor, None] = None,
        *,
        interleaved: bool = False,
        scale: float = 1.,
        inverse: bool = False
) -> Union[np.ndarray, torch.Tensor]:
    """Backward pass of ``rotary``: derivatives with respect to its result in, with respect to ``x`` out (the
    turn the other way, times ``scale``).  Positions and frequencies get no gradient."""
    check_type(inverse, "inverse", bool)
    return _rotate(derivs, frequencies, positions, interleaved, scale, not inverse, "derivs")
