"""Gated linear recurrences along paths: ``linear_recurrence``, its backward pass and its single-row step.

``h_t = a_t h_{t-1} + b_t`` for every channel: a learned memory of a sequence, computed by a parallel scan.
No counterpart in the reference; the conventions (paths ``(..., length, dimension)``, ``*_backprop``, NumPy
or torch) are those of the signature operators."""
from math import prod
from typing import Union

import numpy as np
import torch

from .param_checks import check_type
from .sequence_inputs import (TORCH_TYPES, batched_rows, call, check_like, check_state, contiguous, element_type, empty,
                              on_device, place_of, pointer, raw_stream, state_dtype)

GATE_FORMS = {"value": 0, "log": 1, "logit": 2}
CHECKPOINT_ROWS = 16  # rows between two of the states kept for the backward pass


def _check_gate(x, gate, gate_form, complement):
    """``(element type, gate type, gate form, gates)`` of inputs ``(..., dimension)`` and gates ``(..., G)``."""
    if isinstance(x, torch.Tensor) and isinstance(gate, torch.Tensor) and x.device == gate.device:
        code, gate_code = TORCH_TYPES.get(x.dtype), TORCH_TYPES.get(gate.dtype)
    else:
        code = gate_code = None
    if code is None or gate_code is None:
        code, gate_code = element_type(x, "x"), element_type(gate, "gate")
        check_like(gate, "gate", x, "x")
    if gate_code != code and not (gate_code == 0 and code >= 2):
        raise TypeError("gate.dtype must be that of x, or float32 for 16-bit x; got %s for %s" % (gate.dtype, x.dtype))
    form = GATE_FORMS.get(gate_form) if isinstance(gate_form, str) else None
    if form is None:
        check_type(gate_form, "gate_form", str)
        raise ValueError("gate_form must be one of 'value', 'log' or 'logit', got %r" % gate_form)
    if complement is not True and complement is not False:
        check_type(complement, "complement", bool)
    return code, gate_code, form


def _check_gate_shape(shape, gate_shape):
    dim, gates = shape[-1], gate_shape[-1] if len(gate_shape) else 0
    if dim == 0:
        raise ValueError("x has 0 channels (dimension). Its dimension must be at least 1.")
    if gate_shape[:-1] != shape[:-1] or gates == 0 or dim % gates:
        raise ValueError("gate must have shape %s + (G,) with G dividing %d, got %s" % (tuple(shape[:-1]), dim, tuple(gate_shape)))
    return dim, gates


class _Recurrence:
    """Checked and flattened arguments of one call."""

    def __init__(self, x, gate, initial, gate_form, complement, offsets):
        self.type, self.gate_type, self.form = _check_gate(x, gate, gate_form, complement)
        self.complement = complement
        shape = x.shape
        if len(shape) < 2:
            raise ValueError("x must have at least rank 2, got rank %d." % len(shape))
        self.dim, self.gates = _check_gate_shape(shape, gate.shape)
        self.rows, lead = shape[-2], shape[:-2]
        self.batch = prod(lead)
        self.offsets, self.wide, self.sequences = None, False, 0
        if offsets is None:
            self.state_shape = (*lead, self.dim)
        else:
            self._set_offsets(offsets, x)
        self.initial = check_state(initial, "initial", self.state_shape, x)
        self.x, self.x_batch, self.x_row = batched_rows(x)
        self.gate, self.gate_batch, self.gate_row = batched_rows(gate)
        self.marks_shape = (*lead, -(-self.rows // CHECKPOINT_ROWS), self.dim)
        self.empty = self.batch == 0 or self.rows == 0

    def _set_offsets(self, offsets, x):
        check_type(offsets, "offsets", (np.ndarray, torch.Tensor))
        if len(x.shape) != 2:
            raise ValueError("packed sequences (offsets) need x of shape (rows, dimension), got %s" % (tuple(x.shape),))
        if len(offsets.shape) != 1 or offsets.shape[0] < 2:
            raise ValueError("offsets must be one row of at least 2 values, got shape %s" % (tuple(offsets.shape),))
        self.wide = offsets.dtype == (torch.int64 if isinstance(offsets, torch.Tensor) else np.int64)
        if not self.wide and offsets.dtype != (torch.int32 if isinstance(offsets, torch.Tensor) else np.int32):
            raise TypeError("offsets.dtype must be int32 or int64, got %s instead" % offsets.dtype)
        if not on_device(offsets):
            values = np.asarray(offsets).astype(np.int64)
            if values[0] < 0 or values[-1] > self.rows or (np.diff(values) < 0).any():
                raise ValueError("offsets must not decrease and must lie between 0 and %d" % self.rows)
        if isinstance(x, torch.Tensor):
            if on_device(offsets):
                check_like(offsets, "offsets", x, "x")
            else:
                offsets = torch.as_tensor(offsets).to(x.device)
        elif not isinstance(offsets, np.ndarray):
            check_like(offsets, "offsets", x, "x")
        self.offsets = contiguous(offsets)
        self.sequences = offsets.shape[0] - 1
        self.state_shape = (self.sequences, self.dim)

    def tail(self, x):
        return self.form, self.complement, self.wide, *place_of(x), 0


def linear_recurrence(
        x: Union[np.ndarray, torch.Tensor],
        gate: Union[np.ndarray, torch.Tensor],
        initial: Union[np.ndarray, torch.Tensor, None] = None,
        *,
        gate_form: str = "value",
        complement: bool = False,
        offsets: Union[np.ndarray, torch.Tensor, None] = None,
        return_state: bool = False,
        return_checkpoints: bool = False
):
    """Gated linear recurrence ``h_t = a_t h_{t-1} + b_t`` along axis -2, channel by channel.

    :param x: inputs ``(..., length, dimension)`` of type float32, float64, float16 or bfloat16, fewer than
        2^30 rows long.  CUDA
        tensors are processed on their device and on its current stream, without waiting for the
        result; views with adjacent channels are read in place.  NumPy arrays and CPU tensors go
        through the current CUDA device.
    :param gate: ``(..., length, G)`` with ``G`` dividing ``dimension``: gate ``g`` serves the channels
        ``g * dimension / G`` up to the next gate's.  Its type is that of ``x``, or float32 for 16-bit ``x``.
    :param initial: state before the first row, ``(..., dimension)``, float64 for float64 ``x``, else
        float32; 0 if absent.
    :param gate_form: how ``a`` comes from ``gate``: ``"value"`` a = gate, ``"log"`` a = exp(gate),
        ``"logit"`` a = 1 / (1 + exp(-gate)).
    :param complement: ``b_t = (1 - a_t) x_t`` instead of ``b_t = x_t``.
    :param offsets: packed sequences: ``x`` is ``(rows, dimension)`` and sequence ``i`` holds the rows
        ``offsets[i]`` to ``offsets[i + 1] - 1`` (int32 or int64, ``n + 1`` values that do not decrease).
        Sequences may be empty; rows of no sequence come out as 0.  ``initial`` and the state are
        ``(n, dimension)``.  Values on the host are checked and copied to the device, which waits for the
        copy and cannot be captured; those on the device are trusted: wrong ones give wrong numbers.
    :param return_state: also return the state after the last row (``initial`` for an empty sequence),
        ready for ``linear_recurrence_step``.
    :param return_checkpoints: also return the states before rows 0, 16, 32, .., which
        ``linear_recurrence_backprop`` would otherwise compute again.
    :return: ``h`` like ``x`` (contiguous), or a tuple ``(h, state, checkpoints)`` without the parts not
        asked for.

    States and sums are held in float32 (float64 for float64 ``x``); ``h`` is rounded once, on its way out.
    The scan multiplies the gates of neighbouring rows: where such a product leaves the range of the
    state's type (gates well above 1 over many rows) the result is not finite.

    Example::

        import torch, pysiglib_b200 as psl
        x, g = torch.randn(8, 1000, 64, device="cuda"), torch.randn(8, 1000, 64, device="cuda")
        h, state = psl.linear_recurrence(x, g, gate_form="logit", complement=True, return_state=True)
        y = psl.linear_recurrence_step(x[:, 0], g[:, 0], state, gate_form="logit", complement=True)
    """
    check_type(return_state, "return_state", bool)
    check_type(return_checkpoints, "return_checkpoints", bool)
    r = _Recurrence(x, gate, initial, gate_form, complement, offsets)
    h = empty(x, x.shape, x.dtype)
    wide = state_dtype(x)
    state = empty(x, r.state_shape, wide) if return_state else None
    marks = empty(x, r.marks_shape, wide) if return_checkpoints else None
    if r.empty:
        if return_state:
            state[...] = 0 if r.initial is None else r.initial
    else:
        call("linear_recurrence", r.type, r.gate_type, pointer(r.x), pointer(r.gate), pointer(r.initial),
             pointer(r.offsets), pointer(h), pointer(state), pointer(marks), r.batch, r.rows, r.dim, r.gates,
             r.sequences, r.x_batch, r.x_row, r.gate_batch, r.gate_row, *r.tail(x))
    if return_state:
        return (h, state, marks) if return_checkpoints else (h, state)
    return (h, marks) if return_checkpoints else h


def linear_recurrence_backprop(
        derivs: Union[np.ndarray, torch.Tensor],
        x: Union[np.ndarray, torch.Tensor],
        gate: Union[np.ndarray, torch.Tensor],
        initial: Union[np.ndarray, torch.Tensor, None] = None,
        *,
        gate_form: str = "value",
        complement: bool = False,
        offsets: Union[np.ndarray, torch.Tensor, None] = None,
        state_derivs: Union[np.ndarray, torch.Tensor, None] = None,
        checkpoints: Union[np.ndarray, torch.Tensor, None] = None
):
    """Backward pass of ``linear_recurrence``: from ``dF/dh`` to ``(dF/dx, dF/dgate, dF/dinitial)``.

    :param derivs: derivatives with respect to ``h``, of the shape and type of ``x``.
    :param state_derivs: derivatives with respect to the final state, of its shape and type.
    :param checkpoints: those that ``linear_recurrence`` returned for the same inputs; without them a pass
        over ``x`` and ``gate`` computes them again.
    :return: gradients in the shapes and types of ``x``, ``gate`` and ``initial`` (``None`` without an
        ``initial``); rows of no sequence get 0.

    The other parameters are those of ``linear_recurrence``.  Results do not depend on the order in
    which threads finish: the same call gives the same bits.
    """
    r = _Recurrence(x, gate, initial, gate_form, complement, offsets)
    check_like(derivs, "derivs", x, "x")
    if derivs.dtype != x.dtype:
        raise TypeError("derivs.dtype must be that of x, got %s for %s" % (derivs.dtype, x.dtype))
    if derivs.shape != x.shape:
        raise ValueError("derivs must have the shape of x, %s, got %s" % (tuple(x.shape), tuple(derivs.shape)))
    state_derivs = check_state(state_derivs, "state_derivs", r.state_shape, x)
    checkpoints = check_state(checkpoints, "checkpoints", r.marks_shape, x)
    d, d_batch, d_row = batched_rows(derivs)
    dx, dgate = empty(x, x.shape, x.dtype), empty(gate, gate.shape, gate.dtype)
    dinitial = None if initial is None else empty(x, r.state_shape, state_dtype(x))
    if r.empty:
        if dinitial is not None:
            dinitial[...] = 0 if state_derivs is None else state_derivs
        return dx, dgate, dinitial
    call("linear_recurrence_backprop", r.type, r.gate_type, pointer(d), pointer(r.x), pointer(r.gate),
         pointer(r.initial), pointer(r.offsets), pointer(state_derivs), pointer(checkpoints), pointer(dx),
         pointer(dgate), pointer(dinitial), r.batch, r.rows, r.dim, r.gates, r.sequences, d_batch, d_row, r.x_batch,
         r.x_row, r.gate_batch, r.gate_row, *r.tail(x))
    return dx, dgate, dinitial


def linear_recurrence_step(
        x: Union[np.ndarray, torch.Tensor],
        gate: Union[np.ndarray, torch.Tensor],
        state: Union[np.ndarray, torch.Tensor],
        *,
        gate_form: str = "value",
        complement: bool = False
) -> Union[np.ndarray, torch.Tensor]:
    """One more row for each of a batch of recurrences: ``state`` becomes ``a state + b``.

    :param x: the new rows, ``(..., dimension)``.
    :param gate: their gates, ``(..., G)`` as in ``linear_recurrence``.
    :param state: ``(..., dimension)``, contiguous, float64 for float64 ``x``, else float32.  Overwritten; shares
        no memory with ``x`` and ``gate``.
    :return: the new state in the type of ``x``.

    No gradient passes through a step: with gradients enabled, inputs that require one are refused.

    Stepping through a sequence gives what ``linear_recurrence`` gives for it, up to rounding.
    """
    code, gate_code, form = _check_gate(x, gate, gate_form, complement)
    if not isinstance(state, torch.Tensor) or state.device != getattr(x, "device", None):
        check_like(state, "state", x, "x")
    shape = x.shape
    if len(shape) < 1:
        raise ValueError("x must have at least rank 1, got rank 0.")
    dim, gates = _check_gate_shape(shape, gate.shape)
    torch_state = isinstance(state, torch.Tensor)
    if state.dtype != state_dtype(x):
        raise TypeError("state.dtype must be %s for x of type %s, got %s instead" % (state_dtype(x), x.dtype, state.dtype))
    if state.shape != shape:
        raise ValueError("state must have the shape of x, %s, got %s" % (tuple(shape), tuple(state.shape)))
    if not (state.is_contiguous() if torch_state else state.flags["C_CONTIGUOUS"] and state.flags["WRITEABLE"]):
        raise ValueError("state is overwritten: it must be contiguous and writeable")
    if torch_state and state.requires_grad:
        raise ValueError("state is overwritten: it cannot require a gradient (use linear_recurrence to differentiate)")
    if torch_state and (x.requires_grad or gate.requires_grad) and torch.is_grad_enabled():
        raise ValueError("a step has no gradient: detach x and gate, step under torch.no_grad(), or differentiate "
                         "torch_api.linear_recurrence")
    if torch_state and state.is_cuda:
        x, gate = x.contiguous(), gate.contiguous()
        out = torch.empty_like(x)
        if out.numel():
            device = x.get_device()
            call("linear_recurrence_step", code, gate_code, x.data_ptr(), gate.data_ptr(), state.data_ptr(), out.data_ptr(),
                 out.numel() // dim, dim, gates, dim, gates, form, complement, device, raw_stream(device), 0)
            torch.autograd.graph.increment_version(state)  # a graph that has kept it must not go on with it
        return out
    x, gate = contiguous(x), contiguous(gate)
    out = empty(x, shape, x.dtype)
    batch = prod(shape[:-1])
    if batch:
        call("linear_recurrence_step", code, gate_code, pointer(x), pointer(gate), pointer(state), pointer(out), batch,
             dim, gates, dim, gates, form, complement, *place_of(x), 0)
        if torch_state:
            torch.autograd.graph.increment_version(state)
    return out
