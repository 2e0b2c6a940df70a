"""Arrays of the sequence operators (``linear_recurrence``, ``rotary``): element types, strides, outputs.

Besides float32 and float64 these take float16 and (torch) bfloat16.  Torch views whose channels are
adjacent are read in place, whatever their batch and row strides (an expanded axis included); others are
copied once.  NumPy in gives NumPy out, torch in torch out on the same device."""
import numpy as np
import torch

from . import load_cusig
from .error_codes import err_msg
from .param_checks import check_type

TORCH_TYPES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}
NUMPY_TYPES = {np.dtype(np.float32): 0, np.dtype(np.float64): 1, np.dtype(np.float16): 3}

# handle of a device's current stream, without building a torch.cuda.Stream around it
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def element_type(array, name):
    """Number of the element type in the C ABI."""
    code = TORCH_TYPES.get(array.dtype) if isinstance(array, torch.Tensor) else None
    if code is None:
        check_type(array, name, (np.ndarray, torch.Tensor))
        code = NUMPY_TYPES.get(array.dtype) if isinstance(array, np.ndarray) else None
        if code is None:
            raise TypeError("%s.dtype must be float32, float64, float16 or bfloat16, got %s instead" % (name, array.dtype))
    return code


def state_dtype(array):
    """Type of states: float64 for float64 inputs, else float32."""
    if isinstance(array, torch.Tensor):
        return torch.float64 if array.dtype is torch.float64 else torch.float32
    return np.dtype(np.float64 if array.dtype == np.float64 else np.float32)


def check_like(array, name, like, like_name):
    """Same kind and device as ``like``."""
    if isinstance(array, torch.Tensor) and isinstance(like, torch.Tensor):
        if array.device != like.device:
            raise ValueError("%s and %s must be on the same device" % (name, like_name))
        return
    check_type(array, name, (np.ndarray, torch.Tensor))
    if isinstance(array, torch.Tensor) or isinstance(like, torch.Tensor):
        raise ValueError("%s and %s must both be numpy arrays or both torch tensors" % (name, like_name))


def check_state(array, name, shape, x):
    """A contiguous state-shaped input, or None."""
    if array is None:
        return None
    check_like(array, name, x, "x")
    if array.dtype != state_dtype(x):
        raise TypeError("%s.dtype must be %s for x of type %s, got %s instead" % (name, state_dtype(x), x.dtype, array.dtype))
    if array.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(array.shape)))
    return contiguous(array)


def contiguous(array):
    return array.contiguous() if isinstance(array, torch.Tensor) else np.ascontiguousarray(array)


def on_device(array):
    return isinstance(array, torch.Tensor) and array.is_cuda


def pointer(array):
    if array is None:
        return None
    return array.data_ptr() if isinstance(array, torch.Tensor) else array.ctypes.data


def empty(like, shape, dtype):
    if isinstance(like, torch.Tensor):
        if dtype is like.dtype and shape == like.shape and like.is_contiguous():
            return torch.empty_like(like)
        return like.new_empty(shape, dtype=dtype)
    return np.empty(shape, dtype=dtype)


def batched_rows(array):
    """``(array, batch stride, row stride)`` of (..., L, C) with the batch axes read as one: in place where
    the strides allow it, else a contiguous copy."""
    shape = array.shape
    rank, width, rows = len(shape), shape[-1], shape[-2]
    if isinstance(array, torch.Tensor) and array.is_cuda:
        strides = array.stride()
        if strides[-1] == 1 or width == 1:
            if rank == 2:
                return array, 0, strides[0]
            if rank == 3:
                return array, strides[0], strides[1]
            # axes of one entry take no part: their strides lead nowhere
            batch = [(n, s) for n, s in zip(shape[:-2], strides) if n != 1]
            if all(outer[1] == inner[0] * inner[1] for outer, inner in zip(batch, batch[1:])):
                return array, batch[-1][1] if batch else 0, strides[-2]
    array = contiguous(array)
    return array, rows * width, width


def place_of(array):
    """``(device, stream)`` for a native call: a CUDA tensor's device, all of whose operands this package has
    checked, and its current stream; (-1, None) where the library looks for itself."""
    if not on_device(array):
        return -1, None
    device = array.get_device()
    return device, raw_stream(device)


_natives = {}


def native(name):
    """The native function sigb200_<name>, looked up once."""
    f = _natives.get(name)
    if f is None:
        f = _natives[name] = getattr(load_cusig.library(), "sigb200_" + name)
    return f


def call(name, *args):
    """One native call; raises what the package's other operators raise."""
    code = native(name)(*args)
    if code:
        raise Exception("Error in pysiglib.%s: %s" % (name, err_msg(code)))
