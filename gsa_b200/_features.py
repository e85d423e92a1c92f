# SPDX-License-Identifier: Apache-2.0
"""ctypes binding of the point-feature library (``include/point_features.h``).

The C entries take one struct; ``struct.pack`` builds it in a microsecond,
where a call of forty ctypes arguments would cost more than a small kernel.
"""

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from ._library import load

lib = load("point_features")
for _name in ("rotary_positions", "cross_attention", "cross_attention_grad",
              "neighbor_attention", "neighbor_attention_grad"):
    getattr(lib, _name).argtypes = [ctypes.c_char_p]
    getattr(lib, _name).restype = ctypes.c_int
for _name in ("cross_attention_workspace", "cross_attention_grad_workspace",
              "neighbor_attention_grad_workspace"):
    getattr(lib, _name).argtypes = [ctypes.c_char_p]
    getattr(lib, _name).restype = ctypes.c_int64

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
POSITION_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}

# rotary_args: sizes; x, y; positions and their type and strides, axes,
# pairs, turns; amplitude; interleaved, transposed, stream
pack_rotary = struct.Struct("=4q 6q 7q d 3q").pack
# attention_args: sizes; scale; q, k, v, out, dout; the rest in order
pack_attention = struct.Struct("=9q d 15q 14q").pack


def check(code, what):
    if code == -2:
        raise ValueError(f"{what}: sizes or strides out of range")
    if code:
        raise RuntimeError(f"{what}: CUDA error {code}")


def check_tangents(*tensors):
    """Within a forward-mode level, none of the inputs carries a tangent: the
    kernels would drop it."""
    if forward_ad._current_level >= 0 and any(
        isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors
    ):
        raise ValueError("the operators on points' features have no forward-mode derivatives")


def check_outside_autograd(out, *tensors):
    """With gradients enabled, a call that writes ``out`` neither reads nor
    writes what autograd follows."""
    if out is not None and any(getattr(t, "requires_grad", False) for t in (out, *tensors)):
        raise ValueError("a call with out= takes no part in autograd: give none, or call under torch.no_grad()")


def rows_of(t, what, shape, dtype, device):
    """``(data, row stride, head stride)`` of a CUDA tensor of rows of heads;
    anything but the expected shape, type and device raises."""
    try:
        row, head, element = t.stride()
        fits = t.shape == shape and t.dtype is dtype and t.get_device() == device and (element == 1 or not t.numel())
    except (AttributeError, ValueError):
        fits = False
    if not fits:
        raise ValueError(
            f"{what} must be a {dtype} tensor of shape {tuple(shape)} on the current CUDA device, its last dimension contiguous"
        )
    return t.data_ptr(), row if shape[0] > 1 else 0, head if shape[1] > 1 else 0


_STEP = {torch.float32: 3, torch.float16: 7, torch.bfloat16: 7}  # 16 bytes less one element


def vector_rows_of(t, what, shape, dtype, device):
    """``rows_of`` for kernels that take 16 bytes at a time."""
    data, row, head = found = rows_of(t, what, shape, dtype, device)
    if data & 15 or (row | head) & _STEP[dtype]:
        raise ValueError(f"{what} must start on 16 bytes and have row and head strides that are multiples of 16 bytes")
    return found


def check_written(t, what):
    """A tensor about to be written: no two of its elements share memory."""
    (a, n), (b, m) = sorted(zip(t.stride()[:2], t.shape[:2]))
    least = t.shape[2]
    for stride, size in ((a, n), (b, m)):
        if size > 1:
            if stride < least:
                raise ValueError(f"{what}: elements overlap")
            least = stride * (size - 1) + least
    # a backward pass that saved the tensor learns that it was written
    torch.autograd.graph.increment_version(t)
