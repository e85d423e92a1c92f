# SPDX-License-Identifier: Apache-2.0
"""Rotary positions of points' features.

``Rotary`` turns the first ``part`` elements of every head by angles that grow
with the point's position, so that the products of two turned heads depend on
the difference of their positions only.  Positions are the points' own
coordinates (``axes`` = 2 or 3: an equal share of the pairs for each) or a
place in an order (``axes`` = 1), where ``scaling`` extends a network to
longer orders than it was trained on.
"""

import math
from array import array

import torch

from . import _features as ft
from ._library import current_stream

MAX_PAIRS = 128  # per axis
MAX_DIM = 4096
MAX_AMPLITUDE = torch.finfo(torch.float32).max


def frequencies(pairs, base=10000.0, scaling=None, factor=1.0, length=None, low=1.0, high=32.0):
    """Radians per unit of position of an axis' pairs: ``base ** (-i / pairs)``,
    scaled for positions ``factor`` times as far as those trained on.

    ``None``      as they are;
    ``"linear"``  all divided by ``factor``;
    ``"base"``    the base grown so that the slowest pair is divided by
                  ``factor`` and the fastest kept;
    ``"ramp"``    by how often a pair turns over the ``length`` trained on:
                  kept from ``high`` turns on, divided up to ``low``, and
                  blended linearly between."""
    if scaling == "base" and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    f = [base ** (-i / pairs) for i in range(pairs)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "ramp":
        keep = [min(1.0, max(0.0, (length * x / (2 * math.pi) - low) / (high - low))) for x in f]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, keep)]
    return f


class Rotary:
    """A rotation plan: ``rotary(x, positions)`` returns the turned rows and
    ``rotary.grad(dy, positions)`` the gradient of ``x``.

    ``part``: elements of a head that turn, a multiple of ``2 * axes``; the
    others are copied.  ``layout``: ``"half"`` pairs element p with
    p + part / 2, ``"interleaved"`` 2p with 2p + 1; the pairs of an axis
    follow one another.  ``unit``: the length that counts as one position.
    ``base``, ``scaling``, ``factor``, ``length``: see ``frequencies``.
    ``amplitude``: factor of the turned elements, by default 1, for "ramp"
    0.1 ln(factor) + 1."""

    def __init__(self, part, axes=1, layout="half", base=10000.0, unit=1.0, scaling=None, factor=1.0, length=None,
                 amplitude=None):
        if not (isinstance(part, int) and isinstance(axes, int) and axes >= 1 and part >= 2 and part % (2 * axes) == 0
                and part // (2 * axes) <= MAX_PAIRS):
            raise ValueError("part must be a positive multiple of 2 * axes with at most 128 pairs per axis")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout is 'half' or 'interleaved'")
        if scaling not in (None, "linear", "base", "ramp"):
            raise ValueError("scaling is None, 'linear', 'base' or 'ramp'")
        if not all(math.isfinite(v) and v > 0 for v in (base, unit, factor)):
            raise ValueError("base, unit and factor must be positive")
        if scaling == "ramp" and not (length is not None and math.isfinite(length) and length > 0):
            raise ValueError("scaling 'ramp' needs the length trained on")
        if amplitude is None:
            amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0
        if not abs(amplitude) <= MAX_AMPLITUDE:
            raise ValueError("amplitude must be finite in FP32")
        self.part, self.axes, self.layout, self.amplitude = part, axes, layout, amplitude
        self.pairs = part // (2 * axes)
        self._interleaved = layout == "interleaved"
        f = frequencies(self.pairs, base, scaling, factor, length)
        # copied and pickled with the plan, so its address is asked for per call
        self._turns = array("d", [v / (2 * math.pi) / unit for v in f])

    def _run(self, x, positions, out, transposed):
        try:
            rows, heads, dim = shape = x.shape
            fits = x.is_cuda and x.dtype in ft.TYPES and heads > 0 and self.part <= dim <= MAX_DIM
        except (AttributeError, ValueError):
            fits = False
        if not fits:
            raise ValueError("rows must be CUDA FP32, FP16 or BF16 (N, heads, dim) with dim from part to 4096")
        device, stream = current_stream()
        dtype = x.dtype
        place = ft.rows_of(x, "rows", shape, dtype, device)
        try:
            kind = ft.POSITION_TYPES.get(positions.dtype, -1)
            n, *axes = positions.shape
            fits = kind >= 0 and positions.get_device() == device and n == rows and (
                axes == [self.axes] or (self.axes == 1 and not axes))
        except (AttributeError, ValueError):
            fits = False
        if not fits:
            raise ValueError("positions must be CUDA FP32, int32 or int64 (N, axes) on the rows' device")
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=x.device)
            to = (out.data_ptr(), heads * dim, dim)
        else:
            to = ft.rows_of(out, "out", shape, dtype, device)
            if to[0] == place[0] and to != place and out.numel():
                raise ValueError("out may be the rows themselves, not another view of them")
            ft.check_written(out, "out")
        steps = positions.stride()
        args = ft.pack_rotary(
            ft.TYPES[dtype], rows, heads, dim, *place, *to, positions.data_ptr(), kind, steps[0], steps[1] if axes else 0,
            self.axes, self.pairs, self._turns.buffer_info()[0], self.amplitude, self._interleaved, transposed, stream,
        )
        code = ft.lib.rotary_positions(args)
        if code:
            ft.check(code, "rotary positions")
        return out

    def _turn(self, x, positions, out, transposed):
        ft.check_tangents(x, positions)
        if torch.is_grad_enabled():
            if getattr(positions, "requires_grad", False):
                raise ValueError("positions get no gradient: detach them, or call under torch.no_grad()")
            ft.check_outside_autograd(out, x)
            if getattr(x, "requires_grad", False):
                return _Turn.apply(x, positions, self, transposed)
        return self._run(x, positions, out, transposed)

    def __call__(self, x, positions, out=None):
        """The rows ``x`` (FP32, FP16 or BF16 (N, heads, dim), any row and
        head strides) turned by ``positions`` (FP32, int32 or int64
        (N, axes), or (N,) for one axis).  ``out`` may be ``x`` itself, else it does not
        overlap it.  Differentiable in ``x`` unless ``out`` is given, not in
        the positions; in a captured graph, take the gradient by ``grad``."""
        return self._turn(x, positions, out, False)

    def grad(self, dy, positions, out=None):
        """The gradient of ``x`` from that of ``rotary(x, positions)``; linear
        in ``dy`` and differentiable in it as ``rotary`` is in ``x``."""
        return self._turn(dy, positions, out, True)


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, rotary, transposed):
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.transposed = rotary, transposed
        return rotary._run(x, positions, None, transposed)

    @staticmethod
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        if dy.stride(2) != 1:
            dy = dy.contiguous()
        return ctx.rotary._turn(dy, positions, None, not ctx.transposed), None, None, None
