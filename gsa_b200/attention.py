# SPDX-License-Identifier: Apache-2.0
"""Attention between the points of a hierarchy.

``cross_attention``: the queries of each scene read the states of the same
scene at another level (a decoder level the coarser encoder level, or one
query a whole room).  ``neighbor_attention``: each query reads only the
points that its row of a radius or 3NN query names (``Tree.ball``,
``Forest.ball``, ``QuerySession.ball_into``, ``hierarchy.Batch``).  Both have
a gradient, as a call of its own (``..._grad``) and through autograd.

Rows are packed scene after scene, as in ``Forest``; ``ScenePairs`` holds the
offsets of the query rows and of the key rows of every scene.
"""

import itertools

import torch

from . import _features as ft
from ._library import current_stream

MAX_DIM = 128
MAX_WIDTH = 32
MAX_GROUP = 64  # query heads per head of keys, cross attention
MAX_SCENES = 65535  # of a cross-attention call
_INT_MAX = (1 << 31) - 1


class ScenePairs:
    """Which keys each query may read: queries ``q_seg[i]`` to
    ``q_seg[i + 1]`` read keys ``k_seg[i]`` to ``k_seg[i + 1]``.

    Offsets start at 0, never fall (a scene may have no queries or no keys)
    and end at the number of rows.  They are uploaded once; make the object
    outside a graph capture, and keep it as long as graphs that used it.  A copy
    of it, or one from a pickle, is uploaded anew."""

    def __init__(self, q_seg, k_seg):
        q_seg, k_seg = [int(v) for v in q_seg], [int(v) for v in k_seg]
        if not (len(q_seg) == len(k_seg) >= 2 and all(
            s[0] == 0 and s[-1] < _INT_MAX and all(b >= a for a, b in zip(s, s[1:])) for s in (q_seg, k_seg)
        )):
            raise ValueError("ScenePairs requires equally many ascending query and key offsets from 0 on")
        self.q_seg, self.k_seg = q_seg, k_seg
        self.scenes = len(q_seg) - 1
        self.n_q, self.n_k = q_seg[-1], k_seg[-1]
        self.max_q = max(b - a for a, b in zip(q_seg, q_seg[1:]))
        self.max_k = max(b - a for a, b in zip(k_seg, k_seg[1:]))
        self.device, self.stream = current_stream()
        # both offset lists, and the flag of the kernels' bounded waits
        self._ints = torch.tensor(q_seg + k_seg + [0], dtype=torch.int32).to(f"cuda:{self.device}")
        self._q_at = self._ints.data_ptr()
        self._k_at = self._q_at + 4 * len(q_seg)
        self._error_at = self._k_at + 4 * len(k_seg)

    def __reduce__(self):
        # a copy, or an unpickled one, has offsets and a flag of its own
        return _pairs_on, (self.device, type(self), self.q_seg, self.k_seg)

    @classmethod
    def of_lengths(cls, queries, keys):
        """From the scenes' numbers of query and of key rows."""
        return cls(*([0] + list(itertools.accumulate(n)) for n in (queries, keys)))

    def check(self):
        """Raise if a kernel's bounded wait ran out in any call so far with
        these pairs, on whichever stream (their results are then void).
        Synchronises the device."""
        torch.cuda.synchronize(self.device)
        if int(self._ints[-1]):
            raise RuntimeError("cross attention: a wait for the tensor cores ran out")


def _pairs_on(device, kind, q_seg, k_seg):
    with torch.cuda.device(device):
        return kind(q_seg, k_seg)


class _Call:
    """The checked arguments that one attention call and its gradient share."""

    __slots__ = ("what", "device", "stream", "pairs", "dtype", "q_shape", "k_shape", "on", "sizes", "rows", "mask", "ids",
                 "width", "padded", "copies")

    def __init__(self, what, q, k, v, pairs, scale, types):
        try:
            (n_q, heads, dim), (n_k, kv_heads, _) = q.shape, k.shape
            fits = q.is_cuda and q.dtype in types
        except (AttributeError, ValueError):
            fits = False
        if not fits:
            raise ValueError(f"{what} needs CUDA (N, heads, dim) rows of one type among {[str(t) for t in types]}")
        self.device, self.stream = device, _ = current_stream()
        if not isinstance(pairs, ScenePairs) or pairs.device != device:
            raise ValueError(f"{what} needs ScenePairs made on the current device")
        if not 8 <= dim <= MAX_DIM or dim & 7:
            raise ValueError("the head size must be a multiple of 8, at most 128")
        if not (kv_heads and heads and heads % kv_heads == 0):
            raise ValueError("the query heads must be a multiple of the keys' heads")
        if types is _HALF and heads // kv_heads > MAX_GROUP:
            raise ValueError("at most 64 query heads share a head of keys")
        if types is _HALF and (pairs.scenes > MAX_SCENES or kv_heads > MAX_SCENES):
            raise ValueError("at most 65535 scenes, and heads of keys, in a call")
        if n_q != pairs.n_q or n_k != pairs.n_k:
            raise ValueError("query and key rows must be those of the pairs' offsets")
        if scale is None:
            scale = dim ** -0.5
        if not 2.0**-24 <= scale <= 2.0**24:
            raise ValueError("scale must be positive, from 2^-24 to 2^24")
        if self.stream != pairs.stream:
            # the offsets outlive the pairs until this stream is done with them
            pairs._ints.record_stream(torch.cuda.current_stream())
        self.what, self.dtype, self.pairs, self.on = what, q.dtype, pairs, q.device
        self.q_shape, self.k_shape = (n_q, heads, dim), (n_k, kv_heads, dim)
        self.sizes = (ft.TYPES[q.dtype], pairs.scenes, n_q, n_k, pairs.max_q, pairs.max_k, heads, kv_heads, dim, scale)
        self.copies = [] if types is _HALF else None
        self.rows = self.rows_of(q, "q", self.q_shape) + self.rows_of(k, "k", self.k_shape) + self.rows_of(
            v, "v", self.k_shape)
        self.mask = self.ids = self.width = self.padded = 0

    def rows_of(self, t, name, shape):
        found = ft.vector_rows_of(t, name, shape, self.dtype, self.device)
        if self.copies is not None and ((not found[1] and shape[0] > 1) or (not found[2] and shape[1] > 1)):
            # expanded rows or heads: the cross-attention kernels' copy engine
            # takes no stride of 0
            t = t.contiguous()
            self.copies.append(t)
            found = ft.vector_rows_of(t, name, shape, self.dtype, self.device)
        return found

    def set_mask(self, mask):
        if mask is None:
            return
        if not (isinstance(mask, torch.Tensor) and mask.get_device() == self.device
                and mask.dtype in (torch.bool, torch.uint8) and mask.shape == (self.pairs.n_k,)
                and mask.is_contiguous()):
            raise ValueError("mask must be contiguous CUDA bool (N_k,): the keys that may be read")
        self.mask = mask.data_ptr()

    def set_ids(self, ids, padded):
        if not (isinstance(ids, torch.Tensor) and ids.get_device() == self.device
                and ids.dtype is torch.int32 and ids.ndim == 2 and ids.shape[0] == self.pairs.n_q
                and 1 <= ids.shape[1] <= MAX_WIDTH and ids.is_contiguous()):
            raise ValueError("rows must be contiguous CUDA int32 (N_q, K) with K in [1,32]")
        self.ids, self.width, self.padded = ids.data_ptr(), ids.shape[1], 1 if padded else 0

    def lse_of(self, lse):
        if not (isinstance(lse, torch.Tensor) and lse.get_device() == self.device
                and lse.dtype is torch.float32 and lse.shape == self.q_shape[:2] and lse.is_contiguous()):
            raise ValueError("lse must be contiguous CUDA FP32 (N_q, heads)")
        return lse.data_ptr()

    def run(self, entry, workspace, out, dout, lse, grads):
        p = self.pairs

        def pack(at, size):
            return ft.pack_attention(*self.sizes, *self.rows, *out, *dout, lse, *grads, p._q_at, p._k_at, self.mask, self.ids,
                                     self.width, self.padded, at, size, p._error_at, self.stream)

        args = pack(0, 0)
        if workspace is not None:
            size = workspace(args)
            if size < 0:
                ft.check(size, self.what)
            if size:
                # private to this call: calls on several streams, and
                # captured ones, never share a workspace
                buffer = torch.empty(size, dtype=torch.uint8, device=self.on)
                args = pack(buffer.data_ptr(), size)
        code = entry(args)
        if code:
            ft.check(code, self.what)

    def forward(self, entry, workspace, out, return_lse, inputs):
        if out is None:
            out = torch.empty(self.q_shape, dtype=self.dtype, device=self.on)
            _, heads, dim = self.q_shape
            place = (out.data_ptr(), heads * dim, dim)
        else:
            place = ft.vector_rows_of(out, "out", self.q_shape, self.dtype, self.device)
            if place[0] and place[0] in [t.data_ptr() for t in inputs]:
                raise ValueError("out must not overlap the inputs")
            ft.check_written(out, "out")
        if not return_lse:
            self.run(entry, workspace, place, (0, 0, 0), 0, (0, 0, 0))
            return out
        lse = torch.empty(self.q_shape[:2], dtype=torch.float32, device=self.on)
        self.run(entry, workspace, place, (0, 0, 0), lse.data_ptr(), (0, 0, 0))
        return out, lse

    def backward(self, entry, workspace, dout, out, lse):
        dq = torch.empty(self.q_shape, dtype=self.dtype, device=self.on)
        dk = torch.empty(self.k_shape, dtype=self.dtype, device=self.on)
        dv = torch.empty(self.k_shape, dtype=self.dtype, device=self.on)
        self.run(entry, workspace, self.rows_of(out, "out", self.q_shape), self.rows_of(dout, "dout", self.q_shape),
                 self.lse_of(lse), (dq.data_ptr(), dk.data_ptr(), dv.data_ptr()))
        return dq, dk, dv


_HALF = (torch.bfloat16, torch.float16)
_ALL = (torch.float32, torch.bfloat16, torch.float16)


def _wants_grad(out, *tensors):
    ft.check_tangents(*tensors)
    if not torch.is_grad_enabled():
        return False
    ft.check_outside_autograd(out, *tensors)
    return any(getattr(t, "requires_grad", False) for t in tensors)


def _no_second(dout, *others):
    """A gradient call on a ``dout`` that autograd follows would end its
    derivatives in silence."""
    ft.check_tangents(dout, *others)
    if getattr(dout, "requires_grad", False) and torch.is_grad_enabled():
        raise ValueError("attention has no second derivatives: detach dout, or call under torch.no_grad()")


def _cross(q, k, v, pairs, mask, scale, out, return_lse):
    call = _Call("cross attention", q, k, v, pairs, scale, _HALF)
    call.set_mask(mask)
    return call.forward(ft.lib.cross_attention, ft.lib.cross_attention_workspace, out, return_lse, (q, k, v))


def cross_attention(q, k, v, pairs, mask=None, scale=None, out=None, return_lse=False):
    """``softmax(scale q k^T) v`` of every query over the open keys of its
    scene.

    ``q``: BF16 or FP16 (N_q, heads, dim); ``k``, ``v``: the same type
    (N_k, kv_heads, dim), heads a multiple of kv_heads, at most 64 times (query
    head h reads head h // (heads // kv_heads)); dim a multiple of 8, at most 128.  Row
    and head strides are free in steps of 16 bytes.  ``mask``: bool (N_k,),
    False shuts a key out, whatever it holds.  ``scale``: dim ** -0.5 by
    default, from 2^-24 to 2^24.  A query without open keys gets 0.  Returns ``out`` (written to
    ``out`` if given, which does not overlap the inputs), and with
    ``return_lse`` also the FP32 (N_q, heads) logarithms of the sums of
    exponentials that ``cross_attention_grad`` takes.  Differentiable in q, k
    and v unless ``out`` is given.  In a captured graph, take the gradient by
    ``cross_attention_grad``: torch's autograd may order a captured backward
    pass after work outside the capture."""
    if _wants_grad(out, q, k, v):
        out, lse = _Cross.apply(q, k, v, pairs, mask, scale)
        return (out, lse) if return_lse else out
    return _cross(q, k, v, pairs, mask, scale, out, return_lse)


def cross_attention_grad(dout, q, k, v, out, lse, pairs, mask=None, scale=None):
    """``(dq, dk, dv)`` from the gradient of ``cross_attention``'s ``out``;
    the other arguments are that call's, with its ``out`` and ``lse``.  The
    sums have a fixed order: the same arguments give the same bits.  The
    results take no part in autograd.  Weights are taken again from ``lse``,
    whose 32 bits leave them off by some 2^-22 ``|lse|`` of themselves (FP16:
    beyond an ``|lse|`` of 2^22 they may overflow).  FP16: a row whose ``|lse| / scale`` or
    ``|<dout, out>|`` is 2^31 or more makes dk and dv of its scene NaN."""
    _no_second(dout, q, k, v, out, lse)
    call = _Call("cross attention gradient", q, k, v, pairs, scale, _HALF)
    call.set_mask(mask)
    return call.backward(ft.lib.cross_attention_grad, ft.lib.cross_attention_grad_workspace, dout, out, lse)


def _neighbor(q, k, v, rows, pairs, padded, scale, out, return_lse):
    call = _Call("neighbor attention", q, k, v, pairs, scale, _ALL)
    call.set_ids(rows, padded)
    return call.forward(ft.lib.neighbor_attention, None, out, return_lse, (q, k, v))


def neighbor_attention(q, k, v, rows, pairs, padded=True, scale=None, out=None, return_lse=False):
    """Attention of every query over the keys that its row names.

    ``rows``: int32 (N_q, K), K at most 32: the rows of a radius or 3NN query,
    IDs counted from the first key of the query's scene.  An entry outside the
    scene's keys (a negative one) is absent.  ``padded``: an entry that
    repeats the row's first is absent too, as behind the hits of a radius
    row; else repeats count each time.  (A radius row without hits is all
    zeros and reads key 0, like any such row of a radius query.)  The rows keep
    their values until the gradient is taken: a query that writes the same
    buffer again is not noticed.  ``q``, ``k``, ``v`` and the rest as for
    ``cross_attention``, FP32 too."""
    if _wants_grad(out, q, k, v):
        out, lse = _Neighbor.apply(q, k, v, rows, pairs, padded, scale)
        return (out, lse) if return_lse else out
    return _neighbor(q, k, v, rows, pairs, padded, scale, out, return_lse)


def neighbor_attention_grad(dout, q, k, v, rows, out, lse, pairs, padded=True, scale=None):
    """``(dq, dk, dv)`` from the gradient of ``neighbor_attention``'s
    ``out``, in a fixed order of sums and outside autograd like
    ``cross_attention_grad``."""
    _no_second(dout, q, k, v, out, lse)
    call = _Call("neighbor attention gradient", q, k, v, pairs, scale, _ALL)
    call.set_ids(rows, padded)
    return call.backward(ft.lib.neighbor_attention_grad, ft.lib.neighbor_attention_grad_workspace, dout, out, lse)


def _vectors(t):
    """A gradient as the kernels take it (autograd may hand over an expanded
    or otherwise laid out one, or one that starts anywhere: a contiguous view
    behind other columns, say, of which ``contiguous()`` makes no copy)."""
    size = t.element_size()
    fits = t.stride(2) == 1 and not (t.data_ptr() | t.stride(0) * size | t.stride(1) * size) & 15
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, pairs, mask, scale):
        out, lse = _cross(q, k, v, pairs, mask, scale, None, True)
        ctx.save_for_backward(q, k, v, out, lse, mask)
        ctx.pairs, ctx.scale = pairs, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse, mask = ctx.saved_tensors
        return (*cross_attention_grad(_vectors(dout), q, k, v, out, lse, ctx.pairs, mask, ctx.scale), None, None, None)


class _Neighbor(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rows, pairs, padded, scale):
        out, lse = _neighbor(q, k, v, rows, pairs, padded, scale, None, True)
        ctx.save_for_backward(q, k, v, rows, out, lse)
        ctx.pairs, ctx.padded, ctx.scale = pairs, padded, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, rows, out, lse = ctx.saved_tensors
        return (*neighbor_attention_grad(_vectors(dout), q, k, v, rows, out, lse, ctx.pairs, ctx.padded, ctx.scale),
                None, None, None, None)
