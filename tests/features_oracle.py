# SPDX-License-Identifier: Apache-2.0
"""Plain 64-bit implementations of the point-feature operators, and how far a
16- or 32-bit kernel may be from them.

The bounds follow the kernels' arithmetic.  u is half a step of the type
(``torch.finfo(t).eps / 2``).  Scores are sums of ``dim`` products in 32 bits:
off by at most e = (dim + 8) 2^-24 scale sum |q k|, so a weight p is off by a
factor within 1 +- (2 max e + 2^-19) (numerator and normaliser; exp2 and the
exponent's own rounding, whose argument is below 2^7, take 2^-20 each).  16-bit
kernels round weights (and dS) to the type once more: u each; fp16 below its
normals by half of 2^-24 of its own scale.  Results are rounded once: u.
"""

import math

import torch


def seg_of(lengths):
    seg = [0]
    for n in lengths:
        seg.append(seg[-1] + n)
    return seg


class Attention:
    """Cross attention (ids None) or neighbour attention of packed scenes;
    ``out``, ``lse``, and with ``dout`` also ``dq``, ``dk``, ``dv``, each with
    ``*_off``, the bound of its elements' error (the weights' type: the
    inputs', except for neighbour attention's 32 bits)."""

    def __init__(self, q, k, v, q_seg, k_seg, mask=None, scale=None, ids=None, padded=True, dout=None):
        self.dtype = q.dtype
        u = torch.finfo(q.dtype).eps / 2
        uw = u if ids is None else 2.0**-24  # rounding of the weights
        tiny = 2.0**-25 if q.dtype == torch.float16 and ids is None else 0.0
        n_q, heads, dim = q.shape
        kv = k.shape[1]
        group = heads // kv
        scale = dim**-0.5 if scale is None else scale
        q, k, v = (t.detach().double().cpu() for t in (q, k, v))
        do = None if dout is None else dout.detach().double().cpu()
        mask = None if mask is None else mask.cpu().bool()
        ids = None if ids is None else ids.cpu().long()
        z = lambda t: torch.zeros(t.shape, dtype=torch.float64)  # noqa: E731
        self.out, self.out_off = z(q), z(q)
        self.lse = torch.full((n_q, heads), -math.inf, dtype=torch.float64)
        self.lse_off = torch.zeros(n_q, heads, dtype=torch.float64)
        if do is not None:
            self.dq, self.dk, self.dv = z(q), z(k), z(v)
            self.dq_off, self.dk_off, self.dv_off = z(q), z(k), z(v)
        for i in range(len(q_seg) - 1):
            a, b, c, d = q_seg[i], q_seg[i + 1], k_seg[i], k_seg[i + 1]
            if a == b or c == d:
                continue
            if ids is None:
                kept = torch.arange(c, d)
                kept = kept if mask is None else kept[mask[c:d]]
                count = torch.ones(b - a, len(kept), dtype=torch.float64)
            else:
                kept = torch.arange(c, d)
                count = self.counts(ids[a:b], d - c, padded)
            rows = torch.arange(a, b)[count.sum(1) > 0]
            count = count[count.sum(1) > 0]
            if not len(rows):
                continue
            for h in range(heads):
                g = h // group
                qs, ks, vs = q[rows, h], k[kept, g], v[kept, g]
                s = scale * qs @ ks.T
                e = (dim + 8) * 2.0**-24 * scale * (qs.abs() @ ks.abs().T)
                e = torch.where(count > 0, e, 0.0).amax(1, keepdim=True)
                lse = torch.logsumexp(torch.where(count > 0, s + count.log(), -math.inf), 1, keepdim=True)
                one = (s - lse).exp()  # a single entry's weight
                p = count * one
                off = 2 * e + 2.0**-19 + uw  # relative
                reach = p @ vs.abs()
                flat = (count > 0).double() @ vs.abs()
                o = p @ vs
                o_off = off * reach + tiny * flat
                self.out[rows, h] = o
                self.out_off[rows, h] = o_off + u * (o.abs() + o_off)
                self.lse[rows, h] = lse[:, 0]
                self.lse_off[rows, h] = (e + 2.0**-19 + 2.0**-22 * (lse.abs() + 1))[:, 0]
                if do is None:
                    continue
                ds_ = do[rows, h]
                back = off + 2 * self.lse_off[rows, h][:, None]  # of p from the stored lse
                dp = ds_ @ vs.T
                delta = (ds_ * o).sum(1, keepdim=True)
                x = dp - delta
                ds = p * x
                dp_off = (dim + 8) * 2.0**-24 * (ds_.abs() @ vs.abs().T) + (
                    ds_.abs() * (self.out_off[rows, h] + (dim + 8) * 2.0**-24 * o.abs())).sum(1, keepdim=True)
                ds_off = p * dp_off * (1 + back) + ds.abs() * (back + uw) + tiny * (count > 0)
                many = 2.0**-24 * (count.sum(1).max() + 8)  # long sums in 32 bits
                sums = {
                    "dq": (rows, h, ds @ ks * scale, (ds_off + many * ds.abs()) @ ks.abs() * scale),
                    "dk": (kept, g, ds.T @ qs * scale,
                           (ds_off + 2.0**-24 * (len(rows) + 8) * ds.abs()).T @ qs.abs() * scale),
                    "dv": (kept, g, p.T @ ds_,
                           (p * (back + uw + 2.0**-24 * (len(rows) + 8))).T @ ds_.abs()),
                }
                for name, (at, head, value, value_off) in sums.items():
                    getattr(self, name)[at, head] += value
                    getattr(self, name + "_off")[at, head] += value_off
        if do is not None:
            for name in ("dq", "dk", "dv"):
                x, x_off = getattr(self, name), getattr(self, name + "_off")
                x_off += u * (x.abs() + x_off)
                if self.dtype == torch.float16:  # below 2^-14 its values lie 2^-24 apart
                    x_off += 2.0**-25
        if self.dtype == torch.float16:
            self.out_off += 2.0**-25

    @staticmethod
    def counts(ids, n, padded):
        """How often each row's entries name each of n keys."""
        count = torch.zeros(len(ids), n, dtype=torch.float64)
        for j in range(ids.shape[1]):
            there = (ids[:, j] >= 0) & (ids[:, j] < n)
            if padded and j:
                there &= ids[:, j] != ids[:, 0]
            r = there.nonzero()[:, 0]
            count[r, ids[r, j]] += 1
        return count

    def close(self, name, got):
        want, off = getattr(self, name), getattr(self, name + "_off")
        got = got.detach().double().cpu()
        assert got.shape == want.shape, name
        same = (got == want) | (got.isnan() & want.isnan())
        bad = ~(same | ((got - want).abs() <= off))
        assert not bad.any(), (
            f"{name}: {int(bad.sum())} of {bad.numel()} elements are too far off, worst "
            f"{float(((got - want).abs() / off.clamp(min=1e-300))[bad].max()):.3g} times the bound"
        )


def rotate(x, positions, frequencies, axes, part, layout, unit=1.0, amplitude=1.0, transposed=False):
    """Rotary positions in 64 bits, and the bound of the error: sine and
    cosine within 2^-22 of the 64-bit angle's (its reduction leaves 2^-25 of
    a turn, 2^-22.3 radians), products and sum in 32 bits, one rounding."""
    u = torch.finfo(x.dtype).eps / 2
    y = x.detach().double().cpu().clone()
    off = torch.zeros_like(y)
    place = positions.detach().double().cpu().reshape(len(y), -1) / unit
    f = torch.tensor(frequencies, dtype=torch.float64)
    n = len(f)
    for a in range(axes):
        for i in range(n):
            p = a * n + i
            first, second = (p, p + part // 2) if layout == "half" else (2 * p, 2 * p + 1)
            t = (place[:, a] * f[i])[:, None]
            c, s = t.cos() * amplitude, t.sin() * amplitude * (-1 if transposed else 1)
            u0, v0 = y[..., first].clone(), y[..., second].clone()
            y[..., first], y[..., second] = u0 * c - v0 * s, u0 * s + v0 * c
            # the position's 64-bit turns carry 2^-52 of themselves
            slack = (u0.abs() + v0.abs()) * amplitude * (2.0**-20 + 2.0**-48 * place[:, a].abs()[:, None])
            off[..., first], off[..., second] = slack, slack
    off[..., :part] += u * (y[..., :part].abs() + off[..., :part])
    if x.dtype == torch.float16:
        off[..., :part] += 2.0**-25
    return y, off
