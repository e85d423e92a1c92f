# SPDX-License-Identifier: Apache-2.0
"""Workloads of the point-feature operators: rotary positions, cross
attention between the levels of a hierarchy, and attention along the rows of
a neighbour query.

A case is a dict of plain values.  ``prepare(case, seed)`` makes its inputs,
``run(state)`` makes one pass: in elementary torch operations, or, where
``own`` is true, through the package's operators.  ``exact(case, seed)``
gives the same outputs from the definitions in 64 bits.

Rows are packed scene after scene: rows ``seg[i]`` to ``seg[i + 1]`` belong
to scene ``i``, as in ``gsa_b200.Forest``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROOM = (24000, 6000, 1500, 375, 94)  # the levels of a room hierarchy
PLAIN_SCORES = 1 << 29  # scores that the plain form holds at a time


def listed():
    return [
        # Rotary positions of a coarse level's queries, from the points' own
        # coordinates: a call of a few microseconds.
        dict(name="rotary level 3, xyz", op="rotary", rows=375, heads=8, dim=32, part=30, axes=3, layout="half",
             dtype="bf16", scaling="none", factor=1.0, fused=False, gradient=False),
        # The gradient through the positions of eight rooms at full
        # resolution, of a tensor whose rows hold queries, keys and values
        # together, in a layout whose pairs are neighbours.
        dict(name="rotary 8 rooms, gradient", op="rotary", rows=8 * 24000, heads=8, dim=32, part=30, axes=3,
             layout="interleaved", dtype="bf16", scaling="none", factor=1.0, fused=True, gradient=True),
        # 64 rooms in FP32, positions along a serialised order of all points
        # (a million and more), scaled for that length; half of each head.
        dict(name="rotary 64 rooms, long", op="rotary", rows=64 * 24000, heads=4, dim=64, part=32, axes=1,
             layout="half", dtype="fp32", scaling="ramp", factor=16.0, fused=False, gradient=False),
        # One query (a room's own state, or the next answer about it) reads a
        # whole room's points.
        dict(name="cross 1 row on a room", op="cross", scenes=1, q=1, k=24000, ragged=False, masked=False, heads=8,
             kv_heads=8, dim=64, dtype="bf16", train=False),
        # Two coarse levels of eight scans of unequal sizes, invalid points
        # masked.
        dict(name="cross level 2 to 3, ragged", op="cross", scenes=8, q=1500, k=375, ragged=True, masked=True,
             heads=8, kv_heads=8, dim=32, dtype="fp16", train=False),
        # A decoder level of eight rooms reads the coarser encoder level.
        dict(name="cross level 1 to 2", op="cross", scenes=8, q=6000, k=1500, ragged=False, masked=False, heads=8,
             kv_heads=8, dim=64, dtype="bf16", train=False),
        # The finest levels, keys and values shared by two heads: the largest.
        dict(name="cross level 0 to 1, shared", op="cross", scenes=8, q=24000, k=6000, ragged=False, masked=False,
             heads=4, kv_heads=2, dim=128, dtype="bf16", train=False),
        # A training step's forward and backward pass of the decoder level.
        dict(name="cross level 1 to 2, training", op="cross", scenes=8, q=6000, k=1500, ragged=False, masked=False,
             heads=8, kv_heads=8, dim=64, dtype="bf16", train=True),
        # Training on sixteen small scans of unequal sizes with invalid
        # points, shared heads and a head size between the usual ones.
        dict(name="cross ragged, training", op="cross", scenes=16, q=1500, k=375, ragged=True, masked=True, heads=4,
             kv_heads=2, dim=48, dtype="fp16", train=True),
        # A sampled level of one room attends along its radius rows.
        dict(name="neighbors level 2", op="neighbors", scenes=1, q=1500, k=1500, width=32, ragged=False, heads=4,
             kv_heads=4, dim=32, dtype="bf16", train=False),
        # Eight rooms at full resolution.
        dict(name="neighbors 8 rooms", op="neighbors", scenes=8, q=24000, k=24000, width=32, ragged=False, heads=8,
             kv_heads=8, dim=32, dtype="bf16", train=False),
        # A training step of the first sampled level in FP32.
        dict(name="neighbors level 1, training", op="neighbors", scenes=8, q=6000, k=6000, width=32, ragged=False,
             heads=4, kv_heads=4, dim=32, dtype="fp32", train=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rotary", "cross", "cross", "neighbors"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "rotary":
        axes, dim = rng.choice((1, 1, 2, 3, 3)), 8 * rng.randint(2, 16)
        pairs = rng.randint(1, dim // (2 * axes))
        heads = rng.randint(1, 16)
        return dict(op=op, rows=_log(rng, 1, (1 << 28) // (heads * dim)), heads=heads, dim=dim,
                    part=2 * axes * pairs, axes=axes, layout=rng.choice(("half", "interleaved")),
                    dtype=rng.choice(("bf16", "fp16", "fp32")), scaling=rng.choice(("none", "linear", "base", "ramp")),
                    factor=rng.choice((2.0, 4.0, 16.0)), fused=rng.random() < 0.5, gradient=rng.random() < 0.5)
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    scenes = _log(rng, 1, 32)
    ragged, train = rng.random() < 0.6, rng.random() < 0.5
    if op == "cross":
        dim = 8 * rng.randint(2, 16)
        q = _log(rng, 1, 24000)
        # scores of the largest listed cases, forward and training
        most = 8 * 6000 * 1500 * 8 * 64 if train else 8 * 24000 * 6000 * 4 * 128
        k = _log(rng, 1, max(1, min(24000, most // (scenes * heads * dim * q))))
        return dict(op=op, scenes=scenes, q=q, k=k, ragged=ragged, masked=rng.random() < 0.4, heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, train=train)
    dim = 8 * rng.randint(2, 16)
    most = (8 * 6000 * 32 * 128 if train else 8 * 24000 * 32 * 256) // 2
    width = rng.choice((3, 8, 16, 24, 32, rng.randint(1, 32)))
    q = _log(rng, 1, max(1, min(24000, most // (scenes * heads * dim * width))))
    return dict(op=op, scenes=scenes, q=q, k=_log(rng, max(1, q // 4), 4 * q), width=width, ragged=ragged,
                heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(("bf16", "fp16", "fp32")), train=train)


def _lengths(case):
    """Query and key rows of every scene: all alike, or between a tenth and
    all of the case's; then the third scene of a batch has no keys."""
    n = case["scenes"]
    if not case["ragged"]:
        return [case["q"]] * n, [case["k"]] * n
    share = [0.1 + 0.9 * ((i * 0.6180339887) % 1.0) for i in range(n)]
    q = [max(1, int(case["q"] * s)) for s in share]
    k = [max(1, int(case["k"] * share[-1 - i])) for i in range(n)]
    if n > 2:
        k[2] = 0
    return q, k


def _seg(lengths):
    seg = [0]
    for n in lengths:
        seg.append(seg[-1] + n)
    return seg


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        x = case["rows"] * case["heads"] * case["dim"]
        pairs = case["rows"] * case["part"] // 2
        place = case["rows"] * (12 if case["axes"] == 3 else 4 * case["axes"])
        return {"bytes": 2 * x * size + place, "flops": 6 * pairs * case["heads"]}
    q, k = _lengths(case)
    rows = (sum(q) * case["heads"] * 2 + sum(k) * case["kv_heads"] * 2) * case["dim"] * size
    if case["op"] == "cross":
        kept = 0.875 if case["masked"] else 1.0
        pairs = sum(a * b for a, b in zip(q, k)) * case["heads"] * kept
        extra = sum(k) if case["masked"] else 0
    else:
        pairs = sum(a * case["width"] for a, b in zip(q, k) if b) * case["heads"]
        extra = sum(q) * case["width"] * 4
    if case["train"]:  # the pass forward, and five products backward
        return {"bytes": 2 * rows + extra, "flops": 14 * case["dim"] * pairs}
    return {"bytes": rows + extra, "flops": 4 * case["dim"] * pairs}


# ---------------------------------------------------------------------------
# inputs


def _frequencies(case):
    """Radians per unit of position of every pair of an axis, in 64 bits, and
    the amplitude."""
    n = case["part"] // 2 // case["axes"]
    base, factor = 10000.0, case["factor"]
    i = torch.arange(n, dtype=torch.float64) / n
    if case["scaling"] == "base" and n > 1:
        base = base * factor ** (n / (n - 1))
    f = base ** -i
    if case["scaling"] == "linear":
        f = f / factor
    amplitude = 1.0
    if case["scaling"] == "ramp":
        turns = 65536.0 * f / (2 * math.pi)  # over the length trained on
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f, amplitude


def _rotary_handle(case):
    from gsa_b200 import Rotary

    scaling = None if case["scaling"] == "none" else case["scaling"]
    return Rotary(case["part"], axes=case["axes"], layout=case["layout"], unit=0.02 if case["axes"] > 1 else 1.0,
                  scaling=scaling, factor=case["factor"], length=65536)


def _points(rows, g):
    return torch.rand((rows, 3), generator=g, device="cuda") * torch.tensor([8.0, 6.0, 3.0], device="cuda")


def _morton(x):
    cell = (x * 64.0).long().clamp(0, 1023)
    code = torch.zeros_like(cell[:, 0])
    for bit in range(10):
        for axis in range(3):
            code |= ((cell[:, axis] >> bit) & 1) << (3 * bit + axis)
    return code


def _neighbor_rows(case, seg, k_seg, g):
    """Rows as a radius query gives them: ascending scene-local IDs of nearby
    points, fewer than the row holds in most places, then the first again;
    zeros where no point is near.  Near means close in Morton order."""
    out = []
    for i in range(case["scenes"]):
        q, k = seg[i + 1] - seg[i], k_seg[i + 1] - k_seg[i]
        width = case["width"]
        if k == 0:
            out.append(torch.zeros((q, width), dtype=torch.int32, device="cuda"))
            continue
        x = _points(max(q, k), g)
        codes, order = _morton(x[:k]).sort()
        at = torch.searchsorted(codes, _morton(x[:q]))
        reach = max(width, 48)
        offset = torch.rand((q, 2 * reach), generator=g, device="cuda").argsort(1)[:, :width] - reach
        ids = order[(at[:, None] + offset).remainder(k)].sort(1).values
        found = torch.randint(0, 2 * width + 1, (q, 1), generator=g, device="cuda").clamp(max=width)
        distinct = torch.ones_like(ids, dtype=torch.bool)
        distinct[:, 1:] = ids[:, 1:] > ids[:, :-1]
        column = torch.arange(width, device="cuda")
        ids = torch.where(distinct & (column < found), ids, ids[:, :1])
        out.append(torch.where(found > 0, ids, 0).int())
    return torch.cat(out)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        rows, heads, dim = case["rows"], case["heads"], case["dim"]
        state["x"] = normal(rows, 3, heads, dim)[:, 0] if case["fused"] else normal(rows, heads, dim)
        if case["axes"] == 1:
            order = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda")
            state["positions"] = order.int()
        else:
            state["positions"] = _points(rows, g)[:, : case["axes"]].contiguous()
        f, amplitude = _frequencies(case)
        state["frequencies"], state["amplitude"] = f.cuda(), amplitude
        if own:
            state["rotary"] = _rotary_handle(case)
        return state
    lengths = _lengths(case)
    q_seg, k_seg = _seg(lengths[0]), _seg(lengths[1])
    state["q"] = normal(q_seg[-1], case["heads"], case["dim"])
    kv = normal(k_seg[-1], 2, case["kv_heads"], case["dim"])  # one projection makes both
    state["k"], state["v"] = kv[:, 0], kv[:, 1]
    if case["train"]:
        state["grad"] = normal(q_seg[-1], case["heads"], case["dim"])
    state["q_seg"] = torch.tensor(q_seg, device="cuda")
    state["k_seg"] = torch.tensor(k_seg, device="cuda")
    if case["op"] == "neighbors":
        state["rows"] = _neighbor_rows(case, q_seg, k_seg, g)
    if case["op"] == "cross":
        keep = torch.rand(k_seg[-1], generator=g, device="cuda") < 0.875
        state["mask"] = keep if case["masked"] else None
    if own:
        from gsa_b200 import ScenePairs

        state["pairs"] = ScenePairs(q_seg, k_seg)
    return state


# ---------------------------------------------------------------------------
# one pass


def run(state):
    op, train = state["case"]["op"], state["case"].get("train")
    if op == "rotary":
        gradient = state["case"]["gradient"]
        if not own:
            return _plain_rotary(state)
        return (state["rotary"].grad if gradient else state["rotary"])(state["x"], state["positions"])
    if not own:
        return _plain_cross(state) if op == "cross" else _plain_neighbors(state)
    from gsa_b200 import attention

    q, k, v, pairs = state["q"], state["k"], state["v"], state["pairs"]
    if op == "cross":
        if not train:
            return attention.cross_attention(q, k, v, pairs, mask=state["mask"])
        out, lse = attention.cross_attention(q, k, v, pairs, mask=state["mask"], return_lse=True)
        return (out, *attention.cross_attention_grad(state["grad"], q, k, v, out, lse, pairs, mask=state["mask"]))
    if not train:
        return attention.neighbor_attention(q, k, v, state["rows"], pairs)
    out, lse = attention.neighbor_attention(q, k, v, state["rows"], pairs, return_lse=True)
    return (out, *attention.neighbor_attention_grad(state["grad"], q, k, v, state["rows"], out, lse, pairs))


def _plain_rotary(state):
    """Pairs (a, b) of a head's first ``part`` elements turn by the angle
    position * frequency; angles in 64 bits, for positions are far."""
    case, x = state["case"], state["x"].float()
    part = case["part"]
    place = state["positions"].double().reshape(len(x), -1)
    if case["axes"] > 1:
        place = place / 0.02
    angle = (place[:, :, None] * state["frequencies"]).reshape(len(x), 1, part // 2)
    cos, sin = (angle.cos() * state["amplitude"]).float(), (angle.sin() * state["amplitude"]).float()
    if case["gradient"]:
        sin = -sin
    if case["layout"] == "half":
        a, b = x[..., : part // 2], x[..., part // 2 : part]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., 0:part:2], x[..., 1:part:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, x[..., part:]), -1).to(state["x"].dtype)


def _padded(x, seg, lo, hi, most):
    """Scenes lo..hi of packed rows as (scenes, heads, most, dim) in FP32,
    the rows' places, and which of them are the scene's."""
    start, end = seg[lo:hi, None], seg[lo + 1 : hi + 1, None]
    at = start + torch.arange(most, device=x.device)
    there = at < end
    at = torch.where(there, at, 0)
    return x[at].float().movedim(-2, 1), at, there


def _plain_cross(state):
    case, q, k, v, dtype = state["case"], state["q"], state["k"], state["v"], state["q"].dtype
    lengths = _lengths(case)
    most_q, most_k, group = max(lengths[0]), max(1, max(lengths[1])), case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    out = torch.empty_like(q)
    grads = [torch.empty_like(q), torch.empty(k.shape, dtype=dtype, device=q.device),
             torch.empty(v.shape, dtype=dtype, device=q.device)] if case["train"] else []
    if not len(k):
        return (out.zero_(), grads[0].zero_(), *grads[1:]) if case["train"] else out.zero_()
    step = max(1, PLAIN_SCORES // (case["heads"] * most_q * most_k))
    for lo in range(0, case["scenes"], step):  # as many scenes as fit the card together
        hi = min(lo + step, case["scenes"])
        qs, q_at, q_there = _padded(q, state["q_seg"], lo, hi, most_q)
        ks, k_at, k_there = _padded(k, state["k_seg"], lo, hi, most_k)
        vs = _padded(v, state["k_seg"], lo, hi, most_k)[0]
        ks, vs = ks.repeat_interleave(group, 1), vs.repeat_interleave(group, 1)
        open_ = k_there if state["mask"] is None else k_there & state["mask"][k_at]
        shut = ~open_[:, None, None, :]
        s = torch.matmul(qs, ks.mT) * scale
        s = s.masked_fill_(shut, -math.inf)
        s = s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
        p = s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30))
        o = torch.matmul(p, vs).movedim(1, 2)
        out[q_at[q_there]] = o[q_there].to(dtype)
        if case["train"]:
            do = _padded(state["grad"], state["q_seg"], lo, hi, most_q)[0] * q_there[:, None, :, None]
            dv = torch.matmul(p.mT, do).unflatten(1, (-1, group)).sum(2).movedim(1, 2)
            dp = torch.matmul(do, vs.mT)
            ds = dp.sub_((dp * p).sum(-1, keepdim=True)).mul_(p)
            dq = (torch.matmul(ds, ks) * scale).movedim(1, 2)
            dk = (torch.matmul(ds.mT, qs) * scale).unflatten(1, (-1, group)).sum(2).movedim(1, 2)
            grads[0][q_at[q_there]] = dq[q_there].to(dtype)
            grads[1][k_at[k_there]] = dk[k_there].to(dtype)
            grads[2][k_at[k_there]] = dv[k_there].to(dtype)
    return (out, *grads) if case["train"] else out


def _plain_neighbors(state):
    case, q, k, v, dtype = state["case"], state["q"], state["k"], state["v"], state["q"].dtype
    group, scale = case["heads"] // case["kv_heads"], case["dim"] ** -0.5
    out = torch.empty_like(q)
    dq, dk, dv = None, None, None
    if case["train"]:
        dq = torch.empty_like(q)
        dk = torch.zeros(k.shape, dtype=torch.float32, device=q.device)
        dv = torch.zeros(v.shape, dtype=torch.float32, device=q.device)
    q_seg, k_seg = state["q_seg"], state["k_seg"]
    step = max(1, PLAIN_SCORES // (case["width"] * case["heads"] * case["dim"]))
    for lo in range(0, len(q), step):  # as many rows as fit the card together
        hi = min(lo + step, len(q))
        scene = torch.searchsorted(q_seg[1:], torch.arange(lo, hi, device=q.device), right=True)
        rows = state["rows"][lo:hi].long()
        there = torch.ones_like(rows, dtype=torch.bool)
        there[:, 1:] = rows[:, 1:] != rows[:, :1]  # the rest repeat the first
        there &= (rows >= 0) & (rows < (k_seg[scene + 1] - k_seg[scene])[:, None])
        at = torch.where(there, rows + k_seg[scene][:, None], 0)
        if not len(k):
            out[lo:hi] = 0
            if case["train"]:
                dq[lo:hi] = 0
            continue
        ks = k[at].float().repeat_interleave(group, 2)
        vs = v[at].float().repeat_interleave(group, 2)
        qs = q[lo:hi, None].float()
        s = ((qs * ks).sum(-1) * scale).masked_fill_(~there[..., None], -math.inf)
        s = (s - s.amax(1, keepdim=True).clamp_(min=-1e30)).exp_()
        p = s / s.sum(1, keepdim=True).clamp_(min=1e-30)
        out[lo:hi] = (p[..., None] * vs).sum(1).to(dtype)
        if case["train"]:
            do = state["grad"][lo:hi, None].float()
            dp = (do * vs).sum(-1)
            ds = (dp - (dp * p).sum(1, keepdim=True)) * p * scale
            dq[lo:hi] = (ds[..., None] * ks).sum(1).to(dtype)
            shared = (hi - lo, case["width"], case["kv_heads"], group, case["dim"])
            for total, part in ((dk, ds[..., None] * qs), (dv, p[..., None] * do)):
                total.index_add_(0, at[there], part.view(shared).sum(3)[there])
    return (out, dq, dk.to(dtype), dv.to(dtype)) if case["train"] else out


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    q, k, v = (state[n].double().requires_grad_(case["train"]) for n in ("q", "k", "v"))
    lengths = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    if case["op"] == "cross":
        attend = _exact_cross
        if case["train"] and sum(a * b for a, b in zip(*lengths)) * case["heads"] > 1 << 31:
            return None
    else:
        attend = _exact_neighbors
    q_seg, k_seg = _seg(lengths[0]), _seg(lengths[1])
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    for i in range(case["scenes"]):
        if lengths[1][i] == 0:
            continue
        mine, theirs = slice(q_seg[i], q_seg[i + 1]), slice(k_seg[i], k_seg[i + 1])
        for h in range(case["heads"]):
            for lo in range(mine.start, mine.stop, 8000):
                rows = slice(lo, min(lo + 8000, mine.stop))
                parts = [t.detach()[r, j].requires_grad_(case["train"])
                         for t, r, j in ((q, rows, h), (k, theirs, h // group), (v, theirs, h // group))]
                o = attend(state, *parts, rows, theirs) if case["train"] else attend(
                    state, *(p.detach() for p in parts), rows, theirs)
                if o is None:
                    continue
                out[rows, h] = o.detach()
                if case["train"]:
                    o.backward(state["grad"][rows, h].double())
                    for total, part, r, j in zip(grads, parts, (rows, theirs, theirs), (h, h // group, h // group)):
                        total[r, j] += part.grad if part.grad is not None else 0
    return (out, *grads) if case["train"] else out


def _exact_cross(state, q, k, v, rows, theirs):
    if state["mask"] is not None:
        kept = state["mask"][theirs].nonzero()[:, 0]
        if not len(kept):
            return None
        k, v = k[kept], v[kept]
    return torch.softmax(q @ k.T / math.sqrt(q.shape[1]), 1) @ v


def _exact_neighbors(state, q, k, v, rows, theirs):
    ids = state["rows"][rows].long()
    repeat = torch.zeros_like(ids, dtype=torch.bool)
    repeat[:, 1:] = ids[:, 1:] == ids[:, :1]
    score = torch.einsum("qd,qwd->qw", q, k[ids]) / math.sqrt(q.shape[1])
    weight = torch.softmax(score.masked_fill(repeat, -math.inf), 1)
    return torch.einsum("qw,qwd->qd", weight, v[ids])


def _exact_rotary(case, state):
    f, amplitude = _frequencies(case)
    f = f.cuda()
    n = len(f)
    out = state["x"].double().clone()
    sign = -1.0 if case["gradient"] else 1.0
    for axis in range(case["axes"]):
        place = state["positions"].reshape(len(out), -1)[:, axis].double() / (0.02 if case["axes"] > 1 else 1.0)
        turn = torch.polar(torch.full_like(place, amplitude)[:, None], sign * place[:, None] * f)[:, None]
        pair = torch.arange(axis * n, (axis + 1) * n, device="cuda")
        if case["layout"] == "half":
            first, second = pair, pair + case["part"] // 2
        else:
            first, second = 2 * pair, 2 * pair + 1
        z = torch.complex(out[..., first], out[..., second]) * turn
        out[..., first], out[..., second] = z.real, z.imag
    return out
