# SPDX-License-Identifier: Apache-2.0
"""GPU: rotary positions, cross attention and neighbour attention against
64-bit oracles (``tests/features_oracle.py``, whose bounds are derived there),
and the ways a program calls them."""

import copy
import gc
import math
import pickle

import pytest
import torch

from tests import features_oracle as fo

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=FP32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


# ---------------------------------------------------------------------------
# rotary positions


def check_rotary(x, positions, part, axes, layout, out=None, transposed=False, **plan):
    from gsa_b200 import Rotary, rotary

    r = Rotary(part, axes=axes, layout=layout, **plan)
    before = x.clone()
    got = (r.grad if transposed else r)(x, positions, out=out)
    f = rotary.frequencies(r.pairs, plan.get("base", 10000.0), plan.get("scaling"), plan.get("factor", 1.0),
                           plan.get("length"))
    want, off = fo.rotate(before, positions, f, axes, part, layout, plan.get("unit", 1.0), r.amplitude, transposed)
    bad = (got.double().cpu() - want).abs() > off
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements are too far off"
    assert torch.equal(got[..., part:], before[..., part:])
    return got


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,heads,dim,part,axes", [
    (1, 1, 8, 8, 1), (5, 3, 16, 16, 1), (33, 8, 32, 30, 3), (257, 5, 48, 36, 3), (19, 2, 64, 32, 1), (7, 9, 128, 128, 2),
    (3, 4, 40, 2, 1), (70, 1, 256, 256, 1), (6, 2, 20, 18, 3), (5, 3, 7, 6, 1), (2, 2, 300, 256, 1)])
def test_rotary_shapes(rows, heads, dim, part, axes, dtype, layout):
    x = normal(1, rows, heads, dim, dtype=dtype)
    check_rotary(x, normal(2, rows, axes, scale=4.0), part, axes, layout, unit=0.02)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, FP32])
@pytest.mark.parametrize("scaling", [None, "linear", "base", "ramp"])
def test_rotary_far_positions_and_scalings(kind, scaling):
    x = normal(3, 64, 2, 64, dtype=FP32)
    g = torch.Generator().manual_seed(4)
    far = torch.randint(0, 1 << 24, (64,), generator=g)
    far[0] = 0
    check_rotary(x, far.to(kind).cuda(), 64, 1, "half", scaling=scaling, factor=16.0, length=4096)
    check_rotary(x, far.to(kind).cuda(), 64, 1, "interleaved", transposed=True, scaling=scaling, factor=16.0, length=4096)


def test_rotary_positions_beyond_32_bits():
    x = normal(5, 8, 1, 16)
    far = (torch.arange(8) * 987654321 + (1 << 33)).cuda()
    check_rotary(x, far, 16, 1, "half")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,part", [(32, 30), (64, 48), (14, 12)])
def test_rotary_in_place_strides_and_positions_view(layout, dim, part):
    x = normal(6, 50, 3, 4, dim, dtype=BF16)
    place = normal(7, 50, 7)[:, 2:5]
    separate = check_rotary(x[:, 1], place, part, 3, layout)
    whole = x.clone()
    same = whole[:, 1]
    check_rotary(same, place, part, 3, layout, out=same)
    assert torch.equal(same, separate)
    assert torch.equal(whole[:, 0], x[:, 0]) and torch.equal(whole[:, 2], x[:, 2])
    # heads before rows, in and out; odd addresses
    t = normal(8, 4, 50, dim, dtype=BF16).transpose(0, 1)
    out = torch.empty(4, 50, dim, dtype=BF16, device="cuda").transpose(0, 1)
    check_rotary(t, place, part, 3, layout, out=out)
    odd = normal(9, 50 * 4 * dim + 1, dtype=BF16)[1:].view(50, 4, dim)
    check_rotary(odd, place, part, 3, layout)


def test_rotary_undoes_itself_and_has_its_gradient():
    from gsa_b200 import Rotary

    r = Rotary(30, axes=3)
    x, place = normal(10, 40, 2, 32), normal(11, 40, 3)
    assert torch.allclose(r.grad(r(x, place), place), x, atol=1e-5)
    x.requires_grad_()
    d = normal(12, 40, 2, 32)
    r(x, place).backward(d)
    assert torch.equal(x.grad, r.grad(d, place))
    y = normal(13, 40, 2, 32)  # <turned x, d> = <x, gradient>, by differences
    h = 2.0**-6
    moved = [(r(x.detach() + s * h * y, place).double() * d.double()).sum() for s in (1, -1)]
    # linear in x: only the 32-bit roundings differ, 2^-20 of the sums of |x d| / h
    bound = 2.0**-20 * ((x.detach().abs() + y.abs()).double() * d.abs().double()).sum() * 2 / h
    assert (((moved[0] - moved[1]) / (2 * h)) - (x.grad.double() * y.double()).sum()).abs() < bound


def test_rotary_refuses():
    from gsa_b200 import Rotary

    r = Rotary(32, axes=1)
    x, place = normal(1, 6, 2, 32), torch.arange(6).cuda()
    assert r(x[:0], place[:0]).shape == (0, 2, 32)
    for bad in [(x[..., :16], place), (x[..., ::2], place), (x.double(), place), (x[0], place), (x, place[:5]),
                (x, place.double()), (x, place.cpu()), (x, place[:, None].expand(6, 2)), (x[:, :0], place)]:
        with pytest.raises(ValueError):
            r(*bad)
    for out in (x[:5], x.half(), x.cpu(), x[:, :1].expand(6, 2, 32), x.view(2, 6, 32).transpose(0, 1)):
        with pytest.raises(ValueError):
            r(x, place, out=out)


def test_writes_are_known_to_autograd():
    from gsa_b200 import Rotary, ScenePairs, cross_attention

    q, k, v, q_seg, k_seg = attention_inputs(195, ([40], [60]), 2, 2, 32, BF16)
    pairs, r = ScenePairs(q_seg, k_seg), Rotary(32)
    for write in (lambda t: r(q, torch.arange(40).cuda(), out=t), lambda t: cross_attention(q, k, v, pairs, out=t)):
        buffer = torch.ones_like(q)
        leaf = normal(196, *q.shape, dtype=BF16).requires_grad_()
        product = leaf * buffer
        write(buffer)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
    with torch.inference_mode():
        out = torch.empty_like(q)
        assert cross_attention(q, k, v, pairs, out=out) is out
    empty = q[:0]
    assert r(empty, torch.arange(0).cuda(), out=torch.empty((0, 2, 64), dtype=BF16, device="cuda")[..., :32]).shape == empty.shape
    with pytest.raises(ValueError):
        Rotary(32, amplitude=1e39)


def test_pairs_end_before_another_stream_has_read_them():
    from gsa_b200 import ScenePairs, cross_attention

    q, k, v, q_seg, k_seg = attention_inputs(197, ([500, 700], [900, 400]), 2, 2, 64, BF16)
    pairs = ScenePairs(q_seg, k_seg)
    want = cross_attention(q, k, v, pairs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(50):  # work that the call below waits for
            (q.float() @ q.float().mT)
        got = cross_attention(q, k, v, pairs)
    del pairs
    later = [torch.zeros(7, dtype=torch.int32, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(later) == 64


# ---------------------------------------------------------------------------
# attention


def lengths_case(name):
    return {
        "one": ([1], [1]),
        "row on many": ([1], [3001]),
        "few rows on many": ([3, 2], [1500, 900]),
        "ragged": ([1, 0, 130, 64, 5, 129], [200, 7, 0, 129, 1, 65]),
        "tiles": ([128, 256], [128, 256]),
        "many rows": ([700], [70]),
        "no keys": ([5, 9], [0, 0]),
        "no queries": ([0, 0], [4, 9]),
    }[name]


def attention_inputs(seed, lengths, heads, kv_heads, dim, dtype, layout="packed", scale=1.0):
    q_seg, k_seg = fo.seg_of(lengths[0]), fo.seg_of(lengths[1])
    nq, nk = q_seg[-1], k_seg[-1]
    if layout == "fused":  # one tensor of keys and values, rows of queries inside wider ones
        q = normal(seed, nq, heads + 1, dim, dtype=dtype, scale=scale)[:, 1:]
        kv = normal(seed + 1, nk, 2, kv_heads, dim, dtype=dtype)
        k, v = kv[:, 0], kv[:, 1]
    elif layout == "heads first":
        q = normal(seed, heads, nq, dim, dtype=dtype, scale=scale).transpose(0, 1)
        k = normal(seed + 1, kv_heads, nk, dim, dtype=dtype).transpose(0, 1)
        v = normal(seed + 2, kv_heads, nk, dim, dtype=dtype).transpose(0, 1)
    else:
        q = normal(seed, nq, heads, dim, dtype=dtype, scale=scale)
        k, v = normal(seed + 1, nk, kv_heads, dim, dtype=dtype), normal(seed + 2, nk, kv_heads, dim, dtype=dtype)
    return q, k, v, q_seg, k_seg


def check_cross(q, k, v, q_seg, k_seg, mask=None, scale=None, grads=True, seed=77):
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    out, lse = cross_attention(q, k, v, pairs, mask=mask, scale=scale, return_lse=True)
    dout = normal(seed, *q.shape, dtype=q.dtype) if grads else None
    want = fo.Attention(q, k, v, q_seg, k_seg, mask=mask, scale=scale, dout=dout)
    want.close("out", out)
    want.close("lse", lse)
    if grads:
        got = cross_attention_grad(dout, q, k, v, out, lse, pairs, mask=mask, scale=scale)
        for name, t in zip(("dq", "dk", "dv"), got):
            want.close(name, t)
    pairs.check()
    return want


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [8, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("name", ["one", "row on many", "few rows on many", "ragged", "tiles", "many rows"])
def test_cross_sizes(name, dim, dtype):
    check_cross(*attention_inputs(20, lengths_case(name), 2, 2, dim, dtype))


@pytest.mark.parametrize("dim", [16, 96])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 1), (3, 3), (10, 2)])
@pytest.mark.parametrize("layout", ["packed", "fused", "heads first"])
def test_cross_heads_and_layouts(layout, heads, kv_heads, dim):
    check_cross(*attention_inputs(30, lengths_case("ragged"), heads, kv_heads, dim, BF16, layout))


@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("name", ["no keys", "no queries"])
def test_cross_empty_sides(name, dim):
    from gsa_b200 import ScenePairs, cross_attention

    q, k, v, q_seg, k_seg = attention_inputs(40, lengths_case(name), 4, 2, dim, BF16)
    check_cross(q, k, v, q_seg, k_seg)
    out, lse = cross_attention(q, k, v, ScenePairs(q_seg, k_seg), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (48, FP16), (128, BF16)])
@pytest.mark.parametrize("name", ["ragged", "few rows on many", "tiles"])
def test_cross_masked_keys_may_hold_anything(name, dim, dtype):
    q, k, v, q_seg, k_seg = attention_inputs(50, lengths_case(name), 4, 2, dim, dtype)
    g = torch.Generator().manual_seed(51)
    mask = torch.rand(len(k), generator=g) < 0.6
    mask[k_seg[-2]:] = False  # a whole scene shut
    mask[k_seg[0]:k_seg[0] + min(128, k_seg[1])] = False  # and a first tile
    mask = mask.cuda()
    shut = (~mask).nonzero()[:, 0]
    for i, bad in enumerate((math.nan, math.inf, -math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max)):
        k[shut[i::5]] = bad
        v[shut[i::7]] = bad
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[shut] = 0
    clean_v[shut] = 0
    want = check_cross(q, k, v, q_seg, k_seg, mask=mask)
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    one = cross_attention(q, k, v, pairs, mask=mask, return_lse=True)
    two = cross_attention(q, clean_k, clean_v, pairs, mask=mask.to(torch.uint8), return_lse=True)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    d = normal(52, *q.shape, dtype=dtype)
    dq, dk, dv = cross_attention_grad(d, q, k, v, *one, pairs, mask=mask)
    assert not dk[shut].any() and not dv[shut].any()
    empty = want.lse == -math.inf
    assert empty.any() and not dq[empty.cuda()].any()


@pytest.mark.parametrize("name", ["few rows on many", "many rows", "ragged"])
@pytest.mark.parametrize("dim", [64, 128])
def test_cross_growing_scores(name, dim):
    # scores in the tens that grow along the keys: the running maximum moves
    q, k, v, q_seg, k_seg = attention_inputs(60, lengths_case(name), 2, 1, dim, BF16, scale=3.0)
    k *= torch.linspace(0.1, 2.0, len(k), device="cuda", dtype=torch.float32)[:, None, None].to(BF16)
    check_cross(q, k, v, q_seg, k_seg)
    check_cross(q, k, v, q_seg, k_seg, scale=0.001)


def test_cross_infinities_and_nans_of_open_keys_and_queries():
    from gsa_b200 import ScenePairs, cross_attention

    for n_k in (60, 3000):  # one part, and split keys
        q, k, v, q_seg, k_seg = attention_inputs(70, ([6], [n_k]), 1, 1, 32, BF16)
        q[1] = math.nan
        k[n_k // 2, 0, 3] = math.inf  # scores of +inf, or -inf, by the query's sign
        v[n_k - 1, 0, 5] = math.inf
        out, lse = cross_attention(q, k, v, ScenePairs(q_seg, k_seg), return_lse=True)
        s = (q[:, 0].double() @ k[:, 0].double().T) * 32**-0.5
        want = torch.softmax(s, 1) @ v[:, 0].double()
        for r in range(6):
            if s[r].isnan().any() or (s[r] == math.inf).any():
                assert out[r].isnan().all() and lse[r].isnan().all()
            else:
                assert torch.equal(out[r, 0].isinf(), want[r].isinf())
                rest = ~want[r].isinf()
                assert torch.allclose(out[r, 0].double()[rest], want[r][rest], atol=0.05)
        # nothing but -inf: no softmax
        k[:, 0, :] = 0
        k[:, 0, 0] = -math.inf
        q[:] = 1
        out, lse = cross_attention(q, k, v, ScenePairs(q_seg, k_seg), return_lse=True)
        assert out.isnan().all()


def test_cross_long_keys_of_many_scenes():
    check_cross(*attention_inputs(80, ([1, 3, 1, 2], [9000, 1, 12000, 4097]), 4, 2, 64, FP16))


def test_cross_writes_nothing_but_its_rows():
    from gsa_b200 import ScenePairs, cross_attention

    for lengths in (([130, 5], [300, 70]), ([1], [4000])):
        q, k, v, q_seg, k_seg = attention_inputs(90, lengths, 2, 2, 40, BF16)
        whole = torch.full((len(q) + 6, 4, 48), 7.0, dtype=BF16, device="cuda")
        out = whole[3:-3, 1:3, :40]
        cross_attention(q, k, v, ScenePairs(q_seg, k_seg), out=out)
        assert torch.equal(out, cross_attention(q, k, v, ScenePairs(q_seg, k_seg)))
        out.fill_(7.0)
        assert (whole == 7.0).all()


def test_cross_gradients_by_differences():
    # the 64-bit output moved along a direction, against the kernel's gradient
    q, k, v, q_seg, k_seg = attention_inputs(100, lengths_case("ragged"), 4, 2, 64, BF16)
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    d = normal(101, *q.shape, dtype=BF16)
    out, lse = cross_attention(q, k, v, pairs, return_lse=True)
    grads = cross_attention_grad(d, q, k, v, out, lse, pairs)
    want = fo.Attention(q, k, v, q_seg, k_seg, dout=d)
    for i, (name, t) in enumerate((("dq", q), ("dk", k), ("dv", v))):
        step = torch.randn(t.shape, generator=torch.Generator().manual_seed(102 + i), dtype=torch.float64)
        h = 1e-4
        moved = []
        for s in (1, -1):
            xs = [x.double().cpu() + (s * h * step if x is t else 0) for x in (q, k, v)]
            moved.append((fo.Attention(*xs, q_seg, k_seg).out * d.double().cpu()).sum())
        slope = (moved[0] - moved[1]) / (2 * h)
        bound = (getattr(want, name + "_off") * step.abs()).sum() + 1e-6 * slope.abs() + 1e-4
        assert ((grads[i].double().cpu() * step).sum() - slope).abs() < bound, name


def neighbor_ids(seed, lengths, width, kind):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n, m in zip(*lengths):
        ids = torch.randint(0, max(m, 1), (n, width), generator=g)
        if kind == "radius":  # ascending, then the first again
            ids = ids.sort(1).values
            found = torch.randint(0, width + 1, (n, 1), generator=g)
            ids = torch.where(torch.arange(width) < found, ids, ids[:, :1])
            ids = torch.where(found > 0, ids, 0)
        else:  # absent entries of every sort, whole rows of them
            bad = torch.rand(n, width, generator=g)
            ids = torch.where(bad < 0.1, -1, ids)
            ids = torch.where((bad > 0.1) & (bad < 0.2), m, ids)
            ids = torch.where(bad > 0.95, 2**31 - 1, ids)
            ids = torch.where((bad > 0.9) & (bad < 0.95), -(2**31), ids)
            ids[::5] = -1
        out.append(ids)
    return torch.cat(out).int().cuda()


def check_neighbors(q, k, v, ids, q_seg, k_seg, padded=True, scale=None, seed=78):
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    out, lse = neighbor_attention(q, k, v, ids, pairs, padded=padded, scale=scale, return_lse=True)
    dout = normal(seed, *q.shape, dtype=q.dtype)
    want = fo.Attention(q, k, v, q_seg, k_seg, ids=ids, padded=padded, scale=scale, dout=dout)
    want.close("out", out)
    want.close("lse", lse)
    got = neighbor_attention_grad(dout, q, k, v, ids, out, lse, pairs, padded=padded, scale=scale)
    for name, t in zip(("dq", "dk", "dv"), got):
        want.close(name, t)
    return want


@pytest.mark.parametrize("kind,padded", [("radius", True), ("radius", False), ("absent", True), ("absent", False)])
@pytest.mark.parametrize("dtype,dim,width", [(BF16, 32, 32), (FP16, 8, 3), (FP32, 24, 17), (BF16, 128, 8), (FP32, 128, 32),
                                             (FP16, 72, 1), (FP32, 8, 5), (BF16, 16, 31)])
def test_neighbors(dtype, dim, width, kind, padded):
    lengths = lengths_case("ragged")
    q, k, v, q_seg, k_seg = attention_inputs(110, lengths, 4, 2, dim, dtype)
    check_neighbors(q, k, v, neighbor_ids(111, lengths, width, kind), q_seg, k_seg, padded)


@pytest.mark.parametrize("heads,kv_heads,layout", [(1, 1, "packed"), (6, 1, "fused"), (5, 5, "heads first"), (12, 3, "packed")])
@pytest.mark.parametrize("name", ["one", "few rows on many", "many rows", "no keys", "no queries"])
def test_neighbors_heads_layouts_and_lengths(name, heads, kv_heads, layout):
    lengths = lengths_case(name)
    q, k, v, q_seg, k_seg = attention_inputs(120, lengths, heads, kv_heads, 40, FP32, layout)
    check_neighbors(q, k, v, neighbor_ids(121, lengths, 9, "absent"), q_seg, k_seg)


def test_neighbors_many_keys_and_one_key_for_all():
    # keys of three digits of the sort, and a key that every entry names
    lengths = ([3000], [300_000])
    q, k, v, q_seg, k_seg = attention_inputs(130, lengths, 2, 1, 16, FP32)
    ids = neighbor_ids(131, lengths, 7, "absent")
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    out, lse = neighbor_attention(q, k, v, ids, pairs, return_lse=True)
    d = normal(132, *q.shape)
    _, dk, dv = neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    # the same on the keys that are named, packed
    named, at = ids[(ids >= 0) & (ids < 300_000)].long().unique(return_inverse=True)
    packed = torch.full_like(ids, -1)
    packed[(ids >= 0) & (ids < 300_000)] = at.int()
    want = fo.Attention(q, k[named], v[named], q_seg, [0, len(named)], ids=packed, dout=d)
    want.close("out", out)
    want.close("dk", dk[named])
    want.close("dv", dv[named])
    rest = torch.ones(300_000, dtype=torch.bool, device="cuda")
    rest[named] = False
    assert not dk[rest].any() and not dv[rest].any()
    q, k, v, q_seg, k_seg = attention_inputs(133, ([900], [5]), 2, 1, 16, FP32)
    check_neighbors(q, k, v, torch.full((900, 4), 3, dtype=torch.int32, device="cuda"), q_seg, k_seg, padded=False)


def test_neighbor_gradients_by_differences():
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    lengths = lengths_case("ragged")
    q, k, v, q_seg, k_seg = attention_inputs(140, lengths, 2, 2, 16, FP32)
    ids = neighbor_ids(141, lengths, 6, "radius")
    pairs = ScenePairs(q_seg, k_seg)
    d = normal(142, *q.shape)
    out, lse = neighbor_attention(q, k, v, ids, pairs, return_lse=True)
    grads = neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    h = 2.0**-8
    for i, t in enumerate((q, k, v)):
        step = normal(143 + i, *t.shape)
        moved = [(neighbor_attention(*(x + s * h * step if x is t else x for x in (q, k, v)), ids, pairs).double()
                  * d.double()).sum() for s in (1, -1)]
        slope = ((moved[0] - moved[1]) / (2 * h)).item()
        got = (grads[i].double() * step.double()).sum().item()
        # 32-bit outputs over 2 h: 2^-18 of sum |d| / h; third derivatives: h^2 of sum |d|
        assert abs(got - slope) < d.abs().double().sum().item() * (2.0**-18 / h + h * h)


# ---------------------------------------------------------------------------
# how programs call them


def both(kind, lengths=([130, 64, 1], [70, 129, 900]), dim=32, dtype=BF16, seed=150):
    """A forward and a gradient call of either attention on the same rows."""
    from gsa_b200 import ScenePairs, attention as at

    q, k, v, q_seg, k_seg = attention_inputs(seed, lengths, 4, 2, dim, dtype)
    pairs = ScenePairs(q_seg, k_seg)
    ids = neighbor_ids(seed + 5, lengths, 8, "radius")
    d = normal(seed + 6, *q.shape, dtype=dtype)
    if kind == "cross":
        def forward(**kw):
            return at.cross_attention(q, k, v, pairs, **kw)

        def backward(out, lse):
            return at.cross_attention_grad(d, q, k, v, out, lse, pairs)
    else:
        def forward(**kw):
            return at.neighbor_attention(q, k, v, ids, pairs, **kw)

        def backward(out, lse):
            return at.neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    return (q, k, v), d, forward, backward


@pytest.mark.parametrize("kind", ["cross", "neighbor"])
def test_the_same_bits_again(kind):
    _, _, forward, backward = both(kind, ([400, 9], [1900, 300]))
    out, lse = forward(return_lse=True)
    first = backward(out, lse)
    for _ in range(5):
        o, m = forward(return_lse=True)
        assert torch.equal(o, out) and torch.equal(m, lse)
        assert all(torch.equal(a, b) for a, b in zip(first, backward(o, m)))


@pytest.mark.parametrize("kind", ["cross", "neighbor"])
def test_autograd_is_the_gradient_call(kind):
    leaves, d, forward, backward = both(kind)
    out, lse = forward(return_lse=True)
    want = backward(out, lse)
    for t in leaves:
        t.requires_grad_()
    got = forward()
    assert torch.equal(got, out)
    got.backward(d)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    for t in leaves:
        t.grad = None
    forward().float().sum().backward()  # an expanded gradient
    assert all(t.grad is not None and t.grad.isfinite().all() for t in leaves)
    with torch.no_grad():
        assert not forward().requires_grad


@pytest.mark.parametrize("kind", ["cross", "neighbor"])
def test_streams_and_captured_graphs(kind):
    leaves, d, forward, backward = both(kind, ([5, 300], [3000, 70]))
    out, lse = forward(return_lse=True)
    want = backward(out, lse)
    torch.cuda.synchronize()
    # two streams at once
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                o, m = forward(return_lse=True)
                results.append((o, m, *backward(o, m)))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, (out, lse, *want)))
    # two captured graphs, replayed at once on new inputs
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, m = forward(return_lse=True)
            got = (o, m, *backward(o, m))
        graphs.append((g, got))
    for t in leaves:
        t.copy_(t.flip(-1) * 0.5)
    out, lse = forward(return_lse=True)
    want = backward(out, lse)
    torch.cuda.synchronize()
    for s, (g, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, (out, lse, *want)))


def test_expanded_inputs_and_gradients():
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(170, ([70, 3], [200, 60]), 4, 4, 32, BF16)
    pairs = ScenePairs(q_seg, k_seg)
    one = [q[:1].expand(73, 4, 32), k[:, :1].expand(260, 4, 32), v[:1, :1].expand(260, 4, 32)]
    d = normal(171, 1, 1, 32, dtype=BF16).expand(73, 4, 32)
    same = [t.contiguous() for t in one]
    out, lse = cross_attention(*one, pairs, return_lse=True)
    assert torch.equal(out, cross_attention(*same, pairs))
    got = cross_attention_grad(d, *one, out, lse, pairs)
    assert all(torch.equal(a, b) for a, b in zip(got, cross_attention_grad(d.contiguous(), *same, out, lse, pairs)))
    # broadcast leaves get their sums
    leaf = k[:, :1].clone().requires_grad_()
    cross_attention(q, leaf.expand(260, 4, 32), v, pairs).backward(same[0])
    whole = k[:, :1].expand(260, 4, 32).clone().requires_grad_()
    cross_attention(q, whole, v, pairs).backward(same[0])
    assert torch.equal(leaf.grad, whole.grad.sum(1, keepdim=True))


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (32, FP16), (128, BF16)])
@pytest.mark.parametrize("n_k", [1, 2, 5, 64])
def test_cross_gradients_of_few_keys(n_k, dim, dtype):
    # keys of one tile: delta comes from P and dP, not from the output
    q, k, v, q_seg, k_seg = attention_inputs(180, ([130], [n_k]), 2, 1, dim, dtype)
    want = check_cross(q, k, v, q_seg, k_seg, scale=0.01)
    assert want.dq.abs().max() > 0 or n_k == 1


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16)])
def test_cross_gradients_of_few_keys_beside_many(dim, dtype):
    # a scene of one tile of keys keeps its own path beside one of several, so
    # its gradients are the bits that it has alone
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(185, ([130, 40], [5, 300]), 2, 1, dim, dtype)
    check_cross(q, k, v, q_seg, k_seg)
    d = normal(186, *q.shape, dtype=dtype)

    def gradients(d, q, k, v, pairs):
        out, lse = cross_attention(q, k, v, pairs, return_lse=True)
        return cross_attention_grad(d, q, k, v, out, lse, pairs)

    both = gradients(d, q, k, v, ScenePairs(q_seg, k_seg))
    alone = gradients(d[:130], q[:130], k[:5], v[:5], ScenePairs([0, 130], [0, 5]))
    for got, want in zip(both, alone):
        assert torch.equal(got[: len(want)], want)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (24, FP16)])
@pytest.mark.parametrize("kind", ["one", "masked", "beside"])
def test_cross_gradients_of_a_single_key(kind, dim, dtype):
    # one open key: its weight is 1 whatever the score, so dq and dk are 0
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    n_k = {"one": [1, 1], "masked": [7, 60], "beside": [1, 300]}[kind]
    q, k, v, q_seg, k_seg = attention_inputs(200, ([140, 9], n_k), 4, 2, dim, dtype, scale=8.0)
    mask = None
    if kind == "masked":
        mask = torch.zeros(67, dtype=torch.bool, device="cuda")
        mask[[3, 66]] = True
    check_cross(q, k, v, q_seg, k_seg, mask=mask)
    pairs, d = ScenePairs(q_seg, k_seg), normal(201, *q.shape, dtype=dtype)
    out, lse = cross_attention(q, k, v, pairs, mask=mask, return_lse=True)
    dq, dk, dv = cross_attention_grad(d, q, k, v, out, lse, pairs, mask=mask)
    whole = kind != "beside"
    assert not dq[: None if whole else 140].any() and not dk[: None if whole else 1].any() and dv[:4].any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("width,dim", [(1, 40), (9, 64), (32, 128)])
def test_neighbor_gradients_of_a_single_key(width, dim, dtype):
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(205, ([50, 3], [20, 6]), 4, 2, dim, dtype, scale=8.0)
    ids = (torch.arange(53, device="cuda", dtype=torch.int32) % 6)[:, None].repeat(1, width)
    pairs, d = ScenePairs(q_seg, k_seg), normal(206, *q.shape, dtype=dtype)
    out, lse = neighbor_attention(q, k, v, ids, pairs, return_lse=True)
    dq, dk, dv = neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    assert not dq.any() and not dk.any() and dv.any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("entries", [2, 3, 8])
def test_neighbor_gradients_do_not_see_the_outputs_rounding(entries, dtype):
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    dim, n_k = 48, 40
    q, k, v, q_seg, k_seg = attention_inputs(210, ([300], [n_k]), 2, 2, dim, dtype)
    first = torch.arange(300, device="cuda")[:, None] * 7
    ids = ((first + 3 * torch.arange(entries, device="cuda")) % n_k).int()
    pairs, d = ScenePairs(q_seg, k_seg), normal(211, *q.shape, dtype=dtype)
    out, lse = neighbor_attention(q, k, v, ids, pairs, return_lse=True)
    dq, dk, _ = neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    want = fo.Attention(q, k, v, q_seg, k_seg, ids=ids, dout=d)
    Q, K, V, D = (t.double().cpu().transpose(0, 1) for t in (q, k, v, d))
    count = fo.Attention.counts(ids.cpu().long(), n_k, True)
    p = torch.softmax((Q @ K.mT * dim**-0.5).masked_fill(count == 0, -torch.inf), -1)
    # Besides the result's own half step only 32-bit roundings: sums of 48
    # products, below 2^-17 of the sums of magnitudes, in dp, delta and c, and
    # in p and ds the scores' (below 2^-17 of |q| |k| / sqrt(dim) < 2^3) and
    # lse's: 2^-13 of the magnitudes covers them, where bf16's `out` is rounded
    # by 2^-9 and more of them and fp16's by 2^-12.
    size = p * (D.abs() @ V.abs().mT + (D.abs() * (p @ V.abs())).sum(-1, keepdim=True))
    half = torch.finfo(dtype).eps / 2
    for got, exact, near in ((dq, want.dq, size @ K.abs()), (dk, want.dk, size.mT @ Q.abs())):
        off = half * exact.abs() + 2.0**-13 * dim**-0.5 * near.transpose(0, 1) + 2.0**-25
        error = (got.double().cpu() - exact).abs()
        assert (error <= off).all(), float((error / off).max())
        # and the errors together stay near the half step's alone
        assert error.norm() <= 0.75 * half * exact.norm()


@pytest.mark.parametrize("scale", [2.0**-24, 2.0**-12, 4.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cross_scales(scale, dtype):
    # scores of a few units in each case
    size = (1.0 / scale / 30) ** 0.5 if scale < 1 else 0.2
    q, k, v, q_seg, k_seg = attention_inputs(190, lengths_case("few rows on many"), 2, 1, 64, dtype, scale=min(size, 100.0))
    k *= min(size, 100.0)
    check_cross(q, k, v, q_seg, k_seg, scale=scale)


def test_levels_of_a_hierarchy_together():
    """A step of an attention network on two rooms: rows and levels of the
    batched hierarchy, queries and keys turned by the points' coordinates,
    attention along the radius rows, then of that level's points to the
    coarser one; forward and backward, eager and captured."""
    from gsa_b200 import Rotary, cross_attention, cross_attention_grad, hierarchy as hz, neighbor_attention, neighbor_attention_grad, scenes

    sizes, radii, B, H, D = (3000, 750, 187, 46, 11), (0.2, 0.3, 0.5, 0.9), 2, 4, 32
    X = scenes.room_batch([301, 302], n=sizes[0])
    batch = hz.Batch(sizes, radii)
    rows = batch.run(X)["ball1"]
    near, across = batch.pairs(B, 1, 1), batch.pairs(B, 1, 2)
    place = X[:, : sizes[1]].reshape(-1, 3)
    coarse = X[:, : sizes[2]].reshape(-1, 3)
    turn = Rotary(30, axes=3, unit=0.05)
    n, m = B * sizes[1], B * sizes[2]
    q, k, v = (normal(200 + i, n, H, D, dtype=BF16) for i in range(3))
    k2, v2 = normal(203, m, 2, D, dtype=BF16), normal(204, m, 2, D, dtype=BF16)
    d = normal(205, n, H, D, dtype=BF16)

    def step():
        a, b = turn(q, place), turn(k, place)
        x, lse = neighbor_attention(a, b, v, rows, near, return_lse=True)
        c, e = turn(x, place), turn(k2, coarse)
        y, lse2 = cross_attention(c, e, v2, across, return_lse=True)
        dc, de, dv2 = cross_attention_grad(d, c, e, v2, y, lse2, across)
        dx = turn.grad(dc, place)
        da, db, dv = neighbor_attention_grad(dx, a, b, v, rows, x, lse, near)
        return (x, lse, y, lse2, dx, dv2, dv, turn.grad(da, place), turn.grad(db, place), turn.grad(de, coarse), a, b, c, e, da, db)

    got = step()
    x, lse, y, lse2, dx, dv2, dv = got[:7]
    a, b, c, e, da, db = got[10:]
    near_seg, across_seg = fo.seg_of([sizes[1]] * B), fo.seg_of([sizes[2]] * B)
    want = fo.Attention(a, b, v, near_seg, near_seg, ids=rows, dout=dx)
    for name, t in (("out", x), ("lse", lse), ("dq", da), ("dk", db), ("dv", dv)):
        want.close(name, t)
    want = fo.Attention(c, e, v2, near_seg, across_seg, dout=d)
    for name, t in (("out", y), ("lse", lse2), ("dv", dv2)):
        want.close(name, t)
    # the same through autograd
    leaves = [t.clone().requires_grad_() for t in (q, k, v, k2, v2)]
    f = neighbor_attention(turn(leaves[0], place), turn(leaves[1], place), leaves[2], rows, near)
    cross_attention(turn(f, place), turn(leaves[3], coarse), leaves[4], across).backward(d)
    for leaf, t in zip(leaves, (got[7], got[8], dv, got[9], dv2)):
        assert torch.equal(leaf.grad, t)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step()
    for t in (q, v):
        t.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(captured, step()))
    near.check()
    across.check()


def test_attention_refuses():
    from gsa_b200 import ScenePairs, attention as at

    q, k, v, q_seg, k_seg = attention_inputs(160, ([5, 4], [6, 3]), 4, 2, 16, BF16)
    pairs = ScenePairs(q_seg, k_seg)
    ids = torch.zeros(9, 3, dtype=torch.int32, device="cuda")
    out, lse = at.cross_attention(q, k, v, pairs, return_lse=True)
    odd = normal(1, 9 * 64 + 1, dtype=BF16)[1:].view(9, 4, 16)
    bad = [dict(q=q.float()), dict(q=q.double()), dict(q=q.half()), dict(k=k.half()), dict(v=v[:8]), dict(q=q[:8]),
           dict(q=q[:, :3]), dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), dict(q=odd), dict(q=q.cpu()),
           dict(v=v[:, :1]), dict(k=k[..., :8]), dict(q=q[0]), dict(pairs=None), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=math.nan), dict(pairs=ScenePairs([0, 9], [0, 8])), dict(out=out[:8]), dict(out=out.float()),
           dict(out=q), dict(out=out[:, :1].expand(9, 4, 16)), dict(out=odd)]
    for change in bad + [dict(mask=torch.ones(8, dtype=torch.bool, device="cuda")), dict(mask=torch.ones(9)),
                         dict(mask=torch.ones(9, device="cuda"))]:
        args = dict(q=q, k=k, v=v, pairs=pairs)
        args.update(change)
        with pytest.raises(ValueError):
            at.cross_attention(**args)
    q.requires_grad_()
    for call in (lambda: at.cross_attention(q, k, v, pairs, out=out), lambda: at.neighbor_attention(q, k, v, ids, pairs, out=out)):
        with pytest.raises(ValueError):
            call()
    q.requires_grad_(False)
    with pytest.raises(ValueError):
        at.cross_attention(normal(1, 9, 65, 16, dtype=BF16), normal(1, 9, 1, 16, dtype=BF16), normal(2, 9, 1, 16, dtype=BF16), pairs)
    for change in bad[1:] + [dict(rows=ids[:8]), dict(rows=ids.long()), dict(rows=ids[:, :0]), dict(rows=ids.cpu()),
                             dict(rows=torch.zeros(9, 33, dtype=torch.int32, device="cuda")), dict(rows=ids.T)]:
        if "q" in change and change["q"].dtype == FP16:
            continue  # q alone differs from k: covered by k
        args = dict(q=q, k=k, v=v, rows=ids, pairs=pairs)
        args.update(change)
        with pytest.raises(ValueError):
            at.neighbor_attention(**args)
    for change in [dict(dout=q[:8]), dict(dout=q.float()), dict(out=out[:8]), dict(lse=lse.double()), dict(lse=lse[:8]),
                   dict(lse=lse.T), dict(dout=odd)]:
        args = dict(dout=q, q=q, k=k, v=v, out=out, lse=lse, pairs=pairs)
        args.update(change)
        with pytest.raises(ValueError):
            at.cross_attention_grad(**args)
        with pytest.raises(ValueError):
            at.neighbor_attention_grad(rows=ids, **args)


def test_copies_and_pickles_outlive_their_originals():
    from gsa_b200 import Rotary, ScenePairs, cross_attention

    q, k, v, q_seg, k_seg = attention_inputs(300, ([70, 3], [200, 60]), 2, 2, 32, BF16)
    place = normal(301, 73, 3)
    r, pairs = Rotary(30, axes=3), ScenePairs(q_seg, k_seg)
    turned, want = r(q, place), cross_attention(q, k, v, pairs)
    copies = [(copy.deepcopy(r), copy.deepcopy(pairs)), (copy.copy(r), copy.copy(pairs)), pickle.loads(pickle.dumps((r, pairs)))]
    del r, pairs
    gc.collect()
    later = [torch.full((7,), -1, dtype=torch.int32, device="cuda") for _ in range(64)]
    for turn, twin in copies:
        assert torch.equal(turn(q, place), turned) and torch.equal(cross_attention(q, k, v, twin), want)
        twin.check()
    assert len(later) == 64


@pytest.mark.parametrize("kind", ["cross", "neighbor"])
def test_gradients_that_start_anywhere(kind):
    # one row behind three columns, and a view into a flat buffer: contiguous
    # as torch counts, but not on 16 bytes
    for lengths in (([1], [70]), ([130, 64], [70, 129])):
        leaves, d, forward, backward = both(kind, lengths)
        out, lse = forward(return_lse=True)
        want = backward(out, lse)
        for t in leaves:
            t.requires_grad_()
        n = len(d)
        torch.cat((d.new_zeros(n, 3), forward().flatten(1)), 1).backward(torch.cat((d.new_ones(n, 3), d.flatten(1)), 1))
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
        for t in leaves:
            t.grad = None
        flat = torch.cat((d.new_zeros(1), d.flatten()))[1:].view_as(d)
        assert flat.is_contiguous() and flat.data_ptr() % 16
        forward().backward(flat)
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_rotary_gradients_have_gradients():
    from gsa_b200 import Rotary

    r = Rotary(30, axes=3, layout="interleaved", amplitude=1.5)
    place = normal(321, 40, 3)
    d, e = normal(322, 40, 2, 32).requires_grad_(), normal(323, 40, 2, 32)
    r.grad(d, place).backward(e)  # linear in d, its gradient the turn itself
    assert torch.equal(d.grad, r(e, place))
    x = normal(324, 40, 2, 32).requires_grad_()
    d = d.detach().requires_grad_()
    (dx,) = torch.autograd.grad(r(x, place), x, d, create_graph=True)
    assert torch.equal(dx, r.grad(d.detach(), place))
    dx.backward(e)
    assert torch.equal(d.grad, r(e, place)) and x.grad is None
    with pytest.raises(ValueError):
        r.grad(d, place, out=torch.empty_like(e))


@pytest.mark.parametrize("n_k", [60, 400, 3000])
def test_cross_rows_of_minus_infinity_have_no_gradients(n_k):
    # no softmax: NaN, which the gradient's weights have too, in one part and
    # in several
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(310, ([6, 4], [n_k, 5]), 1, 1, 32, BF16)
    q[:6], k[:n_k] = 1.0, 0.0
    k[:n_k, 0, 0] = -math.inf
    pairs, d = ScenePairs(q_seg, k_seg), normal(311, *q.shape, dtype=BF16)
    out, lse = cross_attention(q, k, v, pairs, return_lse=True)
    assert out[:6].isnan().all() and lse[:6].isnan().all()
    assert out[6:].isfinite().all() and lse[6:].isfinite().all()
    dq, dk, dv = cross_attention_grad(d, q, k, v, out, lse, pairs)
    assert dq[:6].isnan().all() and dk[:n_k].isnan().all() and dv[:n_k].isnan().all()
    assert dq[6:].isfinite().all() and dk[n_k:].isfinite().all() and dv[n_k:].isfinite().all()


def test_the_error_flag_of_another_stream_is_waited_for():
    from gsa_b200 import ScenePairs

    pairs = ScenePairs([0, 4], [0, 4])
    pairs.check()
    x, side = normal(330, 4096, 4096), torch.cuda.Stream()

    def late(flag, times):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(times):  # some milliseconds before the flag is set
                x @ x
            flag.fill_(1)

    late(torch.zeros(1, dtype=torch.int32, device="cuda"), 1)  # kernels loaded
    torch.cuda.synchronize()
    late(pairs._ints[-1:], 40)
    assert not side.query()
    with pytest.raises(RuntimeError):
        pairs.check()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("beside", [1100, 1500, 2100])
@pytest.mark.parametrize("n_k", [1, 2, 5, 64])
def test_cross_gradients_of_few_keys_do_not_see_longer_scenes(n_k, beside, dim, dtype):
    # whatever the longest scene of the batch, a short one has the bits that it
    # has alone, and exactly 0 where its queries have one key
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(340, ([130, 40], [n_k, beside]), 2, 1, dim, dtype)
    d = normal(341, *q.shape, dtype=dtype)

    def gradients(d, q, k, v, pairs):
        out, lse = cross_attention(q, k, v, pairs, return_lse=True)
        return cross_attention_grad(d, q, k, v, out, lse, pairs)

    both = gradients(d, q, k, v, ScenePairs(q_seg, k_seg))
    alone = gradients(d[:130], q[:130], k[:n_k], v[:n_k], ScenePairs([0, 130], [0, n_k]))
    for got, want in zip(both, alone):
        assert torch.equal(got[: len(want)], want)
    if n_k == 1:
        assert not both[0][:130].any() and not both[1][:1].any() and both[2][:1].any()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (24, FP16)])
@pytest.mark.parametrize("n_k", [300, 1500, 2100])
def test_cross_gradients_of_a_single_open_key_among_many(n_k, dim, dtype):
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(345, ([140, 9, 5], [n_k, n_k + 77, 40]), 4, 2, dim, dtype, scale=8.0)
    mask = torch.zeros(len(k), dtype=torch.bool, device="cuda")
    mask[[n_k - 1, n_k + 3]] = True
    mask[k_seg[2]:] = True
    check_cross(q, k, v, q_seg, k_seg, mask=mask)
    pairs, d = ScenePairs(q_seg, k_seg), normal(346, *q.shape, dtype=dtype)
    out, lse = cross_attention(q, k, v, pairs, mask=mask, return_lse=True)
    dq, dk, dv = cross_attention_grad(d, q, k, v, out, lse, pairs, mask=mask)
    assert not dq[:149].any() and not dk[: k_seg[2]].any()
    assert dv[[n_k - 1, n_k + 3]].any() and dq[149:].any() and dk[k_seg[2]:].any()


@pytest.mark.parametrize("dim", [64, 128])
def test_cross_fp16_gradients_of_large_scores_and_outputs(dim):
    # lse of 2^16 and more (320,000 and 2.5 million), and <dout, out> above
    # 2^24: both enter the keys' pass in parts
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(360, ([9], [2]), 1, 1, dim, FP16)
    for size, scale in ((200.0, 0.125), (200.0, 1.0), (25.0, 8.0)):
        q[:], k[:] = size, size
        check_cross(q, k, v, q_seg, k_seg, scale=scale)
    q, k, v, q_seg, k_seg = attention_inputs(365, ([9, 4], [2, 50]), 1, 1, dim, FP16)
    v[:] = v.sign() * 0.5 + 1000.0
    pairs, d = ScenePairs(q_seg, k_seg), torch.full_like(q, 1000.0)
    out, lse = cross_attention(q, k, v, pairs, return_lse=True)
    want = fo.Attention(q, k, v, q_seg, k_seg, dout=d)
    assert (d.double() * out.double()).sum(-1).min() > 2**24
    got = cross_attention_grad(d, q, k, v, out, lse, pairs)
    for name, t in zip(("dq", "dk", "dv"), got):
        assert t.isfinite().all()
        want.close(name, t)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [([130, 9], [64, 5]), ([200, 300], [1500, 90]), ([64, 3], [20000, 4])], ids=str)
def test_cross_fp16_gradients_grow_with_dout(lengths, dim):
    # The gradients are linear in dout, and a power of two of it is exact, so
    # the bounds of their errors grow with it too, but for a result's own step
    # below fp16's normals (half of it 2^-25).  dS at 2^-13 of its usual size
    # loses half its bits, and at 2^12 of it overflows, if it is not brought
    # into fp16's range.
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(350, lengths, 2, 1, dim, FP16, scale=0.125)
    pairs = ScenePairs(q_seg, k_seg)
    d = (normal(351, *q.shape).clamp(-3.9, 3.9) * 8).round() / 8  # six bits each
    d = d.to(FP16)
    out, lse = cross_attention(q, k, v, pairs, scale=1.0, return_lse=True)
    one = cross_attention_grad(d, q, k, v, out, lse, pairs, scale=1.0)
    want = fo.Attention(q, k, v, q_seg, k_seg, scale=1.0, dout=d)
    for name, t in zip(("dq", "dk", "dv"), one):
        want.close(name, t)
    for factor in (2.0**-13, 2.0**-7, 2.0**8, 2.0**12):
        got = cross_attention_grad(d * factor, q, k, v, out, lse, pairs, scale=1.0)
        for name, first, t in zip(("dq", "dk", "dv"), one, got):
            exact, t = getattr(want, name), t.double().cpu()
            fits = exact.abs() * factor < 65000
            assert fits.double().mean() > 0.9
            error = (t - exact * factor).abs()[fits]
            assert (error <= (getattr(want, name + "_off") * factor)[fits] + 2.0**-25).all(), (name, factor)
            # and the errors together grow no faster than dout
            most = 1.5 * factor * (first.double().cpu() - exact).norm() + 2.0**-25 * exact.numel() ** 0.5
            assert error.norm() <= most, (name, factor, float(error.norm() / most))


@pytest.mark.parametrize("dim", [64, 128])
def test_cross_fp16_gradients_of_large_products(dim):
    # two keys among 24,000 share the weight, and dout v is 10,000 and -10,000:
    # dS is 5,000 for results of some hundreds
    q, k, v, q_seg, k_seg = attention_inputs(355, ([3], [24000]), 1, 1, dim, FP16)
    q[:] = 1.0
    k[5], k[20001] = 40.0, 40.0
    k[5, 0, 0], k[5, 0, 1], k[20001, 0, 0], k[20001, 0, 1] = 41.0, 39.0, 39.0, 41.0
    v[5], v[20001] = 1.0, -1.0
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    pairs = ScenePairs(q_seg, k_seg)
    for size in (10000.0 / dim, 60000.0):
        d = torch.full_like(q, size)
        out, lse = cross_attention(q, k, v, pairs, scale=2.0**-6, return_lse=True)
        want = fo.Attention(q, k, v, q_seg, k_seg, scale=2.0**-6, dout=d)
        for name, t in zip(("dq", "dk", "dv"), cross_attention_grad(d, q, k, v, out, lse, pairs, scale=2.0**-6)):
            exact, t = getattr(want, name), t.double().cpu()
            fits = exact.abs() < 65504  # three rows of 30,000 in dk and dv, for one: beyond fp16
            want.close(name, torch.where(fits, t, exact))
            assert torch.equal(t[~fits], exact[~fits].sign() * math.inf)


@pytest.mark.parametrize("dim", [40, 128])
def test_cross_fp16_sizes_are_found_anew(dim):
    # a graph replayed on smaller gradients and values, and calls on two
    # streams: the factors are those of a call of its own
    from gsa_b200 import ScenePairs, cross_attention, cross_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(370, ([70, 0, 300], [700, 40, 9000]), 4, 2, dim, FP16)
    mask = torch.rand(len(k), generator=torch.Generator().manual_seed(371)) < 0.7
    k[~mask], v[~mask] = math.nan, torch.finfo(FP16).max  # shut values count for nothing
    mask, pairs = mask.cuda(), ScenePairs(q_seg, k_seg)
    d = normal(372, *q.shape, dtype=FP16, scale=3000.0)

    def step():
        out, lse = cross_attention(q, k, v, pairs, mask=mask, return_lse=True)
        return cross_attention_grad(d, q, k, v, out, lse, pairs, mask=mask)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for shrink in (1.0, 2.0**-14, 2.0**3):
        d.mul_(shrink)
        v[mask] *= 0.5
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        assert all(t.isfinite().all() and t.any() for t in want)
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in results for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_neighbor_rows_of_minus_infinity_are_nan(dtype):
    from gsa_b200 import ScenePairs, neighbor_attention, neighbor_attention_grad

    q, k, v, q_seg, k_seg = attention_inputs(380, ([6], [9]), 2, 1, 16, dtype)
    q[:], k[:4] = 1.0, 0.0
    k[:4, 0, 0] = -math.inf
    ids = torch.tensor([[0, 1, 2], [3, 3, 3], [-1, 9, -1], [5, 6, 7], [1, 5, 1], [0, -1, 0]], dtype=torch.int32).cuda()
    pairs, d = ScenePairs(q_seg, k_seg), normal(381, *q.shape, dtype=dtype)
    out, lse = neighbor_attention(q, k, v, ids, pairs, return_lse=True)
    lost = torch.tensor([True, True, False, False, False, True]).cuda()  # entries, but no softmax
    assert out[lost].isnan().all() and lse[lost].isnan().all() and out[~lost].isfinite().all()
    assert (lse[2] == -math.inf).all() and not out[2].any() and lse[3:5].isfinite().all()
    dq, dk, dv = neighbor_attention_grad(d, q, k, v, ids, out, lse, pairs)
    assert dq[lost].isnan().all() and not dq[2].any() and dq[3].isfinite().all()
    assert dv[:4].isnan().all() and dv[4:].isfinite().all()
