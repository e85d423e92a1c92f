# SPDX-License-Identifier: Apache-2.0
"""CPU: the point-feature library's symbols and argument structs, what the C
entries and the Python calls refuse before any launch, the frequency tables
and the oracle's own gradients."""

import contextlib
import copy
import ctypes
import gc
import math
import pickle
import re
import struct
import subprocess
import types
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

import gsa_b200
from gsa_b200 import ScenePairs, Rotary, _features as ft, _library, attention, rotary
from tests import features_oracle as fo

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "point_features.h"


def test_exported_symbols_are_the_declared_ones():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"^\s*int(?:64_t)?\s+(\w+)\s*\(", text, flags=re.M))
    out = subprocess.run(["nm", "-D", "--defined-only", str(_library.path("point_features"))], capture_output=True,
                         text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert exported == declared and len(declared) == 9


def test_packed_structs_have_the_headers_sizes(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include "point_features.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) { printf("%zu %zu %zu %zu", '
                   "sizeof(rotary_args), offsetof(rotary_args, amplitude), sizeof(attention_args), "
                   "offsetof(attention_args, scale)); return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    r = ft.pack_rotary(*[0] * 17, 0.5, *[0] * 3)
    a = ft.pack_attention(*[0] * 9, 0.5, *[0] * 29)
    half = (0.5).hex() and ctypes.string_at(ctypes.addressof(ctypes.c_double(0.5)), 8)
    assert [int(s) for s in sizes] == [len(r), r.index(half), len(a), a.index(half)]


def cross_args(**change):
    """A valid call of one scene, 4 queries and 8 keys, with fake addresses."""
    base = 1 << 20
    a = dict(type=2, scenes=1, n_q=4, n_k=8, max_q=4, max_k=8, heads=2, kv_heads=1, dim=16, scale=0.25,
             q=(base, 32, 16), k=(base, 16, 16), v=(base, 16, 16), out=(base, 32, 16), dout=(base, 32, 16), lse=base,
             dq=base, dk=base, dv=base, q_seg=base, k_seg=base, mask=0, ids=base, width=4, padded=1, workspace=base,
             workspace_bytes=1 << 30, error=base, stream=0)
    a.update(change)
    flat = []
    for v in a.values():
        flat += v if isinstance(v, tuple) else [v]
    return ft.pack_attention(*flat)


BAD_SIZES = [dict(type=3), dict(type=-1), dict(scenes=0), dict(n_q=-1), dict(n_k=-1), dict(n_q=1 << 31), dict(heads=0),
             dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(dim=0), dict(dim=12), dict(dim=136), dict(dim=4)]


@pytest.mark.parametrize("bad", BAD_SIZES + [
    dict(type=0), dict(max_q=5), dict(max_q=-1), dict(max_k=9), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=2.0**-25), dict(scale=2.0**25), dict(scenes=65536), dict(heads=65, q=(1 << 20, 65 * 16, 16), out=(1 << 20, 65 * 16, 16)),
    dict(scale=math.inf), dict(scale=math.nan), dict(q=(0, 32, 16)), dict(q=((1 << 20) + 2, 32, 16)),
    dict(q=(1 << 20, 33, 16)), dict(k=(1 << 20, 16, 4)), dict(v=(0, 16, 16)), dict(out=((1 << 20) + 8, 32, 16)),
    dict(q_seg=0), dict(k_seg=0), dict(error=0)], ids=str)
def test_cross_entry_refuses(bad):
    assert ft.lib.cross_attention(cross_args(**bad)) == -2
    if not any(name in bad for name in ("out",)):
        assert ft.lib.cross_attention_grad(cross_args(**bad)) == -2


@pytest.mark.parametrize("bad", [dict(lse=0), dict(dout=(0, 32, 16)), dict(dq=0), dict(dk=0), dict(dv=(1 << 20) + 4),
                                 dict(workspace=0), dict(workspace_bytes=8)], ids=str)
def test_cross_gradient_entry_refuses(bad):
    assert ft.lib.cross_attention_grad(cross_args(**bad)) == -2


@pytest.mark.parametrize("name", ["k", "v", "q", "dout"])
@pytest.mark.parametrize("row", [1 << 31, -32])
def test_neighbor_entry_refuses_rows_too_far_apart(name, row):
    # a gathered tensor's row stride is 32 bits of bytes
    bad = cross_args(**{name: (1 << 20, row, 16)})
    assert ft.lib.neighbor_attention_grad(bad) == -2
    if name in "kv":
        assert ft.lib.neighbor_attention(bad) == -2


@pytest.mark.parametrize("bad", BAD_SIZES + [
    dict(width=0), dict(width=33), dict(ids=0), dict(q=(1 << 20, 33, 16)), dict(k=(0, 16, 16)),
    dict(v=((1 << 20) + 8, 16, 16)), dict(out=(0, 32, 16)), dict(q_seg=0), dict(k_seg=0), dict(scale=0.0)], ids=str)
def test_neighbor_entries_refuse(bad):
    assert ft.lib.neighbor_attention(cross_args(**bad)) == -2
    assert ft.lib.neighbor_attention_grad(cross_args(**bad)) == -2


@pytest.mark.parametrize("bad", [dict(lse=0), dict(dout=(0, 32, 16)), dict(dq=0), dict(dk=0), dict(dv=0),
                                 dict(workspace=0), dict(workspace_bytes=16)], ids=str)
def test_neighbor_gradient_entry_refuses(bad):
    assert ft.lib.neighbor_attention_grad(cross_args(**bad)) == -2


def test_null_arguments_and_workspaces():
    for name in ("cross_attention", "cross_attention_grad", "neighbor_attention", "neighbor_attention_grad",
                 "rotary_positions", "cross_attention_workspace", "cross_attention_grad_workspace",
                 "neighbor_attention_grad_workspace"):
        assert getattr(ft.lib, name)(None) == -2
    assert ft.lib.cross_attention_workspace(cross_args()) == 0  # 8 keys are not split
    assert ft.lib.cross_attention_workspace(cross_args(dim=12)) == -2
    # the values of 4 rows and 2 heads, nothing split
    assert 0 < ft.lib.cross_attention_grad_workspace(cross_args()) <= 256
    many = dict(n_k=24000, max_k=24000, n_q=1, max_q=1)
    size = ft.lib.cross_attention_workspace(cross_args(**many))
    assert size > 0 and size % (4 * 2 * 17) == 0
    assert ft.lib.cross_attention(cross_args(**many, workspace_bytes=size - 1)) == -2
    # empty calls return without a launch
    none = dict(n_q=0, max_q=0, q=(0, 0, 0), out=(0, 0, 0), dout=(0, 0, 0))
    assert ft.lib.cross_attention(cross_args(**none)) == 0
    assert ft.lib.neighbor_attention(cross_args(**none)) == 0


def rotary_call(**change):
    base = 1 << 20
    turns = (ctypes.c_double * 200)()
    a = dict(type=2, rows=4, heads=2, dim=16, x=(base, 32, 16), y=(base, 32, 16), positions=base, pos_type=0,
             pos_row=1, pos_axis=0, axes=1, pairs=8, turns=ctypes.addressof(turns), amplitude=1.0, interleaved=0,
             transposed=0, stream=0)
    a.update(change)
    flat = []
    for v in a.values():
        flat += v if isinstance(v, tuple) else [v]
    return ft.lib.rotary_positions(ft.pack_rotary(*flat))


@pytest.mark.parametrize("bad", [dict(type=3), dict(rows=-1), dict(rows=1 << 31), dict(heads=0), dict(dim=1),
                                 dict(dim=5000), dict(axes=0), dict(pairs=0), dict(pairs=9), dict(axes=2),
                                 dict(pairs=129, dim=1024), dict(pos_type=3), dict(turns=0), dict(x=(0, 32, 16)),
                                 dict(y=(0, 32, 16)), dict(positions=0)], ids=str)
def test_rotary_entry_refuses(bad):
    assert rotary_call(**bad) == -2


def test_rotary_entry_takes_no_rows():
    assert rotary_call(rows=0, x=(0, 0, 0), y=(0, 0, 0), positions=0) == 0


@pytest.mark.parametrize("bad", [dict(part=0), dict(part=7), dict(part=16, axes=3), dict(part=600), dict(part=16, axes=0),
                                 dict(part=16, layout="both"), dict(part=16, scaling="ntk"), dict(part=16, base=0.0),
                                 dict(part=16, unit=-1.0), dict(part=16, factor=math.inf), dict(part=16, scaling="ramp"),
                                 dict(part=16, scaling="ramp", length=0), dict(part=16, amplitude=math.nan)], ids=str)
def test_rotary_plan_refuses(bad):
    with pytest.raises(ValueError):
        Rotary(**bad)


def test_calls_refuse_cpu_tensors():
    x = torch.zeros(4, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        Rotary(16)(x, torch.zeros(4))
    with pytest.raises(ValueError):
        attention.cross_attention(x, x, x, None)
    with pytest.raises(ValueError):
        attention.neighbor_attention(x, x, x, torch.zeros(4, 3, dtype=torch.int32), None)


@pytest.mark.parametrize("q,k", [([0], [0]), ([0, 4], [0, 4, 8]), ([1, 4], [0, 4]), ([0, 4, 3], [0, 1, 2]),
                                 ([0, 4], [0, -1]), ([0, 1 << 31], [0, 4])], ids=str)
def test_scene_pairs_refuse_bad_offsets(q, k):
    with pytest.raises(ValueError):
        ScenePairs(q, k)


def test_written_tensors_do_not_overlap_themselves():
    x = torch.zeros(4, 2, 16)
    ft.check_written(x, "out")
    ft.check_written(x.transpose(0, 1).contiguous().transpose(0, 1), "out")
    ft.check_written(torch.zeros(4, 3, 2, 16)[:, 1], "out")
    ft.check_written(x[:1].expand(1, 2, 16), "out")
    for bad in (x[:, :1].expand(4, 2, 16), x[:1].expand(4, 2, 16), x.as_strided((4, 2, 16), (16, 16, 1)),
                x.as_strided((4, 2, 16), (32, 8, 1))):
        with pytest.raises(ValueError):
            ft.check_written(bad, "out")


def test_public_names():
    for name in ("Rotary", "ScenePairs", "cross_attention", "cross_attention_grad", "neighbor_attention",
                 "neighbor_attention_grad"):
        assert name in gsa_b200.__all__ and getattr(gsa_b200, name)


def test_frequencies():
    n, s = 16, 8.0
    plain = rotary.frequencies(n)
    assert plain[0] == 1.0 and math.isclose(plain[8], 10000.0**-0.5)
    assert rotary.frequencies(n, scaling="linear", factor=s) == [f / s for f in plain]
    grown = rotary.frequencies(n, scaling="base", factor=s)
    assert grown[0] == 1.0 and math.isclose(grown[-1], plain[-1] / s, rel_tol=1e-12)
    ramp = rotary.frequencies(n, scaling="ramp", factor=s, length=4096)
    for f, g in zip(plain, ramp):
        turns = 4096 * f / (2 * math.pi)
        if turns >= 32:
            assert g == f
        elif turns <= 1:
            assert math.isclose(g, f / s)
        else:
            assert f / s < g < f
    assert math.isclose(Rotary(32, scaling="ramp", factor=s, length=4096).amplitude, 0.1 * math.log(s) + 1)
    assert Rotary(32, scaling="linear", factor=s).amplitude == 1.0
    assert rotary.frequencies(1, scaling="base", factor=s) == [1.0]


def test_oracle_gradients_are_those_of_its_output():
    g = torch.Generator().manual_seed(3)
    q_seg, k_seg = [0, 3, 3, 5], [0, 4, 6, 6]
    shapes = [(5, 4, 8), (6, 2, 8), (6, 2, 8)]
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in shapes)
    d = torch.randn(5, 4, 8, generator=g, dtype=torch.float64)
    ids = torch.tensor([[0, 2, 0], [3, -1, 9], [1, 1, 2], [0, 0, 0], [-1, 7, -1]], dtype=torch.int32)
    mask = torch.tensor([1, 0, 1, 1, 1, 1], dtype=torch.bool)
    for kw in (dict(mask=mask), dict(ids=ids), dict(ids=ids, padded=False)):
        o = fo.Attention(q, k, v, q_seg, k_seg, dout=d, **kw)
        for name, t in (("dq", q), ("dk", k), ("dv", v)):
            step = torch.randn(t.shape, generator=g, dtype=torch.float64)
            h = 1e-5
            two = [(fo.Attention(*(x + s * h * step if x is t else x for x in (q, k, v)), q_seg, k_seg, **kw).out * d).sum()
                   for s in (1, -1)]
            got = (two[0] - two[1]) / (2 * h)
            assert torch.isclose(got, (getattr(o, name) * step).sum(), rtol=1e-6, atol=1e-8), (kw, name)


class OnDevice(torch.Tensor):
    """A CPU tensor that passes for one of device 0."""

    is_cuda = True

    def get_device(self):
        return 0


def test_copies_of_a_rotary_plan_have_turns_of_their_own(monkeypatch):
    plan = Rotary(20, axes=2, base=500.0, unit=0.5)
    want, seen = list(plan._turns), []

    def entry(args):
        at = struct.unpack_from("=17q", args)[16]
        seen.append(list((ctypes.c_double * plan_pairs).from_address(at)))
        return 0

    plan_pairs = plan.pairs
    copies = [copy.copy(plan), copy.deepcopy(plan), copy.deepcopy(copy.deepcopy(plan)), pickle.loads(pickle.dumps(plan))]
    del plan
    gc.collect()
    others = [(ctypes.c_double * plan_pairs)(*[7.0] * plan_pairs) for _ in range(500)]
    monkeypatch.setattr(rotary, "current_stream", lambda: (0, 0))
    monkeypatch.setattr(ft, "lib", types.SimpleNamespace(rotary_positions=entry))
    x, y = (torch.zeros(4, 2, 24).as_subclass(OnDevice) for _ in range(2))
    place = torch.zeros(4, 2).as_subclass(OnDevice)
    for twin in copies:
        twin(x, place, out=y)
    assert seen == [want] * 4 and len(others) == 500


def test_copies_of_scene_pairs_have_offsets_of_their_own(monkeypatch):
    monkeypatch.setattr(attention, "current_stream", lambda: (0, 0))
    monkeypatch.setattr(torch.cuda, "device", lambda _: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *_, **__: t.clone())
    pairs = ScenePairs([0, 3, 7], [0, 5, 5])
    for twin in (copy.copy(pairs), copy.deepcopy(pairs), pickle.loads(pickle.dumps(pairs))):
        assert (twin.q_seg, twin.k_seg, twin.device) == (pairs.q_seg, pairs.k_seg, 0)
        at = twin._ints.data_ptr()
        assert at != pairs._ints.data_ptr() and twin._ints.tolist() == [0, 3, 7, 0, 5, 5, 0]
        assert (twin._q_at, twin._k_at, twin._error_at) == (at, at + 12, at + 24)


def test_gradients_are_laid_out_for_the_kernels():
    flat = torch.randn(3 + 2 * 64).to(torch.bfloat16)
    for t in (flat[3:].view(2, 2, 32), flat[3:67].view(1, 2, 32), flat[:128].view(2, 2, 32), flat[:64].view(1, 2, 32).expand(3, 2, 32),
              flat[:128].view(2, 32, 2).transpose(1, 2)):
        got = attention._vectors(t)
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and got.stride(2) == 1


def test_calls_refuse_forward_mode_derivatives():
    x = torch.zeros(4, 2, 16)
    place, ids, lse = torch.zeros(4), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 2)
    turn = Rotary(16)
    with forward_ad.dual_level():
        moved, moved_place = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(place, torch.ones_like(place))
        for call in (lambda: turn(moved, place), lambda: turn.grad(moved, place), lambda: turn(x, moved_place),
                     lambda: turn(moved, place, out=x),
                     lambda: attention.cross_attention(x, moved, x, None), lambda: attention.cross_attention(moved, x, x, None, out=x),
                     lambda: attention.neighbor_attention(x, x, moved, ids, None),
                     lambda: attention.cross_attention_grad(moved, x, x, x, x, lse, None),
                     lambda: attention.neighbor_attention_grad(x, x, moved, x, ids, x, lse, None)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_rotary_refuses_positions_that_want_a_gradient():
    x, place = torch.zeros(4, 2, 16), torch.zeros(4).requires_grad_()
    leaf, turn = x.clone().requires_grad_(), Rotary(16)
    for call in (lambda: turn(x, place), lambda: turn.grad(x, place), lambda: turn(leaf, place), lambda: turn(x, place, out=x)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="rows must be CUDA"):
            call()


def test_attention_gradients_refuse_to_be_differentiated():
    x, lse = torch.zeros(4, 2, 16), torch.zeros(4, 2)
    ids, leaf = torch.zeros(4, 3, dtype=torch.int32), x.clone().requires_grad_()
    for call in (lambda: attention.cross_attention_grad(leaf, x, x, x, x, lse, None),
                 lambda: attention.neighbor_attention_grad(leaf, x, x, x, ids, x, lse, None)):
        with pytest.raises(ValueError, match="second derivatives"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="needs CUDA"):
            call()


def test_written_tensors_that_autograd_follows_are_refused():
    x, place, ids = torch.zeros(4, 2, 16), torch.zeros(4), torch.zeros(4, 3, dtype=torch.int32)
    out, turn = x.clone().requires_grad_(), Rotary(16)
    for call in (lambda: turn(x, place, out=out), lambda: turn.grad(x, place, out=out),
                 lambda: attention.cross_attention(x, x, x, None, out=out), lambda: attention.neighbor_attention(x, x, x, ids, None, out=out)):
        with pytest.raises(ValueError, match="takes no part in autograd"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()


def test_exponential_polynomial_is_as_near_as_it_says():
    text = (ROOT / "gsa_b200" / "csrc" / "cross.cuh").read_text()
    body = text[text.index("void exp2_polynomial"):]
    body = body[: body.index("\n}")]
    stated = re.search(r"without the exponential unit, to 2\^(-\d+)", text).group(1)
    # the Horner steps in their order, each coefficient given twice
    numbers = [float(v) for v in re.findall(r"(\d\.?\d*(?:e-?\d+)?)f", body[body.index("uint64_t p ="):])]
    coefficients = numbers[0::2]
    assert numbers[1::2] == coefficients and len(coefficients) == 6
    x = torch.linspace(-0.5, 0.5, 1_000_001, dtype=torch.float64).float().double()
    p = torch.zeros_like(x)
    for c in coefficients:  # fused: one rounding to 32 bits a step
        p = (p * x + torch.tensor(c, dtype=torch.float32).double()).float().double()
    assert (p / torch.exp2(x) - 1).abs().max() < 2.0 ** int(stated)
