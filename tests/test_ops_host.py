"""Refusals of the operators: every one of them is raised on the host, in front of any device call."""
import ctypes as C
import os
import re

import pytest

from tetris_gymnasium_amd import EngineError, _native as N, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 40  # addresses that nothing ever reads


def V(shape, dtype, strides=None, at=0, device=0):
    return ops.DeviceView(A + at, shape, dtype, strides, device)


def test_library_exports_every_declared_operator():
    lib = N.load()
    header = open(os.path.join(ROOT, "include", "tetris_gym_ops.h")).read()
    declared = set(re.findall(r"^(?:const char\*|int|int64_t|void)\s+\*?(tg_[a-z0-9_]+)\s*\(", header, re.M))
    assert {"tg_linear_i8", "tg_quantize_i8", "tg_beam_select", "tg_beam_reorder"} <= declared and declared == set(N.OPS_SYMBOLS)
    assert N.HAVE_OPS and all(hasattr(lib, n) for n in declared)
    for name, value in (("MAX_K", ops.MAX_K), ("MAX_BEAMS", ops.MAX_BEAMS), ("MAX_STATES", ops.MAX_STATES)):
        assert int(re.search(rf"#define TG_OPS_{name} (\d+)", header).group(1)) == value


def linear(rows=4, k=8, n=3, **kw):
    a = dict(x=V((rows, k), "uint8"), weight=V((n, k), "int8", at=1 << 20), weight_scale=V((n,), "float32", at=2 << 20), out=V((rows, n), "float32", at=3 << 20))
    a.update(kw)
    x, w, s, o = (a.pop(i) for i in ("x", "weight", "weight_scale", "out"))
    return ops.linear_i8(x, w, s, o, **a)


def test_a_good_call_needs_a_gpu():
    if N.load().tg_device_count() > 0:
        pytest.skip("a GPU is present: these addresses must not reach it")
    with pytest.raises(EngineError, match="no CPU fallback"):
        linear()


@pytest.mark.parametrize("kw,msg", [
    (dict(x=V((4, 8), "float32")), "x must be uint8"),
    (dict(weight=V((3, 8), "uint8")), "weight must be int8"),
    (dict(weight=V((3, 7), "int8")), "weight must have shape"),
    (dict(weight=V((3, 8), "int8", (1, 3))), "last axis"),
    (dict(weight_scale=V((4,), "float32")), "weight_scale must have shape"),
    (dict(weight_scale=V((3,), "float32", (2,))), "contiguous"),
    (dict(weight_scale=V((3,), "float16")), "weight_scale must be float32"),
    (dict(out=V((5, 3), "float32", at=3 << 20)), "out has 5 rows"),
    (dict(out=V((4, 3), "int32", at=3 << 20)), "out must be"),
    (dict(out=V((4, 3), "float32", (2, 1), at=3 << 20)), "row stride"),
    (dict(x=V((4, 8), "uint8", (1, 4))), "last axis"),
    (dict(x=V((8,), "uint8")), "two axes"),
    (dict(x=V((2, 2, 8), "uint8", (100, 8, 1))), "flatten"),
    (dict(bias=V((2,), "float32")), "bias must have shape"),
    (dict(x_scale=V((3,), "float32")), "x_scale must have shape"),
    (dict(bias=V((3,), "float32", device=1)), "different devices"),
    (dict(out=V((4, 3), "float32", at=8)), "overlaps"),
    (dict(out=V((4, 3), "float32", at=(3 << 20) + 2)), "not aligned"),
    (dict(x=V((4, 70000), "uint8"), weight=V((3, 70000), "int8", at=1 << 24)), "exact up to"),
    (dict(x=[1, 2]), "device array"),
])
def test_linear_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        linear(**kw)


@pytest.mark.parametrize("x,q,s,msg", [
    (V((4, 8), "int8"), V((4, 8), "int8", at=999), V((4,), "float32", at=4096), "x must be"),
    (V((4, 8), "float32"), V((4, 8), "uint8", at=4096), V((4,), "float32", at=8192), "q must be"),
    (V((4, 8), "float32"), V((4, 9), "int8", at=4096), V((4,), "float32", at=8192), "q must have"),
    (V((4, 8), "float32"), V((4, 8), "int8", at=4096), V((5,), "float32", at=8192), "scale must have"),
    (V((4, 8), "float32"), V((4, 8), "int8", at=4), V((4,), "float32", at=8192), "overlap"),
    (V((4, 8), "float32"), V((4, 8), "int8", (4, 1), at=4096), V((4,), "float32", at=8192), "row strides"),
    (V((4, 8), "float32", (8, 2)), V((4, 8), "int8", at=4096), V((4,), "float32", at=8192), "last axis"),
])
def test_quantize_refusals(x, q, s, msg):
    with pytest.raises(ValueError, match=msg):
        ops.quantize_i8(x, q, s)


def select(g=2, k=3, v=5, b=4, **kw):
    a = dict(logits=V((g, k, v), "float32"), scores=V((g, k), "float32", at=1 << 20), out_scores=V((g, b), "float32", at=2 << 20),
             parents=V((g, b), "int32", at=3 << 20), tokens=V((g, b), "int32", at=4 << 20))
    a.update(kw)
    pos = [a.pop(i) for i in ("logits", "scores", "out_scores", "parents", "tokens")]
    return ops.beam_select(*pos, **a)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=V((2, 3, 5), "int8")), "logits must be"),
    (dict(logits=V((6, 5), "float32")), r"\[G, K, V\]"),
    (dict(logits=V((2, 3, 5), "float32", (30, 10, 2))), "last axis"),
    (dict(scores=V((2, 4), "float32")), "scores must have shape"),
    (dict(scores=V((2, 3), "float16")), "scores must be float32"),
    (dict(out_scores=V((3, 4), "float32", at=2 << 20)), "out_scores must have shape"),
    (dict(parents=V((2, 3), "int32", at=3 << 20)), "parents must have shape"),
    (dict(tokens=V((2, 4), "int64", at=4 << 20)), "tokens must be int32"),
    (dict(mask=V((2, 3, 4), "uint8", at=5 << 20)), "mask must have shape"),
    (dict(mask=V((2, 3, 5), "float32", at=5 << 20)), "mask must be"),
    (dict(finished=V((2, 4), "uint8", at=5 << 20)), "finished must have shape"),
    (dict(finished=V((2, 3), "uint8", at=5 << 20), pad=5), "pad 5 outside"),
    (dict(finished=V((2, 3), "uint8", at=5 << 20), pad=-1), "pad -1 outside"),
    (dict(tokens=V((2, 4), "int32", at=(3 << 20) + 4)), "overlap"),
    (dict(k=65, logits=V((2, 65, 5), "float32"), scores=V((2, 65), "float32", at=1 << 20)), "beams"),
    (dict(b=65), "beams"),
    (dict(v=0), "entry"),
    (dict(logits=V((2, 3, 5), "float32", device=1)), "different devices"),
    (dict(logits=V((2, 3, 5), "float32", (-15, 5, 1))), "negative"),
    (dict(g=1, k=2, v=100000, b=2, logits=V((1, 2, 100000), "bfloat16"), scores=V((1, 2), "float32", at=1 << 20)), "workspace"),
])
def test_select_refusals(kw, msg):
    if msg == "workspace" and ops.beam_select_workspace(1, 2, 100000, 2) == 0:
        pytest.skip("no workspace is used")
    with pytest.raises(ValueError, match=msg):
        select(**kw)


def test_workspace_refusals():
    with pytest.raises(ValueError, match="negative"):
        ops.beam_select_workspace(-1, 2, 3, 4)
    assert ops.beam_select_workspace(8192, 8, 40, 8) == 0


P = V((2, 3), "int32", at=9 << 20)


@pytest.mark.parametrize("states,kw,msg", [
    (V((5, 8), "uint8"), {}, "do not hold 6 rows"),
    (V((6, 8), "uint8"), dict(out=V((6, 7), "uint8", at=4096)), "bytes"),
    (V((6, 8), "uint8"), dict(out=V((6, 8), "uint8", at=4)), "overlap"),
    (V((6, 8), "uint8"), dict(out=[]), "0 outputs"),
    (V((8, 8), "uint8"), dict(beams_in=4), "in place"),
    (V((6, 8), "uint8", (16, 2)), {}, "contiguous"),
    ([V((6, 8), "uint8", at=i << 12) for i in range(25)], {}, "25 arrays"),
    ([V((6, 8), "uint8"), V((6, 8), "uint8", at=16)], {}, "overlap"),
    ([V((6, 8), "uint8"), V((6, 8), "uint8", at=1 << 16)], dict(out=[V((6, 8), "uint8"), V((6, 8), "uint8", at=1 << 20)]), "some arrays in place"),
    (V((6, 8), "uint8", at=9 << 20), {}, "parents"),
    (V((6, 8), "uint8", device=1), {}, "different devices"),
])
def test_reorder_refusals(states, kw, msg):
    with pytest.raises(ValueError, match=msg):
        ops.beam_reorder(states, P, **kw)


def test_reorder_refuses_bad_parents():
    for bad, msg in ((V((2, 3), "int64"), "int32"), (V((6,), "int32"), r"\[G, B\]"), (V((2, 65), "int32"), "beams"), (V((2, 3), "int32", (6, 2)), "contiguous")):
        with pytest.raises(ValueError, match=msg):
            ops.beam_reorder(V((6, 8), "uint8"), bad)


def test_null_pointers_and_types_are_refused_by_the_c_entries():
    lib = N.load()
    assert lib.tg_linear_i8(0, None, None, N.T_U8, 1, 1, 1, None, 1, 1, None, None, None, 0, None, N.T_F32, 1) == N.EINVAL
    assert lib.tg_linear_i8(0, None, None, N.T_F32, 1, 1, 1, None, 1, 1, None, None, None, 0, None, N.T_F32, 1) == N.EINVAL
    assert b"u8 or i8" in lib.tg_ops_last_error()
    assert lib.tg_quantize_i8(0, None, None, N.T_F32, 1, 1, 1, None, 1, None) == N.EINVAL
    assert lib.tg_beam_select(0, None, None, N.T_F32, 1, 1, 1, 1, 1, None, None, 0, 0, None, 0, 1, 1, None, None, None, None, 0) == N.EINVAL
    one = (C.c_int64 * 1)(4)
    assert lib.tg_beam_reorder(0, None, 1, (C.c_void_p * 1)(None), (C.c_void_p * 1)(None), one, one, one, 1, 1, 1, C.c_void_p(64)) == N.EINVAL
    assert lib.tg_reorder_beams(None, None, 1) == N.EINVAL and lib.tg_stream(None, None) == N.EINVAL
    assert lib.tg_linear_i8(0, None, None, N.T_U8, 0, 1, 1, None, 1, 1, None, None, None, 0, None, N.T_F32, 1) == N.OK  # nothing to do


def test_scorer_refusals():
    import numpy as np

    from tetris_gymnasium_amd import PlacementScorer

    w, s = np.ones((1, 13), np.int8), np.ones(1, np.float32)
    assert PlacementScorer([(w, s, None)]).n_features == 13
    for layers in ([], [(w.astype(np.float32), s, None)], [(w, np.ones(2), None)], [(w, s, np.ones(2))], [(np.ones((3, 13), np.int8), np.ones(3), None)],
                   [(np.ones((3, 13), np.int8), np.ones(3), None), (np.ones((1, 4), np.int8), s, None)]):
        with pytest.raises(ValueError):
            PlacementScorer(layers)
    with pytest.raises(ValueError, match="finite"):
        PlacementScorer.from_float([(np.full((1, 13), np.nan), None)])
    f = np.array([[1.0, -2.0, 0.25]], np.float32)
    (q, sc, _), = PlacementScorer.from_float([(f, None)]).layers
    assert q.tolist() == [[64, -127, 16]] and sc[0] == np.float32(2.0) / np.float32(127)  # 63.5 to even, 15.875


@pytest.mark.parametrize("sizes", [(1, 65, 100, 8), (1, 100, 100000, 8), (1, 8, 100, 65), (1, 8, (1 << 20) + 1, 8), (1 << 31, 8, 100000, 8), (1 << 62, 1, 1, 1)])
def test_workspace_of_sizes_beyond_the_limits(sizes):
    with pytest.raises(ValueError, match="are supported"):
        ops.beam_select_workspace(*sizes)


@pytest.mark.parametrize("name", ["logits", "scores", "mask", "finished"])
def test_select_refuses_a_workspace_over_an_input(name):
    g, k, v = 1, 4, 100000
    a = dict(logits=V((g, k, v), "float32"), scores=V((g, k), "float32", at=1 << 24), mask=V((g, k, v), "uint8", at=2 << 24),
             finished=V((g, k), "uint8", at=3 << 24))
    ws = ops.DeviceView(a[name].ptr, (ops.beam_select_workspace(g, k, v, 4),), "uint8")
    with pytest.raises(ValueError, match="workspace overlaps"):
        ops.beam_select(a["logits"], a["scores"], V((g, 4), "float32", at=4 << 24), V((g, 4), "int32", at=5 << 24), V((g, 4), "int32", at=6 << 24),
                        mask=a["mask"], finished=a["finished"], workspace=ws)
