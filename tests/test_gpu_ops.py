"""The operators between observations and actions against their definitions in 64 bits (NumPy)."""
import numpy as np
import pytest

from ops_util import EPS, TINY, Box, rounded
from tetris_gymnasium_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def box():
    b = Box()
    yield b
    b.close()


# ---- linear_i8 ------------------------------------------------------------------------------------------------------
def linear_case(box, rows, k, n, xdt, odt, x_scale, bias, relu, seed, xpitch=None, xbefore=0, wpitch=None, wbefore=0, opitch=None, extreme=False):
    r = np.random.default_rng(seed)
    lo, hi = (0, 255) if xdt == "uint8" else (-128, 127)
    x = r.integers(lo, hi + 1, (rows, k)).astype(xdt)
    w = r.integers(-128, 128, (n, k)).astype(np.int8)
    if extreme:
        x[:], w[:] = hi, -128
    ws = r.uniform(0.5, 2.0, n).astype(np.float32) / np.float32(max(k, 1) * 16384)
    xs = r.uniform(0.5, 2.0, rows).astype(np.float32) if x_scale else None
    b = r.normal(size=n).astype(np.float32) if bias else None
    out = box.put(np.full((rows, n), 77, np.float32), odt, pitch=opitch)
    before = box.get(out, whole=True)
    ops.linear_i8(box.put(x, pitch=xpitch, before=xbefore), box.put(w, pitch=wpitch, before=wbefore), box.put(ws), out,
                  x_scale=None if xs is None else box.put(xs), bias=None if b is None else box.put(b), relu=relu, stream=box.stream)
    got = box.get(out).astype(np.float64)
    exact = np.float32 if k * 255 * 128 < 2**24 else np.float64  # (integers: sums below 2^24 are exact in float32 too)
    acc = (x.astype(exact) @ w.astype(exact).T).astype(np.float64) if k else np.zeros((rows, n))
    p = acc * ws.astype(np.float64) * (1.0 if xs is None else xs.astype(np.float64)[:, None])
    y = p + (0.0 if b is None else b)
    # the sum to float32, the product of the scales, their product with the bias in one fma: 2^-24 of the product each of the first two
    # (and their second order), 2^-24 of the result; then half a step of the output's type
    tol = np.abs(p) * 2.01 * 2.0**-24 + np.abs(y) * (2.0**-24 + (EPS[odt] / 2 if odt != "float32" else 0)) * 1.01 + TINY[odt]
    if relu:
        y = np.maximum(y, 0)
    assert (np.abs(got - y) <= tol).all(), f"off by {np.max(np.abs(got - y) / tol):.3g} tolerances"
    if opitch:
        after = box.get(out, whole=True)
        idx = np.arange(after.size) % opitch >= n
        np.testing.assert_array_equal(after[idx], before[idx])  # what lies between the rows stays


@pytest.mark.parametrize("xdt", ["uint8", "int8"])
@pytest.mark.parametrize("odt", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 200, 256), (2, 13, 1), (17, 13, 64), (16, 64, 16), (33, 65, 63), (5, 200, 40), (130, 129, 257), (64, 800, 100)])
def test_linear_sizes_and_types(box, rows, k, n, xdt, odt):
    linear_case(box, rows, k, n, xdt, odt, x_scale=rows % 2 == 1, bias=k % 2 == 1, relu=n % 2 == 0, seed=rows * 7 + k)


@pytest.mark.parametrize("rows,k,n,odt", [(300, 256, 40, "float32"), (256, 512, 256, "bfloat16"), (257, 1024, 300, "float16"), (8, 4096, 520, "bfloat16"),
                                          (16, 1000, 33, "float32"), (1, 8192, 70, "float16"), (31, 2049, 129, "bfloat16"), (700, 640, 700, "bfloat16"),
                                          (1025, 384, 513, "float32"), (513, 129, 1030, "bfloat16"), (2500, 13, 64, "float16"), (2500, 200, 256, "bfloat16")])
@pytest.mark.parametrize("xdt", ["uint8", "int8"])
def test_linear_larger(box, rows, k, n, odt, xdt):
    linear_case(box, rows, k, n, xdt, odt, True, True, False, seed=rows + k + n)


@pytest.mark.parametrize("rows,k,n,xdt,odt", [(4100, 528, 4000, "int8", "bfloat16"), (4096, 512, 4097, "uint8", "float32"), (4099, 560, 4096, "uint8", "float16"),
                                              (8200, 272, 1024, "uint8", "bfloat16"), (8193, 400, 1001, "int8", "float32"), (4200, 304, 1010, "uint8", "float16"),
                                              (2050, 400, 1000, "int8", "float16"), (1030, 288, 200, "uint8", "float32"), (65, 1024, 8200, "int8", "bfloat16"),
                                              (50, 300, 8200, "uint8", "float16"), (33, 1024, 8192, "int8", "float32"), (20, 2000, 8200, "int8", "bfloat16"),
                                              (32, 333, 8195, "uint8", "float32"), (9, 515, 8200, "uint8", "bfloat16"), (200, 800, 500, "uint8", "bfloat16"),
                                              (256, 130, 1024, "int8", "float32"), (5000, 901, 300, "uint8", "float16"), (20000, 37, 130, "uint8", "bfloat16"),
                                              (20000, 128, 63, "int8", "float16"), (9000, 250, 777, "uint8", "float32"), (9000, 256, 40, "int8", "float32")])
def test_linear_every_variant(box, rows, k, n, xdt, odt):
    """sizes on both sides of the rules that choose a kernel: wide, medium and small tiles, few rows of many columns, short rows"""
    linear_case(box, rows, k, n, xdt, odt, rows % 2 == 0, True, n % 2 == 0, seed=rows + n)


@pytest.mark.parametrize("rows,k,n", [(40, 200, 70), (300, 256, 300), (9, 1024, 64), (260, 640, 130)])
@pytest.mark.parametrize("xpitch,xbefore,wpitch,wbefore,opad", [(3, 0, 0, 0, 0), (0, 1, 5, 3, 1), (16, 16, 16, 16, 8), (8, 8, 0, 0, 4)])
def test_linear_strides_and_alignment(box, rows, k, n, xpitch, xbefore, wpitch, wbefore, opad):
    for odt in ("float32", "bfloat16"):
        linear_case(box, rows, k, n, "uint8", odt, False, True, True, seed=k, xpitch=k + xpitch, xbefore=xbefore, wpitch=k + wpitch, wbefore=wbefore,
                    opitch=n + opad)


@pytest.mark.parametrize("rows,k", [(3, 65536), (40, 65536), (300, 4096)])
@pytest.mark.parametrize("xdt", ["uint8", "int8"])
def test_linear_largest_sums_stay_exact(box, rows, k, xdt):
    linear_case(box, rows, k, 20, xdt, "float32", False, False, False, seed=1, extreme=True)


def test_linear_empty_and_broadcast(box):
    x, w, ws = box.put(np.arange(200, dtype=np.uint8)[None]), box.put(np.ones((3, 200), np.int8)), box.put(np.ones(3, np.float32))
    out = box.put(np.zeros((4, 3), np.float32))
    ops.linear_i8(ops.DeviceView(x.ptr, (4, 200), "uint8", (0, 1)), w, ws, out, stream=box.stream)  # one row read four times
    np.testing.assert_array_equal(box.get(out), np.full((4, 3), np.arange(200).sum(), np.float32))
    ops.linear_i8(ops.DeviceView(x.ptr, (0, 200), "uint8"), w, ws, ops.DeviceView(out.ptr, (0, 3), "float32"), stream=box.stream)
    b = box.put(np.array([-1, 0, 2], np.float32))
    ops.linear_i8(ops.DeviceView(x.ptr, (4, 0), "uint8"), ops.DeviceView(w.ptr, (3, 0), "int8"), ws, out, bias=b, relu=True, stream=box.stream)
    np.testing.assert_array_equal(box.get(out), np.tile(np.array([0, 0, 2], np.float32), (4, 1)))
    s = box.put(np.array([1, np.nan, 1, 1], np.float32))  # a row whose quantisation met a NaN stays NaN, also through relu
    ops.linear_i8(ops.DeviceView(x.ptr, (4, 200), "uint8", (0, 1)), w, ws, out, x_scale=s, relu=True, stream=box.stream)
    assert np.isnan(box.get(out)[1]).all() and np.isfinite(box.get(out)[[0, 2, 3]]).all()


def test_linear_reads_engine_buffers(box):
    """boards and per-placement feature vectors as an engine leaves them"""
    from tetris_gymnasium_amd import Engine, _native as N

    e = Engine(37, 10, 20, obs_mode=N.OBS_BOARD, grouped=True, features=True)
    e.reset(np.arange(1, 38, dtype=np.uint64))
    for t in range(6):
        e.sample_legal_actions(seed=3, counter=t, fetch=False)
        e.step_sampled()
    pf, _ = e.features()
    for view, x in ((e.device_array(N.BUF_PLACEMENT_FEATS), pf.reshape(-1, 13)), (e.device_array(N.BUF_OBS), e.observation().reshape(37, 200))):
        flat = ops.DeviceView(view.ptr, x.shape, "uint8")
        w = np.random.default_rng(0).integers(-128, 128, (5, x.shape[1])).astype(np.int8)
        out = box.put(np.zeros((x.shape[0], 5), np.float32))
        view._ready()
        ops.linear_i8(flat, box.put(w), box.put(np.ones(5, np.float32)), out, stream=box.stream)
        np.testing.assert_array_equal(box.get(out), (x.astype(np.int64) @ w.T.astype(np.int64)).astype(np.float32))
    out = box.put(np.zeros((37, 40, 5), np.float32))
    ops.linear_i8(e.device_array(N.BUF_PLACEMENT_FEATS), box.put(np.ones((5, 13), np.int8)), box.put(np.ones(5, np.float32)), out, stream=box.stream)
    np.testing.assert_array_equal(box.get(out)[..., 2], pf.astype(np.float32).sum(2))
    e.close()


# ---- quantize_i8 ----------------------------------------------------------------------------------------------------
def quantized(x):
    """the definition in 64 bits, x float32 values"""
    bad = ~np.isfinite(x).all(1)
    a = np.where(bad[:, None], 0, x).astype(np.float64)
    s = np.maximum((np.abs(a).max(1, initial=0) / 127).astype(np.float32), np.float32(2.0**-126))
    q = np.rint(a / s.astype(np.float64)[:, None])
    return np.where(bad[:, None], 0, q).astype(np.int8), np.where(bad, np.float32(np.nan), s)


def quantize_case(box, x, dtype, pitch=None, before=0, qpitch=None):
    x = rounded(x, dtype)
    q, s = box.put(np.full(x.shape, 99, np.int8), pitch=qpitch), box.put(np.zeros(x.shape[0], np.float32))
    ops.quantize_i8(box.put(x, dtype, pitch=pitch, before=before), q, s, stream=box.stream)
    eq, es = quantized(x)
    np.testing.assert_array_equal(box.get(s), es)
    np.testing.assert_array_equal(box.get(q), eq)
    if qpitch:
        whole = box.get(q, whole=True)
        idx = np.arange(whole.size) % qpitch >= x.shape[1]
        assert (whole[idx] == 0x5B).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (17, 40), (5, 256), (33, 257), (4, 512), (2, 1000), (9, 1025), (3, 2048), (2, 4100), (2, 8192), (1, 20011), (70, 16), (65, 31), (64, 64), (3, 16384), (2, 16500)])
def test_quantize_sizes(box, rows, k, dtype):
    r = np.random.default_rng(rows * k)
    x = r.normal(size=(rows, k)) * np.exp(2 * r.normal(size=(rows, 1)))
    quantize_case(box, np.clip(x, -6e4, 6e4), dtype)
    quantize_case(box, np.clip(x, -6e4, 6e4), dtype, pitch=k + 3, before=1, qpitch=k + 5)


def test_quantize_borders(box):
    r = np.random.default_rng(5)
    top = r.uniform(0.5, 2.0, 64).astype(np.float32)
    s = (top.astype(np.float64) / 127).astype(np.float32)
    halves = (np.arange(-127, 127) + 0.5)[None] * s[:, None].astype(np.float64)  # as near a half as float32 comes, on both sides
    x = np.concatenate([top[:, None], halves.astype(np.float32), np.nextafter(halves.astype(np.float32), np.float32(9)),
                        np.nextafter(halves.astype(np.float32), np.float32(-9))], 1)
    quantize_case(box, x, "float32")
    exact = np.concatenate([np.full((4, 1), 127.0), np.tile(np.arange(-127, 127) + 0.5, (4, 1))], 1) * np.array([[1], [2.0**-20], [2.0**90], [0.25]])
    quantize_case(box, exact, "float32")  # exact halves: to even
    quantize_case(box, exact[[0, 3]], "float16")
    quantize_case(box, exact[[0, 3]], "bfloat16")


def test_quantize_extremes(box):
    x = np.zeros((12, 70), np.float32)
    x[1, 3] = 1e-45
    x[2, :4] = [1e-40, -3e-39, 5e-45, 2e-38]
    x[3, 5], x[3, 6] = 3.4028235e38, -1.0
    x[4, 2] = np.nan
    x[5, 69] = np.inf
    x[6, 0] = -np.inf
    x[7] = -0.0
    x[8] = np.linspace(-1, 1, 70)
    x[9, 1] = 2.0**-119
    x[10, :2] = [2.0**-126, 2.0**-127]
    quantize_case(box, x, "float32")
    quantize_case(box, x[[0, 4, 5, 6, 7, 8]], "float16")
    quantize_case(box, x[[0, 2, 3, 4, 5, 7, 8]], "bfloat16")
    wide = np.zeros((2, 3000), np.float32)
    wide[0, 2999], wide[1, 1500] = np.nan, 5
    quantize_case(box, wide, "float32")
    s = box.put(np.full(3, 9, np.float32))
    p = box.put(np.zeros((1, 4), np.float32))
    ops.quantize_i8(ops.DeviceView(p.ptr, (3, 0), "float32"), ops.DeviceView(p.ptr, (3, 0), "int8"), s, stream=box.stream)
    np.testing.assert_array_equal(box.get(s), np.full(3, 2.0**-126, np.float32))


# ---- beam_select ----------------------------------------------------------------------------------------------------
def selected(x, sc, beams, mask=None, done=None, pad=0, norm=True):
    """the definition in 64 bits"""
    g, k, v = x.shape
    out = np.full((g, beams), -np.inf), np.full((g, beams), -1, np.int32), np.full((g, beams), -1, np.int32)
    for i in range(g):
        cand = []
        for j in range(k):
            if done is not None and done[i, j]:
                if sc[i, j] > -np.inf:
                    cand.append((-float(sc[i, j]), j, pad))
                continue
            at = np.arange(v) if mask is None else np.flatnonzero(mask[i, j])
            e = x[i, j, at].astype(np.float64)
            with np.errstate(all="ignore"):
                if norm and len(e):
                    m = e.max()
                    e = (e - m) - np.log(np.exp(e - m).sum())  # (m + log first would lose the logarithm beside a maximum of 3e38)
                c = float(sc[i, j]) + e
            first = np.argsort(np.where(c > -np.inf, -c, np.inf), kind="stable")[:beams]
            cand += [(-c[o], j, int(at[o])) for o in first if c[o] > -np.inf]
        for o, (c, j, t) in enumerate(sorted(cand)[:beams]):
            out[0][i, o], out[1][i, o], out[2][i, o] = -c, j, t
    return out


def select_case(box, x, sc, beams, dtype="float32", mask=None, done=None, pad=0, norm=True, xpitch=None, before=0, xv=None, xr=None):
    x = rounded(x, dtype) if xr is None else xr
    g, k, v = x.shape
    outs = [box.put(np.zeros((g, beams), t)) for t in (np.float32, np.int32, np.int32)]
    need = ops.beam_select_workspace(g, k, v, beams)
    ws = box.put(np.full(need, 0xEE, np.uint8)) if need else None
    ops.beam_select(box.put(x, dtype, pitch=xpitch, before=before) if xv is None else xv, box.put(sc.astype(np.float32)), *outs,
                    mask=None if mask is None else box.put(mask.astype(np.uint8)), finished=None if done is None else box.put(done.astype(np.uint8)),
                    pad=pad, normalize=norm, workspace=ws, stream=box.stream)
    es, ep, et = selected(x, sc.astype(np.float32), beams, mask, done, pad, norm)
    gs, gp, gt = (box.get(o) for o in outs)
    np.testing.assert_array_equal(gp, ep)
    np.testing.assert_array_equal(gt, et)
    same = es == gs  # (-inf on both sides too)
    # one rounding to float32 of a score held in 64 bits (its log-sum to 1e-12)
    assert (same | (np.abs(np.where(same, 0, gs) - np.where(same, 0, es)) <= np.abs(np.where(same, 0, es)) * 2.0**-24 * 1.001 + 1e-11)).all()


SIZES = [(1, 1, 1, 1), (1, 4, 40, 4), (3, 1, 5, 3), (5, 8, 40, 8), (2, 3, 7, 16), (4, 16, 128, 16), (2, 64, 9, 64), (3, 2, 300, 64), (1, 8, 1000, 8),
         (2, 5, 1031, 7), (2, 8, 4097, 8), (1, 3, 8192, 33), (1, 2, 20000, 5), (1, 16, 9001, 64), (70, 8, 40, 8), (300, 2, 8, 3), (64, 8, 9000, 64), (130, 4, 3000, 20), (300, 4, 2000, 7), (20, 64, 17, 3),
         (9, 33, 129, 40), (1, 1, 1024, 64), (1, 1, 1025, 1)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("g,k,v,b", SIZES)
def test_select_sizes(box, g, k, v, b, norm, dtype):
    r = np.random.default_rng(g * 1000 + k * 100 + v + b)
    x, sc = r.normal(size=(g, k, v)) * 3, -5 * r.random((g, k))
    select_case(box, x, sc, b, dtype, norm=norm)
    mask = r.random((g, k, v)) < 0.6
    mask[0, 0] = False
    done = r.random((g, k)) < 0.3
    sc[0, -1] = -np.inf
    poisoned = rounded(x, dtype).copy()
    poisoned[~mask] = r.choice([np.nan, np.inf, -np.inf, 3e38 if dtype != "float16" else 6e4], (~mask).sum())
    poisoned = rounded(poisoned, dtype)
    select_case(box, None, sc, b, dtype, mask=mask, done=done, pad=v - 1, norm=norm, xr=poisoned)


@pytest.mark.parametrize("k,v", [(4, 40), (8, 1500), (2, 9000)])
@pytest.mark.parametrize("norm", [True, False])
def test_select_ties_go_to_the_lowest(box, k, v, norm):
    r = np.random.default_rng(v)
    for x in (np.zeros((2, k, v)), r.integers(0, 3, (2, k, v)).astype(np.float64), np.where(r.random((2, k, v)) < 0.5, 0.0, -0.0)):
        x[1] = x[1, :1]  # the beams of the second group are alike
        select_case(box, x, np.zeros((2, k)), 8, norm=norm)
        select_case(box, x, np.zeros((2, k)), 64, "bfloat16", norm=norm)
        select_case(box, x, -r.integers(0, 2, (2, k)).astype(np.float64), 13, done=r.random((2, k)) < 0.4, pad=2, norm=norm)
    asc = np.tile(np.arange(v, dtype=np.float64) / 64, (2, k, 1))  # the best always comes last / first
    select_case(box, asc, np.zeros((2, k)), 9, norm=norm)
    select_case(box, -asc, np.zeros((2, k)), 9, norm=norm)


@pytest.mark.parametrize("k,v", [(26, 2), (8, 40), (4, 1500), (2, 9000)])
def test_select_forced_moves_keep_their_score(box, k, v):
    """one allowed entry: log-probability 0 exactly, so equal scores stay equal and go to the lowest beam"""
    r = np.random.default_rng(v)
    mask = np.zeros((6, k, v), bool)
    for i in range(6):
        mask[i, np.arange(k), r.integers(0, v, k)] = True
    for dtype in ("float32", "bfloat16"):
        select_case(box, r.normal(size=(6, k, v)) * 30, -r.integers(0, 3, (6, k)).astype(np.float64), min(k, 9), dtype, mask=mask)


@pytest.mark.parametrize("v", [40, 1500, 9000])
def test_select_rows_that_differ_by_a_constant_tie(box, v):
    """equal log-probabilities from different logits: the lowest beam first"""
    r = np.random.default_rng(v)
    base = np.round(r.normal(size=v) * 4) / 4
    x = np.stack([base + c for c in (0.0, 1.0, -7.0, 64.0, 0.25)])[None].astype(np.float32)
    outs = [box.put(np.zeros((1, 20), t)) for t in (np.float32, np.int32, np.int32)]
    need = ops.beam_select_workspace(1, 5, v, 20)
    ops.beam_select(box.put(x), box.put(np.zeros((1, 5), np.float32)), *outs, workspace=box.put(np.zeros(need, np.uint8)) if need else None, stream=box.stream)
    order = np.lexsort((np.arange(5 * v) % v, np.arange(5 * v) // v, -np.tile(base, 5)))[:20]
    np.testing.assert_array_equal(box.get(outs[1])[0] * v + box.get(outs[2])[0], order)


@pytest.mark.parametrize("k,v", [(3, 40), (4, 700), (2, 9000)])
def test_select_infinities_and_nan(box, k, v):
    r = np.random.default_rng(v)
    x, sc = r.normal(size=(6, k, v)), -r.random((6, k))
    x[0, 0, 3] = np.nan  # allowed and not a number: no candidate; under a log-sum the whole beam has none
    x[1, 0, 2] = np.inf
    x[2, 0] = -np.inf
    x[3] = -np.inf
    x[4, 1, : v // 2] = -np.inf
    sc[5, 0], sc[5, 1] = -np.inf, np.nan
    select_case(box, x, sc, 5, norm=True)
    select_case(box, x, sc, 5, norm=False)
    low = np.full((1, k, v), np.finfo(np.float32).min)  # masks by the type's lowest value
    low[0, 0, v // 2] = 1.0
    select_case(box, low, np.zeros((1, k)), 4, norm=True)
    big = r.normal(size=(1, k, v)) * 80  # exponentials that under- and overflow 32 bits
    select_case(box, big, np.zeros((1, k)), 6, norm=True)


def test_select_strides(box):
    r = np.random.default_rng(3)
    for v, dtype in ((40, "float32"), (41, "bfloat16"), (3001, "float16"), (9001, "float32"), (9001, "bfloat16")):
        x, sc = r.normal(size=(3, 4, v)), -r.random((3, 4))
        select_case(box, x, sc, 5, dtype, xpitch=v + 3, before=1)
        row = rounded(r.normal(size=(1, 1, v)), dtype)
        p = box.put(row, dtype)
        select_case(box, None, sc, 5, dtype, xv=ops.DeviceView(p.ptr, (3, 4, v), dtype, (0, 0, 1)), xr=np.broadcast_to(row, (3, 4, v)))
    x, sc, m = r.normal(size=(3, 4, 40)).astype(np.float32), -r.random((3, 4)).astype(np.float32), r.random((4, 40)) < 0.5
    outs = [box.put(np.zeros((3, 4), t)) for t in (np.float32, np.int32, np.int32)]
    mp = box.put(m.astype(np.uint8))
    ops.beam_select(box.put(x), box.put(sc), *outs, mask=ops.DeviceView(mp.ptr, (3, 4, 40), "bool", (0, 40, 1)), stream=box.stream)
    np.testing.assert_array_equal(box.get(outs[2]), selected(x, sc, 4, np.broadcast_to(m, (3, 4, 40)))[2])


# ---- beam_reorder ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("g,kin,kout", [(1, 1, 1), (3, 4, 4), (2, 8, 8), (5, 3, 7), (4, 16, 2), (1, 64, 64), (33, 2, 2)])
@pytest.mark.parametrize("rows", [(200, 40, 32, 48), (1,), (13, 7, 3), (4096, 36), (1000, 2), (16, 24, 4, 8, 6), (17, 31, 33, 5001),
                                  tuple(range(5, 29))])
def test_reorder(box, g, kin, kout, rows):
    r = np.random.default_rng(g + kin * 10 + len(rows))
    src = [r.integers(0, 256, (g * kin, n)).astype(np.uint8) for n in rows]
    p = r.integers(0, kin, (g, kout)).astype(np.int32)
    p[r.random((g, kout)) < 0.15] = -1
    p[0, 0] = kin  # out of range: as -1
    dst = [r.integers(0, 256, (g * kout, n)).astype(np.uint8) for n in rows]
    sv, dv = [box.put(a, pitch=a.shape[1] + (i % 2) * 4) for i, a in enumerate(src)], [box.put(a, pitch=a.shape[1] + (i % 3)) for i, a in enumerate(dst)]
    ops.beam_reorder(sv, box.put(p), out=dv, beams_in=kin, stream=box.stream)
    ok = (p >= 0) & (p < kin)
    for a, d, v, s in zip(src, dst, dv, sv):
        e = d.reshape(g, kout, -1).copy()
        for i in range(g):
            e[i, ok[i]] = a.reshape(g, kin, -1)[i, p[i, ok[i]]]
        np.testing.assert_array_equal(box.get(v), e.reshape(d.shape))
        np.testing.assert_array_equal(box.get(s), a)
        pitch = v.strides[0]
        if pitch > d.shape[1]:
            whole = box.get(v, whole=True)
            assert (whole[np.arange(whole.size) % pitch >= d.shape[1]] == 0x5B).all()
    if kin == kout:
        ops.beam_reorder(sv, box.put(p), stream=box.stream)  # in place
        for a, s in zip(src, sv):
            e = a.reshape(g, kin, -1).copy()
            for i in range(g):
                e[i, ok[i]] = a.reshape(g, kin, -1)[i, p[i, ok[i]]]
            np.testing.assert_array_equal(box.get(s), e.reshape(a.shape))


def test_reorder_long_rows_in_place(box):
    r = np.random.default_rng(0)
    a = r.integers(0, 256, (2, 5, 200003)).astype(np.uint8)
    f = r.normal(size=(2, 5, 3, 11)).astype(np.float16)
    p = np.array([[4, 3, 2, 1, 0], [1, 2, 3, 4, 0]], np.int32)  # cycles
    va, vf = box.put(a), box.put(f.reshape(10, 33))
    ops.beam_reorder([va, ops.DeviceView(vf.ptr, (2, 5, 3, 11), "float16")], box.put(p), stream=box.stream)
    for i in range(2):
        np.testing.assert_array_equal(box.get(va)[i], a[i, p[i]])
        np.testing.assert_array_equal(box.get(vf).reshape(f.shape)[i], f[i, p[i]])


# ---- as they are used together --------------------------------------------------------------------------------------
def test_a_quantised_layer_behind_another_and_a_selection(box):
    """observations → hidden (relu) → 8 bits → values of 40 placements → the best of four beams → their rows"""
    r = np.random.default_rng(9)
    g, k, v, h = 6, 4, 40, 64
    x = r.integers(0, 9, (g * k, 200)).astype(np.uint8)
    w1, w2 = r.integers(-127, 128, (h, 200)).astype(np.int8), r.integers(-127, 128, (v, h)).astype(np.int8)
    s1, s2 = (r.uniform(0.5, 2, h) / 2000).astype(np.float32), (r.uniform(0.5, 2, v) / 200).astype(np.float32)
    hid, q, qs, val = (box.put(np.zeros((g * k, h), np.float32)), box.put(np.zeros((g * k, h), np.int8)), box.put(np.zeros(g * k, np.float32)),
                       box.put(np.zeros((g * k, v), np.float32)))
    outs = [box.put(np.zeros((g, k), t)) for t in (np.float32, np.int32, np.int32)]
    mask, sc = r.random((g, k, v)) < 0.7, -r.random((g, k)).astype(np.float32)
    st = box.stream
    xv = box.put(x)
    ops.linear_i8(xv, box.put(w1), box.put(s1), hid, relu=True, stream=st)
    ops.quantize_i8(hid, q, qs, stream=st)
    ops.linear_i8(q, box.put(w2), box.put(s2), val, x_scale=qs, stream=st)
    ops.beam_select(ops.DeviceView(val.ptr, (g, k, v), "float32"), box.put(sc), *outs, mask=box.put(mask.astype(np.uint8)), stream=st)
    ops.beam_reorder(xv, outs[1], stream=st)
    hh = box.get(hid)
    eh = np.maximum(x.astype(np.float64) @ w1.T.astype(np.float64) * s1, 0)
    assert (np.abs(hh - eh) <= np.abs(eh) * 4 * 2.0**-24).all()
    eq, es = quantized(hh)
    np.testing.assert_array_equal(box.get(q), eq)
    vv = box.get(val)
    ev = eq.astype(np.float64) @ w2.T.astype(np.float64) * s2 * es[:, None].astype(np.float64)
    assert (np.abs(vv - ev) <= np.abs(ev) * 4 * 2.0**-24).all()
    _, ep, et = selected(vv.reshape(g, k, v), sc, k, mask)
    np.testing.assert_array_equal(box.get(outs[1]), ep)
    np.testing.assert_array_equal(box.get(outs[2]), et)
    np.testing.assert_array_equal(box.get(xv).reshape(g, k, 200), np.take_along_axis(x.reshape(g, k, 200), ep[:, :, None], 1))


@pytest.mark.parametrize("v", [40, 700, 9000, 70000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_select_sums_over_wide_ranges(box, v, dtype):
    """logits that rise by more than an exponential holds, in either direction, and lie far from zero; sums of equal terms"""
    r = np.random.default_rng(v)
    up = np.sort(r.normal(size=(1, 2, v)) * 2000, axis=2)
    sc = -r.random((1, 2))
    for x in (up, up[:, :, ::-1], up * 1e30 if dtype == "float32" else up * 100, r.normal(size=(1, 2, v)) - 5000, r.normal(size=(1, 2, v)) * 0.01 + 900,
              np.zeros((1, 2, v)), np.where(np.arange(v) < v // 2, -700.0, 3.0) * np.ones((1, 2, 1))):
        mask = r.random((1, 2, v)) < 0.5
        mask[0, 0, -1] = mask[0, 0, 0] = True
        select_case(box, x, sc, 4, dtype)
        select_case(box, x, sc, 4, dtype, mask=mask)


@pytest.mark.parametrize("rows", [4, 300])
def test_linear_without_columns_reads_no_operand(box, rows):
    """rows of no columns have strides too (1 for an empty array of PyTorch's) and no memory"""
    b = box.put(np.array([-1, 0, 2], np.float32))
    out = box.put(np.full((rows, 3), 7, np.float32))
    for stride in (1, 64):
        ops.linear_i8(ops.DeviceView(0, (rows, 0), "uint8", (stride, 1)), ops.DeviceView(0, (3, 0), "int8", (stride, 1)), box.put(np.ones(3, np.float32)),
                      out, bias=b, stream=box.stream)
        np.testing.assert_array_equal(box.get(out), np.tile(np.array([-1, 0, 2], np.float32), (rows, 1)))
