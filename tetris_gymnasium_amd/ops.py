"""Operators between the engine's observations and its actions, on device memory (include/tetris_gym_ops.h):

* `linear_i8`    8-bit observations (or quantised activations) times 8-bit weights, scaled per row and per column
* `quantize_i8`  rows of activations to 8 bits with one scale each — what a second layer takes
* `beam_select`  the best continuations of a group of beams over all entries, under a legal mask
* `beam_reorder` the rows of any number of states that follow their beams

Arrays are device memory of one GPU: a PyTorch tensor, a `DeviceArray` of an Engine, anything with
`__cuda_array_interface__`, or a `DeviceView` around a raw pointer.  Outputs are the caller's; nothing is allocated, kept or
waited for.  Calls run on `stream` (an integer hipStream_t, e.g. `torch.cuda.current_stream().cuda_stream`; 0 = the default
stream) in order with whatever else runs there, and may be captured into a graph.  A `DeviceArray` is exported as to any other
consumer: its engine's stream is waited for first, which a capture does not allow: there, wait for the engine beforehand and pass a
`DeviceView` of the array's `ptr`.  A call runs on its arrays' device, whatever the current one is (an array that is
known by `__cuda_array_interface__` alone does not tell: that of the others, or 0).  Bad arguments raise ValueError, a failed
call EngineError."""
from __future__ import annotations

import ctypes as C

from . import _native as N
from .engine import DeviceArray, EngineError

MAX_BEAMS, MAX_STATES, MAX_K = 64, 24, 65536  # TG_OPS_MAX_*

_TYPES = {"uint8": N.T_U8, "bool": N.T_U8, "int8": N.T_I8, "float32": N.T_F32, "float16": N.T_F16, "bfloat16": N.T_BF16, "int32": -1}
_SIZES = {"uint8": 1, "bool": 1, "int8": 1, "float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8, "int16": 2,
          "float64": 8, "uint16": 2, "uint32": 4, "uint64": 8}
_STR = {"|u1": "uint8", "|b1": "bool", "|i1": "int8", "<f4": "float32", "<f2": "float16", "<i4": "int32", "<i8": "int64", "<i2": "int16",
        "<f8": "float64", "<u2": "uint16", "<u4": "uint32", "<u8": "uint64"}
_names: dict = {}  # dtype object → its name


class DeviceView:
    """A raw device pointer with a shape: dtype by name ("uint8", "int8", "bool", "int32", "float32", "float16", "bfloat16", ...),
    strides in elements (None = contiguous).  The caller keeps the memory alive."""

    __slots__ = ("ptr", "shape", "dtype", "strides", "device", "_meta")

    def __init__(self, ptr, shape, dtype, strides=None, device=0):
        if dtype not in _SIZES:
            raise ValueError(f"DeviceView: unknown dtype {dtype!r}")
        self.ptr, self.shape, self.dtype, self.device = int(ptr), tuple(int(n) for n in shape), dtype, int(device)
        if any(n < 0 for n in self.shape):
            raise ValueError(f"DeviceView: negative size in {self.shape}")
        self.strides = _contiguous(self.shape) if strides is None else tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape):
            raise ValueError("DeviceView: one stride per axis")
        self._meta = (self.shape, self.strides, dtype, self.device)


def _contiguous(shape):
    st, n = [], 1
    for s in reversed(shape):
        st.append(n)
        n *= s
    return tuple(reversed(st))


# An array comes in as (pointer, meta), meta = (shape, strides in elements, dtype, device): a call's metas decide everything that its
# checks and the C entry's sizes depend on, so a call whose metas were seen before reuses their outcome (`_plans`) and only passes the
# pointers on — the checks in Python cost more than a small kernel.  Pointers, values and objects are never kept.
_plans: dict = {}


def _get(a, write=False):
    if hasattr(a, "data_ptr"):  # a torch tensor (torch is not imported here)
        return a.data_ptr(), (a.shape, a.stride(), a.dtype, a.get_device())
    if isinstance(a, DeviceView):
        return a.ptr, a._meta
    if isinstance(a, DeviceArray):
        if write and a._readonly:
            raise ValueError("an output is a read-only DeviceArray")
        a._ready()
        name, item = a.dtype.name, a.dtype.itemsize
        if a.strides is None:
            st = _contiguous(a.shape)
        else:
            if any(s % item for s in a.strides):
                raise ValueError("strides of a DeviceArray are not whole elements")
            st = tuple(s // item for s in a.strides)
        return a.ptr, (a.shape, st, name, int(a.engine.cfg.device))
    cai = getattr(a, "__cuda_array_interface__", None)
    if cai is None:
        raise ValueError(f"a device array is needed (torch tensor, DeviceArray, DeviceView or __cuda_array_interface__), got {type(a).__name__}")
    if write and cai["data"][1]:
        raise ValueError("an output's __cuda_array_interface__ says that it is read-only")
    name = _STR.get(cai["typestr"])
    if name is None:
        raise ValueError(f"unsupported element type {cai['typestr']}")
    shape, item = tuple(cai["shape"]), _SIZES[name]
    st = cai.get("strides")
    if st is not None and any(s % item for s in st):
        raise ValueError(f"strides {tuple(st)} of a {name} array are not whole elements")
    st = _contiguous(shape) if st is None else tuple(s // item for s in st)
    return cai["data"][0], (shape, st, name, None)


def _parse(meta, what):
    """(shape, strides, dtype name, device or None) of a meta"""
    shape, st, dt, dev = meta
    if not isinstance(dt, str):
        name = _names.get(dt)
        if name is None:
            name = _names[dt] = str(dt).rpartition(".")[2]
        dt = name
        if dev is not None and dev < 0:
            raise ValueError(f"{what}: device memory is needed, got a tensor on the host")
    return tuple(shape), tuple(st), dt, dev


def _view(a, what):
    p, meta = _get(a)
    return (p, *_parse(meta, what))


def _plan(key, make, *args):
    plan = _plans.get(key)
    if plan is None:
        plan = make(*args)
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    return plan


def _device(*devs):
    seen = {d for d in devs if d is not None}
    if len(seen) > 1:
        raise ValueError(f"arrays on different devices: {sorted(seen)}")
    return seen.pop() if seen else 0


def _lib():
    lib = N._lib or N.load()
    if not N.HAVE_OPS:
        raise EngineError(f"{N.LIB_PATH} holds no operators (include/tetris_gym_ops.h): build the product library")
    return lib


def _check(lib, rc, what):
    if rc != N.OK:
        msg = f"{what} failed ({rc}): {lib.tg_ops_last_error().decode()}"
        raise ValueError(msg) if rc == N.EINVAL else EngineError(msg)


def _int64(what, *ints):
    """sizes and strides as the C entries take them: ctypes would cut what does not fit"""
    for i in ints:
        if not -(2**63) <= i < 2**63:
            raise ValueError(f"{what}: a size or stride of {i} does not fit 64 bits")


def _type(name, what, allowed):
    if name not in allowed:
        raise ValueError(f"{what} must be {' / '.join(allowed)}, got {name}")
    return _TYPES[name]


_FLOATS = ("float32", "float16", "bfloat16")


def _inner(shape, st, what):
    if shape and shape[-1] > 1 and st[-1] != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")


def _dense(shape, st, want, what):
    """an array of exactly this shape, contiguous"""
    if tuple(shape) != tuple(want):
        raise ValueError(f"{what} must have shape {tuple(want)}, got {tuple(shape)}")
    n = 1
    for s, k in zip(reversed(st), reversed(shape)):
        if k > 1 and s != n:
            raise ValueError(f"{what} must be contiguous")
        n *= k


def _rows(shape, st, what):
    """(rows, columns, row stride) of an array whose leading axes flatten into one"""
    if len(shape) < 2:
        raise ValueError(f"{what} must have at least two axes, got {shape}")
    _inner(shape, st, what)
    rows, stride = 1, 0
    for s, k in zip(reversed(st[:-1]), reversed(shape[:-1])):
        if k == 1:
            continue
        if rows == 1:
            stride = s
        elif s != stride * rows:
            raise ValueError(f"{what}: the leading axes (shape {shape}, strides {tuple(st)}) do not flatten into rows")
        rows *= k
    return rows, shape[-1], stride if rows > 1 else shape[-1]


def linear_i8(x, weight, weight_scale, out, *, x_scale=None, bias=None, relu=False, stream=0):
    """out[..., n] = act((sum_k x[..., k] * weight[n, k]) * (x_scale[...] * weight_scale[n]) + bias[n])

    x uint8 / int8 [..., K] (rows at any stride and alignment: the engine's boards and feature vectors as they lie), weight int8
    [N, K], weight_scale float32 [N], x_scale float32 [rows] or None (1), bias float32 [N] or None, out float32 / float16 /
    bfloat16 [..., N].  The sum is exact (K <= 65 536), the rest float32, rounded once; `relu` clips at zero.  Returns out."""
    xp, xm = _get(x)
    wp, wm = _get(weight)
    sp, sm = _get(weight_scale)
    op, om = _get(out, True)
    xsp, xsm = (None, None) if x_scale is None else _get(x_scale)
    bp, bm = (None, None) if bias is None else _get(bias)
    dev, xtype, rows, k, xs, n, wst, otype, os_ = _plan(("linear", xm, wm, sm, om, xsm, bm), _linear_plan, xm, wm, sm, om, xsm, bm)
    lib = _lib()
    rc = lib.tg_linear_i8(dev, stream, xp, xtype, rows, k, xs, wp, n, wst, sp, xsp, bp, 1 if relu else 0, op, otype, os_)
    if rc:
        _check(lib, rc, "tg_linear_i8")
    return out


def _linear_plan(xm, wm, sm, om, xsm, bm):
    xsh, xst, xt, d0 = _parse(xm, "linear_i8: x")
    wsh, wst, wt, d1 = _parse(wm, "linear_i8: weight")
    ssh, sst, stt, d2 = _parse(sm, "linear_i8: weight_scale")
    osh, ost, ot, d3 = _parse(om, "linear_i8: out")
    xtype = _type(xt, "linear_i8: x", ("uint8", "int8"))
    _type(wt, "linear_i8: weight", ("int8",))
    _type(stt, "linear_i8: weight_scale", ("float32",))
    otype = _type(ot, "linear_i8: out", _FLOATS)
    rows, k, xs = _rows(xsh, xst, "linear_i8: x")
    orows, n, os_ = _rows(osh, ost, "linear_i8: out")
    if wsh != (n, k):
        raise ValueError(f"linear_i8: weight must have shape {(n, k)}, got {wsh}")
    _inner(wsh, wst, "linear_i8: weight")
    if orows != rows:
        raise ValueError(f"linear_i8: out has {orows} rows, x has {rows}")
    _dense(ssh, sst, (n,), "linear_i8: weight_scale")
    devs = [d0, d1, d2, d3]
    if xsm is not None:
        sh, st, t, d = _parse(xsm, "linear_i8: x_scale")
        _type(t, "linear_i8: x_scale", ("float32",))
        _dense(sh, st, (rows,) if len(sh) == 1 else xsh[:-1], "linear_i8: x_scale")
        devs.append(d)
    if bm is not None:
        sh, st, t, d = _parse(bm, "linear_i8: bias")
        _type(t, "linear_i8: bias", ("float32",))
        _dense(sh, st, (n,), "linear_i8: bias")
        devs.append(d)
    _int64("linear_i8", rows, k, xs, n, wst[0], os_)
    return _device(*devs), xtype, rows, k, xs, n, wst[0], otype, os_


def quantize_i8(x, q, scale, *, stream=0):
    """q[..., k] = round(x[..., k] / scale[...]) (half to even), scale = max(max_k |x| / 127, 2^-126)

    x float32 / float16 / bfloat16 [..., K], q int8 [..., K], scale float32 [rows].  q * scale is x to half a step.  A row with a
    NaN or an infinity gets scale NaN and q 0: what is computed from it is NaN, not a plausible number.  Returns (q, scale)."""
    xp, xm = _get(x)
    qp, qm = _get(q, True)
    sp, sm = _get(scale, True)
    dev, xtype, rows, k, xs, qs = _plan(("quantize", xm, qm, sm), _quantize_plan, xm, qm, sm)
    lib = _lib()
    rc = lib.tg_quantize_i8(dev, stream, xp, xtype, rows, k, xs, qp, qs, sp)
    if rc:
        _check(lib, rc, "tg_quantize_i8")
    return q, scale


def _quantize_plan(xm, qm, sm):
    xsh, xst, xt, d0 = _parse(xm, "quantize_i8: x")
    qsh, qst, qt, d1 = _parse(qm, "quantize_i8: q")
    ssh, sst, stt, d2 = _parse(sm, "quantize_i8: scale")
    xtype = _type(xt, "quantize_i8: x", _FLOATS)
    _type(qt, "quantize_i8: q", ("int8",))
    _type(stt, "quantize_i8: scale", ("float32",))
    rows, k, xs = _rows(xsh, xst, "quantize_i8: x")
    qrows, qk, qs = _rows(qsh, qst, "quantize_i8: q")
    if (qrows, qk) != (rows, k):
        raise ValueError(f"quantize_i8: q must have x's shape {xsh}, got {qsh}")
    _dense(ssh, sst, (rows,) if len(ssh) == 1 else xsh[:-1], "quantize_i8: scale")
    _int64("quantize_i8", rows, k, xs, qs)
    return _device(d0, d1, d2), xtype, rows, k, xs, qs


def beam_select_workspace(groups, beams_in, vocab, beams_out):
    """Bytes of device memory beam_select needs as `workspace` for these sizes (0: none)."""
    lib = _lib()
    _int64("beam_select_workspace", groups, beams_in, vocab, beams_out)
    n = lib.tg_beam_select_workspace(groups, beams_in, vocab, beams_out)
    if n < 0:
        _check(lib, N.EINVAL, "tg_beam_select_workspace")
    return n


def beam_select(logits, scores, out_scores, parents, tokens, *, mask=None, finished=None, pad=0, normalize=True, workspace=None, stream=0):
    """One step of a beam search for G independent groups of K beams over V entries.

    Beam k of group g offers entry v at scores[g, k] + logits[g, k, v] - L, with L = log sum exp of the beam's allowed logits
    (`normalize`) or 0 (logits are values that add up as they are).  mask uint8 / bool [G, K, V] (nonzero = allowed; broadcast axes may
    have stride 0); a beam whose `finished` byte [G, K] is set offers only itself, as entry `pad` at its score.  A candidate
    at -inf or NaN does not exist, so a beam of score -inf is dead and a row without allowed entries offers nothing.
    out_scores float32, parents int32, tokens int32 [G, B] receive the B best, best first; equal ones in the order of
    (beam, entry).  Missing ones: -inf, -1, -1.  logits float32 / float16 / bfloat16 [G, K, V].  `workspace`: uint8 memory of
    beam_select_workspace(G, K, V, B) bytes, not shared with a call that may run at the same time.
    Returns (out_scores, parents, tokens)."""
    lp, lm = _get(logits)
    sp, sm = _get(scores)
    op, om = _get(out_scores, True)
    pp, pm = _get(parents, True)
    tp, tm = _get(tokens, True)
    mp, mm = (None, None) if mask is None else _get(mask)
    fp, fm = (None, None) if finished is None else _get(finished)
    wp, wm = (None, None) if workspace is None else _get(workspace, True)
    dev, ltype, g, k, v, lg, lk, mg, mk, b, nws = _plan(("select", lm, sm, om, pm, tm, mm, fm, wm), _select_plan, lm, sm, om, pm, tm, mm, fm, wm)
    if finished is None:
        pad = 0
    else:
        pad = int(pad)
        if not 0 <= pad < v:  # (here, not only behind ctypes, which would cut it to 32 bits)
            raise ValueError(f"beam_select: pad {pad} outside the {v} entries")
    lib = _lib()
    rc = lib.tg_beam_select(dev, stream, lp, ltype, g, k, v, lg, lk, sp, mp, mg, mk, fp, pad, 1 if normalize else 0, b, op, pp, tp, wp, nws)
    if rc:
        _check(lib, rc, "tg_beam_select")
    return out_scores, parents, tokens


def _select_plan(lm, sm, om, pm, tm, mm, fm, wm):
    lsh, lst, lt, d0 = _parse(lm, "beam_select: logits")
    ssh, sst, stt, d1 = _parse(sm, "beam_select: scores")
    osh, ost, ot, d2 = _parse(om, "beam_select: out_scores")
    psh, pst, pt, d3 = _parse(pm, "beam_select: parents")
    tsh, tst, tt, d4 = _parse(tm, "beam_select: tokens")
    ltype = _type(lt, "beam_select: logits", _FLOATS)
    _type(stt, "beam_select: scores", ("float32",))
    _type(ot, "beam_select: out_scores", ("float32",))
    _type(pt, "beam_select: parents", ("int32",))
    _type(tt, "beam_select: tokens", ("int32",))
    if len(lsh) != 3 or len(osh) != 2:
        raise ValueError(f"beam_select: logits must be [G, K, V] and out_scores [G, B], got {lsh} and {osh}")
    g, k, v = lsh
    b = osh[1]
    if not (1 <= k <= MAX_BEAMS and 1 <= b <= MAX_BEAMS and v >= 1):
        raise ValueError(f"beam_select: {k} beams in, {b} out, {v} entries: 1 .. {MAX_BEAMS} beams and at least one entry are supported")
    _inner(lsh, lst, "beam_select: logits")
    _dense(ssh, sst, (g, k), "beam_select: scores")
    for sh, st, what in ((osh, ost, "out_scores"), (psh, pst, "parents"), (tsh, tst, "tokens")):
        _dense(sh, st, (g, b), "beam_select: " + what)
    devs = [d0, d1, d2, d3, d4]
    mst = (0, 0)
    if mm is not None:
        sh, mst, t, d = _parse(mm, "beam_select: mask")
        _type(t, "beam_select: mask", ("uint8", "bool"))
        if sh != (g, k, v):
            raise ValueError(f"beam_select: mask must have shape {(g, k, v)}, got {sh}")
        _inner(sh, mst, "beam_select: mask")
        devs.append(d)
    if fm is not None:
        sh, st, t, d = _parse(fm, "beam_select: finished")
        _type(t, "beam_select: finished", ("uint8", "bool"))
        _dense(sh, st, (g, k), "beam_select: finished")
        devs.append(d)
    nws = 0
    if wm is not None:
        sh, st, t, d = _parse(wm, "beam_select: workspace")
        _type(t, "beam_select: workspace", ("uint8",))
        if len(sh) != 1:
            raise ValueError("beam_select: workspace must have one axis")
        _dense(sh, st, sh, "beam_select: workspace")
        nws = sh[0]
        devs.append(d)
    _int64("beam_select", g, v, *lst, *mst, nws)
    return _device(*devs), ltype, g, k, v, lst[0], lst[1], mst[0], mst[1], b, nws


def _state(meta, rows, what):
    """(bytes of a row, stride of a row in bytes, device) of [G * K, ...] or [G, K, ...]"""
    sh, st, t, d = _parse(meta, what)
    if t not in _SIZES:
        raise ValueError(f"{what}: unsupported element type {t}")
    lead, n = 0, 1
    while lead < len(sh) and (lead == 0 or n != rows):
        n *= sh[lead]
        lead += 1
    if n != rows or lead == 0:
        raise ValueError(f"{what}: the leading axes of {tuple(sh)} do not hold {rows} rows")
    size, cols = _SIZES[t], 1
    for s, k in zip(reversed(st[lead:]), reversed(sh[lead:])):
        if k > 1 and s != cols:
            raise ValueError(f"{what}: a row must be contiguous")
        cols *= k
    flat = _rows(tuple(sh[:lead]) + (1,), tuple(st[:lead]) + (1,), what)
    stride = flat[2] if flat[0] > 1 else cols
    _int64(what, cols * size, stride * size)
    return cols * size, stride * size, d


def beam_reorder(states, parents, *, out=None, beams_in=None, stream=0):
    """Rows that follow their beams: out[i][g, j] = states[i][g, parents[g, j]] for up to 24 arrays in one launch.

    states: an array or a list of arrays [G * K, ...] or [G, K, ...] of integers or floating-point numbers of 8 to 64 bits (other types:
    as a view of their bytes); parents int32 [G, B] as beam_select leaves
    them.  K = beams_in, by default B.  out: the same number of arrays with B rows per group (not overlapping states), or None to
    reorder in place (B = K).
    A parent outside 0 .. K - 1 (the -1 of a missing beam) leaves its row as it was.  Returns out (or states)."""
    src = states if isinstance(states, (list, tuple)) else (states,)
    pp, pm = _get(parents)
    sv = [_get(a, out is None) for a in src]
    dv = sv if out is None else [_get(a, True) for a in (out if isinstance(out, (list, tuple)) else (out,))]
    metas = tuple([m for _, m in sv])
    outs = None if out is None else tuple([m for _, m in dv])
    n, dev, g, k, b, ptrs, rows, ss, ds = _plan(("reorder", pm, metas, outs, beams_in), _reorder_plan, pm, metas, outs, beams_in)
    if n and g:
        lib = _lib()
        rc = lib.tg_beam_reorder(dev, stream, n, ptrs(*[p for p, _ in sv]), ptrs(*[p for p, _ in dv]), rows, ss, ds, g, k, b, pp)
        if rc:
            _check(lib, rc, "tg_beam_reorder")
    return states if out is None else out


def _reorder_plan(pm, metas, outs, beams_in):
    n = len(metas)
    if outs is not None and len(outs) != n:
        raise ValueError(f"beam_reorder: {n} states, {len(outs)} outputs")
    if n > MAX_STATES:
        raise ValueError(f"beam_reorder: {n} arrays: up to {MAX_STATES} go into one call")
    psh, pst, pt, dev = _parse(pm, "beam_reorder: parents")
    _type(pt, "beam_reorder: parents", ("int32",))
    if len(psh) != 2:
        raise ValueError(f"beam_reorder: parents must be [G, B], got {psh}")
    _dense(psh, pst, psh, "beam_reorder: parents")
    g, b = psh
    k = b if beams_in is None else int(beams_in)
    if not (1 <= k <= MAX_BEAMS and 1 <= b <= MAX_BEAMS):
        raise ValueError(f"beam_reorder: {k} beams in, {b} out: 1 .. {MAX_BEAMS} are supported")
    if outs is None and k != b:
        raise ValueError(f"beam_reorder: in place takes as many beams out ({b}) as in ({k})")
    _int64("beam_reorder", g * k, g * b)
    num = C.c_int64 * n
    if g == 0:
        return n, 0, g, k, b, C.c_void_p * n, num(), num(), num()
    sv = [_state(m, g * k, f"beam_reorder: states[{i}]") for i, m in enumerate(metas)]
    dv = sv if outs is None else [_state(m, g * b, f"beam_reorder: out[{i}]") for i, m in enumerate(outs)]
    for i, (s, d) in enumerate(zip(sv, dv)):
        if s[0] != d[0]:
            raise ValueError(f"beam_reorder: rows of states[{i}] hold {s[0]} bytes, of out[{i}] {d[0]}")
    return (n, _device(dev, *(s[2] for s in sv), *(d[2] for d in dv)), g, k, b, C.c_void_p * n, num(*(s[0] for s in sv)), num(*(s[1] for s in sv)),
            num(*(d[1] for d in dv)))
