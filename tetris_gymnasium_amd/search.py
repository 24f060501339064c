"""Beam search over placements, on the device: from the state of every env of an engine, the best sequences of grouped actions
(column * 4 + rotation, wrappers/grouped.py:124-269) under a learned value of the placement's feature vector
(wrappers/observation.py:236-278, the observation examples/train_lin_grouped.py learns from).

Every move of the search runs, without a wait or a copy to the host in between: the features of all 4W placements
(tg_features) → the scorer's 8-bit layers (ops.linear_i8, ops.quantize_i8) → the best continuations of each env's beams under the
legal mask (ops.beam_select) → the beams' environments follow (tg_reorder_beams) → one transition (tg_step)."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _native as N
from . import ops
from .engine import DeviceBuffer, Engine, EngineError


_F16_MAX, _F16_STEP = 65504.0, 2.0**-24


class PlacementScorer:
    """A multi-layer perceptron over feature vectors in 8-bit integers: layers of (weight int8 [out, in], scale float32 [out], bias
    float32 [out] or None), relu between them, one output.  The first layer reads the uint8 features, each later one the rows
    of the layer before quantised to 8 bits.  Layers whose values could pass the range of float32 are refused.

    `hidden` names the type each hidden layer's activations are kept in.  The quantiser behind them rounds to 1/254 of the row's largest,
    so float16's relative 2^-11 is an eighth of that and half the bytes of float32; its range is what decides: float16 where no
    features can take the layer beyond 65 504 and its last step, 2^-24, is not above what one step of one weight adds for
    one unit of one feature (rounding to it then loses no more than rounding that weight to 8 bits did), else float32."""

    def __init__(self, layers):
        self.layers, self.hidden = [], []
        reach, least = 255.0, 1.0  # the most an input of the layer can be, and the least step of one (features: bytes)
        for i, (w, s, b) in enumerate(layers):
            w, s = np.asarray(w), np.ascontiguousarray(s, np.float32)
            b = None if b is None else np.ascontiguousarray(b, np.float32)
            if w.dtype != np.int8 or w.ndim != 2:
                raise ValueError(f"layer {i}: weight must be int8 [out, in], got {w.dtype} {w.shape}")
            if s.shape != (w.shape[0],) or (b is not None and b.shape != (w.shape[0],)):
                raise ValueError(f"layer {i}: scale and bias must have shape {(w.shape[0],)}")
            if self.layers and self.layers[-1][0].shape[0] != w.shape[1]:
                raise ValueError(f"layer {i} takes {w.shape[1]} inputs, layer {i - 1} gives {self.layers[-1][0].shape[0]}")
            self.layers.append((np.ascontiguousarray(w), s, b))
            with np.errstate(all="ignore"):
                # (a weight of 0 counts as 1: the product of the two scales has to be finite too)
                most = np.maximum(np.abs(w.astype(np.float64)).sum(1), 1) * np.abs(s.astype(np.float64)) * reach
                most = float(np.max(most if b is None else most + np.abs(b.astype(np.float64)), initial=0.0))
                least *= float(np.min(np.abs(s), initial=1.0))
            if not most <= float(np.finfo(np.float32).max):  # (also a scale or a bias that is not a number)
                raise ValueError(f"layer {i}: its values are not bounded by the range of float32 (up to {most:.3g})")
            self.hidden.append("float16" if most <= _F16_MAX and least >= _F16_STEP else "float32")
            reach = most * (1 + 2.0**-10)  # (rounded to its type, then scale times 127)
        self.hidden = self.hidden[:-1]
        if not self.layers or self.layers[-1][0].shape[0] != 1:
            raise ValueError("a scorer needs at least one layer, and the last one has one output")

    @classmethod
    def from_float(cls, layers):
        """layers of (weight [out, in], bias [out] or None) in floating point: every output channel's weights to 8 bits with a scale"""
        out = []
        for w, b in layers:
            w = np.asarray(w, np.float32)
            if w.ndim != 2:
                raise ValueError(f"weight must be [out, in], got {w.shape}")
            if not np.isfinite(w).all():
                raise ValueError("weights must be finite")
            s = np.maximum(np.abs(w).max(1, initial=0) / np.float32(127), np.float32(2.0**-126)).astype(np.float32)
            out.append((np.rint(w.astype(np.float64) / s[:, None]).astype(np.int8), s, b))
        return cls(out)

    @property
    def n_features(self):
        return self.layers[0][0].shape[1]


class BeamSearch:
    """`beams` parallel continuations for every env of `engine` (NUMPY rules, stock mappings or its own), on a second engine of
    batch * beams environments next to it; `engine` itself is only read.  plan() may be called any number of times.  States are searched as
    they are, without resets: for an env whose game is over, what a plan says is of no use.  The search steps copies of the
    environments with their generators, so it knows every piece to come, also behind the visible queue: its returns are not those of a
    policy that sees the observation alone."""

    def __init__(self, engine: Engine, scorer: PlacementScorer, beams=8):
        if engine.ruleset != N.RULESET_NUMPY:
            raise EngineError("BeamSearch: the grouped action set belongs to the NUMPY rule-set")
        beams = int(beams)
        if not 1 <= beams <= ops.MAX_BEAMS:
            raise ValueError(f"BeamSearch: 1 .. {ops.MAX_BEAMS} beams, got {beams}")
        if scorer.n_features != engine.W + 3:
            raise ValueError(f"BeamSearch: the scorer takes {scorer.n_features} features, a {engine.W}-column board has {engine.W + 3}")
        engine._need_ops()
        self.engine, self.scorer, self.beams, self.G = engine, scorer, beams, engine.B
        self.device = int(engine.cfg.device)
        self.e = e = Engine(engine.B * beams, engine.W, engine.H, queue_size=engine.Q, gravity=bool(engine.cfg.gravity), obs_mode=N.OBS_NONE,
                            grouped=True, features=True, device=self.device, env_offset=engine.cfg.env_offset,
                            terminate_on_illegal=bool(engine.cfg.grouped_terminate_on_illegal), rewards_mapping=engine.rewards)
        G, K, V, n = self.G, beams, 4 * e.W, e.B
        self.stream = e.stream
        self._bufs = []
        f = lambda shape, dtype: self._view(shape, dtype)  # noqa: E731
        self.cum, self.cum2, self.first = f((G, K), "float32"), f((G, K), "float32"), np.full((G, K), -np.inf, np.float32)
        self.first[:, 0] = 0
        self.values, self.scores = f((G, K, V), "float32"), f((G, K), "float32")
        self.actions = f((n,), "int32")
        p, _ = e.device_ptr(N.BUF_PLACEMENT_FEATS)
        self._x = ops.DeviceView(p, (n * V, e.W + 3), "uint8", device=self.device)
        self._mask_ptr, _ = e.device_ptr(N.BUF_LEGAL_MASK)
        self.mask = ops.DeviceView(self._mask_ptr, (G, K, V), "uint8", device=self.device)
        self._out_ptr, _ = e.device_ptr(N.BUF_STEP_OUT)
        need = ops.beam_select_workspace(G, K, V, K)
        self._ws = f((need,), "uint8") if need else None
        self._layers = []
        x = self._x
        for i, (w, s, b) in enumerate(scorer.layers):
            last = i + 1 == len(scorer.layers)
            y = ops.DeviceView(self.values.ptr, (n * V, 1), "float32", device=self.device) if last else f((n * V, w.shape[0]), scorer.hidden[i])
            q = None if i == 0 else (f((n * V, w.shape[1]), "int8"), f((n * V,), "float32"))
            self._layers.append((x, q, self._put(w), self._put(s), None if b is None else self._put(b), y, not last))
            x = y
        # the state of the searched engine, in its own memory: one row per env
        self._src = [(e.H * e.W, "uint8"), (N.ENV_REC.itemsize, "uint8"), (N.RNG_REC.itemsize, "uint8")]
        self._state = [f((n, b), t) for b, t in self._src]
        self._zero = self._put(np.zeros((G, K), np.int32))
        self._steps = None

    # -- memory ------------------------------------------------------------------------------------
    def _view(self, shape, dtype):
        b = DeviceBuffer(self.e, max(int(np.prod(shape, dtype=np.int64)) * ops._SIZES[dtype], 16))
        self._bufs.append(b)
        return ops.DeviceView(b.ptr, shape, dtype, device=self.device)

    def _put(self, a):
        v = self._view(a.shape, a.dtype.name)
        if a.size:
            self.e.dev_upload(v.ptr, a)
        return v

    def close(self):
        self._bufs = []
        self.e.close()

    def _open(self):
        """in front of every use of the views: they point into memory, and run on a stream, that close() has given back"""
        if not getattr(self.e, "h", None):
            raise EngineError("this BeamSearch has been closed")
        if not getattr(self.engine, "h", None):
            raise EngineError("BeamSearch: the engine it searches has been closed")

    # -- one search --------------------------------------------------------------------------------
    def _load(self):
        """every beam of group g := env g of the searched engine; the first beam alive at 0, the others dead"""
        self._open()
        state = self.engine.get_state_device()
        self.engine.sync()  # (the two engines' streams)
        src = [ops.DeviceView(b.ptr, (self.G, n), t, device=self.device) for b, (n, t) in zip(state, self._src)]
        ops.beam_reorder(src, self._zero, out=self._state, beams_in=1, stream=self.stream)
        self.e.set_state_device(*(v.ptr for v in self._state), unchecked=True)
        self.e.dev_upload(self.cum.ptr, self.first)  # (waits: `state` goes back to its engine's free list behind the copy)
        del state

    def value_placements(self):
        """The scorer's values of all placements of all beams' current states: float32 [G, beams, 4W] device memory."""
        self._open()
        st = self.stream
        self.e._chk(self.e.lib.tg_features(self.e.h), "tg_features")
        for x, q, w, s, b, y, relu in self._layers:
            if q is None:
                ops.linear_i8(x, w, s, y, bias=b, relu=relu, stream=st)
            else:
                ops.quantize_i8(x, q[0], q[1], stream=st)
                ops.linear_i8(q[0], w, s, y, x_scale=q[1], bias=b, relu=relu, stream=st)
        return self.values

    def plan(self, depth):
        """Search `depth` placements ahead.  A beam's rank is the reward collected so far plus the value of its next placement; a beam
        whose game ends is dropped.  Returns {"actions" int32 [G, beams, depth] (-1: no such beam), "scores" float32 [G, beams] (the
        rank of each beam's last placement, best first; -inf: no such beam), "returns" float32 [G, beams] (the rewards collected, -inf
        where the game ended with the last placement)}; "best" int32 [G, depth]: the actions of the best beam still alive (else the
        best of all)."""
        depth = int(depth)
        if depth < 1:
            raise ValueError(f"plan: depth must be at least 1, got {depth}")
        self._open()
        e, G, K, st = self.e, self.G, self.beams, self.stream
        if self._steps is None or self._steps[0].shape[0] < depth:
            self._bufs = [b for b in self._bufs if self._steps is None or b.ptr not in (self._steps[0].ptr, self._steps[1].ptr)]
            self._steps = (self._view((depth, G, K), "int32"), self._view((depth, G, K), "int32"))
        par, tok = self._steps
        self._load()
        lib, h = e.lib, e.h
        for d in range(depth):
            pv, tv = (ops.DeviceView(a.ptr + 4 * d * G * K, (G, K), "int32", device=self.device) for a in (par, tok))
            self.value_placements()
            e._chk(lib.tg_grouped_enumerate(h, None), "tg_grouped_enumerate")
            ops.beam_select(self.values, self.cum, self.scores, pv, tv, mask=self.mask, normalize=False, workspace=self._ws, stream=st)
            ops._check(lib, lib.tg_beam_advance(self.device, st, G, K, pv.ptr, tv.ptr, self.cum.ptr, self.cum2.ptr, self.actions.ptr), "tg_beam_advance")
            e._chk(lib.tg_reorder_beams(h, C.c_void_p(pv.ptr), K), "tg_reorder_beams")
            e.step_device(self.actions.ptr)
            ops._check(lib, lib.tg_beam_collect(self.device, st, G * K, self._out_ptr, self.cum2.ptr), "tg_beam_collect")
            self.cum, self.cum2 = self.cum2, self.cum
        parents, tokens = np.empty((depth, G, K), np.int32), np.empty((depth, G, K), np.int32)
        scores, returns = np.empty((G, K), np.float32), np.empty((G, K), np.float32)
        for v, a in ((par, parents), (tok, tokens), (self.scores, scores), (self.cum, returns)):
            e.dev_download(v.ptr, a)
        e.sync()
        actions = np.full((G, K, depth), -1, np.int32)
        at = np.where(parents[-1] >= 0, np.arange(K), -1)
        for d in range(depth - 1, -1, -1):  # from each last beam back to the root
            ok = at >= 0
            i = np.maximum(at, 0)
            actions[:, :, d] = np.where(ok, np.take_along_axis(tokens[d], i, 1), -1)
            at = np.where(ok, np.take_along_axis(parents[d], i, 1), -1)
        alive = returns > -np.inf
        pick = np.where(alive.any(1), alive.argmax(1), 0)
        return {"actions": actions, "scores": scores, "returns": returns, "best": actions[np.arange(G), pick]}
