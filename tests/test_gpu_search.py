"""Engine.reorder_beams against states permuted on the host, and the beam search over placements against the same search in NumPy."""
import numpy as np
import pytest

from ops_util import Box
from tetris_gymnasium_amd import BeamSearch, Engine, EngineError, PlacementScorer, _native as N, ops
from tetris_gymnasium_amd.engine import DeviceBuffer

pytestmark = pytest.mark.gpu

CONFIGS = {
    "board": dict(obs_mode=N.OBS_BOARD, autoreset=N.AUTORESET_SAME_STEP, episode_stats=True, final_obs=True),
    "dict": dict(obs_mode=N.OBS_DICT, autoreset=N.AUTORESET_NEXT_STEP),
    "rgb": dict(obs_mode=N.OBS_RGB, autoreset=N.AUTORESET_SAME_STEP, episode_stats=True),
    "grouped": dict(obs_mode=N.OBS_BOARD, grouped=True, features=True),
    "functional": dict(ruleset=N.RULESET_FUNCTIONAL, obs_mode=N.OBS_FN, autoreset=N.AUTORESET_SAME_STEP),
    "small": dict(width=6, height=12, obs_mode=N.OBS_BOARD, autoreset=N.AUTORESET_SAME_STEP),
    "inline": dict(obs_mode=N.OBS_BOARD, autoreset=N.AUTORESET_SAME_STEP, ring_fill=0),
}


def everything(e):
    board, rec, rng = e.get_state()
    obs = e.observation()
    obs = {"obs_" + k: v for k, v in obs.items()} if isinstance(obs, dict) else {"obs": obs}
    out = {"b2": board, "rec": rec, "rng": rng, "out": e.fetch_step_out(), **obs}
    return out


def equal(a, b):
    for k in a:
        np.testing.assert_array_equal(a[k], b[k], err_msg=k)


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("packed", [False, True])
def test_reorder_beams_moves_whole_environments(name, packed, monkeypatch):
    if packed:
        if name not in ("board", "grouped", "functional", "small"):
            pytest.skip("this surface has no nibble boards")
        monkeypatch.setenv("TG_PACKED", "1")
    kw = dict(CONFIGS[name])
    if packed:
        kw.pop("final_obs", None)
    w, h = kw.pop("width", 10), kw.pop("height", 20)
    G, K = 30, 6  # (a batch that fills no whole wave; a multiple of 4, as tg_rollout takes it)
    B = G * K
    r = np.random.default_rng(len(name))
    a = Engine(B, w, h, **kw)
    twin = Engine(B, w, h, **kw)  # receives the same states by tg_set_state
    a.reset(np.arange(1, B + 1, dtype=np.uint64))
    for round_ in range(4):
        for _ in range(7 + round_):
            a.step_async(r.integers(0, a.n_actions, B))
        p = r.integers(-1, K, (G, K)).astype(np.int32)
        before = everything(a)
        eps = a.episode_stats() if kw.get("episode_stats") else None
        a.reorder_beams(p, K)
        env = np.where(p < 0, np.arange(K), p) + np.arange(G)[:, None] * K
        env = env.reshape(-1)
        after = everything(a)
        equal(after, {k: v[env] for k, v in before.items()})
        if eps is not None:
            np.testing.assert_array_equal(a.episode_stats(), eps[env])
        twin.set_state(before["b2"][env], before["rec"][env], before["rng"][env])
        for _ in range(9):
            act = r.integers(0, a.n_actions, B)
            equal({k: v for k, v in zip("rtl", a.step(act))}, {k: v for k, v in zip("rtl", twin.step(act))})
        x, y = everything(a), everything(twin)
        x.pop("out"), y.pop("out")
        equal(x, y)
    acts = r.integers(0, a.n_actions, (16, B))  # ... and launches of several transitions go on from there
    a.reorder_beams(p, K)
    b2, rec, rng = a.get_state()
    twin.set_state(b2, rec, rng)
    if not kw.get("grouped"):
        for u, v in zip(a.rollout(acts), twin.rollout(acts)):
            np.testing.assert_array_equal(u, v)
    a.close(), twin.close()


def test_reorder_beams_takes_device_parents_and_refuses_bad_ones():
    e = Engine(12, 10, 20, obs_mode=N.OBS_BOARD)
    with pytest.raises(EngineError, match="never reset"):
        e.reorder_beams(np.zeros(12, np.int32), 4)
    e.reset(np.arange(1, 13, dtype=np.uint64))
    _, rec, rng = e.get_state()
    buf = DeviceBuffer(e, 48)
    e.dev_upload(buf.ptr, np.array([1, 1, 2, 99] * 3, np.int32))
    for p in (buf, buf.ptr, ops.DeviceView(buf.ptr, (3, 4), "int32")):
        e.set_state(None, rec, rng)
        e.reorder_beams(p, 4)
        np.testing.assert_array_equal(e.get_state()[2], rng[[1, 1, 2, 3, 5, 5, 6, 7, 9, 9, 10, 11]])
    for p, k, msg in ((np.zeros(12, np.int32), 5, "divide"), (np.zeros(11, np.int32), 4, "12 integers"), (np.zeros(12), 4, "12 integers"),
                      (ops.DeviceView(buf.ptr, (12,), "float32"), 4, "int32"), (ops.DeviceView(buf.ptr, (11,), "int32"), 1, "int32")):
        with pytest.raises(ValueError, match=msg):
            e.reorder_beams(p, k)
    e.close()


def linear_scorer(w, seed):
    """one layer whose values are exact in float32: integer features times integers times a power of two"""
    r = np.random.default_rng(seed)
    return PlacementScorer([(r.integers(-20, 8, (1, w + 3)).astype(np.int8), np.array([2.0**-6], np.float32), np.array([0.5], np.float32))])


@pytest.mark.parametrize("w,h,G,K,depth,warm,packed", [(10, 20, 5, 4, 5, 0, 0), (6, 12, 7, 8, 12, 9, 0), (10, 20, 3, 1, 3, 4, 0), (10, 24, 2, 16, 6, 20, 0),
                                                       (10, 20, 4, 6, 8, 11, 1)])
def test_plan_is_the_search_done_on_the_host(w, h, G, K, depth, warm, packed, monkeypatch):
    if packed:  # nibble boards
        monkeypatch.setenv("TG_PACKED", "1")
    main = Engine(G, w, h, obs_mode=N.OBS_BOARD, grouped=True)
    main.reset(np.arange(5, 5 + G, dtype=np.uint64))
    for t in range(warm):
        main.sample_legal_actions(seed=1, counter=t, fetch=False)
        main.step_sampled()
    scorer = linear_scorer(w, K)
    s = BeamSearch(main, scorer, K)
    before = main.get_state()
    plans = [s.plan(depth), s.plan(1), s.plan(depth)]
    for a, b in zip(before, main.get_state()):
        np.testing.assert_array_equal(a, b)  # the searched engine is only read
    for k in plans[0]:
        np.testing.assert_array_equal(plans[0][k], plans[2][k])
    got = plans[0]
    # the same in NumPy around an engine that only steps
    e = Engine(G * K, w, h, obs_mode=N.OBS_NONE, grouped=True, features=True)
    st = [np.repeat(a, K, 0) for a in before]
    e.set_state(*st)
    cum = np.full((G, K), -np.inf, np.float32)
    cum[:, 0] = 0
    seq = np.full((G, K, 0), -1, np.int32)
    wt, sc, b = scorer.layers[0]
    for d in range(depth):
        f, _ = e.features()
        mask = e.legal_mask().reshape(G, K, -1)
        val = (f.astype(np.int64) @ wt[0].astype(np.int64) * float(sc[0]) + float(b[0])).reshape(G, K, -1)
        c = np.where(mask != 0, cum[:, :, None] + val, -np.inf).reshape(G, -1)
        first = np.argsort(-c, 1, kind="stable")[:, :K]
        top = np.take_along_axis(c, first, 1)
        par = np.where(top > -np.inf, first // (4 * w), -1)
        tok = np.where(top > -np.inf, first % (4 * w), -1)
        i = np.maximum(par, 0)
        seq = np.concatenate([np.where(par[:, :, None] >= 0, np.take_along_axis(seq, i[:, :, None], 1), -1), tok[:, :, None]], 2)
        cum = np.where(par >= 0, np.take_along_axis(cum, i, 1), -np.inf).astype(np.float32)
        env = (np.where(par >= 0, par, np.arange(K)) + np.arange(G)[:, None] * K).reshape(-1)
        e.set_state(*(a[env] for a in e.get_state()))
        rew, term, _ = e.step(np.maximum(tok, 0).reshape(-1).astype(np.int32))
        cum = np.where(term.reshape(G, K) != 0, -np.inf, cum + rew.reshape(G, K)).astype(np.float32)
    np.testing.assert_array_equal(got["actions"], seq)
    np.testing.assert_array_equal(got["scores"], top.astype(np.float32))
    np.testing.assert_array_equal(got["returns"], cum)
    pick = np.where((cum > -np.inf).any(1), (cum > -np.inf).argmax(1), 0)
    np.testing.assert_array_equal(got["best"], seq[np.arange(G), pick])
    # the planned actions, played by the searched engine, collect the planned rewards
    ret = np.zeros(G, np.float32)
    for d in range(depth):
        ret += np.where(got["best"][:, d] >= 0, main.step(np.maximum(got["best"][:, d], 0))[0], 0)
    alive = got["returns"][np.arange(G), pick] > -np.inf
    np.testing.assert_array_equal(ret[alive], got["returns"][np.arange(G), pick][alive])
    s.close(), e.close(), main.close()


def test_values_of_a_scorer_with_hidden_layers():
    r = np.random.default_rng(3)
    main = Engine(4, 10, 20, obs_mode=N.OBS_BOARD)
    main.reset(np.arange(1, 5, dtype=np.uint64))
    sc = PlacementScorer.from_float([(r.normal(size=(32, 13)) / 13, r.normal(size=32)), (r.normal(size=(17, 32)), None), (r.normal(size=(1, 17)), np.ones(1))])
    s = BeamSearch(main, sc, 3)
    s._load()
    got = np.empty((12 * 40,), np.float32)
    s.e.dev_download(s.value_placements().ptr, got)
    x = s.e.features()[0].reshape(-1, 13).astype(np.float64)
    down = lambda v, dt: s.e.dev_download(v.ptr, np.empty(v.shape, dt))  # noqa: E731
    for i, ((w, ws, b), (_, q, _, _, _, y, _)) in enumerate(zip(sc.layers, s._layers)):  # every layer from what the one before left
        scale = 1.0
        if i:
            amax = np.abs(x).max(1)
            es = np.maximum((amax / 127).astype(np.float32), np.float32(2.0**-126))
            np.testing.assert_array_equal(down(q[1], np.float32), es)
            x = np.rint(x / es[:, None].astype(np.float64))
            np.testing.assert_array_equal(down(q[0], np.int8), x.astype(np.int8))
            scale = es[:, None].astype(np.float64)
        p = (x @ w.T.astype(np.float64)) * ws.astype(np.float64) * scale
        e = p + (0 if b is None else b)
        last = i + 1 == len(sc.layers)
        # float32 as in linear_i8's own test; then half a step of float16 (of its smallest normal value below that)
        tol = np.abs(p) * 2.01 * 2.0**-24 + np.abs(e) * (2.0**-24 + (0 if last else 2.0**-11)) * 1.01 + (2.0**-149 if last else 2.0**-25)
        out = got[:, None] if last else down(y, np.float16)
        assert (np.abs(out.astype(np.float64) - (e if last else np.maximum(e, 0))) <= tol).all()
        x = out.astype(np.float64)
    assert s.plan(3)["actions"].shape == (4, 3, 3)
    s.close(), main.close()


def test_search_refusals():
    sc = linear_scorer(10, 0)
    fn = Engine(2, 10, 20, ruleset=N.RULESET_FUNCTIONAL, obs_mode=N.OBS_FN)
    with pytest.raises(EngineError, match="NUMPY"):
        BeamSearch(fn, sc)
    e = Engine(2, 10, 20, obs_mode=N.OBS_BOARD)
    e.reset(np.array([1, 2], np.uint64))
    for bad in (dict(beams=0), dict(beams=65), dict(scorer=linear_scorer(8, 0))):
        with pytest.raises(ValueError):
            BeamSearch(e, bad.pop("scorer", sc), **bad)
    s = BeamSearch(e, sc, 2)
    with pytest.raises(ValueError, match="depth"):
        s.plan(0)
    s.close(), e.close(), fn.close()


def test_a_full_game_is_played_longer_than_at_random():
    """the search at work: placements planned with a scorer against holes and height (weights by hand: no learning here)"""
    w = np.zeros((1, 13), np.float32)
    w[0, :10], w[0, 10], w[0, 11], w[0, 12] = -0.5, 0, -7.0, -1.8
    e = Engine(8, 10, 20, obs_mode=N.OBS_BOARD, grouped=True)
    e.reset(np.arange(1, 9, dtype=np.uint64))
    s = BeamSearch(e, PlacementScorer.from_float([(w, None)]), 6)
    over = np.zeros(8, bool)
    for _ in range(40):
        over |= e.step(np.maximum(s.plan(2)["best"][:, 0], 0))[1] != 0
    assert not over.any()
    s.close(), e.close()


def test_deeper_plans_do_not_pile_up_memory():
    e = Engine(3, 10, 20, obs_mode=N.OBS_BOARD)
    e.reset(np.array([1, 2, 3], np.uint64))
    s = BeamSearch(e, linear_scorer(10, 0), 2)
    first = [s.plan(d) for d in (1, 2)]
    held = len(s._bufs)
    deeper = [s.plan(d) for d in (3, 4, 5)]
    assert len(s._bufs) == held
    again = s.plan(2)  # shorter ones in the longer buffers
    for k in first[1]:
        np.testing.assert_array_equal(again[k], first[1][k])
    assert [p["actions"].shape[2] for p in deeper] == [3, 4, 5]
    s.close(), e.close()
