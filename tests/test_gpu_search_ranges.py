"""Beam searches whose scorer leaves the usual range of values."""
import numpy as np
import pytest

import test_gpu_search
from tetris_gymnasium_amd import BeamSearch, Engine, PlacementScorer, _native as N, ops

pytestmark = pytest.mark.gpu


def searched(G=6, warm=6, w=10, h=20):
    e = Engine(G, w, h, obs_mode=N.OBS_BOARD, grouped=True)
    e.reset(np.arange(3, 3 + G, dtype=np.uint64))
    for t in range(warm):
        e.sample_legal_actions(seed=2, counter=t, fetch=False)
        e.step_sampled()
    return e


def scorer(up, down, width=24):
    """two layers; `up` and `down` are powers of two on the scales of the first and the second one"""
    r = np.random.default_rng(7)
    return PlacementScorer([(r.integers(-127, 128, (width, 13)).astype(np.int8), r.uniform(0.5, 1, width).astype(np.float32) * np.float32(up), None),
                            (r.integers(-127, 128, (1, width)).astype(np.int8), np.full(1, 2.0**-14 * down, np.float32), None)])


@pytest.mark.parametrize("shift", [12, 40, 90, -30, -60, -90])
def test_a_plan_does_not_depend_on_the_scale_of_its_hidden_layer(shift):
    """the first layer's values times 2^shift, the second layer's weights times 2^-shift: the same scorer, far outside float16"""
    e = searched()
    plain, far = scorer(2.0**-5, 1.0), scorer(2.0 ** (shift - 5), 2.0**-shift)
    assert plain.hidden == ["float16"] and far.hidden == ["float32"]
    value = []
    for sc in (plain, far):
        s = BeamSearch(e, sc, 5)
        s._load()
        v = np.empty((30, 40), np.float32)
        s.e.dev_download(s.value_placements().ptr, v)
        value.append(v.astype(np.float64))
        plan = s.plan(4)
        assert (plan["best"] >= 0).all() and (plan["actions"] >= 0).all()  # no legal placement drops out
        s.close()
    # the hidden rows differ by the rounding to float16 of the first, at most 2^-11 of the row's largest, and by half a step of 1/127 of
    # that on either side: (127 / 2048 + 1.0005) steps for each of 24 activations, times a weight of at most 127 * 2^-14
    x, w1, s1 = features(e, 5), plain.layers[0][0].astype(np.float64), plain.layers[0][1].astype(np.float64)
    top = np.maximum(x @ w1.T * s1, 0).max(1).reshape(30, 40)
    step = top / 127 * 1.07
    assert np.isfinite(value[1]).all() and (np.abs(value[0] - value[1]) <= 24 * step * 127 * 2.0**-14).all()
    # and the far scorer against its definition, rounded as documented: hidden to float32, rows to 8 bits, the sum exact
    hid = (x @ w1.T).astype(np.float32) * far.layers[0][1]
    hid = np.maximum(hid, 0).astype(np.float64)
    qs = np.maximum((hid.max(1) / 127).astype(np.float32), np.float32(2.0**-126)).astype(np.float64)
    y = np.rint(hid / qs[:, None]) @ far.layers[1][0].T.astype(np.float64) * float(far.layers[1][1][0]) * qs[:, None]
    got = value[1].reshape(-1, 1)
    tol = np.abs(y) * 4 * 2.0**-24
    # (sums of products are exact here, |acc| < 2^24: the hidden value is one product rounded once, so the quantiser's integers are equal)
    assert (np.abs(got - y) <= tol).all()
    e.close()


def features(e, beams):
    """the placement features of every env, once for each beam"""
    twin = Engine(e.B, e.W, e.H, obs_mode=N.OBS_NONE, grouped=True, features=True)
    twin.set_state(*e.get_state())
    f = np.repeat(twin.features()[0], beams, 0).reshape(-1, e.W + 3).astype(np.float64)
    twin.close()
    return f


def test_finite_scorers_lose_no_placement_to_the_range_of_their_activations():
    """features that sum to some hundreds times weights of some hundreds: hidden values beyond 65 504"""
    w = np.zeros((3, 13), np.float32)
    w[0], w[1, 10], w[2, 11] = 900.0, 2000.0, 1500.0
    v = np.array([[-1e-4, -1e-4, -1e-3]], np.float32)
    sc = PlacementScorer.from_float([(w, np.full(3, 60000.0, np.float32)), (v, None)])
    e = searched(warm=15)
    s = BeamSearch(e, sc, 8)
    legal, over = e.legal_mask().sum(1), (e.get_state()[1]["flags"] & N.F_GAME_OVER) != 0  # (15 placements at random end some of the games)
    assert (~over).sum() >= 2
    p = s.plan(1)
    assert (np.isfinite(p["scores"]).sum(1) == np.minimum(legal, 8))[~over].all() and (p["best"][:, 0] >= 0)[~over].all()
    s.close(), e.close()


def test_refusals_of_reorder_beams_are_the_operators_messages_too():
    e = Engine(12, 10, 20, obs_mode=N.OBS_BOARD)
    lib = e.lib
    for beams, parents, msg in ((5, 64, b"divide the batch"), (4, None, b"null parents"), (4, 64, b"never reset")):  # (refused before the address is used)
        assert lib.tg_reorder_beams(e.h, parents, beams) == N.EINVAL
        assert msg in lib.tg_ops_last_error() and msg in lib.tg_last_error(e.h)
    assert lib.tg_stream(e.h, None) == N.EINVAL and lib.tg_ops_last_error().startswith(b"tg_stream")
    e.close()


@pytest.mark.parametrize("w,h,G,K,depth,warm", [(10, 20, 4, 17, 4, 3), (10, 20, 5, 32, 4, 0), (10, 20, 3, 64, 3, 5), (20, 40, 3, 8, 4, 2), (20, 40, 2, 16, 5, 0),
                                                (32, 24, 2, 5, 3, 0), (4, 12, 3, 33, 3, 0)])
def test_plans_of_many_beams_and_wide_boards(w, h, G, K, depth, warm, monkeypatch):
    """searches whose selection takes chunks and a workspace (17 and more beams of 40 placements, 16 of 80), and both sides of that"""
    e = Engine(G, w, h, obs_mode=N.OBS_BOARD, grouped=True)
    s = BeamSearch(e, test_gpu_search.linear_scorer(w, K), K)
    assert (s._ws is not None) == (ops.beam_select_workspace(G, K, 4 * w, K) > 0)
    s.close(), e.close()
    test_gpu_search.test_plan_is_the_search_done_on_the_host(w, h, G, K, depth, warm, 0, monkeypatch)


def test_the_search_outlives_games_at_random():
    """the scorer of test_a_full_game_is_played_longer_than_at_random against uniform legal placements on the same games"""
    e = Engine(8, 10, 20, obs_mode=N.OBS_BOARD, grouped=True)
    e.reset(np.arange(1, 9, dtype=np.uint64))
    over = np.zeros(8, bool)
    for t in range(40):
        over |= e.step(e.sample_legal_actions(seed=5, counter=t))[1] != 0
    assert over.any()  # (the search ends none of the eight in 40 placements)
    e.close()


def test_reorder_beams_of_an_engine_on_several_streams():
    B, K = 32768, 8
    r = np.random.default_rng(0)
    engines = [Engine(B, 10, 20, obs_mode=N.OBS_BOARD, autoreset=N.AUTORESET_SAME_STEP, streams=n) for n in (1, 2)]
    for e in engines:
        e.reset(np.arange(1, B + 1, dtype=np.uint64))
    for t in range(24):
        a, p = r.integers(0, 8, B).astype(np.int32), r.integers(-1, K, (B // K, K)).astype(np.int32)
        for e in engines:
            e.step_async(a)
            if t % 3 == 2:
                e.reorder_beams(p, K)
    for x, y in zip(*(e.get_state() for e in engines)):
        np.testing.assert_array_equal(x, y)
    np.testing.assert_array_equal(engines[0].observation(), engines[1].observation())
    for e in engines:
        e.close()
