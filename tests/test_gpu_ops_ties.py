"""beam_select over rows of many equal or ordered logits: what its lists have to be narrowed for, at every chunk size."""
import time

import numpy as np
import pytest

from ops_util import Box, rounded
from test_gpu_ops import select_case
from tetris_gymnasium_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def box():
    b = Box()
    yield b
    b.close()


def rows(kind, g, k, v, r):
    if kind == "equal":
        return np.full((g, k, v), -2.5)
    x = r.normal(size=(g, k, v)) * 3
    if kind == "clipped":  # a quarter of them at the top
        return np.minimum(x, 2.0)
    if kind == "coarse":
        return np.round(x)
    if kind == "two":  # fewer above than are wanted, and many below them
        return np.where(r.random((g, k, v)) < 3.0 / v, 1.0, -1.0)
    if kind == "zeros":
        return np.where(r.random((g, k, v)) < 0.5, 0.0, -0.0)
    if kind == "infinite":
        return np.where(x > 1, np.inf, x)
    x = np.sort(x, 2)
    return x if kind == "rising" else x[:, :, ::-1]


# chunks of 2 048, 4 096 and 8 192 entries, whole ones and a rest
@pytest.mark.parametrize("g,k,v", [(2, 3, 1500), (3, 2, 2048), (130, 8, 3000), (64, 8, 9000), (66, 8, 8192)])
@pytest.mark.parametrize("kind", ["equal", "clipped", "coarse", "two", "zeros", "infinite", "rising", "falling"])
def test_select_among_many_alike(box, g, k, v, kind):
    r = np.random.default_rng(v)
    x = rows(kind, g, k, v, r)
    norm = kind != "infinite"  # (an infinity among a beam's logits leaves it without candidates under a log-sum)
    sc = -r.integers(0, 2, (g, k)).astype(np.float64)
    for beams, dtype in ((1, "float32"), (5, "bfloat16"), (16, "float32"), (17, "float16"), (64, "bfloat16")):
        # log-probabilities of different rows may come nearer to each other than their sums are exact: a beam each
        one = np.where(np.arange(k) == k - 1, 0.0, -np.inf)[None] * np.ones((g, 1)) if norm and kind not in ("equal", "zeros") else sc
        select_case(box, x, one, beams, dtype, norm=norm)
    mask = r.random((g, k, v)) < 0.4
    mask[0, 0] = False
    mask[:, -1, : v // 2] = False
    select_case(box, x, sc, 64, "float32", mask=mask, norm=False)
    select_case(box, x, sc, 16, "bfloat16", mask=mask, done=r.random((g, k)) < 0.2, pad=v - 1, norm=False)


@pytest.mark.parametrize("beams", [8, 16, 64])
def test_equal_logits_cost_no_more_than_a_few_ordinary_calls(box, beams):
    g, k, v = 64, 8, 9000
    outs = [box.put(np.zeros((g, beams), t)) for t in (np.float32, np.int32, np.int32)]
    ws = box.put(np.zeros(ops.beam_select_workspace(g, k, v, beams), np.uint8))
    sc = box.put(np.zeros((g, k), np.float32))

    def spent(x):
        x = box.put(rounded(x, "bfloat16"), "bfloat16")
        best = np.inf
        for _ in range(6):
            box.e.sync()
            t = time.perf_counter()
            for _ in range(5):
                ops.beam_select(x, sc, *outs, workspace=ws, stream=box.stream)
            box.e.sync()
            best = min(best, time.perf_counter() - t)
        return best

    usual = spent(np.random.default_rng(0).normal(size=(g, k, v)) * 3)
    for x in (np.zeros((g, k, v)), np.minimum(np.random.default_rng(1).normal(size=(g, k, v)), 0.5)):
        # (20 - 60 us and 30 - 100 us; 8 000 us where every entry of a chunk is compared with every other)
        assert spent(x) < 12 * usual
