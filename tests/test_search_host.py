"""The scorer of the beam search, as far as it needs no GPU: what it refuses and the types its activations are kept in."""
import numpy as np
import pytest

from tetris_gymnasium_amd import BeamSearch, EngineError, PlacementScorer


def layers(*scales, width=4, biases=None):
    """13 features through hidden layers of `width` units, every weight 100 times its layer's scale"""
    out, k = [], 13
    for i, s in enumerate(scales):
        n = 1 if i + 1 == len(scales) else width
        out.append((np.full((n, k), 100, np.int8), np.full(n, s, np.float32), None if biases is None else np.full(n, biases[i], np.float32)))
        k = n
    return out


def test_hidden_activations_beyond_float16_are_kept_in_float32():
    at = 65504 / (13 * 100 * 255)  # the scale at which 13 features of 255 reach float16's largest value
    assert PlacementScorer(layers(at * 0.99, 1.0)).hidden == ["float16"]
    assert PlacementScorer(layers(at * 1.01, 1.0)).hidden == ["float32"]
    assert PlacementScorer(layers(at * 0.99, 1.0, biases=(0.0, 0.0))).hidden == ["float16"]
    assert PlacementScorer(layers(at * 0.5, 1.0, biases=(40000.0, 0.0))).hidden == ["float32"]
    # the second hidden layer's bound goes by the first one's
    assert PlacementScorer(layers(at * 0.5, 0.9 / 400, 1.0)).hidden == ["float16", "float16"]
    assert PlacementScorer(layers(at * 0.5, 2.1 / 400, 1.0)).hidden == ["float16", "float32"]
    assert PlacementScorer(layers(1.0)).hidden == []


def test_hidden_activations_below_float16_are_kept_in_float32():
    assert PlacementScorer(layers(2.0**-24, 1.0)).hidden == ["float16"]
    assert PlacementScorer(layers(2.0**-25, 1.0)).hidden == ["float32"]
    assert PlacementScorer(layers(2.0**-12, 2.0**-12, 1.0)).hidden == ["float16", "float16"]
    assert PlacementScorer(layers(2.0**-12, 2.0**-13, 1.0)).hidden == ["float16", "float32"]
    assert PlacementScorer(layers(-(2.0**-24), 1.0)).hidden == ["float16"]
    r = np.random.default_rng(0)
    usual = [(r.normal(size=(64, 13)) / 13, r.normal(size=64)), (r.normal(size=(64, 64)) / 8, r.normal(size=64)), (r.normal(size=(1, 64)), None)]
    assert PlacementScorer.from_float(usual).hidden == ["float16", "float16"]


@pytest.mark.parametrize("bad", [
    layers(np.nan), layers(1.0, np.inf), layers(1.0, 1.0, biases=(np.nan, 0.0)), layers(1.0, 1.0, biases=(0.0, np.inf)),
    layers(1e35), layers(1e20, 1e20), layers(1e10, 1e10, 1e10, 1e5),
    [(np.zeros((4, 13), np.int8), np.full(4, 1e30, np.float32), None), (np.zeros((1, 4), np.int8), np.full(1, 1e30, np.float32), None)],
])
def test_values_without_a_bound_are_refused(bad):
    with pytest.raises(ValueError, match="float32"):
        PlacementScorer(bad)


class Closable:
    """an engine as far as close() goes; everything else about it is an error"""

    def __init__(self):
        self.h = object()

    def close(self):
        self.h = None


@pytest.mark.parametrize("which,msg", [("search", "this BeamSearch has been closed"), ("engine", "engine it searches has been closed")])
@pytest.mark.parametrize("use", [lambda s: s.plan(3), lambda s: s.value_placements(), lambda s: s._load()])
def test_a_closed_search_touches_no_memory(which, msg, use):
    """its views hold addresses that close() has freed, and a stream that is gone"""
    s = BeamSearch.__new__(BeamSearch)
    s.engine, s.e, s._bufs, s._steps = Closable(), Closable(), [], None
    s.G, s.beams, s.stream = 2, 3, 0
    s.close() if which == "search" else s.engine.close()
    with pytest.raises(EngineError, match=msg):
        use(s)
