"""Random calls of the operators against their definitions in 64 bits: sizes, types, strides, alignments, masks and ties that no list names.
A slice runs under pytest (tests/test_gpu_ops_fuzz.py); longer runs: python tests/fuzz_ops.py <calls per operator> <seed>."""
import math
import os
import random
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

import numpy as np  # noqa: E402

import test_gpu_ops as T  # noqa: E402
from ops_util import Box, rounded  # noqa: E402

DTYPES = ("float32", "float16", "bfloat16")


def spread(r, lo, hi):
    return int(round(math.exp(r.uniform(math.log(lo), math.log(hi)))))


def linear(r, box):
    rows, n = spread(r, 1, 4000), spread(r, 1, 2000)
    k = r.choice((spread(r, 1, 2500), 16 * spread(r, 1, 100), r.choice((13, 200, 64, 128, 256, 800))))
    while rows * k * n > 2e9:
        rows = max(1, rows // 2)
    a = dict(rows=rows, k=k, n=n, xdt=r.choice(("uint8", "int8")), odt=r.choice(DTYPES), x_scale=r.random() < 0.5, bias=r.random() < 0.5,
             relu=r.random() < 0.5, seed=r.randrange(1 << 30), xpitch=k + r.choice((0, 0, 1, 3, 8, 16)), xbefore=r.choice((0, 0, 1, 5, 16)),
             wpitch=k + r.choice((0, 0, 1, 8, 16)), wbefore=r.choice((0, 0, 3, 16)), opitch=n + r.choice((0, 0, 1, 8)))
    yield a
    T.linear_case(box, **a)


def quantize(r, box):
    rows, k, dt = spread(r, 1, 500), spread(r, 1, 20000), r.choice(DTYPES)
    a = dict(pitch=k + r.choice((0, 1, 7)), before=r.choice((0, 1, 3)), qpitch=k + r.choice((0, 1, 5)))
    seed, coarse = r.randrange(1 << 30), r.random() < 0.3
    yield rows, k, dt, a, seed, coarse
    g = np.random.default_rng(seed)
    x = np.clip(g.normal(size=(rows, k)) * np.exp(g.normal(size=(rows, 1)) * 3), -6e4, 6e4)
    T.quantize_case(box, np.round(x * 8) / 8 if coarse else x, dt, **a)  # (coarse: exact halves)


def select(r, box):
    g, k, v, b = spread(r, 1, 200), spread(r, 1, 64), spread(r, 1, 30000), spread(r, 1, 64)
    while g * k * v > 300000:
        g, k, v = (g // 2, k, v) if g > 1 else (g, k // 2, v) if k > 1 else (g, k, v // 2)
    dt, norm, seed = r.choice(DTYPES), r.random() < 0.6, r.randrange(1 << 30)
    how = dict(spread=r.choice((0.1, 3, 50)), whole=r.random() < 0.3, order=r.choice((0, 0, 0, 1, -1)), ties=not norm and r.random() < 0.3,
               density=r.choice((None, 0.02, 0.5, 0.95)), done=r.random() < 0.5, pad=r.randrange(v))
    a = dict(xpitch=v + r.choice((0, 0, 1, 5)), before=r.choice((0, 1)))
    yield g, k, v, b, dt, norm, seed, how, a
    q = np.random.default_rng(seed)
    x = q.normal(size=(g, k, v)) * how["spread"]
    x = np.round(x) if how["whole"] else x
    if how["order"]:
        x = np.sort(x, 2)[:, :, ::how["order"]]
    x, sc = rounded(np.clip(x, -6e4, 6e4), dt).copy(), -q.random((g, k)) * 5
    sc = np.round(sc) if how["ties"] else sc
    sc[q.random((g, k)) < 0.1] = -np.inf
    mask = None if how["density"] is None else q.random((g, k, v)) < how["density"]
    done = q.random((g, k)) < 0.3 if how["done"] else None
    if mask is not None:
        x[~mask] = np.nan
        x = rounded(x, dt)
    T.select_case(box, None, sc, b, dt, mask=mask, done=done, pad=how["pad"], norm=norm, xr=x, **a)


def reorder(r, box):
    rows = tuple(spread(r, 1, r.choice((40, 3000, 60000))) for _ in range(r.randint(1, 24)))
    kin = spread(r, 1, 64)
    kout = kin if r.random() < 0.5 else spread(r, 1, 64)
    g = max(1, min(spread(r, 1, 300), 2000000 // ((kin + kout) * sum(rows))))
    yield g, kin, kout, rows
    T.test_reorder(box, g, kin, kout, rows)


def run(calls, seed, say=lambda *a: None):
    r = random.Random(seed)
    for i in range(calls):
        for case in (linear, quantize, select, reorder):
            box = Box()
            steps = case(r, box)
            what = next(steps)
            try:
                next(steps, None)
            except Exception as e:
                raise AssertionError(f"{case.__name__} call {i} of seed {seed}: {what}") from e
            finally:
                box.close()
        if i % 100 == 99:
            say(i + 1, "calls of each")


if __name__ == "__main__":
    run(int(sys.argv[1]), int(sys.argv[2]), lambda *a: print(*a, flush=True))
    print("ok")
