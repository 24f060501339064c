"""Calls that need more blocks than one launch holds (2^32 threads along x), and a captured launch, on PyTorch tensors; run in a child process by
test_gpu_ops_launches.py.  Every case stays below 25 GB."""
import gc

import torch  # noqa: F401  (before the engine's library)

import pytest

from tetris_gymnasium_amd import ops

pytestmark = pytest.mark.gpu

BLOCKS = (2**32 - 1) // 256  # blocks of 256 threads


@pytest.fixture(autouse=True)
def memory():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def stream():
    return torch.cuda.current_stream().cuda_stream


def pieces(n, step=1 << 25):
    return (slice(i, min(i + step, n)) for i in range(0, n, step))


def test_more_small_searches():
    g = 4 * BLOCKS + 9
    x, s = torch.randn(g, 1, 1, device="cuda", dtype=torch.bfloat16), torch.randn(g, 1, device="cuda")
    s[::5] = -torch.inf
    out, par, tok = torch.empty(g, 1, device="cuda"), torch.empty(g, 1, device="cuda", dtype=torch.int32), torch.empty(g, 1, device="cuda", dtype=torch.int32)
    ops.beam_select(x, s, out, par, tok, normalize=False, stream=stream())
    for i in pieces(g):
        assert torch.equal(out[i], (x[i, :, 0].double() + s[i].double()).float())
        dead = s[i] == -torch.inf
        assert torch.equal(par[i], torch.where(dead, -1, 0).int()) and torch.equal(tok[i], par[i])


@pytest.mark.parametrize("norm", [False, True])
def test_more_chunks_of_larger_searches(norm):
    g, k, v = BLOCKS // 64 + 3, 64, 17
    x, s = torch.randn(g, k, v, device="cuda", dtype=torch.bfloat16), torch.randn(g, k, device="cuda")
    out, par, tok = torch.empty(g, 1, device="cuda"), torch.empty(g, 1, device="cuda", dtype=torch.int32), torch.empty(g, 1, device="cuda", dtype=torch.int32)
    need = ops.beam_select_workspace(g, k, v, 1)
    assert need
    ops.beam_select(x, s, out, par, tok, normalize=norm, workspace=torch.empty(need, device="cuda", dtype=torch.uint8), stream=stream())
    for i in pieces(g, 1 << 16):
        c = x[i].double()
        c = s[i].double()[:, :, None] + (c - torch.logsumexp(c, 2, keepdim=True) if norm else c)
        c = c.view(-1, k * v)
        best = c.amax(1, keepdim=True)
        # one rounding to float32 of a score good to 1e-11
        assert ((out[i].double() - best).abs() <= best.abs() * 2.0**-24 * 1.001 + 1e-11).all()
        at = par[i].long() * v + tok[i].long()
        near = best - c.gather(1, at)
        assert (near <= 1e-11).all()
        if not norm:  # exact sums: the first of equal ones
            first = torch.where(c == best, torch.arange(k * v, device="cuda"), k * v).amin(1, keepdim=True)
            assert torch.equal(at, first)


def test_more_long_rows_to_quantise():
    rows, k = BLOCKS + 5, 1025  # (a block for each row)
    flat = torch.randn(rows + k - 1, device="cuda")
    x = flat.as_strided((rows, k), (1, 1))  # rows one element apart
    q, s = torch.empty(rows, k, device="cuda", dtype=torch.int8), torch.empty(rows, device="cuda")
    ops.quantize_i8(x, q, s, stream=stream())
    for at in (0, BLOCKS // 2, BLOCKS - 600, rows - 700):
        e = x[at:at + 700].cpu().double()
        es = (e.abs().amax(1) / 127).float()
        assert torch.equal(s[at:at + 700].cpu(), es)
        assert torch.equal(q[at:at + 700].cpu().double(), torch.round(e / es.double()[:, None]))


def test_more_tiles_of_a_product():
    rows, k = 128 * BLOCKS + 300, 257
    x, w = torch.zeros(1, k, device="cuda", dtype=torch.uint8), torch.zeros(1, k, device="cuda", dtype=torch.int8)
    x[0, 256], w[0, 256] = 3, 2
    xs, y = torch.empty(rows, device="cuda"), torch.empty(rows, 1, device="cuda", dtype=torch.float16)
    for i in pieces(rows):
        xs[i] = (torch.arange(i.start, i.stop, device="cuda") % 251).float()
    ops.linear_i8(x.expand(rows, k), w, torch.full((1,), 0.5, device="cuda"), y, x_scale=xs, stream=stream())
    for i in pieces(rows):
        assert torch.equal(y[i, 0], (xs[i] * 3).half())


def test_more_items_to_reorder():
    g, k, n, cols = 4 * BLOCKS // 48 + 5, 64, 24, 9  # (two items a group and array)
    p = torch.randint(0, k, (g, k), device="cuda", dtype=torch.int32)
    p[::7, 3] = -1

    def rows(at, a):  # the bytes of some rows of array a
        return ((at[:, None] * 37 + torch.arange(cols, device="cuda", dtype=torch.int32) * 11 + a * 5) % 251).to(torch.uint8)

    at = torch.arange(g * k, device="cuda", dtype=torch.int32) % 1_000_003
    states = [torch.empty(g * k, cols, device="cuda", dtype=torch.uint8) for _ in range(n)]
    for a, st in enumerate(states):
        for i in pieces(g * k):
            st[i] = rows(at[i], a)
    ops.beam_reorder(states, p, stream=stream())
    own = torch.arange(k, device="cuda", dtype=torch.int32)
    src = (torch.arange(g, device="cuda", dtype=torch.int32)[:, None] * k + torch.where(p < 0, own, p)).view(-1) % 1_000_003
    for a, st in enumerate(states):
        for i in pieces(g * k):
            assert torch.equal(st[i], rows(src[i], a)), a


def test_a_captured_product_reads_an_engines_buffer_at_every_replay():
    import numpy as np

    from tetris_gymnasium_amd import Engine, _native as N

    e = Engine(512, 10, 20, obs_mode=N.OBS_BOARD)
    e.reset(np.arange(1, 513, dtype=np.uint64))
    a = e.device_array(N.BUF_OBS)
    x = ops.DeviceView(a.ptr, a.shape, "uint8")  # (the array itself would wait for its engine inside the capture)
    w = torch.randint(-127, 128, (16, 10), device="cuda", dtype=torch.int32).to(torch.int8)
    y, one = torch.empty(512, 20, 16, device="cuda"), torch.ones(16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    e.sync()
    with torch.cuda.graph(graph):
        ops.linear_i8(x, w, one, y, stream=stream())
    r = np.random.default_rng(0)
    for _ in range(4):
        for _ in range(9):
            e.step_async(r.integers(0, 8, 512))
        e.sync()
        graph.replay()
        torch.cuda.synchronize()
        obs = torch.from_numpy(e.observation()).float()
        assert torch.equal(y.cpu(), obs @ w.cpu().float().T)
    e.close()
