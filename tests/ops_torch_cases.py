"""The operators on PyTorch tensors (run in a child process by test_gpu_ops_torch.py: torch and the engine share one HIP runtime there):
dtypes, views, a stream of their own, a captured graph replayed between eager work, two calls at once."""
import os

import torch  # noqa: F401  (before the engine's library)

import numpy as np
import pytest

from tetris_gymnasium_amd import Engine, _native as N, ops

pytestmark = pytest.mark.gpu


def layer_inputs(m, k, n, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") / 1000 + 1e-4
    return x, w, ws


def layer(x, w, ws, bufs=None, stream=0):
    m, k, n = x.shape[0], x.shape[1], w.shape[0]
    q, s, y = bufs or (torch.empty(m, k, device="cuda", dtype=torch.int8), torch.empty(m, device="cuda"), torch.empty(m, n, device="cuda", dtype=x.dtype))
    ops.quantize_i8(x, q, s, stream=stream)
    ops.linear_i8(q, w, ws, y, x_scale=s, stream=stream)
    return q, s, y


def check_layer(x, w, ws, q, s, y):
    xd = x.cpu().double()
    es = (xd.abs().amax(1) / 127).float().clamp_min(2.0**-126)
    eq = torch.round(xd / es.double()[:, None])
    assert torch.equal(s.cpu(), es) and torch.equal(q.cpu().double(), eq)
    e = (eq @ w.cpu().double().T) * es.double()[:, None] * ws.cpu().double()
    f = torch.finfo(y.dtype)
    # half a step of the output: eps / 2 of a normal value; below the smallest normal one (2^-14 in float16) the step stays
    # smallest_normal * eps whatever the value, so half of that is added
    tol = e.abs() * (f.eps / 2 + 4 * 2.0**-24) * 1.01 + f.smallest_normal * f.eps / 2
    worst = ((y.cpu().double() - e).abs() / tol).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layer_on_torch_tensors(dtype):
    for m, k, n in ((1, 33, 7), (8, 512, 64), (130, 256, 40), (300, 700, 260)):
        x, w, ws = layer_inputs(m, k, n, m, dtype)
        check_layer(x, w, ws, *layer(x, w, ws))
        wide = torch.zeros(m, k + 9, device="cuda", dtype=dtype)
        wide[:, 3:k + 3] = x
        check_layer(x, w, ws, *layer(wide[:, 3:k + 3], w, ws))


def test_a_stream_of_its_own():
    x, w, ws = layer_inputs(4000, 512, 256, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            x = x * 1.5  # the operator has to run behind this stream's own work
        out = layer(x, w, ws, stream=side.cuda_stream)
    side.synchronize()
    check_layer(x, w, ws, *out)


def test_a_captured_graph_replays_on_new_inputs():
    g, k, v, b = 64, 4, 9000, 4
    x, w, ws = layer_inputs(200, 256, 128, 2)
    bufs = layer(x, w, ws)
    lo, sc = torch.randn(g, k, v, device="cuda"), -torch.rand(g, k, device="cuda")
    small = torch.randn(g, k, 40, device="cuda")
    val, par, tok = torch.empty(g, b, device="cuda"), torch.empty(g, b, device="cuda", dtype=torch.int32), torch.empty(g, b, device="cuda", dtype=torch.int32)
    val2, par2, tok2 = torch.empty_like(val), torch.empty_like(par), torch.empty_like(tok)
    need = ops.beam_select_workspace(g, k, v, b)
    wk = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
    st, to = torch.randint(0, 256, (g * k, 600), device="cuda", dtype=torch.uint8), torch.zeros(g * b, 600, device="cuda", dtype=torch.uint8)

    def work(stream):
        layer(x, w, ws, bufs, stream)
        ops.beam_select(lo, sc, val, par, tok, workspace=wk, stream=stream)
        ops.beam_select(small, sc, val2, par2, tok2, normalize=False, stream=stream)
        ops.beam_reorder(st, par, out=to, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        lo.normal_(), small.normal_(), x.normal_(), st.random_(0, 256)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*bufs, val, par, tok, val2, par2, tok2, to)]
        for t in (*bufs, val, par, tok, val2, par2, tok2, to):
            t.zero_()
        work(torch.cuda.current_stream().cuda_stream)  # the same, eagerly
        torch.cuda.synchronize()
        for a, e in zip(got, (*bufs, val, par, tok, val2, par2, tok2, to)):
            assert torch.equal(a, e)
        check_layer(x, w, ws, *bufs)
        c = sc.double()[:, :, None] + torch.log_softmax(lo.double(), 2)
        e = torch.sort(c.view(g, -1), dim=1, descending=True, stable=True)
        assert torch.equal(tok.long(), e.indices[:, :b] % v) and torch.equal(par.long(), e.indices[:, :b] // v)


def test_two_searches_at_once_with_a_workspace_each():
    g, k, v, b = 40, 8, 20000, 8
    streams = [torch.cuda.Stream() for _ in range(2)]
    lo = [torch.randn(g, k, v, device="cuda").bfloat16() for _ in range(2)]
    sc = torch.zeros(g, k, device="cuda")
    need = ops.beam_select_workspace(g, k, v, b)
    outs = [(torch.empty(g, b, device="cuda"), torch.empty(g, b, device="cuda", dtype=torch.int32), torch.empty(g, b, device="cuda", dtype=torch.int32),
             torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for s, l, (a, p, t, wk) in zip(streams, lo, outs):
            ops.beam_select(l, sc, a, p, t, workspace=wk, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for l, (a, p, t, wk) in zip(lo, outs):
        e = torch.sort(torch.log_softmax(l.double(), 2).view(g, -1), dim=1, descending=True, stable=True)
        assert torch.equal(p.long() * v + t.long(), e.indices[:, :b])
        assert (a.double() - e.values[:, :b]).abs().max() < 1e-5


def test_offsets_beyond_32_bits():
    """rows, logits and weights more than 4 GiB apart"""
    big = torch.empty((5 << 30) + 4096, device="cuda", dtype=torch.uint8)
    rows = big[: 2 * (((5 << 30) + 4096) // 2)].view(2, -1)[:, :200]  # two rows 2.5 GiB apart
    rows.random_(0, 256)
    w = torch.randint(-127, 128, (64, 200), device="cuda", dtype=torch.int32).to(torch.int8)
    y = torch.empty(2, 64, device="cuda")
    with pytest.raises(ValueError):  # the documented limit of a row stride
        ops.linear_i8(rows, w, torch.ones(64, device="cuda"), y)
    n = 1 << 20
    m = (1 << 32) // n + 6  # 4 GiB of 1 MiB rows in one reorder, and of logits
    st = big[: m * n].view(m, n)
    st[:, 0] = torch.arange(m, device="cuda") % 251
    st[:, -1] = torch.arange(m, device="cuda") % 241
    k = 7
    par = torch.randint(0, k, (m // k, k), device="cuda", dtype=torch.int32)
    rows0, rows1 = st[:, 0].clone(), st[:, -1].clone()
    ops.beam_reorder(st, par, stream=torch.cuda.current_stream().cuda_stream)
    idx = (torch.arange(m // k, device="cuda")[:, None] * k + par).view(-1)
    assert torch.equal(st[:, 0], rows0[idx]) and torch.equal(st[:, -1], rows1[idx])
    g = m * n // 4 // 40 // 4
    lo = big[: g * 4 * 40 * 4].view(torch.float32).view(g, 4, 40)
    lo.normal_()
    s = torch.zeros(g, 4, device="cuda")
    a, p, t = torch.empty(g, 2, device="cuda"), torch.empty(g, 2, device="cuda", dtype=torch.int32), torch.empty(g, 2, device="cuda", dtype=torch.int32)
    ops.beam_select(lo, s, a, p, t, normalize=False)
    top = lo.view(g, -1).topk(2, 1)
    assert torch.equal(a, top.values)
    last = slice(g - 1000, g)
    same = top.values[last, 0] != top.values[last, 1]
    assert torch.equal((p * 40 + t)[last][same], top.indices[last][same].int())


def test_other_device_stays_current():
    before = torch.cuda.current_device()
    x, w, ws = layer_inputs(4, 16, 4, 0)
    layer(x, w, ws)
    assert torch.cuda.current_device() == before
    with pytest.raises(ValueError, match="device memory"):
        ops.quantize_i8(x.cpu(), torch.empty(4, 16, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda"))


def test_engine_observations_into_a_layer():
    e = Engine(512, 10, 20, obs_mode=N.OBS_BOARD, device=0)
    e.reset(np.arange(1, 513, dtype=np.uint64))
    for _ in range(20):
        e.step_async(np.random.default_rng(1).integers(0, 8, 512))
    obs = torch.as_tensor(e.device_array(N.BUF_OBS), device="cuda")
    w = torch.randint(-127, 128, (64, 200), device="cuda", dtype=torch.int32).to(torch.int8)
    y = torch.empty(512, 64, device="cuda")
    ops.linear_i8(obs.view(512, 200), w, torch.ones(64, device="cuda"), y)
    assert torch.equal(y.cpu(), obs.view(512, 200).cpu().float() @ w.cpu().float().T)
    e.close()
