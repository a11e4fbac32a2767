"""Scratch of the MX4 products, the routed layer and the balance: its checks on the host, and calls that overlap on several streams,
threads and graphs, each against the same call by itself."""
import ctypes
import threading

import pytest
import torch

VP = ctypes.c_void_p
P = VP(0x10000)
F = ctypes.c_float
DEV = "cuda:0"


def test_scratch_sizes(exl3):
    L = exl3.lib()
    assert L.exl3_mx4_linear_scratch(1, 4096, 4096) == 0 and L.exl3_mx4_linear_scratch(40, 4096, 256) > 0
    assert L.exl3_mx4_gemm_scratch(4, 4096, 4096) == 0 and L.exl3_mx4_gemm_scratch(100, 4096, 128) > 0
    assert L.exl3_mx4_moe_scratch(1, 64, 32, 2, 4, -1) > 0 and L.exl3_mx4_moe_scratch(300, 64, 32, 2, 4, 1) > 0
    assert L.exl3_mx4_moe_scratch(5, 64, 32, 0, 4, -1) == 0 and L.exl3_mx4_moe_scratch(5, 64, 32, 0, 4, 0) > 0
    for E, last in ((8, 56), (2048, 56), (2049, 7), (8192, 7)):
        assert L.exl3_route_balance_scratch(last, E) == 0 and L.exl3_route_balance_scratch(last + 1, E) > 0
    for bad in ((-1, 64, 64), (1, 40, 64), (1, 64, 0), (1, 1 << 25, 64)):
        assert L.exl3_mx4_linear_scratch(*bad) == 0 and L.exl3_mx4_gemm_scratch(*bad) == 0
    assert L.exl3_mx4_moe_scratch(1, 48, 32, 2, 4, -1) == 0 and L.exl3_route_balance_scratch(100, 9000) == 0


def test_scratch_refusals(exl3):
    L = exl3.lib()
    n = L.exl3_mx4_linear_scratch(40, 4096, 256)
    lin = [P, 4096, 0, 40, 4096, P, P, 256, 0, None, P, 256, 0]
    g = L.exl3_mx4_gemm_scratch(100, 4096, 128)
    gemm = [P, P, 100, 4096, P, P, 128, None, P, 128, 0]
    m = L.exl3_mx4_moe_scratch(3, 64, 32, 2, 4, -1)
    moe = [P, 64, 0, 3, 64, 32, P, P, 2, 4, P, 0, F(0.0), -1, P, 64, 0]
    w = L.exl3_mx4_moe_scratch(200, 64, 32, 2, 4, -1)
    wide = [P, 64, 0, 200, 64, 32, P, P, 2, 4, P, 0, F(0.0), -1, P, 64, 0]
    b = L.exl3_route_balance_scratch(100, 64)
    bal = [P, 64, 100, 64, P, 2, None, 0, F(1.0), P, P, P, P]
    for fn, args, need in ((L.exl3_mx4_linear_in, lin, n), (L.exl3_mx4_gemm_in, gemm, g), (L.exl3_mx4_moe_forward_in, moe, m),
                           (L.exl3_mx4_moe_forward_in, wide, w), (L.exl3_route_balance_in, bal, b)):
        for scratch, size in ((P, need - 1), (None, need), (VP(0x10080), need), (P, -1), (P, 0)):
            assert fn(*args, scratch, size, None) == 1, (fn, size)
            assert b"scratch" in L.exl3_last_error()


def _calls(exl3, seed):
    """name -> a call on inputs of this seed that takes scratch."""
    from test_mx4_gpu import layer, mx, routing, rows
    w, _ = mx(exl3, (256, 8192), 1)
    lin = exl3.MX4Linear(w)
    x = rows((96, 8192), torch.bfloat16, seed).to(DEV)
    q = exl3.mx4_quantize(x)
    ex, _, _ = layer(exl3, 16, 512, 640, 2)
    h = {M: rows((M, 512), torch.float16, seed + M, 0.3).to(DEV) for M in (6, 300)}
    r = {M: [torch.from_numpy(v).to(DEV) for v in routing(M, 4, 16, seed + M)] for M in h}
    z = torch.randn(3000, 64, generator=torch.Generator().manual_seed(seed)).to(DEV)
    ids = torch.topk(z, 4)[1].to(torch.int32)
    return {"linear": lambda: lin.run_alloc(x, 256, True), "gemm": lambda: exl3.mx4_gemm(q, w, out_dtype=torch.float32),
            "moe_pairs": lambda: exl3.mx4_moe_forward(h[6], *r[6], ex), "moe_blocks": lambda: exl3.mx4_moe_forward(h[300], *r[300], ex),
            "balance": lambda: torch.cat([t.float() for t in exl3.route_balance(z, ids)])}


NAMES = ["linear", "gemm", "moe_pairs", "moe_blocks", "balance"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_calls_overlap_on_streams(exl3, name):
    calls = [_calls(exl3, s)[name] for s in (10, 20, 30)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    out = [[] for _ in calls]
    for _ in range(25):
        for s, c, o in zip(streams, calls, out):
            with torch.cuda.stream(s):
                o.append(c())
    torch.cuda.synchronize()
    for w, o in zip(want, out):
        assert all(torch.equal(y, w) for y in o)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_calls_of_threads(exl3, name):
    """Two threads, on a stream each and on one together."""
    calls = [_calls(exl3, s)[name] for s in (10, 20)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.Stream()] * 2):
        out = [[], []]

        def work(i):
            with torch.cuda.stream(streams[i]):
                for _ in range(25):
                    out[i].append(calls[i]())

        ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        torch.cuda.synchronize()
        for w, o in zip(want, out):
            assert len(o) == 25 and all(torch.equal(y, w) for y in o)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_graphs_replay_beside_each_other_and_eager_calls(exl3, name):
    calls = [_calls(exl3, s)[name] for s in (10, 20, 30)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c() for _ in range(3)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(6):
        eager = []
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [calls[2]() for _ in range(9)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[2]) for y in eager)
        for w, o in zip(want, outs):
            assert all(torch.equal(y, w) for y in o)
            for y in o:
                y.zero_()
        torch.cuda.synchronize()
