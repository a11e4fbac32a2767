"""Calls whose grids leave one launch (2^24 workgroups of 256 threads): run in several, or refused before any."""
import ctypes

import numpy as np
import pytest
import torch

import mx4_util as U

VP = ctypes.c_void_p
P = VP(0x10000)
F = ctypes.c_float
DEV = "cuda:0"


def test_refused_before_a_launch(exl3):
    L = exl3.lib()
    big = 1 << 40
    assert L.exl3_mx4_quantize(P, big, 1, big, 0, P, P, None) == 1                       # one row of 2^40 values
    assert L.exl3_mx4_dequantize(P, P, 1, big, P, big, 0, None) == 1
    assert L.exl3_mx4_linear(P, 32, 0, 1 << 33, 32, P, P, 1, 0, None, P, 1, 0, None) == 1           # an output per thread
    assert L.exl3_mx4_linear(P, 32, 0, 1 << 32, 32, P, P, 256, 0, None, P, 256, 0, None) == 1       # tiles of rows
    assert L.exl3_mx4_gemm(P, P, 1 << 33, 32, P, P, 128, None, P, 128, 0, None) == 1
    assert L.exl3_mx4_gemm(P, P, 1, 64, P, P, 1 << 33, None, P, 1 << 33, 0, None) == 1
    assert L.exl3_mx4_moe_forward_in(P, 64, 0, 1 << 24, 64, 1 << 20, P, P, 1, 4, P, 0, F(0.0), -1, P, 64, 0, P, 1 << 60, None) == 1
    assert b"grid" in L.exl3_last_error()


def test_other_calls_are_refused_too(exl3):
    """2^32 threads of an activation, a workgroup of 64 for each of 2^27 rows of logits."""
    L = exl3.lib()
    for n in (1 << 32, (1 << 32) - 255):
        assert L.exl3_act_mul(P, P, P, n, 0, 0, F(0.0), None) == 1
    assert b"grid" in L.exl3_last_error()
    assert L.exl3_route_topk(P, 8, 1 << 27, 8, None, 2, 0, 1, F(1.0), P, P, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_more_rows_than_a_launch_has_workgroups(exl3, dtype):
    m, k = (1 << 24) + 3, 32
    buf = torch.zeros(m, 40, dtype=dtype, device=DEV)
    at = [0, 5, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, m - 1]
    x = torch.randn(len(at), k, generator=torch.Generator().manual_seed(1)).to(dtype)
    buf[at, :k] = x.to(DEV)
    t = exl3.mx4_quantize(buf[:, :k])
    c, s = U.quantise(x.double().numpy())
    assert np.array_equal(t.codes[at].cpu().numpy(), c) and np.array_equal(t.scales[at].cpu().numpy(), s)
    assert int(t.codes.count_nonzero()) == np.count_nonzero(c) and int(t.scales.count_nonzero()) == np.count_nonzero(s)
    buf.fill_(7)
    exl3.mx4_dequantize(t, out=buf[:, :k])
    assert np.array_equal(buf[at, :k].cpu().double().numpy(), U.values(c, s)) and (buf[:, k:] == 7).all()
    buf[at, :k] = 0
    assert int(buf[:, :k].count_nonzero()) == 0


@pytest.mark.gpu
def test_more_tokens_than_a_launch_has_workgroups(exl3):
    """The sum of a token's rows takes two workgroups for 1056 columns: 2^23 tokens and a few."""
    M, H, I = (1 << 23) + 2, 1056, 32
    ts = [exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV))
          for c, s in (U.random_mx4(sh, i, 118, 122) for i, sh in enumerate(((1, I, H), (1, I, H), (1, H, I))))]
    ex = exl3.MX4Experts.stacked(*ts)
    x = torch.zeros(M, H, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 9, (1 << 23) - 2, (1 << 23) - 1, 1 << 23, M - 1], device=DEV)
    x[at] = (torch.randn(len(at), H, generator=torch.Generator().manual_seed(2)) * 0.1).bfloat16().to(DEV)
    ids, w = torch.zeros(M, 1, dtype=torch.int32, device=DEV), torch.ones(M, 1, device=DEV)
    y = torch.full((M, H), 9.0, dtype=torch.bfloat16, device=DEV)
    exl3.mx4_moe_forward(x, ids, w, ex, out=y)
    few = [0] * 200                                                      # (as many rows as take the same kernels)
    want = exl3.mx4_moe_forward(torch.cat([x[at], x[few]]), ids[:206], w[:206], ex, out_dtype=torch.bfloat16)[:len(at)]
    assert want.abs().min(1)[0].lt(1).all() and torch.equal(y[at], want)
    y[at] = 0
    assert not y.view(torch.int16).any()
