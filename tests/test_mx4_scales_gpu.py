"""Products of MX4 matrices at the ends of the scale bytes, on the kernels for small matrices, few rows and many rows."""
import numpy as np
import pytest
import torch

import mx4_util as U
from test_mx4_gpu import mx, rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# small matrices (m k / 32 < 16), few rows, tiles
SHAPES = [(1, 96, 40), (1, 480, 33), (7, 64, 20), (1, 512, 48), (6, 1056, 50), (20, 544, 100), (200, 288, 130)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("a_bytes,b_bytes", [((0, 2), (250, 252)), ((0, 2), (252, 254)), ((252, 254), (0, 3)), ((0, 0), (200, 254)),
                                             ((60, 70), (185, 190))])
def test_gemm_of_scales_at_either_end(exl3, m, k, n, a_bytes, b_bytes):
    """One scale times a code may leave fp32 (4 at byte 253, 2 at 254), or be 2^-127, where the product of both does neither."""
    a, av = mx(exl3, (m, k), m + k, *a_bytes)
    w, wv = mx(exl3, (n, k), n + k, *b_bytes)
    ref, mag = av @ wv.T, np.abs(av) @ np.abs(wv).T
    U.check(exl3.mx4_gemm(a, w, out_dtype=torch.float32), ref, mag, k, torch.float32)
    # and the other way round, every output in the other matrix's place
    U.check(exl3.mx4_gemm(w, a, out_dtype=torch.float32), ref.T, mag.T, k, torch.float32)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gemm_nan_blocks_beside_any_codes(exl3, m, k, n):
    a, av = mx(exl3, (m, k), 3)
    w, wv = mx(exl3, (n, k), 4)
    want = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
    a.scales[m - 1, k // 32 - 1] = 255
    y = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
    assert torch.isnan(y[m - 1]).all() and torch.equal(y[:m - 1], want[:m - 1])
    w.scales[5, 0] = 255
    y = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
    keep = torch.arange(n, device=DEV) != 5
    assert torch.isnan(y[:, 5]).all() and torch.isnan(y[m - 1]).all() and torch.equal(y[:m - 1][:, keep], want[:m - 1][:, keep])


@pytest.mark.parametrize("k,n", [(32, 1), (64, 7), (480, 1), (96, 5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_of_small_matrices_over_the_scales(exl3, dtype, k, n):
    x = rows((9, k), dtype, k)
    xv = x.double().numpy()
    for lo, hi in ((0, 20), (110, 130), (216, 252)):
        w, wv = mx(exl3, (n, k), lo + n, lo, hi)
        y = exl3.MX4Linear(w).run_alloc(x.to(DEV), n, True)
        ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
        # a partial sum is at most mag: none leaves fp32 where that does not; a result past fp32's largest, 2^128 (1 - 2^-24), is inf
        fits, past = mag < 2.0 ** 127, np.abs(ref) > 2.0 ** 128 * (1 + U.sum_bound(k)) + U.sum_bound(k) * mag
        U.check(y[torch.from_numpy(fits).to(DEV)], ref[fits], mag[fits], k, torch.float32, extra=k * 2.0 ** -149)
        assert np.array_equal(y.cpu().double().numpy()[past], np.sign(ref[past]) * np.inf)
    w.scales[n - 1, 0] = 255
    y = exl3.MX4Linear(w).run_alloc(x.to(DEV), n, True)
    assert torch.isnan(y[:, n - 1]).all() and not torch.isnan(y[:, :n - 1]).any()   # (those past 2^128 are infinite)
