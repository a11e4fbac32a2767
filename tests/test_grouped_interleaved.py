"""Weights' gradients into matrices that lie inside one another without overlapping: row n of every expert together ([N, E, K] and
[K, E, N] in memory)."""
import ctypes

import pytest
import torch

from grouped_util import check, ends_of, sizes_for, weights_gradient

P = ctypes.c_void_p(0x10000)


def test_which_matrices_overlap(exl3):
    """dw_ld and dw_es of E matrices of n x k (2 of 64 x 32); the scratch is refused behind these checks."""
    L = exl3.lib()

    def call(ld, es, E=2):
        assert L.exl3_grouped_mm_dw_scratch(4096, 64, 32, E) > 0
        rc = L.exl3_grouped_mm_dw_in(P, 64, P, 32, 2, 4096, 64, 32, P, E, P, ld, es, 1, 0, None, 0, None)
        assert rc == 1
        return L.exl3_last_error()

    for ld, es, E in ((32, 2048, 2), (64, 32, 2), (96, 40, 2), (96, 32, 3), (96, 64, 2)):
        assert b"scratch" in call(ld, es, E), (ld, es, E)
    for ld, es, E in ((32, 2047, 2), (63, 32, 2), (64, 31, 2), (95, 32, 3), (64, 33, 2), (64, 0, 2)):
        assert b"strides" in call(ld, es, E), (ld, es, E)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("T,N,K", ((100, 40, 64), (5000, 33, 24)))
def test_gradient_into_interleaved_matrices(exl3, T, N, K, out_dtype):
    E = 3
    sizes = sizes_for(T, E, T)
    ends = ends_of(sizes)
    g = torch.Generator(device="cuda").manual_seed(T)
    x, dy = (torch.randn(T, c, device="cuda", generator=g).bfloat16() for c in (K, N))
    ref, mag = weights_gradient(dy, x, ends)
    n = max(sizes) + 16
    for turned in (False, True):
        big = torch.full((K if turned else N, E + 2, (N if turned else K) + 8), 9.0, device="cuda").to(out_dtype)
        inner = big[:, 1:1 + E, 3:3 + (N if turned else K)]
        out = inner.permute(1, 2, 0) if turned else inner.transpose(0, 1)
        exl3.grouped_mm_dw(dy, x, ends, out=out)
        check(out, ref, mag, n, "gradient")
        old = out.double()
        exl3.grouped_mm_dw(dy, x, ends, out=out, accumulate=True)
        check(out, ref + old, mag + old.abs(), n + 1, "sum")
        rest = torch.ones_like(big, dtype=torch.bool)
        rest[:, 1:1 + E, 3:3 + inner.shape[2]] = False
        assert bool((big[rest] == 9).all())
