"""Operands of the grouped products and of G4 rows whose rows lie further apart than the kernels' offsets reach (2^22 elements): a copy,
not a refusal."""
import importlib

import pytest
import torch

from grouped_util import check, ends_of, rows_product, weights_gradient

G4 = importlib.import_module("b70-inference_amd.g4")
GROUPED = importlib.import_module("b70-inference_amd.grouped")
MOST = 1 << 22


@pytest.mark.parametrize("ld", (MOST - 8, MOST, MOST + 8))
def test_rows_far_apart(ld):
    x = torch.arange(3 * ld, dtype=torch.int32).view(3, ld).to(torch.float16)[:, 8:72]
    for rows in (lambda: GROUPED._rows2("t", "x", x), lambda: (lambda y, m, s: (y, s))(*G4._g4_rows(x, 64))):
        y, s = rows()
        assert torch.equal(y, x) and s == y.stride(0) and s <= MOST
        assert (s == ld) == (ld <= MOST)                       # read in place where that works


@pytest.mark.parametrize("turned", (False, True))
@pytest.mark.parametrize("E", (64, 65))
def test_matrices_far_apart(E, turned):
    """Experts of [N, E, K], whose rows are E K apart: 2^22 for 64 of them."""
    w = torch.arange(2 * E * (MOST // 64), dtype=torch.int32).view(2, E, MOST // 64).to(torch.float16).transpose(0, 1)
    if turned:
        w = w.transpose(1, 2)
    v, layout, ld, es = GROUPED._matrices("t", w)
    assert ld <= MOST and (v is w) == (E == 64)
    n, k = w.shape[1:]
    shape, strides = ((E, n, k), (es, ld, 1)) if layout == 0 else ((E, n, k), (es, 1, ld))
    assert torch.equal(v.as_strided(shape, strides), w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_products_of_rows_far_apart(exl3, dtype):
    sizes, E, N, K = [2, 0, 5], 3, 40, 64
    ends = ends_of(sizes)
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(7, MOST + 8, device="cuda", generator=g).to(dtype)
    x, dy = wide[:, 16:16 + K], wide[:, 800:800 + N]
    apart = torch.randn(N, MOST // K + 1, K, device="cuda", generator=g).to(dtype)
    w = apart[:, 5:5 + E].transpose(0, 1)
    check(exl3.grouped_mm(x, w, ends), *rows_product(x, w, ends, 7), K, "forward")
    check(exl3.grouped_mm_dx(dy, w, ends), *rows_product(dy, w.transpose(1, 2), ends, 7), N, "dx")
    check(exl3.grouped_mm_dw(dy, x, ends), *weights_gradient(dy, x, ends), 5, "dw")
    codes = torch.randint(0, 256, (E, N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.rand(E, N, 2, device="cuda", generator=g).half()
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (2, -1))
    w64 = ((q - 8) * scales.double()[..., None]).flatten(-2)
    check(exl3.grouped_mm(x, exl3.G4Tensor(codes, scales), ends), *rows_product(x, w64, ends, 7), K, "4-bit experts")
    y = exl3.G4Linear(exl3.G4Tensor(codes[0], scales[0])).run_alloc(x, N, True)
    check(y, *rows_product(x, w64[:1], ends_of([7]), 7), K, "4-bit linear")
