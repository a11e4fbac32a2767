"""MX4 on the host: the checks of the C entry points and of the Python layer (they return before any GPU work), and the
tests' own 64-bit quantiser."""
import ctypes

import numpy as np
import pytest
import torch

from mx4_util import GRID, quantise, random_mx4, values

VP = ctypes.c_void_p
P = VP(0x10000)
ODD = VP(0x10002)
F = ctypes.c_float


def test_oracle_quantiser_rounds_to_nearest_even():
    x = np.zeros(32)
    x[:16] = [4, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -5, -0.25, 6, 7.9, 0.2501, 0.7499, 5.01, -3.4999]
    codes, scales = quantise(x)
    assert scales.tolist() == [127]
    want = np.zeros(32)
    want[:16] = [4, 4, 4, 2, 2, 1, 1, 0, -4, 0, 6, 6, 0.5, 0.5, 6, -3]
    assert np.array_equal(values(codes, scales), want)
    c, s = random_mx4((3, 64), 1)
    c[:, ::16] |= 7                                    # every block holds a 6: its scale is recovered
    c2, s2 = quantise(values(c, s))
    assert np.array_equal(s, s2) and np.array_equal(values(c, s), values(c2, s2)) and len(GRID) == 8


def test_c_refusals(exl3):
    L = exl3.lib()
    q = L.exl3_mx4_quantize
    assert q(P, 64, 1, 40, 0, P, P, None) == 1         # k not a multiple of 32
    assert q(P, 32, 1, 64, 0, P, P, None) == 1         # stride below k
    assert q(P, 64, 1, 64, 7, P, P, None) == 1         # type
    assert q(ODD, 64, 1, 64, 0, P, P, None) == 1       # alignment
    assert q(P, 68, 2, 64, 0, P, P, None) == 1         # second row misaligned
    assert q(None, 64, 1, 64, 0, P, P, None) == 1
    assert q(None, 64, 0, 64, 0, None, None, None) == 0
    assert q(P, 64, -1, 64, 0, P, P, None) == 1
    d = L.exl3_mx4_dequantize
    assert d(P, P, 1, 48, P, 64, 0, None) == 1
    assert d(P, P, 1, 64, ODD, 64, 0, None) == 1
    assert d(P, P, 1, 64, P, 64, 3, None) == 1
    assert d(P, P, 0, 64, P, 64, 0, None) == 0
    ln = L.exl3_mx4_linear
    assert ln(P, 64, 1, 1, 64, P, P, 16, 0, None, P, 16, 0, None) == 1      # fp32 rows
    assert b"fp16 or bf16" in L.exl3_last_error()
    assert ln(P, 64, 0, 1, 40, P, P, 16, 0, None, P, 16, 0, None) == 1
    assert ln(P, 64, 0, 1, 64, ODD, P, 16, 0, None, P, 16, 0, None) == 1
    assert ln(ODD, 64, 0, 1, 64, P, P, 16, 0, None, P, 16, 0, None) == 1
    assert ln(P, 68, 0, 2, 64, P, P, 16, 0, None, P, 16, 0, None) == 1
    assert ln(P, 64, 0, 1, 64, P, P, 16, 0, None, P, 8, 0, None) == 1       # output stride
    assert ln(P, 64, 0, 1, 64, P, P, 16, 500, None, P, 16, 0, None) == 1
    assert ln(P, 64, 0, 1, 64, P, P, 0, 0, None, P, 16, 0, None) == 1
    assert ln(P, 64, 0, 0, 64, P, P, 16, 0, None, P, 16, 0, None) == 0
    assert ln(P, 64, 0, 1, 64, P, None, 16, 0, None, P, 16, 0, None) == 1
    wide = (1 << 24) + 32                                                   # longer sums than fp32 is good for
    assert ln(P, wide, 0, 1, wide, P, P, 16, 0, None, P, 16, 0, None) == 1
    g = L.exl3_mx4_gemm
    assert g(P, P, 1, wide, P, P, 16, None, P, 16, 0, None) == 1
    assert g(P, P, 1, 48, P, P, 16, None, P, 16, 0, None) == 1
    assert g(ODD, P, 1, 64, P, P, 16, None, P, 16, 0, None) == 1
    assert g(P, None, 1, 64, P, P, 16, None, P, 16, 0, None) == 1
    assert g(P, P, 0, 64, P, P, 16, None, P, 16, 0, None) == 0
    m = L.exl3_mx4_moe_forward
    ok = [P, 64, 0, 1, 64, 32, P, P, 2, 4, P, 0, F(0.0), -1, P, 64, 0, None]
    for i, v in ((2, 1), (4, 48), (5, 40), (1, 32), (8, 65), (9, 0), (9, 5000), (11, 9), (13, 4), (15, 32), (16, 5), (0, ODD),
                 (6, None), (10, None), (14, None)):
        a = list(ok)
        a[i] = v
        assert m(*a) == 1, i
    assert m(*[0 if i == 3 else v for i, v in enumerate(ok)]) == 0


def test_tensor_and_linear_refusals(exl3):
    E = exl3.Exl3Error
    u8 = torch.uint8
    ok = exl3.MX4Tensor(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 2, dtype=u8))
    assert tuple(ok.shape) == (4, 64) and ok.k == 64
    for c, s in ((torch.zeros(4, 32), torch.zeros(4, 2, dtype=u8)), (torch.zeros(4, 31, dtype=u8), torch.zeros(4, 2, dtype=u8)),
                 (torch.zeros(4, 32, dtype=u8), torch.zeros(3, 2, dtype=u8)),
                 (torch.zeros(32, 4, dtype=u8).t(), torch.zeros(4, 2, dtype=u8)),
                 (torch.zeros(4 * 32 + 1, dtype=u8)[1:].view(4, 32), torch.zeros(4, 2, dtype=u8)),
                 (torch.zeros(4, 0, dtype=u8), torch.zeros(4, 0, dtype=u8))):
        with pytest.raises(E):
            exl3.MX4Tensor(c, s)
    with pytest.raises(E):
        exl3.mx4_quantize(torch.zeros(2, 40))
    with pytest.raises(E):
        exl3.mx4_quantize(torch.zeros(2, 64, dtype=torch.int32))
    with pytest.raises(E):
        exl3.mx4_quantize(torch.zeros(2, 64))          # not on a GPU
    with pytest.raises(E):
        exl3.mx4_dequantize(ok, torch.float64)
    with pytest.raises(E):
        exl3.mx4_gemm(ok, exl3.MX4Tensor(torch.zeros(4, 16, dtype=u8), torch.zeros(4, 1, dtype=u8)))
    lin = exl3.MX4Linear(ok)
    with pytest.raises(E):
        lin.run(torch.zeros(1, 32, dtype=torch.float16), torch.zeros(1, 4))
    with pytest.raises(E):
        exl3.MX4Linear(ok, torch.zeros(3))
    with pytest.raises(E):
        exl3.MX4Linear(exl3.MX4Tensor(torch.zeros(32, dtype=u8), torch.zeros(2, dtype=u8)))


def test_scale_base(exl3):
    def base(scales, codes=0x22):
        s = torch.tensor(scales, dtype=torch.uint8).view(1, -1)
        c = torch.full((1, 16 * s.shape[1]), codes, dtype=torch.uint8)
        lin = exl3.MX4Linear(exl3.MX4Tensor(c, s))
        return lin.scale_base, lin.fp16_rows

    assert base([104, 140]) == (0, True)
    assert base([103, 120]) == (-20, True)             # 2^-24 .. 2^-7 fits after 2^-20 is taken out
    assert base([60, 96]) == (-44, True)
    assert base([60, 97]) == (-43, False)
    assert base([200, 210]) == (70, True)
    assert base([255, 120]) == (0, True)               # a NaN block fits anywhere
    assert base([0, 200], codes=0x88) == (0, True)     # zeros (of either sign) too


def test_experts_refusals(exl3):
    u8 = torch.uint8

    def t(*shape):
        return exl3.MX4Tensor(torch.zeros(*shape[:-1], shape[-1] // 2, dtype=u8), torch.zeros(*shape[:-1], shape[-1] // 32, dtype=u8))

    e = exl3.MX4Experts([t(64, 96)] * 2, [t(64, 96)] * 2, [t(96, 64)] * 2)
    s = exl3.MX4Experts.stacked(t(2, 64, 96), t(2, 64, 96), t(2, 96, 64))
    assert (e.E, e.H, e.I) == (s.E, s.H, s.I) == (2, 96, 64) and tuple(e.tables.shape) == (9, 2)
    with pytest.raises(exl3.Exl3Error):
        exl3.MX4Experts([t(64, 96)], [t(64, 96)], [t(64, 96)])
    with pytest.raises(exl3.Exl3Error):
        exl3.MX4Experts([t(64, 96)], [t(64, 64)], [t(96, 64)])
    with pytest.raises(exl3.Exl3Error):
        exl3.MX4Experts([], [], [])
    with pytest.raises(NotImplementedError):
        exl3.MX4Experts([exl3.MX4Linear(t(64, 96), torch.zeros(64))], [t(64, 96)], [t(96, 64)])
    with pytest.raises(exl3.Exl3Error):
        exl3.MX4Experts.stacked(t(2, 64, 96), t(2, 64, 96), t(2, 64, 96))
    ids, w = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2)
    with pytest.raises(exl3.Exl3Error):
        exl3.mx4_moe_forward(torch.zeros(1, 64, dtype=torch.float16), ids, w, e)
    with pytest.raises(exl3.Exl3Error):
        exl3.mx4_moe_forward(torch.zeros(1, 96, dtype=torch.float16), ids.long(), w, e)
    with pytest.raises(exl3.Exl3Error):
        exl3.mx4_moe_forward(torch.zeros(1, 96, dtype=torch.float16), ids, w, e)     # not on a GPU


def test_balance_refusals(exl3):
    L = exl3.lib()
    ok = [P, 64, 4, 64, P, 2, None, 0, F(1.0), P, P, P, P, None]
    for i, v in ((1, 32), (3, 0), (3, 9000), (5, 0), (5, 65), (2, -1), (0, None), (4, None), (9, None), (12, None)):
        a = list(ok)
        a[i] = v
        assert L.exl3_route_balance(*a) == 1, i
    assert L.exl3_route_balance(*[5 if i == 7 else v for i, v in enumerate(ok)]) == 2
    ok = [P, 64, 4, 64, 2, None, 0, F(1.0), P, P, None, P, 64, None]
    for i, v in ((1, 32), (8, None), (9, None), (11, None), (12, 32), (4, 0)):
        a = list(ok)
        a[i] = v
        assert L.exl3_route_balance_grad(*a) == 1, i
    assert L.exl3_route_balance_grad(*[0 if i == 2 else v for i, v in enumerate(ok)]) == 0
    z, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(exl3.Exl3Error):
        exl3.route_balance(z, ids)                     # not on a GPU
