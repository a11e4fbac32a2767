"""Products grouped by expert and 4-bit weights with group scales on the host: the checks of the C entry points and of the Python layer
(they return before any GPU work)."""
import ctypes

import pytest
import torch

VP = ctypes.c_void_p
P = VP(0x10000)
ODD = VP(0x10001)
HALF = VP(0x10002)


def test_grouped_mm_refusals(exl3):
    f = exl3.lib().exl3_grouped_mm

    def call(x=P, x_ld=64, dtype=0, T=4, k=64, w=P, w_ld=64, w_es=4096, layout=0, n=64, ends=P, E=2, out=P, out_ld=64, out_dtype=0,
             rest=0):
        return f(x, x_ld, dtype, T, k, w, w_ld, w_es, layout, n, ends, E, out, out_ld, out_dtype, rest, None)

    assert call(T=0) == 0 and call(T=0, x=None, w=None, out=None) == 0
    for bad in (dict(T=-1), dict(T=1 << 30), dict(k=0), dict(n=0), dict(k=(1 << 22) + 1, x_ld=1 << 23), dict(n=(1 << 22) + 1), dict(E=0),
                dict(E=65537), dict(dtype=1), dict(dtype=7), dict(out_dtype=3), dict(ends=None), dict(ends=HALF), dict(layout=2),
                dict(rest=2), dict(x_ld=63), dict(x_ld=(1 << 22) + 8), dict(w_ld=63), dict(w_ld=(1 << 22) + 8), dict(w_es=-1),
                dict(out_ld=63), dict(x=None), dict(w=None), dict(out=None), dict(x=ODD), dict(w=ODD), dict(out=ODD),
                dict(out=HALF, out_dtype=1)):
        assert call(**bad) == 1, bad
        assert b"exl3_grouped_mm" in exl3.lib().exl3_last_error()
    assert call(layout=1, w_ld=63) == 1 and call(layout=1, k=32, x_ld=32, n=64, w_ld=63) == 1
    assert call(T=(1 << 30) - 1, n=1 << 22, out_ld=1 << 22, w_es=0) == 1          # more tiles than a launch has workgroups
    assert b"grid" in exl3.lib().exl3_last_error()


def test_grouped_dw_refusals(exl3):
    L = exl3.lib()

    def call(dy=P, dy_ld=64, x=P, x_ld=32, dtype=2, T=4, n=64, k=32, ends=P, E=2, dw=P, dw_ld=32, dw_es=2048, dw_dtype=1, acc=0, s=None,
             size=0):
        return L.exl3_grouped_mm_dw_in(dy, dy_ld, x, x_ld, dtype, T, n, k, ends, E, dw, dw_ld, dw_es, dw_dtype, acc, s, size, None)

    for bad in (dict(T=-1), dict(n=0), dict(k=0), dict(E=0), dict(dtype=1), dict(dw_dtype=5), dict(ends=None), dict(acc=2), dict(dy_ld=63),
                dict(x_ld=31), dict(dw_ld=31), dict(dw_es=2047), dict(dw_es=-1), dict(dy=None), dict(x=None), dict(dw=None), dict(dw=HALF),
                dict(dy=ODD)):
        assert call(**bad) == 1, bad
        assert b"exl3_grouped_mm_dw" in L.exl3_last_error()
    need = L.exl3_grouped_mm_dw_scratch(4096, 64, 32, 2)
    assert need > 0 and L.exl3_grouped_mm_dw_scratch(4, 64, 32, 2) == 0
    assert L.exl3_grouped_mm_dw_scratch(16384, 4096, 7168, 16) == 0 and L.exl3_grouped_mm_dw_scratch(-1, 64, 32, 2) == 0
    for s, size in ((P, need - 1), (None, need), (VP(0x10080), need), (P, -1), (P, 0)):
        assert call(T=4096, s=s, size=size) == 1
        assert b"scratch" in L.exl3_last_error()


def test_g4_refusals(exl3):
    L = exl3.lib()

    def call(x=P, x_ld=128, dtype=0, m=2, k=128, codes=P, scales=P, sdt=0, zeros=None, group=64, n=16, bias=None, C=P, c_ld=16, cdt=0,
             s=None, size=0):
        return L.exl3_g4_linear_in(x, x_ld, dtype, m, k, codes, scales, sdt, zeros, group, n, bias, C, c_ld, cdt, s, size, None)

    assert call(m=0) == 0
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(k=144, x_ld=144), dict(dtype=1), dict(sdt=1), dict(cdt=4), dict(x_ld=127),
                dict(x_ld=132), dict(x=HALF), dict(codes=HALF), dict(scales=ODD), dict(C=ODD), dict(c_ld=15), dict(bias=HALF), dict(x=None),
                dict(codes=None), dict(scales=None), dict(C=None), dict(k=192, x_ld=192, group=128), dict(k=(1 << 22) + 128, x_ld=1 << 23)):
        assert call(**bad) == 1, bad
        assert b"exl3_g4_linear" in L.exl3_last_error()
    for group in (16, 48, 96, 0, -64):
        assert call(group=group) == 2, group
    need = L.exl3_g4_linear_scratch(100, 16384, 256, 128)
    assert need > 0 and L.exl3_g4_linear_scratch(1, 4096, 4096, 128) == 0 and L.exl3_g4_linear_scratch(100, 8192, 256, 0) == 0
    for s, size in ((P, need - 1), (None, need), (VP(0x10080), need), (P, 0)):
        assert call(m=100, k=16384, x_ld=16384, n=256, c_ld=256, group=128, s=s, size=size) == 1
        assert b"scratch" in L.exl3_last_error()
    g = L.exl3_grouped_g4
    args = [P, 128, 0, 2, 128, P, P, 0, None, 64, 16, P, 3, P, 16, 0, 0, None]
    for i, v in ((11, None), (12, 0), (16, 2), (9, 96), (1, 120)):
        bad = list(args)
        bad[i] = v
        assert g(*bad) in (1, 2), i


def test_python_refusals(exl3):
    h, f, i32 = torch.float16, torch.float32, torch.int32
    x, w, ends = torch.zeros(4, 64, dtype=h), torch.zeros(2, 32, 64, dtype=h), torch.zeros(2, dtype=i32)
    dy = torch.zeros(4, 32, dtype=h)
    err = exl3.Exl3Error
    for bad in (dict(x=x.float()), dict(x=x[0]), dict(x=x.bfloat16()), dict(x=torch.zeros(4, 32, dtype=h)), dict(w=w.float()), dict(w=w[0]),
                dict(w=w[:, :0]), dict(w=w[:0]), dict(ends=ends.long()), dict(ends=ends[:1]), dict(ends=ends[None]),
                dict(out_dtype=torch.int32), dict(out=torch.zeros(4, 31, dtype=h)), dict(out=torch.zeros(4, 32, dtype=i32)),
                dict(out=torch.zeros(32, 4, dtype=h).t()), dict(out=torch.zeros(1, 32, dtype=h).expand(4, 32)), dict()):
        args = dict(x=x, w=w, ends=ends, out=None, out_dtype=None)
        args.update(bad)
        with pytest.raises(err):                               # (the last: tensors on the CPU)
            exl3.grouped_mm(**args)
    with pytest.raises(err):
        exl3.grouped_mm_dx(x, w, ends)
    for bad in (dict(dy=dy.bfloat16()), dict(dy=dy[:3]), dict(ends=ends.long()), dict(ends=ends[:0]), dict(accumulate=True),
                dict(out=torch.zeros(2, 32, 63)), dict(out=torch.zeros(1, 32, 64).expand(2, 32, 64)), dict(out_dtype=torch.int8), dict()):
        args = dict(dy=dy, x=x, ends=ends, out=None, out_dtype=None, accumulate=False)
        args.update(bad)
        with pytest.raises(err):
            exl3.grouped_mm_dw(**args)


def test_g4_python_refusals(exl3):
    u8, h = torch.uint8, torch.float16
    codes, scales = torch.zeros(32, 64, dtype=u8), torch.ones(32, 2, dtype=h)
    err = exl3.Exl3Error
    for bad in ((codes.int(), scales), (codes, scales.float()), (codes[0], scales[0]), (codes, scales[:31]), (codes, torch.ones(32, 0, dtype=h)),
                (codes, scales, torch.zeros(32, 2)), (codes, scales, torch.zeros(32, 1, dtype=u8)), (codes.t().contiguous().t(), scales),
                (torch.zeros(32 * 64 + 8, dtype=u8)[8:].view(32, 64), scales)):
        with pytest.raises(err):
            exl3.G4Tensor(*bad)
    for groups in (8, 128, 4 * 3):
        with pytest.raises((NotImplementedError, err)):
            exl3.G4Tensor(codes, torch.ones(32, groups, dtype=h))
    t = exl3.G4Tensor(codes, scales)
    assert tuple(t.shape) == (32, 128) and t.group == 64 and t.k == 128
    lin = exl3.G4Linear(t)
    with pytest.raises(err):
        exl3.G4Linear(codes)
    with pytest.raises(err):
        exl3.G4Linear(t, torch.zeros(31))
    with pytest.raises(err):
        exl3.G4Linear(exl3.G4Tensor(codes[None], scales[None]))
    with pytest.raises(err):
        lin.run(torch.zeros(1, 64, dtype=h), torch.zeros(1, 32))
    with pytest.raises(err):
        lin.run(torch.zeros(1, 128, dtype=h), torch.zeros(1, 32))                  # on the CPU
    ends = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(err):
        exl3.grouped_mm(torch.zeros(1, 128, dtype=h), t, ends)                     # one matrix
    e = exl3.G4Tensor(codes[None], scales[None])
    with pytest.raises(err):
        exl3.grouped_mm(torch.zeros(1, 64, dtype=h), e, ends)
    with pytest.raises(NotImplementedError, match="gradient"):
        exl3.grouped_mm_dx(torch.zeros(1, 32, dtype=h), e, ends)
    with pytest.raises(NotImplementedError, match="grouped_mm"):
        exl3.ExpertTables([lin], [lin], [lin])
    with pytest.raises(NotImplementedError, match="grouped_mm"):
        exl3.BlockSparseMLP(e, 2)
    with pytest.raises(NotImplementedError, match="MX4"):
        exl3.MX4Experts([t], [t], [t])
