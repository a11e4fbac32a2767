"""MX4 kernels against 64-bit counterparts: quantisation bit for bit, products within the rounding of their type and the
bound of an fp32 sum."""
import numpy as np
import pytest
import torch

import mx4_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T16 = (torch.float16, torch.bfloat16)
T3 = T16 + (torch.float32,)


def rows(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(spread * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


def mx(exl3, shape, seed, lo=110, hi=130):
    c, s = U.random_mx4(shape, seed, lo, hi)
    return exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)), U.values(c, s)


# ------------------------------------------------------------------------------------------------ quantise
@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("m,k", [(1, 32), (1, 64), (3, 96), (5, 4096), (2, 4128), (257, 160), (7, 21504)])
def test_quantize_bits(exl3, dtype, m, k):
    x = rows((m, k), dtype, m * 1000 + k)
    x[0, ::7] = 0
    t = exl3.mx4_quantize(x.to(DEV))
    c, s = U.quantise(x.double().numpy())
    assert np.array_equal(t.scales.cpu().numpy(), s)
    assert np.array_equal(t.codes.cpu().numpy(), c)
    for dt in T3:
        v = exl3.mx4_dequantize(t, dt)
        assert np.array_equal(v.cpu().double().numpy(), U.values(c, s)), dt


@pytest.mark.parametrize("dtype", T3)
def test_quantize_ties_and_extremes(exl3, dtype):
    g = np.concatenate([U.GRID, (U.GRID[1:] + U.GRID[:-1]) / 2, [5.0, 7.0, 7.9375]])
    lo, hi = {torch.float16: (-20, 12), torch.bfloat16: (-130, 124), torch.float32: (-145, 124)}[dtype]
    blocks = []
    for e in range(lo, hi + 1):
        b = np.concatenate([[4.0], g, -g])[:32] * 2.0 ** e
        blocks.append(np.pad(b, (0, 32 - len(b))))
    x = torch.from_numpy(np.stack(blocks)).to(dtype)
    x = torch.cat([x, torch.zeros(1, 32, dtype=dtype), -torch.zeros(1, 32, dtype=dtype),
                   torch.full((1, 32), torch.finfo(dtype).max, dtype=dtype),
                   torch.full((1, 32), torch.finfo(dtype).smallest_normal / 64, dtype=dtype)])
    t = exl3.mx4_quantize(x.to(DEV))
    c, s = U.quantise(x.double().numpy())
    assert np.array_equal(t.scales.cpu().numpy(), s)
    assert np.array_equal(t.codes.cpu().numpy(), c)


def test_dequantize_rounds_once_to_fp16(exl3):
    """Scales beyond fp16's exact range: the value rounded as numpy rounds it, infinite above the largest."""
    codes = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 16))
    scales = np.arange(0, 256, dtype=np.uint8)[:, None]
    for roll in (0, 3, 8, 100):
        s = np.roll(scales, roll, 0)
        t = exl3.MX4Tensor(torch.from_numpy(codes).to(DEV), torch.from_numpy(s.copy()).to(DEV))
        with np.errstate(over="ignore"):
            want = U.values(codes, s).astype(np.float16)
        assert np.array_equal(exl3.mx4_dequantize(t, torch.float16).cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_not_finite(exl3, dtype, bad):
    x = rows((3, 128), dtype, 5)
    x[1, 70] = bad
    t = exl3.mx4_quantize(x.to(DEV))
    c, s = U.quantise(x.double().numpy())
    assert s[1, 2] == 255 and np.array_equal(t.scales.cpu().numpy(), s) and np.array_equal(t.codes.cpu().numpy(), c)
    v = exl3.mx4_dequantize(t, dtype).cpu()
    assert torch.isnan(v[1, 64:96]).all() and torch.isfinite(v[1, :64]).all() and torch.isfinite(v[0]).all()


def test_quantize_strides_shapes_and_out(exl3):
    base = rows((9, 256), torch.bfloat16, 9).to(DEV)
    want = exl3.mx4_quantize(base[:, :96].contiguous())
    for x in (base[:, :96], rows((9, 256), torch.bfloat16, 9).to(DEV).t().contiguous().t()[:, :96]):
        t = exl3.mx4_quantize(x)
        assert torch.equal(t.codes, want.codes) and torch.equal(t.scales, want.scales)
    wide = torch.zeros(9, 97, dtype=torch.bfloat16, device=DEV)          # rows (and the first value) off 16 bytes
    wide[:, 1:] = base[:, :96]
    t = exl3.mx4_quantize(wide[:, 1:])
    assert torch.equal(t.codes, want.codes)
    one = base[:1, :96].expand(4, 96)                                    # rows on top of one another
    t = exl3.mx4_quantize(one)
    assert torch.equal(t.codes, want.codes[:1].expand(4, 48))
    x3 = base[:8, :96].reshape(2, 4, 96)
    t3 = exl3.mx4_quantize(x3)
    assert tuple(t3.shape) == (2, 4, 96) and torch.equal(t3.codes.view(8, 48), want.codes[:8])
    buf = exl3.MX4Tensor(torch.empty(9, 48, dtype=torch.uint8, device=DEV), torch.empty(9, 3, dtype=torch.uint8, device=DEV))
    assert exl3.mx4_quantize(base[:, :96], out=buf) is buf and torch.equal(buf.codes, want.codes)
    assert exl3.mx4_quantize(base[:0, :96]).codes.numel() == 0
    o = torch.full((9, 128), 7.0, device=DEV)
    exl3.mx4_dequantize(want, out=o[:, :96])
    assert torch.equal(o[:, :96], exl3.mx4_dequantize(want, torch.float32)) and (o[:, 96:] == 7).all()
    with pytest.raises(exl3.Exl3Error):
        exl3.mx4_dequantize(want, out=o[:, 1:97])


# ------------------------------------------------------------------------------------------------ dense products
SHAPES = [(1, 32, 1), (1, 64, 17), (2, 96, 33), (3, 160, 130), (16, 128, 64), (17, 544, 100), (31, 4096, 48), (33, 1056, 96),
          (48, 512, 31), (64, 2080, 160), (65, 1024, 257), (100, 4096, 128), (129, 288, 384), (257, 640, 300), (520, 1024, 520), (4, 8192, 50), (8, 8192, 50), (16, 4096, 48), (7, 21504, 40)]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(exl3, dtype, m, k, n):
    w, wv = mx(exl3, (n, k), m + k + n)
    x = rows((m, k), dtype, m * k)
    xv = x.double().numpy()
    ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    lin = exl3.MX4Linear(w)
    for out in (dtype, torch.float32):
        y = torch.full((m, n), float("nan"), dtype=out, device=DEV)
        lin.run(x.to(DEV), y)
        U.check(y, ref, mag, k, out)
    b = rows((n,), torch.float32, 3)
    y = exl3.MX4Linear(w, b.to(DEV)).run_alloc(x.to(DEV), n, True)
    U.check(y, ref + b.double().numpy(), mag + np.abs(b.double().numpy()), k, torch.float32)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gemm(exl3, m, k, n):
    a, av = mx(exl3, (m, k), 7 * m + k + n)
    w, wv = mx(exl3, (n, k), m + k + n)
    ref, mag = av @ wv.T, np.abs(av) @ np.abs(wv).T
    for out in T3:
        y = exl3.mx4_gemm(a, w, out_dtype=out)
        U.check(y, ref, mag, k, out)
    b = rows((n,), torch.bfloat16, 4)
    y = exl3.mx4_gemm(a, w, bias=b.to(DEV), out_dtype=torch.float32)
    U.check(y, ref + b.double().numpy(), mag + np.abs(b.double().numpy()), k, torch.float32)


# One shape for every tile of the two plans, without and with k-splits (test_mx4_plan.py pins which they take), ragged in every
# dimension. The reference covers the first, last and some other columns.
TILES = [("linear", 3000, 160, 2601), ("linear", 2001, 8224, 70), ("linear", 1001, 160, 12301), ("linear", 1501, 4128, 2602),
         ("gemm", 97, 544, 16401), ("gemm", 1501, 8224, 70), ("gemm", 1001, 160, 12301), ("gemm", 201, 8224, 16402)]


@pytest.mark.parametrize("kind,m,k,n", TILES)
def test_every_tile(exl3, kind, m, k, n):
    w, wv = mx(exl3, (n, k), m + n)
    cols = np.unique(np.r_[:40, n - 40:n, np.random.default_rng(m).integers(0, n, 40)] % n)
    wv = wv[cols]
    b = rows((n,), torch.float32, m).to(DEV)
    bv = b.cpu().double().numpy()[cols]
    for dtype in T16 if kind == "linear" else (torch.bfloat16,):
        x = rows((m, k), dtype, m).to(DEV)
        if kind == "linear":
            xv = x.cpu().double().numpy()
            y = exl3.MX4Linear(w, b).run_alloc(x, n, True)
        else:
            q = exl3.mx4_quantize(x)
            xv = U.values(q.codes.cpu().numpy(), q.scales.cpu().numpy())
            y = exl3.mx4_gemm(q, w, bias=b, out_dtype=torch.float32)
        U.check(y[:, torch.from_numpy(cols).to(DEV)], xv @ wv.T + bv, np.abs(xv) @ np.abs(wv).T + np.abs(bv), k, torch.float32)
        assert torch.isfinite(y).all()
        # 16-bit outputs, rows of a multiple of eight of them: the same sums, rounded
        n8 = n // 8 * 8
        w8 = exl3.MX4Tensor(w.codes[:n8], w.scales[:n8])
        for out in T16:
            buf = torch.full((m, n8 + 8), 3.0, dtype=out, device=DEV)
            if kind == "linear":
                exl3.MX4Linear(w8, b[:n8]).run(x, buf[:, :n8])
            else:
                exl3.mx4_gemm(q, w8, bias=b[:n8], out=buf[:, :n8])
            assert torch.equal(buf[:, :n8], y[:, :n8].to(out)) and (buf[:, n8:] == 3).all()


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_scales_over_the_whole_range(exl3, m):
    k, n = 256, 48
    x = rows((m, k), torch.bfloat16, 1)
    for lo, hi in ((0, 40), (60, 96), (100, 150), (150, 186), (200, 236)):
        w, wv = mx(exl3, (n, k), lo, lo, hi)
        lin = exl3.MX4Linear(w)
        for dt in T16:
            xd = x.to(dt)
            if dt == torch.float16 and not lin.fp16_rows:
                with pytest.raises(NotImplementedError):
                    lin.run(xd.to(DEV), torch.empty(m, n, device=DEV))
                continue
            xv = xd.double().numpy()
            y = lin.run_alloc(xd.to(DEV), n, True)
            # (sums below the normal range lose bits of their own: half the smallest step for each addition)
            U.check(y, xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.float32, extra=k * 2.0 ** -149)
    a, av = mx(exl3, (m, k), 11, 20, 60)                                 # products with scales far apart, up to 2^8 to 2^-107
    w, wv = mx(exl3, (n, k), 12, 100, 235)
    U.check(exl3.mx4_gemm(a, w, out_dtype=torch.float32), av @ wv.T, np.abs(av) @ np.abs(wv).T, k, torch.float32)


@pytest.mark.parametrize("m", [1, 40, 200])
@pytest.mark.parametrize("lo", [20, 85, 130, 190])
def test_blocks_of_zeros_take_any_scale(exl3, m, lo):
    k, n = 256, 255
    w, _ = mx(exl3, (n, k), 15, lo, lo + 15)                              # fp16 rows take a power of two out of these
    w.codes[:, 32:48] = torch.tensor([0, 8, 128, 136], dtype=torch.uint8, device=DEV).repeat(4)
    w.scales[:, 2] = torch.arange(n, device=DEV).to(torch.uint8)          # 0 .. 254 beside zeros of either sign
    lin = exl3.MX4Linear(w)
    assert lin.fp16_rows
    wv = U.values(w.codes.cpu().numpy(), w.scales.cpu().numpy())
    for dt in T16:
        x = rows((m, k), dt, 16)
        y = lin.run_alloc(x.to(DEV), n, True)
        xv = x.double().numpy()
        U.check(y, xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.float32, extra=k * 2.0 ** -149)


@pytest.mark.parametrize("m", [1, 3, 20, 200])
@pytest.mark.parametrize("k", [96, 512])
def test_not_finite_stays_in_its_row(exl3, m, k):
    n = 48
    w, _ = mx(exl3, (n, k), 21)
    w.scales[5, k // 32 - 1] = 255                                        # a NaN block: column 5 is NaN
    lin = exl3.MX4Linear(w)
    for dt in T16:
        x = rows((m, k), dt, 22).to(DEV)
        y0 = lin.run_alloc(x, n, True)
        assert torch.isnan(y0[:, 5]).all() and torch.isfinite(y0[:, :5]).all() and torch.isfinite(y0[:, 6:]).all()
        x[m - 1, k - 1] = float("inf")
        y = lin.run_alloc(x, n, True)
        assert not torch.isfinite(y[m - 1]).any()
        assert torch.equal(y[:m - 1, :5], y0[:m - 1, :5]) and torch.equal(y[:m - 1, 6:], y0[:m - 1, 6:])
    a = exl3.mx4_quantize(x)
    y = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
    assert torch.isnan(y[m - 1]).all() and torch.isnan(y[:, 5]).all()
    assert torch.isfinite(y[:m - 1, :5]).all() and torch.isfinite(y[:m - 1, 6:]).all()


@pytest.mark.parametrize("m", [1, 6, 33, 130])
def test_linear_strides_types_and_neighbours(exl3, m):
    k, n = 288, 72
    w, wv = mx(exl3, (n, k), 31)
    lin = exl3.MX4Linear(w)
    x = rows((m, 2 * k), torch.bfloat16, 32).to(DEV)
    want = lin.run_alloc(x[:, :k].contiguous(), n, True)
    assert torch.equal(lin.run_alloc(x[:, :k], n, True), want)
    off = torch.zeros(m, k + 3, dtype=torch.bfloat16, device=DEV)
    off[:, 3:] = x[:, :k]
    assert torch.equal(lin.run_alloc(off[:, 3:], n, True), want)
    for ld, at in ((n + 5, 3), (n + 8, 4)):                               # output rows inside a larger buffer
        for dt in T3:
            buf = torch.full((m + 2, ld), 5.0, dtype=dt, device=DEV)
            lin.run(x[:, :k], buf[1:m + 1, at:at + n])
            assert torch.equal(buf[1:m + 1, at:at + n], want.to(dt))
            assert (buf[0] == 5).all() and (buf[m + 1] == 5).all() and (buf[:, :at] == 5).all() and (buf[:, at + n:] == 5).all()
    f = x[:, :k].float()
    assert torch.equal(lin.run_alloc(f, n, True), lin.run_alloc(f.half(), n, True))
    y3 = lin.run_alloc(x[:, :k].reshape(1, m, k), n, False)
    assert tuple(y3.shape) == (1, m, n) and y3.dtype == torch.bfloat16 and torch.equal(y3[0], want.bfloat16())
    assert lin.run_alloc(x[:0, :k], n, False).shape == (0, n)


@pytest.mark.parametrize("m", [1, 16, 130])
def test_products_are_repeatable_and_rows_independent(exl3, m):
    k, n = 2048, 256
    w, _ = mx(exl3, (n, k), 41)
    lin = exl3.MX4Linear(w)
    x = rows((m, k), torch.bfloat16, 42).to(DEV)
    y = lin.run_alloc(x, n, True)
    p = torch.randperm(m)
    for _ in range(3):
        assert torch.equal(lin.run_alloc(x, n, True), y)
    assert torch.equal(lin.run_alloc(x[p], n, True), y[p])
    a = exl3.mx4_quantize(x)
    g = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
    assert torch.equal(exl3.mx4_gemm(exl3.mx4_quantize(x[p]), w, out_dtype=torch.float32), g[p])


def test_offsets_past_32_bits(exl3):
    """A weight of 2^32 codes and more, rows of more than 2^31 values: only the last rows are checked."""
    n, k = 66000, 65536                                                   # 2.16e9 bytes of codes
    w = exl3.MX4Tensor(torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV), torch.full((n, k // 32), 127, dtype=torch.uint8, device=DEV))
    c, s = U.random_mx4((64, k), 51)
    w.codes[-64:] = torch.from_numpy(c).to(DEV)
    w.scales[-64:] = torch.from_numpy(s).to(DEV)
    for m in (1, 20, 200):
        x = rows((m, k), torch.bfloat16, 52)
        a = exl3.mx4_quantize(x.to(DEV))
        xv, wv = x.double().numpy(), U.values(c, s)
        y = torch.empty(m, n, device=DEV)
        exl3.MX4Linear.run(_bare(exl3, w), x.to(DEV), y)
        U.check(y[:, -64:], xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.float32)
        assert (y[:, :-64] == 0).all()
        av = exl3.mx4_dequantize(a, torch.float32).cpu().double().numpy()
        y = exl3.mx4_gemm(a, w, out_dtype=torch.float32)
        U.check(y[:, -64:], av @ wv.T, np.abs(av) @ np.abs(wv).T, k, torch.float32)
    del w, y
    v = torch.zeros(33000, 65536 + 64, dtype=torch.bfloat16, device=DEV)  # 2.17e9 values
    v[-1, :96] = rows((96,), torch.bfloat16, 53).to(DEV)
    t = exl3.mx4_quantize(v)
    c, s = U.quantise(v[-1:, :96].cpu().double().numpy())
    assert np.array_equal(t.codes[-1:, :48].cpu().numpy(), c) and np.array_equal(t.scales[-1:, :3].cpu().numpy(), s)
    assert int(t.codes[:-1].amax()) == 0
    out = torch.empty_like(v)
    exl3.mx4_dequantize(t, out=out)
    assert np.array_equal(out[-1:, :96].cpu().double().numpy(), U.values(c, s)) and (out[:-1] == 0).all()


def _bare(exl3, w):
    """An MX4Linear without the constructor's pass over the weights (bf16 rows need nothing from it)."""
    lin = exl3.MX4Linear.__new__(exl3.MX4Linear)
    lin.weight, (lin.out_features, lin.in_features) = w, w.shape
    lin.bias, lin.scale_base, lin.fp16_rows = None, 0, False
    return lin


# ------------------------------------------------------------------------------------------------ routed experts
def act64(g, u, act, limit):
    if act == "gelu_tanh":
        return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
    s = g / (1 + np.exp(-g))
    return np.minimum(s, limit) * np.clip(u, -limit, limit) if limit else s * u


def moe64(x, ids, w, gv, uv, dv, act, limit, shared, half):
    """The layer in float64 and a bound on the kernel's error (without the output's rounding): sums_bound for every product, the
    middle's rounding (half step `half`), 8 steps of fp32 for the activation."""
    M, H = x.shape
    E, I = gv.shape[:2]
    out, err = np.zeros((M, H)), np.zeros((M, H))
    for t in range(M):
        todo = [(e, wt) for e, wt in zip(ids[t], w[t]) if 0 <= e < E] + ([(shared, 1.0)] if shared >= 0 else [])
        for e, wt in todo:
            g, u = gv[e] @ x[t], uv[e] @ x[t]
            dg, du = (U.sum_bound(H) * (np.abs(v[e]) @ np.abs(x[t])) for v in (gv, uv))
            h = act64(g, u, act, limit)
            sg = np.abs(act64(g, np.ones_like(u), act, 0.0))
            # |silu'|, |gelu'| <= 1.13
            dh = np.abs(h) * (half + 8 * 2.0 ** -23) + 1.13 * dg * (np.abs(u) + du) + sg * du
            y = dv[e] @ h
            out[t] += wt * y
            err[t] += abs(wt) * (np.abs(dv[e]) @ dh + U.sum_bound(I) * (np.abs(dv[e]) @ (np.abs(h) + dh))) + abs(wt * y) * 2.0 ** -23
        err[t] += len(todo) * 2.0 ** -23 * np.abs(out[t]) + len(todo) * 2.0 ** -24 * err[t]
    return out, err


def layer(exl3, E, H, I, seed, lo=118, hi=122):
    ts, vs = zip(*[mx(exl3, s, seed + i, lo, hi) for i, s in enumerate(((E, I, H), (E, I, H), (E, H, I)))])
    return exl3.MX4Experts.stacked(*ts), ts, vs


def routing(M, k, E, seed, distinct=True):
    g = np.random.default_rng(seed)
    ids = np.stack([g.permutation(E)[:k] if distinct else g.integers(0, E, k) for _ in range(M)]).astype(np.int32)
    return ids.reshape(M, k), g.random((M, k)).astype(np.float32)


MOE = [(1, 64, 32, 4, 2), (1, 512, 160, 16, 4), (3, 96, 64, 8, 3), (8, 256, 128, 32, 4), (17, 160, 96, 3, 2), (40, 128, 256, 2, 2),
       (70, 288, 160, 5, 1), (200, 256, 96, 4, 2), (150, 1056, 32, 64, 4), (300, 288, 160, 5, 1), (130, 128, 256, 2, 2),
       (97, 96, 64, 30, 2), (4, 7168, 2048, 3, 2)]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("M,H,I,E,k", MOE)
def test_moe(exl3, dtype, M, H, I, E, k):
    ex, _, (gv, uv, dv) = layer(exl3, E, H, I, M + H)
    x = rows((M, H), dtype, M, 0.3) * 0.25
    ids, w = routing(M, k, E, M)
    for act, limit, shared in (("silu", 0.0, -1), ("gelu_tanh", 0.0, E - 1), ("silu", 0.5, 0)):
        ref, err = moe64(x.double().numpy(), ids, w, gv, uv, dv, act, limit, shared, U.HALF_STEP[dtype])
        for out in (torch.float32, dtype):
            y = exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex, act, limit, shared,
                                     out_dtype=out)
            U.check(y, ref, 0.0, H, out, extra=err)


@pytest.mark.parametrize("M", [1, 4, 30, 130])
def test_moe_inactive_repeated_and_empty(exl3, M):
    E, H, I, k = 6, 128, 64, 4
    ex, _, (gv, uv, dv) = layer(exl3, E, H, I, 60)
    x = rows((M, H), torch.bfloat16, 61, 0.3) * 0.25
    ids, w = routing(M, k, E, 62, distinct=False)                         # the same expert twice in a token
    ids[::3, 1] = -1
    ids[::5, 2] = E
    ids[M // 2] = -7                                                      # a token with no expert
    for shared in (-1, 2):
        ref, err = moe64(x.double().numpy(), ids, w, gv, uv, dv, "silu", 0.0, shared, 2.0 ** -8)
        out = torch.full((M, H + 8), 3.0, dtype=torch.float16, device=DEV)
        exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex, shared=shared, out=out[:, :H])
        U.check(out[:, :H], ref, 0.0, H, torch.float16, extra=err)
        assert (out[:, H:] == 3).all()
        if shared < 0:
            assert (out[M // 2, :H] == 0).all()
    none = torch.empty(M, 0, dtype=torch.int32, device=DEV), torch.empty(M, 0, device=DEV)
    ref, err = moe64(x.double().numpy(), np.empty((M, 0)), np.empty((M, 0)), gv, uv, dv, "silu", 0.0, 1, 2.0 ** -8)
    U.check(exl3.mx4_moe_forward(x.to(DEV), *none, ex, shared=1), ref, 0.0, H, torch.float32, extra=err)
    assert (exl3.mx4_moe_forward(x.to(DEV), *none, ex) == 0).all()
    assert exl3.mx4_moe_forward(x[:0].to(DEV), none[0][:0], none[1][:0], ex).shape == (0, H)


def test_moe_skewed_load(exl3):
    """Most tokens on one expert (many row blocks), a few on others, most experts idle."""
    E, H, I, M, k = 40, 256, 96, 333, 2
    ex, _, (gv, uv, dv) = layer(exl3, E, H, I, 70)
    x = rows((M, H), torch.float16, 71, 0.3) * 0.25
    ids = np.full((M, k), 7, np.int32)
    ids[:, 1] = np.where(np.arange(M) % 11 == 0, 30, -1)
    w = np.random.default_rng(1).random((M, k)).astype(np.float32)
    ref, err = moe64(x.double().numpy(), ids, w, gv, uv, dv, "silu", 0.0, -1, 2.0 ** -11)
    y = exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex)
    U.check(y, ref, 0.0, H, torch.float32, extra=err)


def test_moe_lists_scales_and_ranges(exl3):
    E, H, I, M, k = 3, 96, 64, 5, 2
    ts, (gv, uv, dv) = zip(*[mx(exl3, sh, 80 + i, *r) for i, (sh, r) in enumerate(
        (((E, I, H), (118, 122)), ((E, I, H), (118, 122)), ((E, H, I), (60, 90))))])   # down far below fp16
    ex = exl3.MX4Experts.stacked(*ts)
    one = [[exl3.MX4Tensor(t.codes[e], t.scales[e]) for e in range(E)] for t in ts]
    lists = exl3.MX4Experts([exl3.MX4Linear(t) for t in one[0]], one[1], one[2])
    assert (ex.tables[8] < 0).all() and (ex.tables[2] == 0).all()
    ids, w = routing(M, k, E, 82)
    i, ww = torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV)
    for dt in T16:
        x = rows((M, H), dt, 81, 0.3) * 0.25
        y = exl3.mx4_moe_forward(x.to(DEV), i, ww, ex)
        assert torch.equal(y, exl3.mx4_moe_forward(x.to(DEV), i, ww, lists))
        ref, err = moe64(x.double().numpy(), ids, w, gv, uv, dv, "silu", 0.0, -1, U.HALF_STEP[dt])
        U.check(y, ref, 0.0, H, torch.float32, extra=err)
    ts[0].scales[1, 0, 0] = 200
    wide = exl3.MX4Experts.stacked(*ts)
    assert not wide.fp16_rows
    with pytest.raises(NotImplementedError):
        exl3.mx4_moe_forward(x.half().to(DEV), i, ww, wide)
    exl3.mx4_moe_forward(x.to(DEV), i, ww, wide)


def test_moe_repeatable_and_rows_independent(exl3):
    E, H, I, M, k = 16, 256, 128, 90, 4
    ex, _, _ = layer(exl3, E, H, I, 90)
    x = rows((M, H), torch.bfloat16, 91, 0.3).to(DEV)
    ids, w = (torch.from_numpy(v).to(DEV) for v in routing(M, k, E, 92))
    y = exl3.mx4_moe_forward(x, ids, w, ex)
    p = torch.randperm(M).to(DEV)
    for _ in range(3):
        assert torch.equal(exl3.mx4_moe_forward(x, ids, w, ex), y)
    assert torch.equal(exl3.mx4_moe_forward(x[p], ids[p], w[p], ex), y[p])


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("M", [2, 40, 100])
def test_block_sparse_mlp_over_mx4_experts(exl3, dtype, M):
    E, H, I, k = 8, 256, 96, 2
    ex, _, _ = layer(exl3, E + 1, H, I, 100)
    gate = (rows((H, E), torch.float32, 101, 0.0) / 16).half().to(DEV)
    mlp = exl3.BlockSparseMLP(ex, k, has_shared=True, router_weight=gate, scoring="sigmoid", routed_scaling=1.5)
    x = (rows((M, H), dtype, 102, 0.3) * 0.25).to(DEV)
    y = mlp.forward(x.view(1, M, H))
    logits = exl3.router_logits(x.half(), gate)
    ids, w = exl3.route_topk(logits, k, None, "sigmoid", True, 1.5)
    assert y.dtype == torch.float32 and tuple(y.shape) == (1, M, H)
    assert torch.equal(y[0], exl3.mx4_moe_forward(x, ids, w, ex, shared=E))
    soft = exl3.BlockSparseMLP(ex, k, has_shared=True, router_weight=gate)
    ids, w = exl3.route_topk(logits, k)
    assert torch.equal(soft.forward(x, out_dtype=dtype), exl3.mx4_moe_forward(x, ids, w, ex, shared=E).to(dtype))


def test_quantise_then_multiply_together(exl3):
    """Weights quantised from full precision, rows quantised per call, against the product of the quantised values; the
    linear over the same weights against the unquantised rows."""
    m, k, n = 37, 512, 96
    wf, x = rows((n, k), torch.float32, 110, 0.2) / 20, rows((m, k), torch.bfloat16, 111)
    w = exl3.mx4_quantize(wf.to(DEV))
    wv = U.values(*U.quantise(wf.double().numpy()))
    xv = U.values(*U.quantise(x.double().numpy()))
    y = exl3.mx4_gemm(exl3.mx4_quantize(x.to(DEV)), w, out_dtype=torch.bfloat16)
    U.check(y, xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.bfloat16)
    xf = x.double().numpy()
    U.check(exl3.MX4Linear(w).run_alloc(x.to(DEV), n, False), xf @ wv.T, np.abs(xf) @ np.abs(wv).T, k, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 7, 150])
def test_captured_layer_replays(exl3, M):
    """Quantise, product, linear and the routed layer captured together and replayed on changed inputs, with eager calls and
    synchronisations between; a second graph over the same workspace."""
    E, H, I, k, n = 8, 256, 128, 2, 160
    ex, _, _ = layer(exl3, E, H, I, 120)
    w, _ = mx(exl3, (n, H), 121)
    lin = exl3.MX4Linear(w)
    x = (rows((M, H), torch.bfloat16, 122, 0.3) * 0.25).to(DEV)
    ids, wt = (torch.from_numpy(v).to(DEV) for v in routing(M, k, E, 123))

    def step():
        return (exl3.mx4_gemm(exl3.mx4_quantize(x), w, out_dtype=torch.float32), lin.run_alloc(x, n, True),
                exl3.mx4_moe_forward(x, ids, wt, ex))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for r in range(4):
        x.copy_((rows((M, H), torch.bfloat16, 200 + r, 0.3) * 0.25).to(DEV))
        ids.copy_(torch.from_numpy(routing(M, k, E, 300 + r)[0]).to(DEV))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graphs[r % 2].replay()
        graphs[1 - r % 2].replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want)), r


def test_other_stream(exl3):
    """Calls follow the caller's current stream."""
    k, n, m = 4096, 512, 64
    w, _ = mx(exl3, (n, k), 130)
    lin = exl3.MX4Linear(w)
    x0 = rows((m, k), torch.bfloat16, 131).to(DEV)
    want = lin.run_alloc(x0, n, True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.zeros_like(x0)
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            big = big @ big / 64                                          # the copy below waits behind this
        x.copy_(x0)
        y = lin.run_alloc(x, n, True)
    s.synchronize()
    assert torch.equal(y, want)
