"""Products grouped by expert and their gradients against 64-bit products: sizes, tiles, types, strides, empty experts, rows of no
expert."""
import pytest
import torch

from grouped_util import HALF, check, ends_of, rows_product, sizes_for, spans, weights_gradient

pytestmark = pytest.mark.gpu
OUTS = (torch.float16, torch.bfloat16, torch.float32)


def _data(T, E, N, K, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, K, device="cuda", generator=g).to(dtype)
    dy = torch.randn(T, N, device="cuda", generator=g).to(dtype)
    w = (torch.randn(E, N, K, device="cuda", generator=g) / K ** 0.5).to(dtype)
    return x, dy, w


# rows, experts, N, K, rows of no expert: single rows and columns, odd sizes, a block more or less, many and few rows per expert
SIZES = [(1, 1, 1, 1, 0), (1, 8, 64, 128, 0), (5, 3, 7, 9, 0), (17, 4, 33, 65, 3), (64, 1, 128, 64, 0), (33, 2, 130, 72, 31),
         (200, 5, 256, 264, 0), (257, 1, 264, 520, 0), (300, 130, 96, 64, 11), (511, 2, 513, 127, 1), (700, 3, 136, 1000, 0)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T,E,N,K,pad", SIZES)
def test_products_and_gradients(exl3, T, E, N, K, pad, dtype):
    sizes = sizes_for(T, E, 7 * T + N, empty=(1,) if E > 2 else ())
    ends = ends_of(sizes)
    x, dy, w = _data(T + pad, E, N, K, dtype, T + N + K)
    for out_dtype in OUTS:
        y = exl3.grouped_mm(x, w, ends, out_dtype=out_dtype)
        ref, mag = rows_product(x, w, ends, T + pad)
        check(y[:T], ref[:T], mag[:T], K, "forward")
        assert bool((y[T:] == 0).all())
        dx = exl3.grouped_mm_dx(dy, w, ends, out_dtype=out_dtype)
        ref, mag = rows_product(dy, w.transpose(1, 2), ends, T + pad)
        check(dx[:T], ref[:T], mag[:T], N, "dx")
        assert bool((dx[T:] == 0).all())
        dw = exl3.grouped_mm_dw(dy, x, ends, out_dtype=out_dtype)
        ref, mag = weights_gradient(dy, x, ends)
        check(dw, ref, mag, max(sizes), "dw")
    assert exl3.grouped_mm(x, w, ends).dtype == dtype and exl3.grouped_mm_dw(dy, x, ends).dtype == dtype


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tile", (1, 2, 3, 4, 5))
def test_every_tile(exl3, monkeypatch, tile, dtype):
    """Each tile over blocks that are full, end early, or hold a row, a contraction of one step and of many, and its tail."""
    monkeypatch.setenv("EXL3MI_GROUPED_TILE", str(tile))
    for sizes, N, K in (([256, 1, 0, 300, 31], 272, 64), ([3, 0, 65, 129, 600], 520, 408), ([0, 0, 40], 8, 8), ([16, 1, 0, 33], 24, 5000)):
        ends = ends_of(sizes)
        x, dy, w = _data(sum(sizes), len(sizes), N, K, dtype, tile + N)
        y = exl3.grouped_mm(x, w, ends)
        check(y, *rows_product(x, w, ends, len(x)), K, "forward")
        dx = exl3.grouped_mm_dx(dy, w, ends)
        check(dx, *rows_product(dy, w.transpose(1, 2), ends, len(x)), N, "dx")
        dw = exl3.grouped_mm_dw(dy, x, ends)
        check(dw, *weights_gradient(dy, x, ends), max(sizes), "dw")


@pytest.mark.parametrize("N,K", ((64, 96), (33, 57)))
def test_rows_in_parts(exl3, N, K):
    """Small matrices of many rows: an expert's rows go to several workgroups, some of which have none."""
    sizes = [3000, 0, 20, 64]
    ends = ends_of(sizes)
    x, dy, w = _data(sum(sizes), 4, N, K, torch.bfloat16, 2)
    assert exl3.lib().exl3_grouped_mm_dw_scratch(sum(sizes), N, K, 4) > 0
    ref, mag = weights_gradient(dy, x, ends)
    for out_dtype in OUTS:
        check(exl3.grouped_mm_dw(dy, x, ends, out_dtype=out_dtype), ref, mag, 3000 + 16, "parts")
    old = torch.randn(4, N, K, device="cuda")
    out = old.clone()
    exl3.grouped_mm_dw(dy, x, ends, out=out, accumulate=True)
    check(out, ref + old.double(), mag + old.double().abs(), 3000 + 17, "sum")


def test_given_out_keeps_other_rows(exl3):
    ends = ends_of([3, 0, 70])
    x, dy, w = _data(100, 3, 64, 128, torch.bfloat16, 1)
    for call, wide in ((lambda o: exl3.grouped_mm(x, w, ends, out=o), 64), (lambda o: exl3.grouped_mm_dx(dy, w, ends, out=o), 128)):
        big = torch.full((100, wide + 24), 5.0, device="cuda")
        call(big[:, 8:8 + wide])
        assert bool((big[73:] == 5).all()) and bool((big[:, :8] == 5).all()) and bool((big[:, 8 + wide:] == 5).all())
        assert not bool((big[:73, 8:8 + wide] == 5).any())
    # no rows at all, and no expert with rows
    none = ends_of([0, 0, 0])
    assert exl3.grouped_mm(x[:0], w, none).shape == (0, 64)
    assert bool((exl3.grouped_mm(x, w, none) == 0).all())
    assert bool((exl3.grouped_mm_dw(dy, x, none) == 0).all())
    assert bool((exl3.grouped_mm_dw(dy[:0], x[:0], none) == 0).all())


@pytest.mark.parametrize("dtype", HALF)
def test_strides(exl3, dtype):
    """Slices of wider rows, halves of stacked weights, transposed weights and gradients, one matrix for all experts, unaligned
    rows."""
    sizes = [40, 0, 33, 100]
    T, E, N, K = sum(sizes), 4, 72, 136
    ends = ends_of(sizes)
    x, dy, w = _data(T, E, N, K, dtype, 3)
    want, mag = rows_product(x, w, ends, T)
    wide = torch.full((T, K + 16), 9.0, dtype=dtype, device="cuda")
    for off in (8, 1, 3):
        wide[:, off:off + K] = x
        check(exl3.grouped_mm(wide[:, off:off + K], w, ends), want, mag, K, f"rows from {off}")
    stacked = torch.full((E, 2 * N, K), 9.0, dtype=dtype, device="cuda")
    stacked[:, N:] = w
    check(exl3.grouped_mm(x, stacked[:, N:], ends), want, mag, K, "half of stacked weights")
    turned = w.transpose(1, 2).contiguous().transpose(1, 2)
    check(exl3.grouped_mm(x, turned, ends), want, mag, K, "transposed weights")
    dref, dmag = rows_product(dy, w.transpose(1, 2), ends, T)
    check(exl3.grouped_mm_dx(dy, turned, ends), dref, dmag, N, "dx, transposed weights")
    spread = torch.zeros(E, N, K, 2, dtype=dtype, device="cuda")
    spread[..., 0] = w
    check(exl3.grouped_mm(x, spread[..., 0], ends), want, mag, K, "weights with gaps")
    check(exl3.grouped_mm(x.t().contiguous().t(), w, ends), want, mag, K, "columns of rows")
    one = w[1:2].expand(E, N, K)
    check(exl3.grouped_mm(x, one, ends), *rows_product(x, one, ends, T), K, "one matrix")
    gref, gmag = weights_gradient(dy, x, ends)
    out = torch.empty(E, K, N, device="cuda").transpose(1, 2)
    check(exl3.grouped_mm_dw(dy, x, ends, out=out), gref, gmag, 100, "transposed gradient")
    out = torch.full((E, N + 3, K + 5), 9.0, device="cuda")
    check(exl3.grouped_mm_dw(dy, x, ends, out=out[:, 1:1 + N, 2:2 + K]), gref, gmag, 100, "gradient inside a larger one")
    assert bool((out[:, 0] == 9).all()) and bool((out[:, 1 + N:] == 9).all()) and bool((out[..., :2] == 9).all()) and bool((out[..., 2 + K:] == 9).all())


@pytest.mark.parametrize("out_dtype", OUTS)
@pytest.mark.parametrize("N,K", ((64, 128), (33, 57)))
def test_accumulate(exl3, N, K, out_dtype):
    sizes = [5, 0, 90]
    ends = ends_of(sizes)
    x, dy, w = _data(95, 3, N, K, torch.bfloat16, 5)
    old = torch.randn(3, N, K, device="cuda").to(out_dtype)
    out = old.clone()
    assert exl3.grouped_mm_dw(dy, x, ends, out=out, accumulate=True) is out
    ref, mag = weights_gradient(dy, x, ends)
    check(out, ref + old.double(), mag + old.double().abs(), 91, "sum")
    assert torch.equal(out[1], old[1])


@pytest.mark.parametrize("dtype", HALF)
def test_rows_do_not_mix(exl3, dtype):
    """Infinities and NaN of a row, of an expert's weights and of rows behind stay where they are."""
    sizes = [20, 3, 41]
    ends = ends_of(sizes)
    for N, K in ((64, 96), (35, 41)):
        x, dy, w = _data(70, 3, N, K, dtype, 6)
        x[7] = float("nan")
        x[22, 3] = float("inf")
        x[64:] = float("nan")
        dy[64:] = float("inf")
        w[1] = float("nan")
        y = exl3.grouped_mm(x, w, ends)
        ref, mag = rows_product(x, w, ends, 70)
        keep = [t for t in range(64) if t != 7 and not 20 <= t < 23]
        check(y[keep], ref[keep], mag[keep], K, "finite rows")
        assert bool(y[7].isnan().all()) and bool(y[20:23].isnan().all()) and bool((y[64:] == 0).all())
        dx = exl3.grouped_mm_dx(dy, w, ends)
        ref, mag = rows_product(dy, w.transpose(1, 2), ends, 70)
        keep = [t for t in range(64) if not 20 <= t < 23]
        check(dx[keep], ref[keep], mag[keep], N, "dx")
        dw = exl3.grouped_mm_dw(dy, x, ends)
        ref, mag = weights_gradient(dy, x, ends)
        check(dw[2], ref[2], mag[2], 41, "dw of the expert behind")
        assert bool(dw[0].isnan().all())


def test_gradients_against_differences(exl3):
    """The gradients of a sum c . y: a step along each in fp32 outputs changes it as they say (the product is linear, so a step of
    any size does; steps are powers of two, exact in the rows' type)."""
    sizes = [9, 0, 30]
    ends = ends_of(sizes)
    N, K = 24, 40
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randint(-8, 9, (39, K), device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randint(-8, 9, (3, N, K), device="cuda", generator=g).to(torch.bfloat16)
    c = torch.randint(-8, 9, (39, N), device="cuda", generator=g).to(torch.bfloat16)

    def total(x, w):                                           # whole numbers: exact
        return float((exl3.grouped_mm(x, w, ends, out_dtype=torch.float32).double() * c.double()).sum())

    dx = exl3.grouped_mm_dx(c, w, ends, out_dtype=torch.float32)
    dw = exl3.grouped_mm_dw(c, x, ends, out_dtype=torch.float32)
    base = total(x, w)
    for t, k in ((0, 0), (8, 39), (9, 1), (38, 20)):
        x2 = x.clone()
        x2[t, k] += 4
        assert total(x2, w) - base == 4 * float(dx[t, k])
    for e, n, k in ((0, 0, 0), (1, 3, 3), (2, 23, 39), (0, 11, 7)):
        w2 = w.clone()
        w2[e, n, k] += 4
        assert total(x, w2) - base == 4 * float(dw[e, n, k])


def test_ends_out_of_range_reach_nothing_else(exl3):
    """Ends below 0, above the rows or not ascending: no access out of range, rows outside out untouched."""
    x, dy, w = _data(50, 4, 32, 64, torch.float16, 8)
    for bad in ([-5, 10, 60, 1 << 30], [40, 10, 50, 20], [50, 0, 50, 0]):
        ends = torch.tensor(bad, dtype=torch.int32, device="cuda")
        big = torch.full((70, 32), 5.0, device="cuda")
        exl3.grouped_mm(x, w, ends, out=big[10:60])
        assert bool((big[:10] == 5).all()) and bool((big[60:] == 5).all())
        assert exl3.grouped_mm_dw(dy, x, ends).shape == (4, 32, 64)


def test_repeats_and_permutations(exl3):
    """Repeated calls give the same bits, and a row's result does not depend on the rows beside it."""
    sizes = [100, 7, 64]
    ends = ends_of(sizes)
    x, dy, w = _data(171, 3, 200, 328, torch.bfloat16, 10)
    y = exl3.grouped_mm(x, w, ends)
    assert torch.equal(y, exl3.grouped_mm(x, w, ends))
    dw = exl3.grouped_mm_dw(dy, x, ends)
    assert torch.equal(dw, exl3.grouped_mm_dw(dy, x, ends))
    order = torch.cat([a + torch.randperm(b - a) for _, a, b in spans(ends)]).cuda()
    assert torch.equal(exl3.grouped_mm(x[order], w, ends), y[order])


def test_timing_that_repeats_launches_adds_once(exl3):
    from importlib import import_module
    lib = import_module(exl3.__name__ + "._lib")
    for N, K in ((96, 40), (256, 264)):                        # in one part and in parts
        ends = ends_of([3000, 20])
        x, dy, _ = _data(3020, 2, N, K, torch.bfloat16, N)
        dw = torch.ones(2, N, K, device="cuda")
        lib.profile_enable(True, repeat=3)
        try:
            exl3.grouped_mm_dw(dy, x, ends, out=dw, accumulate=True)
            torch.cuda.synchronize()
        finally:
            lib.profile_enable(False)
        ref, mag = weights_gradient(dy, x, ends)
        check(dw, ref + 1, mag + 1, 3001, f"{N} x {K}")


@pytest.mark.parametrize("m", (10, 300))
def test_offsets_past_32_bits(exl3, m):
    """Weights of 9 GB, then rows and outputs of more than 4 GB each, whose last expert's rows lie at the end."""
    E, N, K = 1100, 2048, 2048
    w = torch.zeros(E, N, K, dtype=torch.bfloat16, device="cuda")
    x, dy, last = _data(m, 1, N, K, torch.bfloat16, m)
    w[-1] = last[0]
    ends, one = ends_of([0] * (E - 1) + [m]), ends_of([m])
    ref, mag = rows_product(x, last, one, m)
    rdx, mdx = rows_product(dy, last.transpose(1, 2), one, m)
    check(exl3.grouped_mm(x, w, ends), ref, mag, K, "forward")
    check(exl3.grouped_mm_dx(dy, w, ends), rdx, mdx, N, "dx")
    rdw, mdw = weights_gradient(dy, x, one)
    exl3.grouped_mm_dw(dy, x, ends, out=w)
    check(w[-1:], rdw, mdw, m, "dw")
    assert not bool(w[:-1].any())
    del w
    T = (1 << 31) // K + 700
    xs, dys = (torch.cat((torch.zeros(T - m, K, dtype=torch.bfloat16, device="cuda"), v)) for v in (x, dy))
    two = torch.cat((torch.zeros_like(last), last))
    ends = ends_of([T - m, m])
    y = exl3.grouped_mm(xs, two, ends)
    check(y[-m:], ref, mag, K, "forward, many rows")
    assert not bool(y[:-m].any())
    y = exl3.grouped_mm_dx(dys, two, ends)
    check(y[-m:], rdx, mdx, N, "dx, many rows")
    dw = exl3.grouped_mm_dw(dys, xs, ends)
    check(dw[1:], rdw, mdw, m, "dw, many rows")
    assert not bool(dw[0].any())


@pytest.mark.parametrize("tile", ("0", "1", "4", "5"))
def test_many_experts(exl3, monkeypatch, tile):
    """As many experts as a step of the search for a block's takes, and one more or less, with rows of none behind them."""
    monkeypatch.setenv("EXL3MI_GROUPED_TILE", tile)
    N, K, pad = 16, 32, 3
    for E in (63, 64, 65, 575, 576, 577, 1152, 2500):
        sizes = sizes_for(3 * E // 2, E, E, empty=range(0, E, 5))
        T, ends = sum(sizes), ends_of(sizes)
        x, _, w = _data(T + pad, E, N, K, torch.float16, E)
        of = torch.repeat_interleave(torch.arange(E), torch.tensor(sizes)).cuda()
        prod = w.double()[of] * x[:T].double()[:, None]
        for y in (exl3.grouped_mm(x, w, ends), exl3.grouped_mm(x, w, ends, out=torch.full((T + pad, N), 7.0, device="cuda"))):
            check(y[:T], prod.sum(-1), prod.abs().sum(-1), K, f"{E} experts")
            assert bool((y[T:] == (7 if y.dtype == torch.float32 else 0)).all())
