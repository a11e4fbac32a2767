"""Products grouped by expert of small whole numbers without zeros, whose sums are exact in fp32: every input that is left out, taken
twice or taken from elsewhere shows. All tiles and layouts, long contractions, parts of rows, and tiles that a workgroup goes round to."""
from importlib import import_module

import pytest
import torch

from grouped_util import HALF, ends_of, spans

pytestmark = pytest.mark.gpu


def whole(*shape, dtype, seed):
    """-3, -2, -1, 1, 2, 3: sums of fewer than 2^20 products stay below 2^24."""
    v = torch.randint(0, 6, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return (v - 3 + (v > 2)).to(dtype)


def data(sizes, N, K, dtype, pad=0):
    T, E = sum(sizes) + pad, len(sizes)
    return (ends_of(sizes), whole(T, K, dtype=dtype, seed=T + K), whole(T, N, dtype=dtype, seed=T + N + 1), whole(E, N, K, dtype=dtype, seed=N + K))


def products(rows, w, ends):
    y = torch.zeros(rows.shape[0], w.shape[1], device="cuda")
    for e, a, b in spans(ends):
        y[a:b] = (rows[a:b].double() @ w[e].double().t().contiguous()).float()
    return y


def gradients(dy, x, ends):
    return torch.stack([(dy[a:b].double().t().contiguous() @ x[a:b].double()).float() for _, a, b in spans(ends)])


def turned(w):
    """The same matrices, stored across."""
    return w.transpose(1, 2).contiguous().transpose(1, 2)


f32 = torch.float32


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tile", (0, 1, 2, 3, 4, 5))
@pytest.mark.parametrize("K", (2048, 4096, 4104, 8192, 8200, 21504))
def test_long_contractions(exl3, monkeypatch, K, tile, dtype):
    """Inputs at the ends of what a wave, a workgroup or a step of the few rows' kernel and of each tile takes."""
    monkeypatch.setenv("EXL3MI_GROUPED_TILE", str(tile))
    ends, x, _, w = data([1, 0, 19, 40], 72, K, dtype, 3)
    want = products(x, w, ends)
    assert torch.equal(exl3.grouped_mm(x, w, ends, out_dtype=f32), want)
    assert torch.equal(exl3.grouped_mm(x, turned(w), ends, out_dtype=f32), want)
    for m in (x, w):                                           # and read at odd places
        m.copy_(whole(*m.shape, dtype=dtype, seed=K + tile))
    odd = torch.empty(x.shape[0], K + 3, dtype=dtype, device="cuda")[:, 1:1 + K].copy_(x)
    assert torch.equal(exl3.grouped_mm(odd, w, ends, out_dtype=f32), products(x, w, ends))


# Rows of five experts whose tiles of 256 rows fill the 256 workgroups once and leave the last round in halves of tiles (27 blocks by
# 12 columns of tiles, 68 left over), and once where it is too full for that (35 by 12, 164).
ROUNDS = ([2100, 0, 900, 2999, 1], [2100, 0, 900, 4999, 1])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("sizes", ROUNDS)
def test_tiles_that_a_workgroup_goes_round_to(exl3, monkeypatch, sizes, dtype):
    monkeypatch.setenv("EXL3MI_GROUPED_TILE", "1")
    N = K = 2824
    tiles = (sum((s + 255) // 256 for s in sizes) + 1) * ((N + 255) // 256)
    assert tiles > 256 and (2 * (tiles % 256) <= 256) == (sizes is ROUNDS[0])
    ends, x, dy, w = data(sizes, N, K, dtype, 77)
    assert torch.equal(exl3.grouped_mm(x, w, ends, out_dtype=f32), products(x, w, ends))
    assert torch.equal(exl3.grouped_mm(x, turned(w), ends, out_dtype=f32), products(x, w, ends))
    assert torch.equal(exl3.grouped_mm_dx(dy, w, ends, out_dtype=f32), products(dy, w.transpose(1, 2), ends))
    y = torch.full((len(x), N), 5.0, device="cuda")
    exl3.grouped_mm(x, w, ends, out=y)
    assert torch.equal(y[:-77], products(x, w, ends)[:-77]) and bool((y[-77:] == 5).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tile", (1, 2))
def test_gradients_that_a_workgroup_goes_round_to(exl3, monkeypatch, tile, dtype):
    """Twelve by twelve tiles of 256 for each of five experts, one of them without rows."""
    monkeypatch.setenv("EXL3MI_GROUPED_TILE", str(tile))
    ends, x, dy, _ = data(ROUNDS[0], 2824, 2824, dtype, 77)
    want = gradients(dy, x, ends)
    dw = exl3.grouped_mm_dw(dy, x, ends, out_dtype=f32)
    assert torch.equal(dw, want)
    exl3.grouped_mm_dw(dy, x, ends, out=dw, accumulate=True)
    assert torch.equal(dw, 2 * want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("N,K", ((64, 96), (33, 57), (512, 512), (264, 40)))
def test_gradients_of_many_rows(exl3, N, K, dtype):
    """Small matrices of many rows: an expert's rows in parts that do and do not end with the step of 64 rows."""
    sizes = [4096, 0, 4097, 63, 5000, 1]
    ends, x, dy, _ = data(sizes, N, K, dtype, 5)
    assert exl3.lib().exl3_grouped_mm_dw_scratch(len(x), N, K, len(sizes)) > 0
    want = gradients(dy, x, ends)
    dw = exl3.grouped_mm_dw(dy, x, ends, out_dtype=f32)
    assert torch.equal(dw, want)
    exl3.grouped_mm_dw(dy, x, ends, out=dw, accumulate=True)
    assert torch.equal(dw, 2 * want)


@pytest.mark.parametrize("sizes,parts", (([40, 20], False), ([3000, 20], True)))
@pytest.mark.parametrize("N,K", ((96, 40), (256, 264), (33, 57)))
def test_timing_that_repeats_launches_adds_once_in_one_part_and_in_parts(exl3, N, K, sizes, parts):
    lib = import_module(exl3.__name__ + "._lib")
    ends, x, dy, _ = data(sizes, N, K, torch.bfloat16)
    assert (exl3.lib().exl3_grouped_mm_dw_scratch(len(x), N, K, 2) > 0) == parts
    dw = torch.ones(2, N, K, device="cuda")
    lib.profile_enable(True, repeat=3)
    try:
        exl3.grouped_mm_dw(dy, x, ends, out=dw, accumulate=True)
        torch.cuda.synchronize()
    finally:
        lib.profile_enable(False)
    assert torch.equal(dw, gradients(dy, x, ends) + 1)
