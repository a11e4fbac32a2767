"""Products with 4-bit weights whose scales are powers of two and whose rows are small whole numbers without zeros: every sum is exact in
fp32, so every input, code, scale or zero that is left out, taken twice or taken from elsewhere shows. All kernels, groups, splits."""
import pytest
import torch

from grouped_util import HALF, ends_of, spans

pytestmark = pytest.mark.gpu


def whole(m, k, dtype, seed):
    v = torch.randint(0, 6, (m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return (v - 3 + (v > 2)).to(dtype)


def make(lead, n, k, group, zeros, scale_dtype, seed):
    """Codes, scales 1/2, 1 or 2 and zeros. At most 21504 inputs: halves below 21504 * 15 * 3 * 2 < 2^21, or (bf16 rows without zeros)
    32nds below 2^17, all in 24 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-1, 2, (*lead, n, k // group), device="cuda", generator=g).float()).to(scale_dtype)
    z = torch.randint(0, 16, scales.shape, device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    q = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double().unflatten(-1, (scales.shape[-1], -1))
    w = ((q - (8.0 if z is None else z.double()[..., None])) * scales.double()[..., None]).flatten(-2)
    return (codes, scales, z), w


def product(x, w):
    return (x.double() @ w.t().contiguous()).float()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("k,group", ((8192, 32), (8192, 128), (8320, 64), (8320, 128), (21504, 128), (21504, 21504), (5376, 32), (4608, 256)))
def test_long_rows(exl3, k, group, zeros, dtype):
    """1 to 40 rows of up to and above 8192 inputs, and each input of them alone."""
    t, w = make((), 40, k, group, zeros, dtype, k + group)
    lin = exl3.G4Linear(exl3.G4Tensor(*t))
    for m in (1, 3, 16, 40):
        x = whole(m, k, dtype, m)
        assert torch.equal(lin.run_alloc(x, 40, True), product(x, w)), m
    x = torch.zeros(512, k, dtype=dtype, device="cuda")
    y = torch.empty(k, 40, device="cuda")
    for i in range(0, k, 512):                                 # (the last one's rows behind k stay 0)
        m = min(512, k - i)
        one = x.clone()
        one[torch.arange(m), torch.arange(i, i + m)] = 1
        y[i:i + m] = lin.run_alloc(one, 40, True)[:m]
    assert torch.equal(y, w.t().float())
    for i in sorted({p for b in (32, 128, 512, 2048, 4096, 8192, k) for p in (b - 1, b, b - 33) if 0 <= p < k} | {0}):
        one = x[:5].clone()
        one[3, i] = 1
        assert torch.equal(lin.run_alloc(one, 40, True)[3], w[:, i].float()), i


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128, 256))
@pytest.mark.parametrize("tile", (0, 1, 2, 3, 4))
def test_experts_every_tile_and_group(exl3, monkeypatch, tile, group, zeros, dtype):
    """Ten chunks of 128 inputs: scales of a row come four at a time."""
    monkeypatch.setenv("EXL3MI_G4_TILE", str(tile))
    sizes, k, n = [130, 0, 16, 17, 1, 64], 1280, 268
    ends, T = ends_of(sizes), sum(sizes)
    t, w = make((6,), n, k, group, zeros, HALF[tile % 2], tile + group)
    x = whole(T + 5, k, dtype, 2)
    y = exl3.grouped_mm(x, exl3.G4Tensor(*t), ends, out_dtype=torch.float32)
    for e, a, b in spans(ends):
        assert torch.equal(y[a:b], product(x[a:b], w[e])), e
    assert bool((y[T:] == 0).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128, 512))
@pytest.mark.parametrize("m", (139, 200, 515))
def test_inputs_in_splits(exl3, m, group, zeros, dtype):
    n = k = 4096
    assert exl3.lib().exl3_g4_linear_scratch(m, k, n, group) > 0
    t, w = make((), n, k, group, zeros, HALF[m % 2], m + group)
    x, bias = whole(m, k, dtype, m), torch.arange(n, device="cuda") % 64 - 32.0
    y = torch.full((m, n), float("nan"), device="cuda")
    exl3.G4Linear(exl3.G4Tensor(*t), bias).run(x, y)
    assert torch.equal(y, product(x, w) + bias)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T", (40, 130))
def test_one_expert_of_long_rows_keeps_rows_of_none(exl3, T, dtype):
    """Sizes at which a linear's inputs are split over workgroups, whose sums know no rows of no expert: an expert's are not split."""
    n, k = 256, 16384
    assert exl3.lib().exl3_g4_linear_scratch(T + 9, k, n, 128) > 0
    t, w = make((1,), n, k, 128, True, dtype, T)
    x, ends = whole(T + 9, k, dtype, T), ends_of([T])
    y = torch.full((T + 9, n), 5.0, device="cuda")
    exl3.grouped_mm(x, exl3.G4Tensor(*t), ends, out=y)
    assert torch.equal(y[:T], product(x[:T], w[0])) and bool((y[T:] == 5).all())
    y = exl3.grouped_mm(x, exl3.G4Tensor(*t), ends, out_dtype=torch.float32)
    assert torch.equal(y[:T], product(x[:T], w[0])) and bool((y[T:] == 0).all())
