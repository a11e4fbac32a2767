"""Products with 4-bit weights and group scales against 64-bit products: sizes, tiles, groups, zeros, types, strides, experts."""
import pytest
import torch

from grouped_util import HALF, check, ends_of, sizes_for, spans

pytestmark = pytest.mark.gpu
OUTS = (torch.float16, torch.bfloat16, torch.float32)


def make(lead, n, k, group, zeros, scale_dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = (torch.exp2(torch.randn(*lead, n, k // group, device="cuda", generator=g)) / (4 * k ** 0.5)).to(scale_dtype)
    z = torch.randint(0, 16, scales.shape, device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def values(codes, scales, zeros):
    """The weights in 64 bits."""
    q = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double().unflatten(-1, (scales.shape[-1], -1))
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((q - z) * scales.double()[..., None]).flatten(-2)


def rows(m, k, dtype, seed):
    return torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def product(x, w):
    return x.double() @ w.t().contiguous(), x.double().abs() @ w.abs().t().contiguous()


# rows, n, k: one to many rows, odd n, a chunk of 128 or less, blocks more or less, several slices of 512
SIZES = [(1, 1, 32), (1, 3, 64), (2, 17, 96), (1, 256, 4096), (7, 65, 640), (16, 130, 1056), (17, 64, 128), (33, 300, 544), (100, 257, 256),
         (130, 40, 1152), (300, 520, 384)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
def test_linear(exl3, group, zeros, dtype):
    for m, n, k in SIZES:
        if k % group:
            k = -(-k // group) * group
        w = make((), n, k, group, zeros, HALF[(m + n) % 2], m + n + k)
        x = rows(m, k, dtype, m)
        bias = torch.randn(n, device="cuda") if n % 2 else None
        ref, mag = product(x, values(*w))
        if bias is not None:
            ref, mag = ref + bias.double(), mag + bias.double().abs()
        lin = exl3.G4Linear(exl3.G4Tensor(*w), bias)
        for out_dtype in OUTS:
            y = torch.full((m, n), float("nan"), dtype=out_dtype, device="cuda")
            lin.run(x, y)
            check(y, ref, mag, k, f"{m} x {n} x {k}")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tile", (1, 2, 3, 4))
def test_every_tile(exl3, monkeypatch, tile, dtype):
    monkeypatch.setenv("EXL3MI_G4_TILE", str(tile))
    for m, n, k, group, zeros in ((150, 272, 512, 32, False), (40, 40, 1984, 64, True), (129, 300, 768, 128, True),
                                  (17, 64, 768, 256, False), (33, 260, 1152, 1152, True), (5, 8, 160, 32, True)):
        w = make((), n, k, group, zeros, torch.float16, m + n)
        x = rows(m, k, dtype, m)
        y = exl3.G4Linear(exl3.G4Tensor(*w)).run_alloc(x, n, True)
        check(y, *product(x, values(*w)), k, f"{m} x {n} x {k}, groups of {group}")


def test_more_inputs_than_a_workgroup_holds(exl3):
    """More than 8192 inputs leave the few-rows kernel."""
    w = make((), 40, 8192 + 128, 128, True, torch.float16, 1)
    x = rows(3, 8192 + 128, torch.bfloat16, 1)
    check(exl3.G4Linear(exl3.G4Tensor(*w)).run_alloc(x, 40, True), *product(x, values(*w)), 8320)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T,E,n,k,group,pad", ((1, 8, 64, 128, 32, 0), (10, 200, 96, 512, 64, 0), (50, 3, 33, 256, 128, 7), (300, 5, 130, 192, 64, 40),
                                               (700, 4, 264, 256, 256, 0), (3, 2, 1, 32, 32, 2), (2, 1, 3, 32, 32, 1)))
def test_experts(exl3, T, E, n, k, group, pad, dtype):
    for zeros in (False, True):
        codes, scales, z = make((E,), n, k, group, zeros, dtype, T + n)
        ends = ends_of(sizes_for(T, E, T + k, empty=(1,) if E > 2 else ()))
        x = rows(T + pad, k, dtype, T)
        w = values(codes, scales, z)
        t = exl3.G4Tensor(codes, scales, z)
        ref = torch.zeros(T + pad, n, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(ref)
        for e, a, b in spans(ends):
            ref[a:b], mag[a:b] = product(x[a:b], w[e])
        for out_dtype in OUTS:
            y = exl3.grouped_mm(x, t, ends, out_dtype=out_dtype)
            check(y[:T], ref[:T], mag[:T], k)
            assert bool((y[T:] == 0).all())
        big = torch.full((T + pad, n + 16), 5.0, device="cuda")
        exl3.grouped_mm(x, t, ends, out=big[:, 8:8 + n])
        assert bool((big[T:] == 5).all()) and bool((big[:, :8] == 5).all()) and bool((big[:, 8 + n:] == 5).all())
        check(big[:T, 8:8 + n], ref[:T], mag[:T], k)


@pytest.mark.parametrize("tile", (1, 2, 3, 4))
def test_experts_every_tile(exl3, monkeypatch, tile):
    monkeypatch.setenv("EXL3MI_G4_TILE", str(tile))
    sizes = [130, 0, 16, 17, 1, 64]
    ends = ends_of(sizes)
    codes, scales, z = make((6,), 268, 448, 64, True, torch.bfloat16, tile)
    x = rows(sum(sizes) + 5, 448, torch.bfloat16, 2)
    y = exl3.grouped_mm(x, exl3.G4Tensor(codes, scales, z), ends, out_dtype=torch.float32)
    for e, a, b in spans(ends):
        check(y[a:b], *product(x[a:b], values(codes[e], scales[e], z[e])), 448)
    assert bool((y[sum(sizes):] == 0).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("zeros", (False, True))
def test_every_code_and_zero_is_exact(exl3, zeros, dtype):
    """One input at a time: the weights themselves, every q against every z, exact in fp32."""
    n, k = 16, 512
    codes = torch.arange(n * k, device="cuda").remainder(16).reshape(n, k)
    codes = codes.roll(3, 1)
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)
    scales = torch.exp2(torch.arange(n * k // 32, device="cuda").remainder(9) - 4.0).reshape(n, -1).to(torch.bfloat16)
    z = torch.arange(n, device="cuda").to(torch.uint8)[:, None].expand(n, k // 32).contiguous() if zeros else None
    w = exl3.G4Tensor(packed, scales, z)
    for m in (16, 512):
        x = torch.eye(k, device="cuda")[:m].to(dtype)
        y = exl3.G4Linear(w).run_alloc(x, n, True)
        assert torch.equal(y.double(), values(packed, scales, z)[:, :m].t())


def test_scales_near_the_types_ends(exl3):
    """bf16 scales of 2^125 beside rows of 2^-100, and of 2^-120 beside rows of 2^60."""
    for s, x0 in ((2.0 ** 125, 2.0 ** -100), (2.0 ** -120, 2.0 ** 60)):
        for zeros in (False, True):
            codes, scales, z = make((), 20, 128, 64, zeros, torch.bfloat16, 3)
            scales = torch.full_like(scales, s)
            for m in (2, 40):
                x = (rows(m, 128, torch.float32, m) * x0).to(torch.bfloat16)
                y = exl3.G4Linear(exl3.G4Tensor(codes, scales, z)).run_alloc(x, 20, True)
                check(y, *product(x, values(codes, scales, z)), 128)


@pytest.mark.parametrize("dtype", HALF)
def test_rows_do_not_mix(exl3, dtype):
    """Infinities and NaN of a row, and of another output's scales, stay where they are; an infinite input gives what the sum does."""
    for m in (5, 40, 200):
        codes, scales, _ = make((), 24, 160, 32, False, torch.float16, m)
        codes[3, 8] = 0x9F                                     # inputs 16 and 17 of output 3: 15 and 9
        scales[7, 2] = float("nan")
        scales[11, 4] = float("inf")
        x = rows(m, 160, dtype, m)
        x[1] = float("nan")
        x[2, 16] = float("inf")
        y = exl3.G4Linear(exl3.G4Tensor(codes, scales)).run_alloc(x, 24, True)
        keep_m, keep_n = [i for i in range(m) if i not in (1, 2)], [i for i in range(24) if i not in (7, 11)]
        ref, mag = product(x[keep_m], values(codes, scales, None)[keep_n])
        check(y[keep_m][:, keep_n], ref, mag, 160)
        assert bool(y[1].isnan().all()) and bool(y[:, 7].isnan().all()) and float(y[2, 3]) == float("inf")


def test_strided_rows_and_outputs(exl3):
    w = make((), 40, 256, 64, True, torch.float16, 4)
    lin, x = exl3.G4Linear(exl3.G4Tensor(*w)), rows(9, 256, torch.bfloat16, 5)
    ref, mag = product(x, values(*w))
    wide = torch.zeros(9, 300, dtype=torch.bfloat16, device="cuda")
    for off in (0, 8, 3):
        wide[:, off:off + 256] = x
        check(lin.run_alloc(wide[:, off:off + 256], 40, True), ref, mag, 256)
    big = torch.full((9, 60), 5.0, device="cuda")
    lin.run(x, big[:, 7:47])
    check(big[:, 7:47], ref, mag, 256)
    assert bool((big[:, :7] == 5).all()) and bool((big[:, 47:] == 5).all())
    check(lin.run_alloc(x.reshape(3, 3, 256), 40, True).reshape(9, 40), ref, mag, 256)
    assert lin.run_alloc(x[:0], 40, True).shape == (0, 40)
    x32 = x.float()
    check(lin.run_alloc(x32, 40, True), *product(x32.half(), values(*w)), 256)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T", (40, 130))
def test_one_expert_keeps_rows_of_none(exl3, T, dtype):
    """One expert of few outputs and many inputs, where a linear's inputs would be split over workgroups."""
    codes, scales, z = make((1,), 256, 4096, 128, True, dtype, T)
    x = rows(T + 9, 4096, dtype, T)
    ends = ends_of([T])
    y = torch.full((T + 9, 256), 5.0, device="cuda")
    exl3.grouped_mm(x, exl3.G4Tensor(codes, scales, z), ends, out=y)
    check(y[:T], *product(x[:T], values(codes[0], scales[0], z[0])), 4096)
    assert bool((y[T:] == 5).all())
    y = exl3.grouped_mm(x, exl3.G4Tensor(codes, scales, z), ends)
    assert bool((y[T:] == 0).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,group,zeros", ((15, 40, 2048, 128, False), (14, 50, 2048, 64, True), (6, 33, 4608, 32, False), (1, 700, 8192, 64, True),
                                               (3, 4200, 1536, 128, True), (9, 70, 512, 512, False)))
def test_few_rows(exl3, m, n, k, group, zeros, dtype):
    """Rows that fill their share of a CU's LDS and rows that do not, groups of inputs that waves take in turn, many tiles."""
    w = make((), n, k, group, zeros, dtype, m + n)
    x = rows(m, k, dtype, m)
    y = torch.full((m, n), float("nan"), device="cuda")
    exl3.G4Linear(exl3.G4Tensor(*w)).run(x, y)
    check(y, *product(x, values(*w)), k)


def test_offsets_past_32_bits(exl3):
    """Codes of 5.4 GB, rows and outputs of more than 4 GB."""
    E, n, k, m = 640, 4096, 4096, 20
    codes = torch.zeros(E, n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(E, n, k // 128, dtype=torch.float16, device="cuda")
    w = make((), n, k, 128, False, torch.float16, 1)
    codes[-1], scales[-1] = w[0], w[1]
    x = rows(m, k, torch.float16, 2)
    ref, mag = product(x, values(*w))
    for T in (m, 600):                                         # few rows of the last expert, and all experts in blocks of them
        xs = torch.cat((torch.ones(T - m, k, dtype=torch.float16, device="cuda"), x))
        ends = ends_of([0] * (E - 2) + [T - m, m])
        check(exl3.grouped_mm(xs, exl3.G4Tensor(codes, scales), ends)[T - m:], ref, mag, k)
    T = (1 << 31) // k + 1000                                  # x 4.3 GB, y 4.3 GB
    xs = torch.zeros(T, k, dtype=torch.float16, device="cuda")
    xs[-m:] = x
    y = torch.empty(T, n, dtype=torch.float16, device="cuda")
    exl3.G4Linear(exl3.G4Tensor(*w)).run(xs, y)
    check(y[-m:], ref, mag, k)
    assert not bool(y[:-m].any())


@pytest.mark.parametrize("dtype", HALF)
def test_last_tiles_in_splits(exl3, dtype):
    """More tiles than the CUs take in a round: the last ones' inputs are split over workgroups, the others' are not."""
    m, n, k = 1037, 14850, 4096
    need = exl3.lib().exl3_g4_linear_scratch(m, k, n, 128)
    assert 0 < need < 2 * 4 * m * n
    w = make((), n, k, 128, True, torch.float16, 3)
    x, bias = rows(m, k, dtype, 4), torch.randn(n, device="cuda")
    ref, mag = product(x, values(*w))
    y = torch.full((m, n), float("nan"), device="cuda")
    exl3.G4Linear(exl3.G4Tensor(*w), bias).run(x, y)
    check(y, ref + bias.double(), mag + bias.double().abs(), k)
