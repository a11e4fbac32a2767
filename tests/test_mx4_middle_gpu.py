"""The routed layer's middle, act(gate, up): values that fp16 does not hold, on every path."""
import numpy as np
import pytest
import torch

import mx4_util as U
from test_mx4_gpu import act64, routing, rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def shifted(exl3, shape, seed, by, axis):
    """Codes with scale bytes 118 .. 122, those of block b (or of the rows of block b) `by(b)` higher."""
    c, s = U.random_mx4(shape, seed, 118, 122)
    n = shape[axis] // 32
    b = np.array([by(i) for i in range(n)])
    s = (s.astype(np.int32) + (np.repeat(b, 32)[None, :, None] if axis == 1 else b)).astype(np.uint8)
    return exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)), U.values(c, s)


def exponent(top):
    """Largest power of two by which a group whose largest magnitude is within 1 % of `top` may be held."""
    e = [0 if 2.0 ** -8 <= t < 2.0 ** 15 else np.frexp(t)[1] - 15 for t in (0.99 * top, 1.01 * top) if t > 0]
    return max(e, default=-126)


def underflow(h, group):
    """What fp16's range costs the values of a row h held in groups with a power of two each: half its least step, 2^-25, once where a
    group is rounded and once more where it is brought to the largest power of the row."""
    a = [exponent(np.abs(h[i:i + group]).max()) for i in range(0, len(h), group)]
    return np.repeat([2.0 ** (e - 25) + 2.0 ** (max(a) - 25) for e in a], group)[:len(h)]


def reference(x, ids, w, gv, uv, dv, act, half, group):
    """The layer in float64 and a bound on the kernel's error: sums_bound for every product, the middle's rounding (half a step
    `half`, and with fp16 in groups of `group` columns its range), 8 steps of fp32 for the activation."""
    M, H = x.shape
    out, err = np.zeros((M, H)), np.zeros((M, H))
    for t in range(M):
        for e, wt in zip(ids[t], w[t]):
            g, u = gv[e] @ x[t], uv[e] @ x[t]
            dg, du = (U.sum_bound(H) * (np.abs(v[e]) @ np.abs(x[t])) for v in (gv, uv))
            h = act64(g, u, act, 0.0)
            sg = np.abs(act64(g, np.ones_like(u), act, 0.0))
            dh = np.abs(h) * (half + 8 * 2.0 ** -23) + 1.13 * dg * (np.abs(u) + du) + sg * du + (underflow(h, group) if group else 0.0)
            y = dv[e] @ h
            out[t] += wt * y
            err[t] += abs(wt) * (np.abs(dv[e]) @ dh + U.sum_bound(gv.shape[1]) * (np.abs(dv[e]) @ (np.abs(h) + dh)))
            err[t] += abs(wt * y) * 2.0 ** -23
        err[t] += ids.shape[1] * (2.0 ** -23 * np.abs(out[t]) + 2.0 ** -24 * err[t])
    return out, err


# pairs as they stand; blocks of 32, 64 and 128 rows
PATHS = [(3, 256, 160, 4, 2), (2, 96, 1120, 3, 2), (100, 256, 160, 16, 2), (100, 128, 320, 4, 2), (150, 96, 288, 2, 2)]
# powers of two of the up projection's blocks of 32 rows, taken back by the down projection's blocks
SHIFTS = {"large": lambda b: 24, "small": lambda b: -40, "mixed": lambda b: (12, 0, -10)[b % 3], "one": lambda b: 20 if b == 1 else 0,
          "rising": lambda b: min(2 * b - 8, 12),
          "huge": lambda b: 60}


@pytest.mark.parametrize("kind", list(SHIFTS))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,H,I,E,k", PATHS)
def test_moe_middle_of_any_magnitude(exl3, dtype, M, H, I, E, k, kind):
    by = SHIFTS[kind]
    g, gv = shifted(exl3, (E, I, H), 1, lambda b: 0, 1)
    u, uv = shifted(exl3, (E, I, H), 2, by, 1)
    d, dv = shifted(exl3, (E, H, I), 3, lambda b: -by(b), 2)
    ex = exl3.MX4Experts.stacked(g, u, d)
    x = rows((M, H), dtype, M, 0.3)
    ids, w = routing(M, k, E, M)
    for act in ("silu", "gelu_tanh"):
        group = 0 if dtype == torch.bfloat16 else 16 if M < 10 else 128
        ref, err = reference(x.double().numpy(), ids, w, gv, uv, dv, act, U.HALF_STEP[dtype], group)
        for out in (torch.float32, dtype):
            y = exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex, act, out_dtype=out)
            U.check(y, ref, 0.0, H, out, extra=err)


@pytest.mark.parametrize("M,H,I,E,k", PATHS)
def test_moe_middle_not_finite_stays_in_its_token(exl3, M, H, I, E, k):
    """A NaN or an infinity in a row of x makes its own outputs not finite and leaves the others' bits."""
    (g, _), (u, _), (d, _) = (shifted(exl3, s, i, lambda b: 0, a) for i, (s, a) in enumerate((((E, I, H), 1), ((E, I, H), 1), ((E, H, I), 2))))
    ex = exl3.MX4Experts.stacked(g, u, d)
    ids, w = (torch.from_numpy(v).to(DEV) for v in routing(M, k, E, M))
    x = rows((M, H), torch.float16, M, 0.3).to(DEV)
    want = exl3.mx4_moe_forward(x, ids, w, ex)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[M // 2, H - 1] = bad
        y = exl3.mx4_moe_forward(z, ids, w, ex)
        keep = torch.arange(M, device=DEV) != M // 2
        assert torch.equal(y[keep], want[keep]) and not torch.isfinite(y[M // 2]).any()
    assert (exl3.mx4_moe_forward(torch.zeros_like(x), ids, w, ex) == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,H,I,E,k", [(90, 4640, 96, 8, 2), (90, 96, 2336, 8, 2), (100, 2592, 2144, 4, 2), (130, 2208, 64, 2, 2)])
def test_moe_wide_blocks_of_long_rows(exl3, dtype, M, H, I, E, k):
    """More steps of k than a wave holds scales of (16; 8 in blocks of 128 rows), in either product."""
    g, gv = shifted(exl3, (E, I, H), 4, lambda b: 0, 1)
    u, uv = shifted(exl3, (E, I, H), 5, lambda b: 0, 1)
    d, dv = shifted(exl3, (E, H, I), 6, lambda b: b % 5, 2)
    ex = exl3.MX4Experts.stacked(g, u, d)
    x = rows((M, H), dtype, M, 0.3) * 0.25
    ids, w = routing(M, k, E, M)
    ref, err = reference(x.double().numpy(), ids, w, gv, uv, dv, "silu", U.HALF_STEP[dtype], 0 if dtype == torch.bfloat16 else 128)
    y = exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex)
    U.check(y, ref, 0.0, H, torch.float32, extra=err)


@pytest.mark.parametrize("M,H,I,E,k", [(2, 64, 8224, 2, 1), (3, 32, 8736, 3, 1), (100, 96, 1120, 4, 2), (90, 64, 1312, 8, 2), (260, 64, 2208, 2, 1)])
def test_moe_middle_whose_groups_change(exl3, M, H, I, E, k):
    """Pairs: a wave takes two groups of 512 columns of a row, each smaller, larger or like the other; blocks: more steps than lanes
    that share a row."""
    def by(b):
        g = b // 16 if M < 10 else b // 4
        return (0, 14, -14)[(g % 9) % 3 if g < 9 else (g % 9) // 3]

    g, gv = shifted(exl3, (E, I, H), 7, lambda b: 0, 1)
    u, uv = shifted(exl3, (E, I, H), 8, by, 1)
    d, dv = shifted(exl3, (E, H, I), 9, lambda b: -by(b), 2)
    ex = exl3.MX4Experts.stacked(g, u, d)
    assert ex.fp16_rows
    x = rows((M, H), torch.float16, M, 0.3)
    ids, w = routing(M, k, E, M)
    ref, err = reference(x.double().numpy(), ids, w, gv, uv, dv, "silu", U.HALF_STEP[torch.float16], 16 if M < 10 else 128)
    y = exl3.mx4_moe_forward(x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV), ex)
    U.check(y, ref, 0.0, H, torch.float32, extra=err)
