"""MX4 values in 64 bits, written from the format: the tests' counterpart of the kernels."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def quantise(x):
    """(codes uint8 [..., k / 2], scales uint8 [..., k / 32]) of float64 rows: nearest value by search, ties to the even code."""
    v = np.asarray(x, np.float64)
    blk = v.reshape(v.shape[:-1] + (-1, 32))
    top = np.abs(blk).max(-1)
    bad = ~np.isfinite(blk).all(-1)
    _, e = np.frexp(np.where(bad | (top == 0), 1.0, top))
    s = np.where(top == 0, 0, np.clip(e - 1 - 2 + 127, 0, 254))
    a = np.abs(np.where(bad[..., None], 0, blk)) * 2.0 ** (127.0 - s)[..., None]
    d = np.abs(a[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    cand = d == best                                   # one value, or two neighbours at a tie
    code = np.argmax(np.where(cand, 2 - np.arange(8) % 2, 0), -1)
    code = code | np.where(np.signbit(blk), 8, 0)
    code = np.where(bad[..., None], 0, code)
    s = np.where(bad, 255, s)
    code = code.reshape(v.shape[:-1] + (-1, 2))
    return (code[..., 0] | code[..., 1] << 4).astype(np.uint8), s.astype(np.uint8)


def values(codes, scales):
    """float64 values of codes and scales."""
    c = np.asarray(codes)
    q = np.stack([c & 15, c >> 4], -1).reshape(c.shape[:-1] + (-1,))
    v = np.where(q & 8, -1.0, 1.0) * GRID[q & 7]
    s = np.asarray(scales).astype(np.float64)
    f = np.where(s == 255, np.nan, 2.0 ** (s - 127))
    return v * np.repeat(f, 32, -1)


def random_mx4(shape, seed, lo=110, hi=130):
    """Random codes and scales (bytes lo .. hi) of values [..., k]."""
    g = np.random.default_rng(seed)
    codes = g.integers(0, 256, shape[:-1] + (shape[-1] // 2,), dtype=np.uint8)
    scales = g.integers(lo, hi + 1, shape[:-1] + (shape[-1] // 32,), dtype=np.uint8)
    return codes, scales


def sum_bound(k):
    """Error of an fp32 sum of k products on the matrix instructions over the sum of their magnitudes: the products are
    exact, an instruction adds 32 of them (at most 32 half steps of its own part, which is a 32nd of k), the chain of
    instructions k / 32 times, and 8 waves add their sums; each addition is off by at most a whole step of 2^-23."""
    return (k / 32 + 8 + 32) * 2.0 ** -23


def check(y, ref, mag, k, dtype, extra=0.0):
    """y (tensor of dtype) within its rounding and the sums' bound of ref (float64); mag: sums of magnitudes."""
    y = y.detach().cpu().double().numpy()
    tol = np.abs(ref) * HALF_STEP[dtype] + SMALLEST[dtype] + (sum_bound(k) * mag + extra) * (1 + HALF_STEP[dtype])
    err = np.abs(y - ref)
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(bad)[:5].tolist())
