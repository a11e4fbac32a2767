"""Products grouped by expert in 64 bits, and how far a kernel's may be from them."""
import torch

HALF = (torch.float16, torch.bfloat16)


def ends_of(sizes, device="cuda"):
    return torch.tensor(sizes, dtype=torch.int64).cumsum(0).to(torch.int32).to(device)


def sizes_for(T, E, seed, empty=()):
    """T rows over E experts, some more than others; those of `empty` have none."""
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(torch.randn(E, generator=g))
    for e in empty:
        w[e] = 0
    return torch.bincount(torch.multinomial(w, T, replacement=True, generator=g), minlength=E).tolist() if T else [0] * E


def spans(ends):
    at = 0
    for e, end in enumerate(ends.tolist()):
        yield e, at, end
        at = end


def rows_product(x, w, ends, T_out):
    """x[t] @ w[e]^T in 64 bits, and the same of the magnitudes; NaN in rows of no expert."""
    y = torch.full((T_out, w.shape[1]), float("nan"), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for e, a, b in spans(ends):
        if b > a:
            y[a:b] = x[a:b].double() @ w[e].double().t().contiguous()
            mag[a:b] = x[a:b].double().abs() @ w[e].double().abs().t().contiguous()
    return y, mag


def weights_gradient(dy, x, ends):
    E = ends.shape[0]
    dw = torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(dw)
    for e, a, b in spans(ends):
        if b > a:
            dw[e] = dy[a:b].double().t().contiguous() @ x[a:b].double()
            mag[e] = dy[a:b].double().abs().t().contiguous() @ x[a:b].double().abs()
    return dw, mag


def bound(ref, mag, c, dtype):
    """Products of 16-bit values are exact in fp32; c of them added in any order are off by at most c units of 2^-23 of the sum of
    their magnitudes (2^-24 for rounding, twice that where an addition cuts off); the result is rounded once, by half a step."""
    off = c * 2.0 ** -23 * mag
    eps = torch.finfo(dtype).eps / 2
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return off + eps * (ref.abs() + off) + least


def check(out, ref, mag, c, what=""):
    assert out.shape == ref.shape, (out.shape, ref.shape)
    lim = bound(ref, mag, c, out.dtype)
    err = (out.double() - ref).abs()
    bad = ~(err <= lim)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by {float((err / lim).nan_to_num(1e30).max()):.2f} bounds, first at {bad.nonzero()[0].tolist()}"
