"""A routed layer of bf16 experts: gate and up products with fp32 outputs, which the activation takes (it refuses bf16), the middle
converted to bf16."""
import pytest
import torch

from grouped_util import spans

pytestmark = pytest.mark.gpu
M, H, I, E, TOPK = 60, 128, 96, 7, 2


def test_routed_layer_of_bf16_experts(exl3):
    """Against 64 bits. gate and up: sums of H products, off by at most da and db (units of 2^-23 of the magnitudes' sum). The middle
    h = silu(a) b: silu's slope is below 1.1, fp32's evaluation below 2^-20, so off by eh before it is rounded to fp16 (2^-11, at
    least 2^-25) and to bf16 (2^-8). down: these times the weights, sums of I products, then two picks' weights and sums."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(M, H, device="cuda", generator=g).bfloat16()
    gate, up = ((torch.randn(E, I, H, device="cuda", generator=g) / H ** 0.5).bfloat16() for _ in range(2))
    down = (torch.randn(E, H, I, device="cuda", generator=g) / I ** 0.5).bfloat16()
    ids, w = exl3.route_topk(torch.randn(M, E, device="cuda", generator=g), TOPK)
    counts, tok, pw, _ = exl3.moe_align(ids, w, E)
    tok, ends = tok.long(), counts.cumsum(0, dtype=torch.int32)
    rows = x[tok]
    a, b = (exl3.grouped_mm(rows, m, ends, out_dtype=torch.float32) for m in (gate, up))
    h = torch.empty(len(tok), I, dtype=torch.float16, device="cuda")
    for wrong in (a.bfloat16(), exl3.grouped_mm(rows, gate, ends)):
        with pytest.raises(exl3.Exl3Error, match="fp16 or fp32"):
            exl3.silu_mul(wrong, wrong, h, 0.0)
    exl3.silu_mul(a, b, h, 0.0)
    y = exl3.grouped_mm(h.bfloat16(), down, ends, out_dtype=torch.float32)
    out = torch.zeros(M, H, device="cuda").index_add_(0, tok, y * pw[:, None])

    ref = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    lim = torch.full_like(ref, 1e-30)
    for e, lo, hi in spans(ends):
        if hi == lo:
            continue
        r, p, t = rows[lo:hi].double(), pw[lo:hi, None].double(), tok[lo:hi]
        wg, wu, wd = (m[e].double().t().contiguous() for m in (gate, up, down))
        u, v = r @ wg, r @ wu
        da, db = H * 2.0 ** -23 * (r.abs() @ wg.abs()), H * 2.0 ** -23 * (r.abs() @ wu.abs())
        s = u * torch.sigmoid(u)
        m = s * v
        eh = 1.1 * da * (v.abs() + db) + s.abs() * db + 2.0 ** -20 * m.abs()
        eh = eh + (m.abs() + eh) * (2.0 ** -11 + 2.0 ** -8 * (1 + 2.0 ** -11)) + 2.0 ** -24
        mag = ((m.abs() + eh) @ wd.abs()) * p
        ref.index_add_(0, t, (m @ wd) * p)
        lim.index_add_(0, t, (eh @ wd.abs()) * p + (I + 4) * 2.0 ** -23 * mag)
    err = (out.double() - ref).abs()
    assert bool((err <= lim).all()), float((err / lim).max())
    assert bool((lim <= 0.05 * ref.abs().max()).all())
