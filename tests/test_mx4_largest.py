"""MX4 weights at bf16's and fp32's upper end: which matrices take bf16 rows (on the host), and their products."""
import numpy as np
import pytest
import torch

import mx4_util as U

DEV = "cuda:0"


def tensor(exl3, scales, code):
    """One row of blocks with these scale bytes, every code `code`, of alternating sign."""
    c = torch.full((1, 16 * len(scales)), code | (code | 8) << 4, dtype=torch.uint8)
    return exl3.MX4Tensor(c, torch.tensor([scales], dtype=torch.uint8))


@pytest.mark.parametrize("scale,code,fits", [(252, 7, True), (253, 5, True), (253, 6, False), (253, 7, False), (254, 3, True),
                                             (254, 4, False), (254, 7, False), (254, 0, True), (255, 7, True)])
def test_which_weights_bf16_holds(exl3, scale, code, fits):
    for scales in ([scale], [120, scale, 100]):
        w = tensor(exl3, scales, code)
        v = U.values(w.codes.numpy(), w.scales.numpy())
        with np.errstate(over="ignore"):
            assert fits == (not np.isinf(v.astype(np.float32)).any())
        assert exl3.MX4Linear(w).bf16_rows is fits
    big = exl3.MX4Tensor(w.codes.repeat(96, 1), w.scales.repeat(96, 1))                  # [96, 96]
    one = exl3.MX4Tensor(big.codes & 0x99, big.scales.clamp(max=250))
    stack = [exl3.MX4Tensor(torch.stack([t.codes for t in ts]), torch.stack([t.scales for t in ts])) for ts in ([one, big], [one, one])]
    assert exl3.MX4Experts([one, big], [one, one], [one, one]).bf16_rows is fits
    assert exl3.MX4Experts.stacked(stack[1], stack[1], stack[0]).bf16_rows is fits
    assert exl3.MX4Experts([one], [one], [one]).bf16_rows


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_products_with_the_largest_weights(exl3, m):
    k, n = 256, 48
    c, s = U.random_mx4((n, k), 1, 245, 252)
    x = (torch.randn(m, k, generator=torch.Generator().manual_seed(2)) * 2.0 ** -20).bfloat16()
    xv = x.double().numpy()
    w, wv = exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)), U.values(c, s)
    U.check(exl3.MX4Linear(w).run_alloc(x.to(DEV), n, True), xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.float32)
    for dt in (torch.bfloat16, torch.float32):
        assert np.array_equal(exl3.mx4_dequantize(w, dt).cpu().double().numpy(), wv)
    s[3, 1], c[3, 16:32] = 254, 0x93                                                     # 1.5 and -.5
    wv = U.values(c, s)
    w = exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV))
    U.check(exl3.MX4Linear(w).run_alloc(x.to(DEV), n, True), xv @ wv.T, np.abs(xv) @ np.abs(wv).T, k, torch.float32)
    w.codes[3, 20] = 4
    lin = exl3.MX4Linear(w)
    with pytest.raises(NotImplementedError, match="2\\^128"):
        lin.run_alloc(x.to(DEV), n, True)
    assert torch.isinf(exl3.mx4_dequantize(w, torch.bfloat16)[3, 40])


@pytest.mark.gpu
def test_routed_layer_refuses_what_bf16_does_not_hold(exl3):
    c, s = U.random_mx4((2, 96, 96), 3, 118, 122)
    t = [exl3.MX4Tensor(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)) for _ in range(3)]
    ids, w = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), torch.ones(1, 2, device=DEV)
    x = torch.ones(1, 96, dtype=torch.bfloat16, device=DEV)
    exl3.mx4_moe_forward(x, ids, w, exl3.MX4Experts.stacked(*t))
    t[2].scales[1, 5, 2] = 254
    t[2].codes[1, 5, 40] = 7
    with pytest.raises(NotImplementedError, match="2\\^128"):
        exl3.mx4_moe_forward(x, ids, w, exl3.MX4Experts.stacked(*t))
