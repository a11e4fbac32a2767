"""Rows of the router balance whose logits all lie far below zero: their shares stay what the scores' ratios are."""
import pytest
import torch

from test_balance_gpu import DEV, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["sigmoid", "sqrt_softplus"])
@pytest.mark.parametrize("M,E,k", [(3, 8, 2), (24, 33, 2), (300, 160, 8), (9, 2500, 4)])
def test_balance_of_low_rows(exl3, score, M, E, k):
    z, ids = make(M, E, k, M + E)
    low = torch.tensor([-90.0, -120.0, -16.0, -17.0, -30.0, -75.0, -87.0, -103.0, -200.0, -400.0, 0.0])
    z = z + low[torch.arange(M) % len(low)][:, None]
    compare(exl3, z, ids, score, None, 1.0)
    mask = torch.arange(M) % 3 != 2
    compare(exl3, z, ids, score, mask, 0.1)
    # in place, over a row's own logits
    dz = z.to(DEV)
    l, c, p, n = exl3.route_balance(dz, ids.to(DEV), score=score)
    assert abs(float(p.sum()) - 1) < 1e-4                        # every row counts whole
    want = exl3.route_balance_grad(dz, c, n, k, score=score)
    assert torch.equal(exl3.route_balance_grad(dz, c, n, k, score=score, out=dz), want)


@pytest.mark.parametrize("score", ["sigmoid", "sqrt_softplus"])
def test_balance_of_equal_low_logits(exl3, score):
    E = 40
    ids = torch.arange(4, dtype=torch.int32).expand(5, 4).contiguous().to(DEV)
    for level in (-20.0, -88.0, -89.0, -104.0, -110.0, -1e4, -1e30):
        l, c, p, n = exl3.route_balance(torch.full((5, E), level, device=DEV), ids, score=score)
        assert (p - 1 / E).abs().max() < 1e-6 and abs(float(l) - 1) < 1e-5


@pytest.mark.parametrize("score", ["sigmoid", "sqrt_softplus"])
def test_balance_of_far_apart_logits(exl3, score):
    """One expert near 0, the others down to -160: their shares are small, not zero, as far as fp32 goes."""
    z, ids = make(30, 24, 3, 5)
    z[:, 1:] -= torch.linspace(0, 160, 23)
    compare(exl3, z, ids, score, None, 1.0)
