"""MX4 projections where EXL3 ones are expected: refused by name, on the host."""
import pytest
import torch


def test_mx4_projections_are_refused_by_exl3_tables(exl3):
    def t(n, k):
        return exl3.MX4Linear(exl3.MX4Tensor(torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // 32, dtype=torch.uint8)))

    g, u, d = t(256, 128), t(256, 128), t(128, 256)
    with pytest.raises(NotImplementedError, match="MX4Experts"):
        exl3.ExpertTables([g], [u], [d])
    with pytest.raises(NotImplementedError, match="MX4Experts"):
        exl3.BC_GatedMLP(None, None, None, None, None, None, None, 0, False, True, True, False, False, g, u, d, 0.0)
    assert exl3.MX4Experts([g], [u], [d]).E == 1
