"""The activations take two matrices of fp16 or of fp32: other types are refused before the library is called (which would read them
as fp32, past their end where they are narrower)."""
import importlib

import pytest
import torch

MOE = importlib.import_module("b70-inference_amd.moe")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float64, torch.int8, torch.int32, torch.uint8))
def test_other_types_are_refused(exl3, monkeypatch, dtype):
    calls = []
    fake = type("Fake", (), {"exl3_act_mul": staticmethod(lambda *a: calls.append(a) or 0)})()
    monkeypatch.setattr(MOE, "lib", lambda: fake)
    monkeypatch.setattr(MOE, "require_device", lambda *t: None)
    monkeypatch.setattr(MOE, "stream_of", lambda t: None)
    x, z = torch.zeros(4, 64, dtype=dtype), torch.zeros(4, 64, dtype=torch.float16)
    for act in (lambda x: exl3.silu_mul(x, x, z, 0.0), lambda x: exl3.gelu_mul(x, x, z)):
        with pytest.raises(exl3.Exl3Error, match="fp16 or fp32"):
            act(x)
        assert not calls
        act(x.half())
        act(x.float())
        assert [a[4] for a in calls] == [0, 1]                 # EXL3_F16, EXL3_F32
        calls.clear()
