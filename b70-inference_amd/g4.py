"""4-bit weights with group scales (G4) on the HIP kernels: the linear, and what grouped_mm takes as experts.

w = (q - z) s: whole numbers q from 0 to 15, and for each `group` neighbouring inputs of an output (32, 64 or a multiple of 128) one
16-bit scale s and one whole number z from 0 to 15 (8 where no zeros are given).

  * G4Tensor(codes, scales, zeros)                 weights [..., n, k] as they lie in memory
  * G4Linear(weight, bias): run(x, y) / run_alloc  y = x @ W^T (+ bias), 16-bit rows (run and run_alloc as BC_LinearEXL3's; no
    projection for ExpertTables or BC_GatedMLP)
  * grouped_mm(x, G4Tensor [E, n, k], ends)        rows sorted by expert
No weight is rounded: q - z is exact in the rows' type and the scales multiply fp32 sums. Tensors live on the GPU; every op is
asynchronous on the current stream of its tensors' device and has scratch of its own where it needs some (calls may overlap on streams
and threads, and can be captured without a warm-up). The reference has no counterpart: its weights are EXL3
only.
"""
from __future__ import annotations

import torch

from ._lib import EXL3_BF16, EXL3_F16, Exl3Error, check, lib, on_device, ptr, scratch, stream_of
from .mx4 import DTYPES, _bias, _out2, _rows

_HALF = {torch.float16: EXL3_F16, torch.bfloat16: EXL3_BF16}
_MOST_LD = 1 << 22                     # elements from row to row that the kernels' 32-bit offsets inside a block of rows allow


def _g4_rows(x: torch.Tensor, k: int):
    """_rows, in the kernels' reach (a copy where the rows are further apart)."""
    x2, m, ld = _rows(x, k)
    return (x2, m, ld) if ld <= _MOST_LD or ld == k else (x2.contiguous(), m, k)


class G4Tensor:
    """codes uint8 [..., n, k / 2] (two q to a byte, the even one in the low half), scales fp16 or bf16 [..., n, k / group] and zeros
    uint8 [..., n, k / group] (0 .. 15) or None, all contiguous."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None):
        if codes.dtype != torch.uint8 or scales.dtype not in _HALF or codes.dim() not in (2, 3) or codes.dim() != scales.dim():
            raise Exl3Error("G4Tensor: codes uint8 [(E,) n, k / 2] and scales fp16 or bf16 [(E,) n, k / group] expected")
        if codes.shape[:-1] != scales.shape[:-1] or 0 in codes.shape or 0 in scales.shape or 2 * codes.shape[-1] % scales.shape[-1]:
            raise Exl3Error(f"G4Tensor: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not belong together")
        group = 2 * codes.shape[-1] // scales.shape[-1]
        if group not in (32, 64) and group % 128:
            raise NotImplementedError(f"G4Tensor: groups of {group} inputs (32, 64 and multiples of 128)")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise Exl3Error(f"G4Tensor: zeros must be uint8 {tuple(scales.shape)}")
        ts = [t for t in (codes, scales, zeros) if t is not None]
        if len({t.device for t in ts}) > 1:
            raise Exl3Error("G4Tensor: codes, scales and zeros on different devices")
        if not all(t.is_contiguous() for t in ts):
            raise Exl3Error("G4Tensor: codes, scales and zeros must be contiguous")
        if codes.data_ptr() % 16:
            raise Exl3Error("G4Tensor: codes must be 16-byte aligned")
        self.codes, self.scales, self.zeros, self.group = codes, scales, zeros, group

    @property
    def k(self) -> int:
        return 2 * self.codes.shape[-1]

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape[:-1] + (self.k,)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, dev) -> G4Tensor:
        return G4Tensor(self.codes.to(dev), self.scales.to(dev), None if self.zeros is None else self.zeros.to(dev))


class G4Linear:
    """y = x @ W^T (+ bias) with W [n, k] in G4 and 16-bit rows x; the weights are read as they are at each call."""

    def __init__(self, weight: G4Tensor, bias: torch.Tensor | None = None):
        if not isinstance(weight, G4Tensor) or weight.codes.dim() != 2:
            raise Exl3Error("G4Linear: weight must be a G4Tensor [n, k]")
        self.weight = weight
        self.out_features, self.in_features = weight.shape
        self.bias = _bias("G4Linear", bias, self.out_features)

    def run(self, x: torch.Tensor, y: torch.Tensor) -> None:
        """x [..., k] fp16 or bf16 (other types become fp16) -> y (fp16, bf16 or fp32, preallocated) [..., n]."""
        k, n, w = self.in_features, self.out_features, self.weight
        if x.dim() < 1 or x.shape[-1] != k:
            raise Exl3Error(f"G4Linear: x must be [..., {k}], got {tuple(x.shape)}")
        where = on_device("G4Linear", x, y, w.codes, self.bias)
        if x.dtype not in _HALF:
            x = x.half()
        x2, m, ld = _g4_rows(x, k)
        y2, y_ld = _out2("G4Linear", y, m, n)
        ws, need = scratch("exl3_g4_linear", x, m, k, n, w.group)
        with where:
            rc = lib().exl3_g4_linear_in(x2.data_ptr(), ld, _HALF[x.dtype], m, k, w.codes.data_ptr(), w.scales.data_ptr(),
                                         _HALF[w.scales.dtype], ptr(w.zeros), w.group, n, ptr(self.bias), y2.data_ptr(), y_ld,
                                         DTYPES[y.dtype], ptr(ws), need, stream_of(x))
        if rc:
            check(rc, "g4_linear")

    def run_alloc(self, x: torch.Tensor, out_features: int, output_fp32: bool) -> torch.Tensor:
        dt = torch.float32 if output_fp32 else x.dtype if x.dtype == torch.bfloat16 else torch.float16
        y = x.new_empty(x.shape[:-1] + (out_features,), dtype=dt)
        self.run(x, y)
        return y
