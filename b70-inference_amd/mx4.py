"""Microscaled 4-bit values (MX4) on the HIP kernels: quantisation, linears and routed experts with MX4 weights.

32 consecutive values of a row share a scale 2^(s - 127) held in a byte (255: not a number); a value is sign, two exponent
bits and one mantissa bit (0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte, the even one in the low half: 4.25 bits per weight.

  * mx4_quantize(x) / mx4_dequantize(t, dtype)     rows of fp16, bf16 or fp32 to MX4Tensor and back
  * MX4Linear(weight, bias): run(x, y) / run_alloc  y = x @ W^T (+ bias), 16-bit rows, weights exact in the rows' type (run
    and run_alloc as BC_LinearEXL3's; as a projection it belongs into MX4Experts, not into ExpertTables or BC_GatedMLP)
  * mx4_gemm(A, B)                                  A @ B^T of two MX4Tensors on the scaled matrix instructions
  * MX4Experts, mx4_moe_forward(x, ids, w, experts) the routed layer of moe_forward over MX4 experts (BlockSparseMLP takes
    MX4Experts too)
Tensors live on the GPU; every op is asynchronous on the current stream of its tensors' device and has scratch of its own (calls may
overlap on several streams, and with replays of graphs that hold some). The reference has no
counterpart: its weights are EXL3 only.
"""
from __future__ import annotations

import torch

from ._lib import ACT_GELU_TANH, ACT_SILU, EXL3_BF16, EXL3_F16, EXL3_F32, Exl3Error, check, lib, on_device, ptr, scratch, \
    stream_of

ACTS = {"silu": ACT_SILU, "gelu_tanh": ACT_GELU_TANH, ACT_SILU: ACT_SILU, ACT_GELU_TANH: ACT_GELU_TANH}
DTYPES = {torch.float16: EXL3_F16, torch.float32: EXL3_F32, torch.bfloat16: EXL3_BF16}

# Scale bytes whose blocks are exact in fp16: 0.5 * 2^-23 is its smallest magnitude, 6 * 2^13 below its largest.
_F16_LO, _F16_HI = 104, 140
_BF16_HI = 252                         # 6 * 2^125 is below bf16's largest magnitude (and fp32's)


class MX4Tensor:
    """codes uint8 [..., k / 2] and scales uint8 [..., k / 32] of values [..., k], both contiguous."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() < 1 or codes.dim() != scales.dim():
            raise Exl3Error("MX4Tensor: codes uint8 [..., k / 2] and scales uint8 [..., k / 32] expected")
        if codes.shape[:-1] != scales.shape[:-1] or scales.shape[-1] == 0 or codes.shape[-1] != 16 * scales.shape[-1]:
            raise Exl3Error(f"MX4Tensor: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not belong together")
        if codes.device != scales.device:
            raise Exl3Error("MX4Tensor: codes and scales on different devices")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise Exl3Error("MX4Tensor: codes and scales must be contiguous")
        if codes.data_ptr() % 16:
            raise Exl3Error("MX4Tensor: codes must be 16-byte aligned")
        self.codes, self.scales = codes, scales

    @classmethod
    def empty(cls, shape, like: torch.Tensor) -> MX4Tensor:
        """Uninitialised values of `shape` (the last dimension a multiple of 32) on like's device."""
        t = cls.__new__(cls)
        lead, k = tuple(shape[:-1]), shape[-1]
        t.codes = like.new_empty(lead + (k // 2,), dtype=torch.uint8)
        t.scales = like.new_empty(lead + (k // 32,), dtype=torch.uint8)
        return t

    @property
    def k(self) -> int:
        return 32 * self.scales.shape[-1]

    @property
    def shape(self) -> torch.Size:
        return self.scales.shape[:-1] + (self.k,)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, dev) -> MX4Tensor:
        return MX4Tensor(self.codes.to(dev), self.scales.to(dev))


# One row of 4096 x 4096 takes 4.7 us on the GPU and quantising four of them 2: the host path is the bound, so few calls and no views
# beyond those the shapes need.
def _rows(x: torch.Tensor, k: int):
    """x as [M, k] with 16-byte aligned, contiguous, non-overlapping rows (a copy where it is not), M and its row stride."""
    if x.is_contiguous():
        if x.data_ptr() % 16 == 0:
            return x, x.numel() // k, k
        x2 = x
    else:
        x2 = x if x.dim() == 2 else x.reshape(-1, k)
        m, ld = x2.shape[0], x2.stride(0) if x2.shape[0] > 1 else k
        if x2.stride(1) == 1 and ld >= k and ld * x2.element_size() % 16 == 0 and x2.data_ptr() % 16 == 0:
            return x2, m, ld
    x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2, x2.numel() // k, k


def _out2(what: str, out: torch.Tensor, m: int, n: int):
    """Output rows [m, n] of `out` [..., n], and their stride."""
    if out.dtype not in DTYPES or out.dim() < 1 or out.shape[-1] != n or out.numel() != m * n:
        raise Exl3Error(f"{what}: out must be fp16, bf16 or fp32 [..., {n}] with {m} rows")
    if out.is_contiguous():
        return out, n
    o2 = out if out.dim() == 2 else out.view(-1, n)
    ld = o2.stride(0) if m > 1 else n
    if (n > 1 and o2.stride(1) != 1) or ld < n:
        raise Exl3Error(f"{what}: rows of out must be contiguous and must not overlap")
    return o2, ld


def mx4_quantize(x: torch.Tensor, out: MX4Tensor | None = None) -> MX4Tensor:
    """MX4 of x (fp16, bf16 or fp32 [..., k], k a multiple of 32): per 32 values a scale 2^(floor(log2 max|x|) - 2), each
    value rounded to the nearest (ties to the even code, magnitudes above 6 scales to 6). A block with an infinity or a
    NaN becomes NaN."""
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise Exl3Error(f"mx4_quantize: x must be fp16, bf16 or fp32, got {x.dtype}")
    shape = x.shape
    if len(shape) < 1 or shape[-1] == 0 or shape[-1] % 32:
        raise Exl3Error(f"mx4_quantize: the last dimension of {tuple(shape)} must be a multiple of 32")
    if out is None:
        where = on_device("mx4_quantize", x)
        out = MX4Tensor.empty(shape, x)
    else:
        where = on_device("mx4_quantize", x, out.codes, out.scales)
        if out.shape != shape:
            raise Exl3Error(f"mx4_quantize: out is {tuple(out.shape)}, x {tuple(shape)}")
    k = shape[-1]
    x2, m, ld = _rows(x, k)
    with where:
        rc = lib().exl3_mx4_quantize(x2.data_ptr(), ld, m, k, dt, out.codes.data_ptr(), out.scales.data_ptr(), stream_of(x))
    if rc:
        check(rc, "mx4_quantize")
    return out


def mx4_dequantize(t: MX4Tensor, dtype: torch.dtype = torch.float16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of t [..., k], exact in bf16 and fp32 up to their largest magnitude (scales to 2^125; infinite from 2^128 on),
    in fp16 for scales 2^-23 .. 2^13, else rounded once."""
    codes, scales = t.codes, t.scales
    shape = t.shape
    k = shape[-1]
    if out is None:
        if dtype not in DTYPES:
            raise Exl3Error(f"mx4_dequantize: fp16, bf16 or fp32, got {dtype}")
        out = codes.new_empty(shape, dtype=dtype)
    elif out.shape != shape:
        raise Exl3Error(f"mx4_dequantize: out is {tuple(out.shape)}, the values {tuple(shape)}")
    where = on_device("mx4_dequantize", codes, scales, out)
    m = scales.numel() * 32 // k
    o2, ld = _out2("mx4_dequantize", out, m, k)
    with where:
        rc = lib().exl3_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), m, k, o2.data_ptr(), ld, DTYPES[out.dtype],
                                       stream_of(out))
    if rc:
        check(rc, "mx4_dequantize")
    return out


def _bias(what: str, bias, n: int):
    if bias is None:
        return None
    if bias.numel() != n or not bias.is_floating_point():
        raise Exl3Error(f"{what}: bias must be floating point [{n}]")
    return bias.detach().reshape(-1).float().contiguous()


def mx4_gemm(A: MX4Tensor, B: MX4Tensor, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """A [..., k] @ B^T (+ bias [n]) for B [n, k], both MX4: [..., n] with fp32 sums, one rounding."""
    k = A.k
    if B.scales.dim() != 2 or B.k != k:
        raise Exl3Error(f"mx4_gemm: A {tuple(A.shape)} and B {tuple(B.shape)} must share k, B [n, k]")
    n, m = B.scales.shape[0], A.scales.numel() * 32 // k
    bias = None if bias is None else _bias("mx4_gemm", bias, n)
    if out is None:
        if out_dtype not in DTYPES:
            raise Exl3Error(f"mx4_gemm: out_dtype fp16, bf16 or fp32, got {out_dtype}")
        out = o2 = A.codes.new_empty(A.codes.shape[:-1] + (n,), dtype=out_dtype)
        ld = n
        where = on_device("mx4_gemm", A.codes, A.scales, B.codes, B.scales, bias)
    else:
        where = on_device("mx4_gemm", A.codes, A.scales, B.codes, B.scales, bias, out)
        o2, ld = _out2("mx4_gemm", out, m, n)
    if n == 0:
        return out
    ws, need = scratch("exl3_mx4_gemm", out, m, k, n)
    with where:
        rc = lib().exl3_mx4_gemm_in(A.codes.data_ptr(), A.scales.data_ptr(), m, k, B.codes.data_ptr(), B.scales.data_ptr(), n,
                                    ptr(bias), o2.data_ptr(), ld, DTYPES[out.dtype], ptr(ws), need, stream_of(out))
    if rc:
        check(rc, "mx4_gemm")
    return out


def _scale_bases(w: MX4Tensor):
    """Per leading matrix of w [..., n, k]: the power of two to take out of its scales so that every block that is not all
    zeros is exact in fp16 (0 where none is needed), whether there is one, and whether every value fits bf16 (of magnitudes
    2^128 and more, which the two largest scales have, none does). Reads the weights once, on the host's time."""
    s = w.scales.flatten(-2).to(torch.int16)
    blk = (w.codes.view(torch.int64) & 0x7777777777777777).unflatten(-1, (-1, 2)).ne(0).any(-1).flatten(-2)
    live = blk & (s < 255)                                     # (NaN blocks stay NaN under any base)
    lo = torch.where(live, s, torch.full_like(s, 255)).amin(-1).reshape(-1).tolist()
    hi = torch.where(live, s, torch.full_like(s, -1)).amax(-1).reshape(-1).tolist()
    base = [0 if b < 0 or (a >= _F16_LO and b <= _F16_HI) else b - _F16_HI for a, b in zip(lo, hi)]
    ok = [b < 0 or a - e >= _F16_LO for a, b, e in zip(lo, hi, base)]
    fits = [True] * len(hi)
    if max(hi) > _BF16_HI:
        c = w.codes.unflatten(-1, (-1, 16))
        top = torch.maximum(c & 7, c >> 4 & 7).amax(-1).flatten(-2)
        past = ((s == 253) & (top >= 6)) | ((s == 254) & (top >= 4))           # from 4 2^126 and 2 2^127 on
        fits = past.any(-1).logical_not().reshape(-1).tolist()
    return base, ok, fits


class MX4Linear:
    """y = x @ W^T (+ bias) with W [n, k] in MX4 and 16-bit rows x. The weights are exact in the rows' type; fp16 rows need
    the matrix's scales (of blocks that are not all zeros) to span at most 2^36: MX4Linear finds the power of two to take
    out once, here, and refuses fp16 rows of a wider matrix (bf16 rows take any) and bf16 rows of one with values of 2^128 and
    more. A weight that is changed afterwards needs an MX4Linear of its own."""

    bf16_rows = True

    def __init__(self, weight: MX4Tensor, bias: torch.Tensor | None = None):
        if len(weight.shape) != 2 or weight.shape[0] == 0:
            raise Exl3Error(f"MX4Linear: weight must be MX4 [n, k], got {tuple(weight.shape)}")
        self.weight = weight
        self.out_features, self.in_features = weight.shape
        self.bias = _bias("MX4Linear", bias, self.out_features)
        (self.scale_base,), (self.fp16_rows,), (self.bf16_rows,) = _scale_bases(weight)

    def run(self, x: torch.Tensor, y: torch.Tensor) -> None:
        """x [..., k] fp16 or bf16 (other types become fp16) -> y (fp16, bf16 or fp32, preallocated) [..., n]."""
        k, n, w = self.in_features, self.out_features, self.weight
        if x.dim() < 1 or x.shape[-1] != k:
            raise Exl3Error(f"MX4Linear: x must be [..., {k}], got {tuple(x.shape)}")
        where = on_device("MX4Linear", x, y, w.codes, self.bias)
        if x.dtype != torch.float16 and x.dtype != torch.bfloat16:
            x = x.half()
        if x.dtype == torch.float16 and not self.fp16_rows:
            raise NotImplementedError("MX4Linear: the weight's scales span more than fp16 holds; use bf16 rows")
        if x.dtype == torch.bfloat16 and not self.bf16_rows:
            raise NotImplementedError("MX4Linear: the weight has values of 2^128 and more, which bf16 does not hold")
        x2, m, ld = _rows(x, k)
        y2, y_ld = _out2("MX4Linear", y, m, n)
        ws, need = scratch("exl3_mx4_linear", x, m, k, n)
        with where:
            rc = lib().exl3_mx4_linear_in(x2.data_ptr(), ld, DTYPES[x.dtype], m, k, w.codes.data_ptr(), w.scales.data_ptr(), n,
                                          self.scale_base, ptr(self.bias), y2.data_ptr(), y_ld, DTYPES[y.dtype], ptr(ws), need,
                                          stream_of(x))
        if rc:
            check(rc, "mx4_linear")

    def run_alloc(self, x: torch.Tensor, out_features: int, output_fp32: bool) -> torch.Tensor:
        dt = torch.float32 if output_fp32 else x.dtype if x.dtype == torch.bfloat16 else torch.float16
        y = x.new_empty(x.shape[:-1] + (out_features,), dtype=dt)
        self.run(x, y)
        return y


class MX4Experts:
    """Device table of E experts with MX4 weights: int64 [9, E] = (codes address, scales address, scale base) of gate [I, H],
    up [I, H] and down [H, I]. Holds references to every tensor that it points at. Lists of MX4Tensor or MX4Linear (without
    biases), one per expert; MX4Experts.stacked takes one MX4Tensor [E, rows, k] per projection. Weights that are changed afterwards need
    a table of their own."""

    def __init__(self, gates, ups, downs):
        if not (len(gates) == len(ups) == len(downs)) or not gates:
            raise Exl3Error("MX4Experts: gate/up/down lists must be non-empty and equally long")
        projs = []
        for plist in (gates, ups, downs):
            ts = []
            for p in plist:
                if isinstance(p, MX4Linear):
                    if p.bias is not None:
                        raise NotImplementedError("MX4Experts: experts with biases")
                    p = p.weight
                ts.append(p)
            projs.append(ts)
        shape = projs[0][0].shape
        if len(shape) != 2:
            raise Exl3Error("MX4Experts: projections must be MX4 [rows, k]")
        shapes = (tuple(shape), tuple(shape), (shape[1], shape[0]))
        bases = [[_scale_bases(t) for t in ts] for ts in projs]
        rows = []
        for ts, bs, want in zip(projs, bases, shapes):
            if any(tuple(t.shape) != want for t in ts):
                raise Exl3Error(f"MX4Experts: every gate and up must be {shapes[0]}, every down {shapes[2]}")
            rows += [[t.codes.data_ptr() for t in ts], [t.scales.data_ptr() for t in ts], [b[0][0] for b in bs]]
        self._finish([t for ts in projs for t in ts], rows, shapes[0], all(b[1][0] for bs in bases for b in bs),
                     all(b[2][0] for bs in bases for b in bs))

    def _finish(self, tensors, rows, shape, fp16_rows, bf16_rows):
        self.tensors = tensors
        if len({t.device for t in tensors}) > 1:
            raise Exl3Error("MX4Experts: weights on several devices")
        self.E, (self.I, self.H) = len(rows[0]), shape
        if self.I % 32:
            raise Exl3Error(f"MX4Experts: {self.I} intermediate columns are not a multiple of 32")
        self.fp16_rows, self.bf16_rows = fp16_rows, bf16_rows
        self.tables = torch.tensor(rows, dtype=torch.int64).to(tensors[0].device)

    @classmethod
    def stacked(cls, gate: MX4Tensor, up: MX4Tensor, down: MX4Tensor) -> MX4Experts:
        """E experts from gate and up [E, I, H] and down [E, H, I]."""
        if len(gate.shape) != 3 or gate.shape[0] == 0 or up.shape != gate.shape \
                or tuple(down.shape) != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise Exl3Error("MX4Experts.stacked: gate and up [E, I, H] and down [E, H, I] expected")
        rows, fine, fits = [], True, True
        for t in (gate, up, down):
            base, ok = [], True
            for e0 in range(0, t.shape[0], 16):                # a few experts at a time: the check's scratch stays small
                b, o, f = _scale_bases(MX4Tensor(t.codes[e0:e0 + 16], t.scales[e0:e0 + 16]))
                base, ok, fits = base + b, ok and all(o), fits and all(f)
            n, c, s = t.shape[0], t.codes[0].numel(), t.scales[0].numel()
            rows += [[t.codes.data_ptr() + e * c for e in range(n)], [t.scales.data_ptr() + e * s for e in range(n)], base]
            fine = fine and ok
        self = cls.__new__(cls)
        self._finish([gate, up, down], rows, gate.shape[1:], fine, fits)
        return self


def mx4_moe_forward(x: torch.Tensor, topk_ids: torch.Tensor, topk_w: torch.Tensor, experts: MX4Experts, act=ACT_SILU,
                    act_limit: float = 0.0, shared: int = -1, out: torch.Tensor | None = None,
                    out_dtype=torch.float32) -> torch.Tensor:
    """out[t] = sum_j topk_w[t, j] * expert_{topk_ids[t, j]}(x[t]) (+ expert `shared` with weight 1), fp32 sums, expert(x) =
    down(act(gate(x), up(x))) with act(gate, up) rounded to x's type (its magnitude may leave fp16's range). x fp16 or bf16 [M, H]; topk_ids int32 [M, k] (outside
    [0, E): inactive); topk_w fp32 [M, k]; out fp16, bf16 or fp32. The arguments are moe_forward's."""
    H = experts.H
    if x.dim() != 2 or x.dtype not in (torch.float16, torch.bfloat16) or x.shape[1] != H:
        raise Exl3Error(f"mx4_moe_forward: x must be fp16 or bf16 [M, {H}]")
    if x.dtype == torch.float16 and not experts.fp16_rows:
        raise NotImplementedError("mx4_moe_forward: an expert's scales span more than fp16 holds; use bf16 rows")
    if x.dtype == torch.bfloat16 and not experts.bf16_rows:
        raise NotImplementedError("mx4_moe_forward: an expert has values of 2^128 and more, which bf16 does not hold")
    M = x.shape[0]
    if topk_ids.dtype != torch.int32 or topk_w.dtype != torch.float32:
        raise Exl3Error("mx4_moe_forward: topk_ids int32 and topk_w fp32 expected")
    if topk_ids.shape != topk_w.shape or topk_ids.dim() != 2 or topk_ids.shape[0] != M:
        raise Exl3Error("mx4_moe_forward: topk_ids / topk_w must be [M, k]")
    if out is None:
        if out_dtype not in DTYPES:
            raise Exl3Error(f"mx4_moe_forward: out_dtype fp16, bf16 or fp32, got {out_dtype}")
        out = o2 = x.new_empty((M, H), dtype=out_dtype)
        o_ld = H
        where = on_device("mx4_moe_forward", x, topk_ids, topk_w, experts.tables)
    else:
        where = on_device("mx4_moe_forward", x, topk_ids, topk_w, experts.tables, out)
        o2, o_ld = _out2("mx4_moe_forward", out, M, H)
    a = ACTS.get(act)
    if a is None:
        raise NotImplementedError(f"mx4_moe_forward: activation {act!r}")
    topk_ids, topk_w = topk_ids.contiguous(), topk_w.contiguous()
    x2, _, ld = _rows(x, H)
    k, shared = topk_ids.shape[1], int(shared)
    ws, need = scratch("exl3_mx4_moe", x, M, H, experts.I, k, experts.E, shared)
    with where:
        rc = lib().exl3_mx4_moe_forward_in(x2.data_ptr(), ld, DTYPES[x.dtype], M, H, experts.I, topk_ids.data_ptr(),
                                           topk_w.data_ptr(), k, experts.E, experts.tables.data_ptr(), a, float(act_limit), shared,
                                           o2.data_ptr(), o_ld, DTYPES[out.dtype], ptr(ws), need, stream_of(x))
    if rc:
        check(rc, "mx4_moe_forward")
    return out
