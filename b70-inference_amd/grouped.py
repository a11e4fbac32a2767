"""Products of rows grouped by expert, and their gradients, on the HIP kernels.

Rows are sorted by expert: `ends` int32 [E] (on the GPU, ascending) says behind which row each expert's rows end, so expert e
has rows ends[e - 1] .. ends[e] - 1 (from 0 for e = 0), none where two ends are equal; rows behind the last end belong to no
expert. moe_align sorts a routing: ends = counts.cumsum(0, dtype=torch.int32), x[pair_tok] the rows.

  * grouped_mm(x, w, ends)       y[t] = w[e] @ x[t]; w 16-bit [E, N, K] or a G4Tensor (4-bit weights with group scales)
  * grouped_mm_dx(dy, w, ends)   dx[t] = dy[t] @ w[e], the gradient with respect to the rows
  * grouped_mm_dw(dy, x, ends)   dw[e] = dy[rows of e]^T @ x[rows of e], the gradient with respect to the weights
There is no autograd graph: pass the gradients on. Rows and weights fp16 or bf16, sums fp32 in an order fixed by the sizes, layouts and alignments, one rounding
to out's type. Tensors live on the GPU; every op is asynchronous on the current stream of its tensors' device and has scratch of its
own where it needs some (calls may overlap on streams and threads, and can be captured without a warm-up). The reference has no counterpart: its experts are
EXL3 only.
"""
from __future__ import annotations

import torch

from ._lib import EXL3_BF16, EXL3_F16, Exl3Error, check, lib, on_device, ptr, scratch, stream_of
from .g4 import _MOST_LD, G4Tensor, _g4_rows
from .mx4 import DTYPES

_HALF = {torch.float16: EXL3_F16, torch.bfloat16: EXL3_BF16}
_W_NK, _W_KN = 0, 1                    # exl3_grouped_w


def _ends(what: str, ends: torch.Tensor, E: int) -> torch.Tensor:
    if ends.dtype != torch.int32 or ends.dim() != 1 or ends.shape[0] != E:
        raise Exl3Error(f"{what}: ends must be int32 [{E}], got {ends.dtype} {tuple(ends.shape)}")
    return ends.contiguous()


def _rows2(what: str, name: str, x: torch.Tensor):
    """x [T, k] with contiguous, non-overlapping rows in the kernels' reach (a copy where they are not) and their stride."""
    if x.dim() != 2 or x.dtype not in _HALF:
        raise Exl3Error(f"{what}: {name} must be fp16 or bf16 [T, columns], got {x.dtype} {tuple(x.shape)}")
    T, k = x.shape
    if k == 0:
        raise Exl3Error(f"{what}: {name} has no columns")
    ld = x.stride(0) if T > 1 else k
    if (k > 1 and x.stride(1) != 1) or ld < k or ld > _MOST_LD:
        x = x.contiguous()
        ld = k
    return x, ld


def _matrices(what: str, w: torch.Tensor):
    """w [E, N, K] as (tensor, layout, row stride, expert stride): rows of K or, for transposed matrices, of N (a copy of w where
    neither is contiguous, or where they are further apart than the kernels reach)."""
    E, n, k = w.shape
    se, sn, sk = w.stride()
    se = se if E > 1 else 0
    if se >= 0:
        if (sk == 1 or k == 1) and (n == 1 or k <= sn <= _MOST_LD):
            return w, _W_NK, sn if n > 1 else k, se
        if (sn == 1 or n == 1) and (k == 1 or n <= sk <= _MOST_LD):
            return w, _W_KN, sk if k > 1 else n, se
    return w.contiguous(), _W_NK, k, n * k


def _out_rows(what: str, x: torch.Tensor, T: int, n: int, out, out_dtype):
    """out [T, n] (allocated where it is None), and its row stride."""
    if out is None:
        dt = x.dtype if out_dtype is None else out_dtype
        if dt not in DTYPES:
            raise Exl3Error(f"{what}: out_dtype fp16, bf16 or fp32, got {dt}")
        return x.new_empty((T, n), dtype=dt), n
    if out.dtype not in DTYPES or tuple(out.shape) != (T, n):
        raise Exl3Error(f"{what}: out must be fp16, bf16 or fp32 [{T}, {n}], got {out.dtype} {tuple(out.shape)}")
    ld = out.stride(0) if T > 1 else n
    if (n > 1 and out.stride(1) != 1) or ld < n:
        raise Exl3Error(f"{what}: rows of out must be contiguous and must not overlap")
    return out, ld


def _mm(what: str, x, w, ends, transpose: bool, out, out_dtype):
    if isinstance(w, G4Tensor):
        raise NotImplementedError(f"{what}: 4-bit weights have no gradient of their rows")
    if w.dim() != 3 or w.dtype not in _HALF or 0 in w.shape:
        raise Exl3Error(f"{what}: w must be fp16 or bf16 [E, N, K], got {w.dtype} {tuple(w.shape)}")
    x, ld = _rows2(what, "dy" if transpose else "x", x)
    E, n, k = w.shape
    if transpose:
        n, k = k, n
    T = x.shape[0]
    if x.dtype != w.dtype or x.shape[1] != k:
        raise Exl3Error(f"{what}: rows {x.dtype} {tuple(x.shape)} and weights {w.dtype} {tuple(w.shape)} do not belong together")
    ends = _ends(what, ends, E)
    rest = out is None
    out, o_ld = _out_rows(what, x, T, n, out, out_dtype)
    where = on_device(what, x, w, ends, out)
    w, layout, w_ld, w_es = _matrices(what, w)
    if transpose:
        layout ^= 1
    with where:
        rc = lib().exl3_grouped_mm(x.data_ptr(), ld, _HALF[x.dtype], T, k, w.data_ptr(), w_ld, w_es, layout, n, ends.data_ptr(),
                                   E, out.data_ptr(), o_ld, DTYPES[out.dtype], int(rest), stream_of(x))
    if rc:
        check(rc, what)
    return out


def _mm_g4(what: str, x, w: G4Tensor, ends, out, out_dtype):
    if w.codes.dim() != 3:
        raise Exl3Error(f"{what}: w must be a G4Tensor [E, N, K], got {tuple(w.shape)}")
    E, n, k = w.shape
    if x.dim() != 2 or x.dtype not in _HALF or x.shape[1] != k:
        raise Exl3Error(f"{what}: x must be fp16 or bf16 [T, {k}], got {x.dtype} {tuple(x.shape)}")
    ends = _ends(what, ends, E)
    rest = out is None
    x2, T, ld = _g4_rows(x, k)
    out, o_ld = _out_rows(what, x, T, n, out, out_dtype)
    with on_device(what, x, w.codes, ends, out):
        rc = lib().exl3_grouped_g4(x2.data_ptr(), ld, _HALF[x.dtype], T, k, w.codes.data_ptr(), w.scales.data_ptr(),
                                   _HALF[w.scales.dtype], ptr(w.zeros), w.group, n, ends.data_ptr(), E, out.data_ptr(), o_ld,
                                   DTYPES[out.dtype], int(rest), stream_of(x))
    if rc:
        check(rc, what)
    return out


def grouped_mm(x: torch.Tensor, w, ends: torch.Tensor, out: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[t] = w[e] @ x[t] for the rows t of every expert e: x fp16 or bf16 [T, K], w of x's type [E, N, K] (any strides; matrices
    whose rows or columns are contiguous are read in place) or a G4Tensor [E, N, K], ends int32 [E]. Returns [T, N] of out_dtype (fp16, bf16 or fp32; None:
    x's type), 0 in rows of no expert, or writes out, which keeps such rows as they are."""
    if isinstance(w, G4Tensor):
        return _mm_g4("grouped_mm", x, w, ends, out, out_dtype)
    return _mm("grouped_mm", x, w, ends, False, out, out_dtype)


def grouped_mm_dx(dy: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped_mm with respect to x: dx[t] = dy[t] @ w[e], dy fp16 or bf16 [T, N], w as there [E, N, K]. Returns [T, K]
    of out_dtype (None: dy's type), 0 in rows of no expert, or writes out, which keeps such rows as they are."""
    return _mm("grouped_mm_dx", dy, w, ends, True, out, out_dtype)


def grouped_mm_dw(dy: torch.Tensor, x: torch.Tensor, ends: torch.Tensor, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of grouped_mm with respect to w: dw[e] = sum over the rows t of expert e of dy[t] (x) x[t], dy [T, N] and x [T, K] fp16
    or bf16 alike, ends int32 [E]. Returns [E, N, K] of out_dtype (fp16, bf16 or fp32; None: x's type), 0 for an expert without rows,
    or writes out; with accumulate it is added to what out holds."""
    what = "grouped_mm_dw"
    dy, dy_ld = _rows2(what, "dy", dy)
    x, x_ld = _rows2(what, "x", x)
    if dy.dtype != x.dtype or dy.shape[0] != x.shape[0]:
        raise Exl3Error(f"{what}: dy {dy.dtype} {tuple(dy.shape)} and x {x.dtype} {tuple(x.shape)} do not belong together")
    if ends.dim() != 1 or ends.shape[0] == 0:
        raise Exl3Error(f"{what}: ends must be int32 [E], got {ends.dtype} {tuple(ends.shape)}")
    E, T, n, k = ends.shape[0], x.shape[0], dy.shape[1], x.shape[1]
    ends = _ends(what, ends, E)
    if out is None:
        if accumulate:
            raise Exl3Error(f"{what}: accumulate needs out")
        dt = x.dtype if out_dtype is None else out_dtype
        if dt not in DTYPES:
            raise Exl3Error(f"{what}: out_dtype fp16, bf16 or fp32, got {dt}")
        out = x.new_empty((E, n, k), dtype=dt)
    elif out.dtype not in DTYPES or tuple(out.shape) != (E, n, k):
        raise Exl3Error(f"{what}: out must be fp16, bf16 or fp32 [{E}, {n}, {k}], got {out.dtype} {tuple(out.shape)}")
    where = on_device(what, dy, x, ends, out)
    se, sn, sk = out.stride()
    a, a_ld, b, b_ld, m = dy, dy_ld, x, x_ld, n
    if not (k == 1 or sk == 1) and (n == 1 or sn == 1):        # transposed matrices: the transposed product
        a, a_ld, b, b_ld, m, k, sn, sk = x, x_ld, dy, dy_ld, k, n, sk, sn
    ld = sn if m > 1 else k
    es = se if E > 1 else m * ld
    if (k > 1 and sk != 1) or ld < k or (es < (m - 1) * ld + k and (es < k or ld < (E - 1) * es + k)):
        raise Exl3Error(f"{what}: matrices of out must have contiguous rows or columns and must not overlap")
    ws, need = scratch("exl3_grouped_mm_dw", x, T, m, k, E)
    with where:
        rc = lib().exl3_grouped_mm_dw_in(a.data_ptr(), a_ld, b.data_ptr(), b_ld, _HALF[x.dtype], T, m, k, ends.data_ptr(), E,
                                         out.data_ptr(), ld, es, DTYPES[out.dtype], int(bool(accumulate)), ptr(ws), need, stream_of(x))
    if rc:
        check(rc, what)
    return out
