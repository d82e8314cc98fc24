"""MXFP4 rows and their product (kernels: ``csrc/fp4.cu``, ``csrc/gemm_fp4.cu``): the 4-bit counterpart of ``ops/mx.py``.

``quant_rows`` packs activation rows (e2m1 values, one UE8M0 scale per 32 inputs: ``formats.codecs.mxfp4_quant``'s numbers),
``gemm`` multiplies such rows with weights of the same form on the block-scaled tensor-core instruction, ``dequant_rows``
gives the numbers back.  A checkpoint's MXFP4 matrix (packed bytes, row-major scales) becomes an operand with
``rows_from_mxfp4``, once.

    w = fp4.rows_from_mxfp4(packed, scales)          # [N, K / 2], [N, K / 32]
    y = fp4.gemm(fp4.quant_rows(x), w)               # [rows, N] bf16

Packed rows: ``q`` [rows, Kp / 2], the even element in the low nibble, ``Kp`` = K rounded up to 256, zeros behind K.  Scales:
``sf`` [Kp / 128, units, 128] in the unit layout of ``ops/mx.py``; ``units`` covers the rows in whole blocks of 256.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import native

_KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
K_BLOCK = 256                  # packed rows are whole multiples of it
ROW_BLOCK = 256                # so are the rows that scale units cover


def padded(n: int, unit: int) -> int:
    return -(-n // unit) * unit


class Fp4Rows:
    """``rows`` x ``K`` numbers in MXFP4: ``q`` and ``sf`` as described above."""
    __slots__ = ("q", "sf", "rows", "K")

    def __init__(self, q: torch.Tensor, sf: torch.Tensor, rows: int, K: int):
        kp = padded(K, K_BLOCK)
        if not (rows >= 0 and K >= 1):
            raise ValueError("Fp4Rows: rows and K")
        if not (q.dtype == torch.uint8 and q.is_contiguous() and q.numel() == rows * (kp // 2)):
            raise ValueError(f"Fp4Rows: q holds {rows} rows of {kp // 2} bytes")
        if not (sf.dtype == torch.uint8 and sf.is_contiguous() and sf.dim() == 3 and sf.shape[0] == kp // 128 and sf.shape[2] == 128
                and sf.shape[1] * 32 >= padded(rows, ROW_BLOCK)):
            raise ValueError(f"Fp4Rows: sf is [{kp // 128}, at least {padded(rows, ROW_BLOCK) // 32}, 128]")
        if not (q.device == sf.device):
            raise ValueError("Fp4Rows: q and sf on one device")
        self.q, self.sf, self.rows, self.K = q, sf, rows, K


def empty_rows(rows: int, K: int, device) -> Fp4Rows:
    kp = padded(K, K_BLOCK)
    q = torch.empty(rows, kp // 2, dtype=torch.uint8, device=device)
    sf = torch.empty(kp // 128, padded(rows, ROW_BLOCK) // 32, 128, dtype=torch.uint8, device=device)
    r = Fp4Rows.__new__(Fp4Rows)
    r.q, r.sf, r.rows, r.K = q, sf, rows, K
    return r


def quant_rows(x: torch.Tensor, out: Optional[Fp4Rows] = None) -> Fp4Rows:
    """Rows of ``x`` [rows, K] (f32 / f16 / bf16, last dim contiguous) in MXFP4.  A block of 32 with a NaN or an infinity becomes NaN."""
    if not (x.dim() == 2 and x.dtype in _KIND):
        raise ValueError("quant_rows: x is [rows, K] in f32, f16 or bf16")
    rows, K = x.shape
    if not (K >= 1 and (K == 1 or x.stride(1) == 1) and x.stride(0) >= 0):
        raise ValueError("quant_rows: the last dimension is contiguous")
    if out is None:
        out = empty_rows(rows, K, x.device)
    else:
        if not (out.rows == rows and out.K == K and out.q.device == x.device):
            raise ValueError("quant_rows: out has another size or device")
    if rows:
        native.launch("tf_fp4_quant_rows", x, x.data_ptr(), _KIND[x.dtype], x.stride(0), out.q.data_ptr(), out.sf.data_ptr(), out.sf.shape[1],
                      rows, K)
    return out


def dequant_rows(r: Fp4Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that ``r`` stands for, [rows, K] (exact in bf16 and f32)."""
    if not (dtype in _KIND):
        raise ValueError("dequant_rows: f32, f16 or bf16")
    y = torch.empty(r.rows, r.K, dtype=dtype, device=r.q.device)
    if r.rows:
        native.launch("tf_fp4_dequant_rows", y, r.q.data_ptr(), r.sf.data_ptr(), r.sf.shape[1], y.data_ptr(), _KIND[dtype], r.K, r.rows, r.K)
    return y


def rows_from_mxfp4(packed: torch.Tensor, scales: torch.Tensor) -> Fp4Rows:
    """A checkpoint's matrix: packed e2m1 [N, K / 2] and row-major UE8M0 scales [N, K / 32] (K a multiple of 32)."""
    if not (packed.dim() == 2 and packed.dtype == torch.uint8 and scales.dtype == torch.uint8):
        raise ValueError("rows_from_mxfp4: bytes [N, K / 2] and [N, K / 32]")
    N, K = packed.shape[0], packed.shape[1] * 2
    if not (K > 0 and K % 32 == 0 and tuple(scales.shape) == (N, K // 32)):
        raise ValueError("rows_from_mxfp4: scales [N, K / 32] of a K that 32 divides")
    kp, rows = padded(K, K_BLOCK), padded(N, ROW_BLOCK)
    q = packed if kp == K else torch.nn.functional.pad(packed, (0, (kp - K) // 2))
    s = torch.nn.functional.pad(scales, (0, (kp - K) // 32, 0, rows - N))
    sf = s.view(rows // 32, 32, kp // 128, 4).permute(2, 0, 1, 3).reshape(kp // 128, rows // 32, 128)
    return Fp4Rows(q.contiguous(), sf.contiguous(), N, K)


def gemm(a: Fp4Rows, w: Fp4Rows, out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16, status=None) -> torch.Tensor:
    """``a`` [M, K] x ``w`` [N, K] transposed -> [M, N]; fp32 sums, rounded once to bf16 / f16 / f32.  ``out``: its last dimension
    contiguous, rows at any pitch."""
    if not (a.K == w.K):
        raise ValueError(f"gemm: K of the operands: {a.K} and {w.K}")
    if not (a.q.device == w.q.device):
        raise ValueError("gemm: both operands on one device")
    if out is None:
        if not (dtype in _KIND):
            raise ValueError("gemm: f32, f16 or bf16")
        out = torch.empty(a.rows, w.rows, dtype=dtype, device=a.q.device)
    else:
        if not (out.dtype in _KIND and tuple(out.shape) == (a.rows, w.rows) and out.device == a.q.device):
            raise ValueError("gemm: out has another size, type or device")
        if not (w.rows <= 1 or out.stride(1) == 1):
            raise ValueError("gemm: out's last dimension is contiguous")
        if not (a.rows <= 1 or out.stride(0) >= w.rows):
            raise ValueError("gemm: out's rows overlap")
    if a.rows and w.rows:
        native.launch("tf_gemm_fp4", out, a.q.data_ptr(), a.sf.data_ptr(), a.sf.shape[1], w.q.data_ptr(), w.sf.data_ptr(), w.sf.shape[1],
                      out.data_ptr(), max(out.stride(0), w.rows), _KIND[out.dtype], a.rows, w.rows, padded(a.K, K_BLOCK),
                      None if status is None else status.data_ptr())
    return out


def linear(x: torch.Tensor, w: Fp4Rows, status=None) -> torch.Tensor:
    """``x`` [rows, K] quantised to MXFP4 and multiplied with ``w`` [N, K], in x's type."""
    return gemm(quant_rows(x), w, dtype=x.dtype, status=status)
