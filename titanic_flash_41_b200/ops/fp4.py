"""MXFP4 rows and their product (kernels: ``csrc/fp4.cu``, ``csrc/gemm_fp4.cu``): the 4-bit counterpart of ``ops/mx.py``.

``quant_rows`` packs activation rows (e2m1 values, one UE8M0 scale per 32 inputs: ``formats.codecs.mxfp4_quant``'s numbers),
``gemm`` multiplies such rows with weights of the same form on the block-scaled tensor-core instruction, ``dequant_rows``
gives the numbers back.  A checkpoint's MXFP4 matrix (packed bytes, row-major scales) becomes an operand with
``rows_from_mxfp4``, once.

    w = fp4.rows_from_mxfp4(packed, scales)          # [N, K / 2], [N, K / 32]
    y = fp4.gemm(fp4.quant_rows(x), w)               # [rows, N] bf16

Packed rows: ``q`` [rows, Kp / 2], the even element in the low nibble, ``Kp`` = K rounded up to 256, zeros behind K.  Scales:
``sf`` [Kp / 128, units, 128] in the unit layout of ``ops/mx.py``; ``units`` covers the rows in whole blocks of 256.

The product's waits are bounded.  One that runs out leaves a void result and reports it, to the caller's ``status`` (``native.StatusWord.t``) or, without
one, to a word of the device that ``check`` reads.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch

from . import native

_KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
K_BLOCK = 256                  # packed rows are whole multiples of it
ROW_BLOCK = 256                # so are the rows that scale units cover


def padded(n: int, unit: int) -> int:
    return -(-n // unit) * unit


class Fp4Rows:
    """``rows`` x ``K`` numbers in MXFP4: ``q`` and ``sf`` as described above."""
    __slots__ = ("_q", "_sf", "_both", "q_at", "sf_at", "rows", "K", "units", "device")

    def __init__(self, q: torch.Tensor, sf: torch.Tensor, rows: int, K: int):
        half = -(-K // K_BLOCK) * (K_BLOCK // 2)         # bytes of a row
        if rows < 0 or K < 1:
            raise ValueError("Fp4Rows: rows and K")
        if q.dtype is not torch.uint8 or not q.is_contiguous() or q.numel() != rows * half:
            raise ValueError(f"Fp4Rows: q holds {rows} rows of {half} bytes")
        least = -(-rows // ROW_BLOCK) * (ROW_BLOCK // 32)
        shape, device = sf.shape, q.device
        if sf.dtype is not torch.uint8 or not sf.is_contiguous() or len(shape) != 3 or shape[0] != half // 64 or shape[2] != 128 \
                or shape[1] < least:
            raise ValueError(f"Fp4Rows: sf is [{half // 64}, at least {least}, 128]")
        if device != sf.device:
            raise ValueError("Fp4Rows: q and sf on one device")
        self._q, self._sf, self._both = q, sf, None
        self.q_at, self.sf_at = q.data_ptr(), sf.data_ptr()
        if self.q_at & 15 or self.sf_at & 3:
            raise ValueError("Fp4Rows: q starts on a 16-byte boundary, sf on one of 4 (16 in a product)")
        self.rows, self.K, self.units, self.device = rows, K, shape[1], device

    # Rows that are made here lie in one buffer; tensors over its parts are made when somebody asks for them.
    @property
    def q(self) -> torch.Tensor:
        if self._q is None:
            self._q = self._both[:self.sf_at - self.q_at].view(self.rows, padded(self.K, K_BLOCK) // 2)
        return self._q

    @property
    def sf(self) -> torch.Tensor:
        if self._sf is None:
            self._sf = self._both[self.sf_at - self.q_at:].view(padded(self.K, K_BLOCK) // 128, self.units, 128)
        return self._sf


def empty_rows(rows: int, K: int, device) -> Fp4Rows:
    if rows < 0 or K < 1:
        raise ValueError("empty_rows: rows and K")
    half = -(-K // K_BLOCK) * (K_BLOCK // 2)             # bytes of a row; a row's 2 * half / 32 scale bytes, in whole blocks of rows
    r = Fp4Rows.__new__(Fp4Rows)
    r.rows, r.K, r.units = rows, K, -(-rows // ROW_BLOCK) * (ROW_BLOCK // 32)
    r._q = r._sf = None
    r._both = both = torch.empty(rows * half + 2 * half * r.units, dtype=torch.uint8, device=device)
    r.q_at = both.data_ptr()
    r.sf_at = r.q_at + rows * half
    r.device = both.device
    return r


def quant_rows(x: torch.Tensor, out: Optional[Fp4Rows] = None) -> Fp4Rows:
    """Rows of ``x`` [rows, K] (f32 / f16 / bf16, last dim contiguous) in MXFP4.  A block of 32 with a NaN or an infinity becomes NaN."""
    kind = _KIND.get(x.dtype)
    if x.dim() != 2 or kind is None:
        raise ValueError("quant_rows: x is [rows, K] in f32, f16 or bf16")
    rows, K = x.shape
    row, one = x.stride()
    if K < 1 or (K > 1 and one != 1) or row < 0:
        raise ValueError("quant_rows: the last dimension is contiguous")
    if out is None:
        out = empty_rows(rows, K, x.device)
    elif not (out.rows == rows and out.K == K and out.device == x.device):
        raise ValueError("quant_rows: out has another size or device")
    if rows:
        native.launch("tf_fp4_quant_rows", x, x.data_ptr(), kind, row, out.q_at, out.sf_at, out.units, rows, K)
    return out


def dequant_rows(r: Fp4Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that ``r`` stands for, [rows, K] (exact in bf16 and f32)."""
    if dtype not in _KIND:
        raise ValueError("dequant_rows: f32, f16 or bf16")
    y = torch.empty(r.rows, r.K, dtype=dtype, device=r.device)
    if r.rows:
        native.launch("tf_fp4_dequant_rows", y, r.q_at, r.sf_at, r.units, y.data_ptr(), _KIND[dtype], r.K, r.rows, r.K)
    return y


def rows_from_mxfp4(packed: torch.Tensor, scales: torch.Tensor) -> Fp4Rows:
    """A checkpoint's matrix: packed e2m1 [N, K / 2] and row-major UE8M0 scales [N, K / 32] (K a multiple of 32)."""
    if packed.dim() != 2 or packed.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("rows_from_mxfp4: bytes [N, K / 2] and [N, K / 32]")
    N, K = packed.shape[0], packed.shape[1] * 2
    if K < 1 or K % 32 or scales.shape != (N, K // 32):
        raise ValueError("rows_from_mxfp4: scales [N, K / 32] of a K that 32 divides")
    kp, rows = padded(K, K_BLOCK), padded(N, ROW_BLOCK)
    q = packed if kp == K else torch.nn.functional.pad(packed, (0, (kp - K) // 2))
    s = torch.nn.functional.pad(scales, (0, (kp - K) // 32, 0, rows - N))
    sf = s.view(rows // 32, 32, kp // 128, 4).permute(2, 0, 1, 3).reshape(kp // 128, rows // 32, 128)
    q, sf = (x if x.data_ptr() % 16 == 0 else x.clone() for x in (q.contiguous(), sf.contiguous()))       # (bytes of a file begin anywhere)
    return Fp4Rows(q, sf, N, K)


_WORDS: Dict[torch.device, native.StatusWord] = {}


def _word_at(device: torch.device) -> Optional[int]:
    """Address of the device's status word.  It is made by the first product outside of a graph's capture (whose memory and work are the graph's): a
    graph captured before any reports nowhere."""
    word = _WORDS.get(device)
    if word is None:
        if device.type == "cuda":
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    return None
            word = native.StatusWord(device)
            torch.cuda.current_stream(device).synchronize()                     # (products on other streams use it too)
        else:
            word = native.StatusWord(device)
        word.at = word.t.data_ptr()
        word = _WORDS.setdefault(device, word)
    return word.at


def check(device=None) -> None:
    """Raise if a wait of a product ran out on this device (on any) since the last call."""
    one = None if device is None else torch.empty(0, device=device).device
    for at, word in list(_WORDS.items()):
        if one is None or at == one:
            word.check()


def gemm(a: Fp4Rows, w: Fp4Rows, out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16, status=None) -> torch.Tensor:
    """``a`` [M, K] x ``w`` [N, K] transposed -> [M, N]; fp32 sums, rounded once to bf16 / f16 / f32.  ``out``: its last dimension
    contiguous, rows at any pitch.  ``status``: see the top of this module."""
    if a.K != w.K:
        raise ValueError(f"gemm: K of the operands: {a.K} and {w.K}")
    if a.device != w.device:
        raise ValueError("gemm: both operands on one device")
    if (a.sf_at | w.sf_at) & 15:
        raise ValueError("gemm: scales start on 16-byte boundaries")
    if status is not None and (status.dtype is not torch.int32 or status.numel() < 4 or not status.is_contiguous() or status.device != a.device):
        raise ValueError("gemm: status is int32 [4] on the operands' device")
    M, N = a.rows, w.rows
    if out is None:
        if dtype not in _KIND:
            raise ValueError("gemm: f32, f16 or bf16")
        out, pitch = torch.empty(M, N, dtype=dtype, device=a.device), N
    else:
        dtype = out.dtype
        if dtype not in _KIND or out.shape != (M, N) or out.device != a.device:
            raise ValueError("gemm: out has another size, type or device")
        pitch, one = out.stride()
        if N > 1 and one != 1:
            raise ValueError("gemm: out's last dimension is contiguous")
        if M > 1 and pitch < N:
            raise ValueError("gemm: out's rows overlap")
        pitch = max(pitch, N)
    if M and N:
        if status is None:
            word = _WORDS.get(a.device)
            status_at = _word_at(a.device) if word is None else word.at
        else:
            status_at = status.data_ptr()
        native.launch("tf_gemm_fp4", out, a.q_at, a.sf_at, a.units, w.q_at, w.sf_at, w.units, out.data_ptr(), pitch, _KIND[dtype], M, N,
                      -(-a.K // K_BLOCK) * K_BLOCK, status_at)
    return out


def linear(x: torch.Tensor, w: Fp4Rows, status=None) -> torch.Tensor:
    """``x`` [rows, K] quantised to MXFP4 and multiplied with ``w`` [N, K], in x's type."""
    return gemm(quant_rows(x), w, dtype=x.dtype, status=status)
