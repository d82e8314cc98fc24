"""Paged KV cache held in 4 bits, and attention over it (kernels: ``csrc/paged.cu``, ``csrc/paged_attn.cu``).

A cache is two byte buffers of pages; a page holds ``page`` tokens (16, 32, 64, 128 or 256), for every kv head a block of
keys and a block of values: packed e2m1, one e4m3 scale per 16 numbers (the arithmetic of the compressed KV rows,
``formats.codecs.kv_v41fp4_encode``), 72 bytes a token and head of 128 channels, for keys and values each.  A block's
scale is 2^-6 to 448: blocks whose largest number is below 0.094 share the grid of 2^-6 (steps of 2^-7 next to zero; up to 2^-8 becomes
zero), and what is above 2,688 becomes 2,688.  Keys and values far from 1 are scaled by the caller, keys against ``scale``, values
against what the attention gives.

    cache = PagedCache.allocate(pages, kv_heads, head_dim, page=64)
    q = append(cache, k, v, table, lengths, cu, q=q, rope=table_of_angles)     # rotate, quantise, store; rotated queries back
    o = attention(cache, q, table, lengths, cu)

A batch is ``total`` rows of ``S`` sequences: ``cu`` int32 [S + 1] holds the sequences' row offsets (None: one row each),
``lengths`` int32 [S] the tokens of every sequence once the rows are in the cache, ``table`` int32 [S, W] its pages in order.  Row
i of sequence s is token ``lengths[s] - (cu[s + 1] - i)``.  All three stay on the device, so a captured graph follows them; rows
behind the last sequence's are left as they were (in an output that a call makes itself: whatever the memory held).

No position, page or offset takes a call out of its buffers, and the cache's status word (``cache.check()``) has the first one that was
out of range:

* ``append`` and ``read`` skip a row whose position is negative, behind the table or behind the table of angles, or whose page
  is none of the cache's, and report it.  ``read`` gives zeros there, ``append`` the row's query (rotated, if its position has
  angles).  They also report offsets that leave 0 .. ``total`` or run backwards.
* ``attention`` reports pages that it cannot read and counts them as zeros.  It reports no position: a row before the first token sees
  no key, and one behind the table sees the tokens that the table has pages for.  Nor does it report offsets: a range is clipped
  to the batch, and of rows that two ranges claim, or that stand in ranges of more than ``total`` rows in all, some get no result.

A cache over a user's own buffers (``PagedCache(k, v, head_dim)``) has a status word if it is given one, and reports nothing without.

Layout of a head's blocks, T = page, D = head_dim.  Keys: ``[T][D / 2]`` bytes, the even channel in the low nibble, then ``[T][D / 16]``
scales.  Values by pairs of tokens: ``[T / 2][D]`` bytes, byte c channel c of the even token in the low nibble and of the odd one in
the high nibble, then ``[T / 2][D / 16][2]`` scales.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native

_KIND = {torch.float16: 1, torch.bfloat16: 2}
PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
_MOST_TOKENS = (1 << 31) - 1024
_MOST_HEADS = 1024                                       # of rows that are appended or read back


class PagedCache:
    """``k`` and ``v``: uint8 [pages, kv_heads, page * (D / 2 + D / 16)], contiguous and 16-byte aligned."""
    __slots__ = ("k", "v", "pages", "kv_heads", "page", "head_dim", "device", "status", "args", "status_ptr")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, head_dim: int, status: Optional[native.StatusWord] = None):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"PagedCache: head_dim is one of {HEAD_DIMS}")
        shape, device = k.shape, k.device
        if not (len(shape) == 3 and shape == v.shape and k.dtype is torch.uint8 and v.dtype is torch.uint8 and device == v.device
                and k.is_contiguous() and v.is_contiguous()):
            raise ValueError("PagedCache: k and v are byte buffers [pages, kv_heads, bytes] of one shape and device")
        pages, kv_heads, size = shape
        token = head_dim // 2 + head_dim // 16
        page = size // token
        if not (page in PAGES and page * token == size and pages >= 1 and kv_heads >= 1):
            raise ValueError(f"PagedCache: a block holds {PAGES} tokens of {token} bytes")
        k_at, v_at = k.data_ptr(), v.data_ptr()
        if (k_at | v_at) & 15:
            raise ValueError("PagedCache: buffers start on a 16-byte boundary")
        if status is not None and status.t.device != device:
            raise ValueError("PagedCache: status on the buffers' device")
        self.k, self.v, self.pages, self.kv_heads, self.page, self.head_dim = k, v, pages, kv_heads, page, head_dim
        self.device, self.status = device, status
        # what every call hands to the library
        self.args = (k_at, v_at, pages, kv_heads, page, head_dim)
        self.status_ptr = None if status is None else status.t.data_ptr()

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda") -> "PagedCache":
        if not (page in PAGES and head_dim in HEAD_DIMS and pages >= 1 and kv_heads >= 1):
            raise ValueError(f"PagedCache: pages of {PAGES} tokens, heads of {HEAD_DIMS} channels")
        k, v = (torch.zeros(pages, kv_heads, page * (head_dim // 2 + head_dim // 16), dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, head_dim, native.StatusWord(device))

    def check(self) -> None:
        """Raise if a call on this cache met an index out of range, a number that is not finite or a wait that ran out (a cache without a
        status word knows of none)."""
        if self.status is not None:
            self.status.check()


def rope_table(positions: int, freqs: torch.Tensor) -> torch.Tensor:
    """Cosines and sines of ``position * freqs`` (``models.oracle.rope_frequencies``), fp32 [positions, 2 * len(freqs)], for ``append``.
    The angles are formed and reduced in 64 bits."""
    a = torch.arange(positions, dtype=torch.float64, device=freqs.device)[:, None] * freqs.double()
    return torch.cat([a.cos(), a.sin()], 1).float()


def _batch(cache: PagedCache, total: int, table: torch.Tensor, lengths: torch.Tensor, cu: Optional[torch.Tensor], name: str) -> tuple:
    """Checks a batch's metadata: what the library takes of it, the number of sequences next to last."""
    dev = cache.device
    if table.dtype is not torch.int32 or table.dim() != 2 or table.device != dev or not table.is_contiguous():
        raise ValueError(f"{name}: table is int32 [S, W] on the cache's device")
    S, width = table.shape
    if S and not 0 < width * cache.page <= _MOST_TOKENS:
        raise ValueError(f"{name}: a table " + ("of more than 2^31 - 1024 tokens" if width else "without pages"))
    if lengths.dtype is not torch.int32 or lengths.shape != (S,) or lengths.device != dev or not lengths.is_contiguous():
        raise ValueError(f"{name}: lengths is int32 [{S}] on the cache's device")
    if cu is None:
        if total > S:
            raise ValueError(f"{name}: {total} rows of {S} sequences need cu")
        return table.data_ptr(), width, lengths.data_ptr(), None, S, total
    if cu.dtype is not torch.int32 or cu.shape != (S + 1,) or cu.device != dev or not cu.is_contiguous():
        raise ValueError(f"{name}: cu is int32 [{S + 1}] on the cache's device")
    return table.data_ptr(), width, lengths.data_ptr(), cu.data_ptr(), S, total


def _rows3(cache: PagedCache, x: torch.Tensor, total: int, heads: Optional[int], dtype, name: str) -> Tuple[int, int, int]:
    """Address, row and head strides of rows of heads [total, heads, D]."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != total or (heads is not None and shape[1] != heads) or shape[2] != cache.head_dim:
        raise ValueError(f"{name}: [{total}, {heads or 'heads'}, {cache.head_dim}], got {tuple(shape)}")
    if x.dtype is not dtype or x.device != cache.device:
        raise ValueError(f"{name}: {dtype} on the cache's device")
    row, head, one = x.stride()
    at = x.data_ptr()
    if one != 1 or row & 7 or head & 7 or row < 0 or head < 0 or at & 15:
        raise ValueError(f"{name}: channels contiguous, rows of heads on 16-byte boundaries")
    return at, row, head


def _end(at: tuple, x: torch.Tensor) -> int:
    """Address behind rows of heads of 16-bit numbers (``_rows3``)."""
    rows, heads, D = x.shape
    return at[0] + 2 * ((rows - 1) * at[1] + (heads - 1) * at[2] + D)


def _overlap(rows: int, heads: int, row: int, head: int, D: int) -> bool:
    """Whether rows of heads of these strides lie over each other."""
    if (heads < 2 or head >= D) and (rows < 2 or row >= (heads - 1) * head + D):
        return False                                     # the usual case: one row behind the other
    if (heads > 1 and head < D) or (rows > 1 and row < D):
        return True
    # two of them meet where some rows are as far apart as some heads, to less than D
    return any(1 <= i < rows and abs(i * row - j * head) < D for j in range(1, heads) for i in (j * head // row, j * head // row + 1))


def _meets(at: tuple, x: torch.Tensor, start: int, size: int) -> bool:
    """Whether ``size`` bytes from ``start`` on lie over rows of heads (not between two of them)."""
    if start >= _end(at, x) or start + size <= at[0]:
        return False
    pitch, extent = 2 * at[1], _end(at, x[:1]) - at[0]
    gap = (start - at[0]) % pitch if pitch else 0
    return gap < extent or gap + size > pitch


def _like(x: torch.Tensor, at: tuple) -> torch.Tensor:
    """Contiguous rows of x's shape and type (``empty_like`` takes the least host time, where x is contiguous itself)."""
    rows, heads, D = x.shape
    if at[2] == D and at[1] == heads * D:
        return torch.empty_like(x)
    return torch.empty(rows, heads, D, dtype=x.dtype, device=x.device)


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
           cu: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
           interleaved: bool = True, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Store keys and values [total, kv_heads, D] (f16 / bf16, any row and head strides) at their positions; ``rope`` (``rope_table``;
    its width a multiple of 32, at most D) rotates the last channels of every key, in neighbouring pairs or, with ``interleaved`` false, the
    first half with the second.  ``q`` [total, heads, D] is rotated alike and returned (contiguous, in its own type; ``q_out`` shares no memory
    with queries, keys and values).  At most 1,024 heads of each.

    A key is rotated exactly and rounded once, to the 4-bit grid.  A NaN is stored as zero and an infinity as the largest number,
    and both are reported.  A page that is written belongs to one sequence, once: two sequences (or calls in flight at one time) may share only
    pages that neither writes."""
    if k.dim() != 3:
        raise ValueError("append: k is [total, kv_heads, D]")
    total, dt = k.shape[0], k.dtype
    if dt not in _KIND:
        raise ValueError("append: f16 or bf16")
    batch = _batch(cache, total, table, lengths, cu, "append")
    k_at = _rows3(cache, k, total, cache.kv_heads, dt, "append: k")
    v_at = _rows3(cache, v, total, cache.kv_heads, dt, "append: v")
    angles = (None, 0, 0)
    if rope is not None:
        if rope.dtype is not torch.float32 or rope.dim() != 2 or not rope.is_contiguous() or rope.device != cache.device or not rope.shape[0] \
                or rope.data_ptr() & 15:
            raise ValueError("append: rope is fp32 [positions, channels] on the cache's device")
        positions, rd = rope.shape
        if rd % 32 or not 0 < rd <= cache.head_dim:
            raise ValueError("append: rope rotates a multiple of 32 channels, at most head_dim")
        angles = (rope.data_ptr(), positions, rd)
    q_at, out_at = (None, 0, 0, 0), None
    if cache.kv_heads > _MOST_HEADS or (q is not None and q.dim() == 3 and q.shape[1] > _MOST_HEADS):
        raise ValueError("append: at most 1,024 heads and kv heads")
    if q is not None:
        q_at = (*_rows3(cache, q, total, None, dt, "append: q"), q.shape[1])
        if q_out is None:
            q_out = _like(q, q_at)
            out_at = q_out.data_ptr()
        elif not (q_out.shape == q.shape and q_out.dtype == dt and q_out.device == q.device and q_out.is_contiguous() and q_out.data_ptr() % 16 == 0):
            raise ValueError("append: q_out is contiguous, of q's shape and type")
        else:
            out_at, size = q_out.data_ptr(), 2 * q_out.numel()
            for at, x, name in ((q_at, q, "q"), (k_at, k, "k"), (v_at, v, "v")):
                if size and _meets(at, x, out_at, size):
                    raise ValueError(f"append: q_out overlaps {name}")
    elif q_out is not None:
        raise ValueError("append: q_out without q")
    if total and batch[4]:
        native.launch("tf_paged_append", k, *q_at, *k_at, *v_at, _KIND[dt], out_at, *cache.args, *batch, *angles, 1 if interleaved else 0, cache.status_ptr)
    return q_out


def read(cache: PagedCache, total: int, table: torch.Tensor, lengths: torch.Tensor, cu: Optional[torch.Tensor] = None
         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of a batch's rows out of the cache, bf16 [total, kv_heads, D] each (exact; rows behind the last sequence's are zeros)."""
    if cache.kv_heads > _MOST_HEADS:
        raise ValueError("read: at most 1,024 heads")
    batch = _batch(cache, total, table, lengths, cu, "read")
    k = (torch.empty if batch[4] else torch.zeros)(total, cache.kv_heads, cache.head_dim, dtype=torch.bfloat16, device=cache.device)
    v = torch.empty_like(k) if batch[4] else k.clone()
    if total and batch[4]:
        native.launch("tf_paged_read", k, k.data_ptr(), v.data_ptr(), *cache.args, *batch, cache.status_ptr)
    return k, v


_WORK = {}


def _workspace(*shape: int) -> int:
    """Floats of workspace of a call (a function of its sizes alone)."""
    if len(_WORK) > 4096:
        _WORK.clear()
    n = _WORK[shape] = native.lib().tf_paged_attention_workspace(*shape)
    return n


def attention(cache: PagedCache, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, cu: Optional[torch.Tensor] = None, *,
              scale: Optional[float] = None, window: int = 0, first: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of ``q`` [total, heads, D] (f16 / bf16; heads a multiple of kv_heads) over the sequences' pages, in q's type.

    A row at position p sees the keys ``max(first[s], p - window + 1) .. p`` (window 0: no lower bound; ``first`` int32 [S]: none).  ``sink``
    fp32 [heads]: a logit per head that takes part in the softmax and has no value.  A row without keys gives zeros.  ``scale`` is positive, by
    default ``D ** -0.5``; logits are fp32 numbers, and a row whose logits pass their range gives NaN.  ``out`` (rows and heads at any distance that keeps them apart) may be ``q`` itself, and shares no memory with it
    otherwise.  With ``return_lse`` also the logarithm of every row's softmax sum, fp32 [total, heads]."""
    dt = q.dtype
    if q.dim() != 3 or dt not in _KIND:
        raise ValueError("attention: q is [total, heads, D] in f16 or bf16")
    total, heads, D = q.shape
    batch = _batch(cache, total, table, lengths, cu, "attention")
    q_at = _rows3(cache, q, total, None, dt, "attention: q")
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"attention: {heads} heads over {cache.kv_heads} kv heads")
    if scale is None:
        scale = D ** -0.5
    if not 0.0 < scale <= 1e30:
        raise ValueError("attention: scale is positive")
    if not 0 <= window < 1 << 31:
        raise ValueError("attention: window")
    S = batch[4]
    if first is not None and (first.dtype is not torch.int32 or first.shape != (S,) or not first.is_contiguous() or first.device != cache.device):
        raise ValueError(f"attention: first is int32 [{S}] on the cache's device")
    if sink is not None and (sink.dtype is not torch.float32 or sink.shape != (heads,) or not sink.is_contiguous() or sink.device != cache.device):
        raise ValueError(f"attention: sink is fp32 [{heads}] on the cache's device")
    if out is None:
        out = _like(q, q_at)
        out_at = (out.data_ptr(), heads * D, D)
    else:
        out_at = _rows3(cache, out, total, heads, dt, "attention: out")
        if _overlap(total, heads, out_at[1], out_at[2], D):
            raise ValueError("attention: rows of out overlap")
        if out_at != q_at and out_at[0] < _end(q_at, q) and q_at[0] < _end(out_at, out):
            pitch, extent = 2 * q_at[1], 2 * ((heads - 1) * q_at[2] + D)     # (columns of one buffer, as a fused projection has them)
            gap = (out_at[0] - q_at[0]) % pitch if pitch else 0
            if out_at[1] != q_at[1] or gap < extent or gap + 2 * ((heads - 1) * out_at[2] + D) > pitch:
                raise ValueError("attention: out overlaps q")
    lse = torch.empty(total, heads, dtype=torch.float32, device=cache.device) if return_lse else None
    if total and S:
        shape = (total, S, heads, cache.kv_heads, D, table.shape[1] * cache.page)
        size = _WORK.get(shape)
        if size is None:
            size = _workspace(*shape)
        work = torch.empty(size, dtype=torch.float32, device=cache.device) if size else None
        native.launch("tf_paged_attention", q, *q_at, heads, _KIND[dt], *out_at, None if lse is None else lse.data_ptr(), *cache.args, *batch,
                      scale, window, None if first is None else first.data_ptr(), None if sink is None else sink.data_ptr(),
                      None if work is None else work.data_ptr(), cache.status_ptr)
        if size:
            native.LAUNCHES[0] += 1                      # the parts of items that were cut are joined in a launch of its own
    return (out, lse) if return_lse else out
