"""Paged 4-bit KV cache (``ops/paged.py``): append with rotation, reading back, attention; against their formulas in 64 bits."""
import math
import pathlib
import subprocess

import pytest
import torch

from titanic_flash_41_b200.formats import codecs
from titanic_flash_41_b200.models import oracle
from titanic_flash_41_b200.ops import fp4, native, paged

DEV = "cuda"


# ------------------------------------------------------------------------------------------ the formulas
def kv4(x):
    """x [..., D] in 64 bits -> what its cached form stands for: blocks of 16, scale e4m3(max(amax / 6, 2^-6))."""
    b = x.double().reshape(-1, 16)
    grid = torch.tensor([(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64, device=x.device)
    s = nearest(b.abs().amax(1) / 6, grid)[:, None]
    vals = torch.tensor(codecs.E2M1_VALUES, dtype=torch.float64, device=x.device)
    return (nearest((b / s).abs(), vals) * s * torch.sign(b)).view(x.shape)


def nearest(a, grid):
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    return grid[torch.where(lo % 2 == 0, lo, hi)]


def rotate(x, table, pos, interleaved):
    x = x.double().clone()
    half = table.shape[1] // 2
    cos, sin = table[pos].double()[:, None].split(half, -1)
    t0 = x.shape[-1] - 2 * half
    i = torch.arange(half, device=x.device)
    a, b = (t0 + 2 * i, t0 + 2 * i + 1) if interleaved else (t0 + i, t0 + half + i)
    x[..., a], x[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    return x


class Batch:
    """Sequences with their page tables over one cache, every byte of which was poisoned (scales that are NaN) before."""

    def __init__(self, rows, lengths, kv, D, page, dtype=torch.bfloat16, seed=0, spare=2):
        self.rows, self.lens, self.page, self.dtype = rows, lengths, page, dtype
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        need = [-(-max(n, 0) // page) for n in lengths]
        width = max(max(need), 1) + 1
        pages = sum(need) + spare
        self.cache = paged.PagedCache.allocate(pages, kv, D, page, DEV)
        self.cache.k.fill_(255)
        self.cache.v.fill_(255)
        order = torch.randperm(pages, generator=self.gen, device=DEV).int()
        self.table = torch.full((len(rows), width), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        self.cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=DEV)
        self.total = sum(rows)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEV).to(self.dtype)

    def fill(self):
        """Random keys and values at every position; what the cache then holds, per sequence, in 64 bits."""
        c = self.cache
        n = sum(max(x, 0) for x in self.lens)
        cu = torch.tensor([sum(max(x, 0) for x in self.lens[:i]) for i in range(len(self.lens) + 1)], dtype=torch.int32, device=DEV)
        k, v = self.randn(n, c.kv_heads, c.head_dim), self.randn(n, c.kv_heads, c.head_dim)
        if n:
            paged.append(c, k, v, self.table, self.lengths.clamp(min=0), cu)
        ends = cu.tolist()
        return [(kv4(k[a:b]), kv4(v[a:b])) for a, b in zip(ends, ends[1:])]


def attend(b, kv, q, scale, window=0, first=None, sink=None):
    """Per row: output, its softmax's logarithm, and what ``check`` needs to say how far rounding may take both."""
    D, H = q.shape[2], q.shape[1]
    grp = H // b.cache.kv_heads
    outs, lses, spreads, logits, floors = [], [], [], [], []
    at = 0
    for i, (n, length) in enumerate(zip(b.rows, b.lens)):
        k, v = kv[i]
        x = q[at:at + n].double()
        at += n
        pos = torch.arange(length - n, length, device=DEV)
        key = torch.arange(k.shape[0], device=DEV)
        seen = key[None] <= pos[:, None]
        if window:
            seen &= key[None] > pos[:, None] - window
        if first is not None:
            seen &= key[None] >= int(first[i])
        kk, vv = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
        s = torch.einsum("nhd,lhd->nhl", x, kk) * scale
        size = torch.einsum("nhd,lhd->nhl", x.abs(), kk.abs()) * scale
        s = s.masked_fill(~seen[:, None], -math.inf)
        lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((n, H), -math.inf, dtype=torch.float64, device=DEV)
        if sink is not None:
            lse = torch.logaddexp(lse, sink.double()[None])
        p = torch.exp(s - lse[..., None]).nan_to_num(0.0)
        outs.append(torch.einsum("nhl,lhd->nhd", p, vv))
        # p is held relative to a maximum m that the row's largest logit is not below, so the sum of the p is at least 1; a p below 2^-14 is a
        # subnormal f16 and off by up to 2^-25 whatever its size: that adds up to 2^-25 |v| a key to the numerator, and no more to the quotient
        spreads.append(torch.einsum("nhl,lhd->nhd", p, vv.abs()))
        floors.append((seen.sum(-1)[:, None] * 2.0 ** -25 * (vv.abs().amax() if k.shape[0] else 0)).expand(n, H))
        # (a query's elements below 2^-14 of the row's largest keep 2^-25 of it)
        small = D * 2.0 ** -2 * x.abs().amax(-1) * (k.abs().amax() if k.shape[0] else 0) * scale / (D + 2)
        logits.append(small + (size.masked_fill(~seen[:, None], 0.0).amax(-1) if k.shape[0] else 0))
        lses.append(lse)
    return [torch.cat(x) for x in (outs, lses, spreads, logits, floors)]


def check(b, kv, q, out, lse=None, **more):
    """A logit is a sum of D exact products in fp32 and a multiplication: off by at most e = (D + 2) 2^-23 sum |q k| scale, and its exponential by
    that and 2^-21 (the unit's error and that of the subtraction of logits below 8).  A probability is rounded to f16 (2^-11; below
    2^-14 of the largest by 2^-25), the sums to fp32, the output to its type.  Both the numerator and the sum carry the logits' error."""
    scale = more.pop("scale", q.shape[2] ** -0.5)
    want, wlse, spread, size, floor = attend(b, kv, q, scale, **more)
    length = max(max(b.lens), 1)
    e = (q.shape[2] + 2) * 2.0 ** -23 * size + 2.0 ** -21 + 2.0 ** -22 * size
    bound = torch.finfo(out.dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2 * e + length * 2.0 ** -23)[..., None] * spread + floor[..., None] + 2.0 ** -24
    diff = (out.double() - want).abs()
    assert torch.isfinite(out).all() and (diff <= bound).all(), float((diff - bound).max())
    if lse is not None:
        none = torch.isinf(wlse)
        assert torch.equal(torch.isneginf(lse), none)
        off = (lse.double() - wlse)[~none].abs()
        assert (off <= (e + length * 2.0 ** -23 + 2.0 ** -22 * wlse.abs().nan_to_num(posinf=0.0) + 2.0 ** -20)[~none]).all(), float(off.max())


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def cpu_batch(total=3):
    c = paged.PagedCache.allocate(4, 2, 64, 16, "cpu")
    return (c, torch.zeros(total, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
            torch.zeros(3, dtype=torch.int32))


def test_refusals_of_caches():
    for page, D in ((24, 64), (8, 64), (512, 64), (16, 96), (16, 512)):
        with pytest.raises(ValueError, match="PagedCache"):
            paged.PagedCache.allocate(4, 2, D, page, "cpu")
    k = torch.zeros(4, 2, 16 * 36, dtype=torch.uint8)
    for a, b, D in ((k, k[:, :1], 64), (k, k.to(torch.int8), 64), (k[:, :, :-1], k[:, :, :-1], 64), (k, k, 128), (k[:, ::2], k[:, ::2], 64),
                    (k.view(-1)[8:8 + 576].view(1, 1, 576), k.view(-1)[:576].view(1, 1, 576), 64), (k[:0], k[:0], 64)):
        with pytest.raises(ValueError, match="PagedCache"):
            paged.PagedCache(a, b, D)


def test_refusals_of_status_words():
    """A report is a write through the word's address: one on another device is none that a kernel may write."""
    k = torch.zeros(4, 2, 16 * 36, dtype=torch.uint8)
    word = native.StatusWord("cpu")
    assert paged.PagedCache(k, k.clone(), 64, word).status is word
    word.t = word.t.to("meta")
    with pytest.raises(ValueError, match="PagedCache: status"):
        paged.PagedCache(k, k.clone(), 64, word)


def test_refusals_of_append_and_read():
    c, x, table, lengths, cu = cpu_batch()
    rope = torch.zeros(8, 32)
    ok = dict(q=x, rope=rope)
    for args, kw, what in (
            ((x.float(), x.float(), table, lengths, cu), {}, "f16 or bf16"),
            ((x[:, :1], x, table, lengths, cu), {}, "append: k"),
            ((x, x[:2], table, lengths, cu), {}, "append: v"),
            ((x, x.half(), table, lengths, cu), {}, "append: v"),
            ((x, x, table.long(), lengths, cu), {}, "table"),
            ((x, x, table.t(), lengths, cu), {}, "table"),
            ((x, x, table, lengths[:1], cu), {}, "lengths"),
            ((x, x, table, lengths, cu[:2]), {}, "cu"),
            ((x, x, table, lengths, None), {}, "need cu"),
            ((x, x, table, lengths, cu), dict(rope=rope[:, :16].contiguous()), "multiple of 32"),
            ((x, x, table, lengths, cu), dict(rope=torch.zeros(8, 128)), "multiple of 32"),
            ((x, x, table, lengths, cu), dict(rope=rope.double()), "rope is fp32"),
            ((x, x, table, lengths, cu), dict(q=x[:, :, :32]), "append: q"),
            ((x, x, table, lengths, cu), dict(q=x, q_out=x.half()), "q_out"),
            ((x, x, table, lengths, cu), dict(q_out=x), "q_out without q"),
            ((torch.zeros(3, 2, 68, dtype=torch.bfloat16)[:, :, 4:], x, table, lengths, cu), {}, "16-byte"),
            ((x, x, table, lengths, cu), ok, "CUDA")):
        with pytest.raises(ValueError, match=what):
            paged.append(c, *args, **kw)
    with pytest.raises(ValueError, match="need cu"):
        paged.read(c, 3, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        paged.read(c, 3, table, lengths, cu)


def test_refusals_of_more_heads_than_a_row_may_have():
    x = torch.zeros(1, 1025, 64, dtype=torch.float16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for kv, heads, what in ((1024, 1024, "CUDA"), (1025, 1, "1,024 heads"), (1, 1025, "1,024 heads")):
        c = paged.PagedCache.allocate(1, kv, 64, 16, "cpu")
        with pytest.raises(ValueError, match=what):
            paged.append(c, x[:, :kv], x[:, :kv], table, lengths, q=x[:, :heads])
        with pytest.raises(ValueError, match=what if kv > 1 else "CUDA"):
            paged.read(c, 1, table, lengths)


def test_refusals_of_attention():
    c, x, table, lengths, cu = cpu_batch()
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    for args, kw, what in (
            ((q.float(), table, lengths, cu), {}, "f16 or bf16"),
            ((q[:, :3], table, lengths, cu), {}, "kv heads"),
            ((q[:, :, :32], table, lengths, cu), {}, "attention: q"),
            ((q.transpose(0, 1).contiguous().transpose(1, 2), table, lengths, cu), {}, "attention: q"),
            ((q, table, lengths, None), {}, "need cu"),
            ((q, table[:, :0], lengths, cu), {}, "without pages"),
            ((q, table, lengths, cu), dict(scale=0.0), "scale"),
            ((q, table, lengths, cu), dict(scale=-1.0), "scale"),
            ((q, table, lengths, cu), dict(scale=math.nan), "scale"),
            ((q, table, lengths, cu), dict(scale=math.inf), "scale"),
            ((q, table, lengths, cu), dict(window=-1), "window"),
            ((q, table, lengths, cu), dict(first=lengths[:1]), "first"),
            ((q, table, lengths, cu), dict(sink=torch.zeros(3)), "sink"),
            ((q, table, lengths, cu), dict(sink=torch.zeros(4, dtype=torch.float16)), "sink"),
            ((q, table, lengths, cu), dict(out=q.bfloat16()), "attention: out"),
            ((q, table, lengths, cu), {}, "CUDA")):
        with pytest.raises(ValueError, match=what):
            paged.attention(c, *args, **kw)


def test_rope_table_is_the_frequencies_angles():
    f = oracle.rope_frequencies(64, 160000.0, 16.0)
    t = paged.rope_table(70000, f)
    a = torch.arange(70000, dtype=torch.float64)[:, None] * f.double()
    assert t.shape == (70000, 64) and t.dtype == torch.float32
    assert (t.double() - torch.cat([a.cos(), a.sin()], 1)).abs().max() <= 2.0 ** -24


def test_divisions_are_exact(tmp_path):
    """The kernels' division by a multiplication (``csrc/divide.h``): append divides by up to 1,024 heads x 8 blocks, reading back by twice as much;
    around every multiple that a CTA of 32 rows meets (a quotient that is one too large is so at its multiple's end first), and around larger ones."""
    src = tmp_path / "divide.cc"
    src.write_text("""
#include "divide.h"
#include <stdio.h>
int main() {
  long bad = 0;
  for (int n = 1; n <= 16384; ++n) {
    const Divide by(n);
    auto look = [&](long i) {
      int rest;
      if (i < 0 || i + n >= 1l << 31) return;
      if (by((int)i, &rest) != i / n || rest != i % n) ++bad;
      const int k = by.small((int)i, &rest);
      if (n <= 8192 && i < 33l * n ? k != i / n || rest != i % n : k < i / n) ++bad;
    };
    for (long x = 0; x <= 64; ++x)
      for (long d = -1; d <= 1; ++d) look(x * n + d);
    for (long x = 128; x * n < 1l << 31; x *= 2)
      for (long d = -1; d <= 1; ++d) look(x * n + d);
  }
  printf("%ld", bad);
}
""")
    csrc = pathlib.Path(paged.__file__).resolve().parent.parent / "csrc"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(csrc), "-o", str(tmp_path / "divide"), str(src)], check=True)
    assert subprocess.run([str(tmp_path / "divide")], check=True, capture_output=True, text=True).stdout == "0"


# ------------------------------------------------------------------------------------------ append
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page,rope,interleaved", [(128, 64, 64, True), (64, 16, 64, False), (128, 32, 32, False), (128, 16, 128, False),
                                                     (64, 256, 32, True), (64, 128, 0, True)])
def test_append_rotates_and_rounds_once(dtype, D, page, rope, interleaved):
    b = Batch([1, 7, 70, 2, 1], [1, 8, 300, 35, 64], 2, D, page, dtype, seed=D + page + rope)
    h, kv = 6, 2
    qkv = b.randn(b.total + 2, (h + 2 * kv) * D)              # (two rows behind the last sequence)
    qkv[:, h * D:] *= torch.exp(2 * torch.randn(qkv.shape[0], 2 * kv * D, generator=b.gen, device=DEV)).to(dtype)
    q, k, v = (qkv[:, a * D:e * D].view(-1, e - a, D) for a, e in ((0, h), (h, h + kv), (h + kv, h + 2 * kv)))
    table = paged.rope_table(320, oracle.rope_frequencies(rope, 160000.0).to(DEV)) if rope else None
    kb, vb = b.cache.k.clone(), b.cache.v.clone()
    q_out = torch.full((b.total + 2, h, D), 3.0, dtype=dtype, device=DEV)
    assert paged.append(b.cache, k, v, b.table, b.lengths, b.cu, q=q, rope=table, interleaved=interleaved, q_out=q_out) is q_out
    b.cache.check()
    pos = torch.cat([torch.arange(l - n, l, device=DEV) for n, l in zip(b.rows, b.lens)])
    turned = [rotate(x[:b.total], table, pos, interleaved) if rope else x[:b.total].double() for x in (q, k)]
    kk, vv = paged.read(b.cache, b.total, b.table, b.lengths, b.cu)
    assert torch.equal(kk.double(), kv4(turned[1]))           # bit for bit: one rounding of the exact rotation
    assert torch.equal(vv.double(), kv4(v[:b.total]))
    # a query is rounded to its type, from fp32 products and a sum
    off = (q_out[:b.total].double() - turned[0]).abs()
    assert (off <= torch.finfo(dtype).eps / 2 * turned[0].abs() + 2.0 ** -22 * q[:b.total].double().abs().amax(-1, keepdim=True)).all()
    assert (q_out[b.total:] == 3.0).all()
    # all else in the pool is as it was
    seq = torch.repeat_interleave(torch.arange(len(b.rows), device=DEV), torch.tensor(b.rows, device=DEV))
    at, slot = b.table[seq, pos // page].long(), pos % page
    vals = page * D // 2
    for buf, old, name in ((b.cache.k, kb, "k"), (b.cache.v, vb, "v")):
        mine = torch.zeros(buf.shape[0], page, dtype=torch.bool, device=DEV)
        mine[at, slot] = True
        if name == "k":
            keep = [(buf[..., :vals].view(-1, kv, page, D // 2), old[..., :vals].view(-1, kv, page, D // 2)),
                    (buf[..., vals:].view(-1, kv, page, D // 16), old[..., vals:].view(-1, kv, page, D // 16))]
            for new, was in keep:
                assert torch.equal(new.transpose(1, 2)[~mine], was.transpose(1, 2)[~mine])
        else:
            for odd in (0, 1):
                new, was = (x[..., :vals].view(-1, kv, page // 2, D) >> 4 * odd & 15 for x in (buf, old))
                assert torch.equal(new.transpose(1, 2)[~mine[:, odd::2]], was.transpose(1, 2)[~mine[:, odd::2]])
                new, was = (x[..., vals:].view(-1, kv, page // 2, D // 16, 2)[..., odd] for x in (buf, old))
                assert torch.equal(new.transpose(1, 2)[~mine[:, odd::2]], was.transpose(1, 2)[~mine[:, odd::2]])


@pytest.mark.gpu
def test_tokens_one_by_one_equal_the_prompt_at_once():
    """Odd and even tokens of a pair written by different calls, and rows that are written again (a rejected draft)."""
    D, kv, n = 128, 3, 37
    a, b = (Batch([n], [n], kv, D, 16, seed=4) for _ in range(2))
    b.table = a.table
    k, v = a.randn(n, kv, D), a.randn(n, kv, D)
    paged.append(a.cache, k, v, a.table, a.lengths, a.cu)
    for i in range(n):
        if i % 5 == 0:                                        # a draft of two tokens that is rejected
            junk = torch.full((2, kv, D), 9.0, device=DEV, dtype=k.dtype)
            if i + 2 <= n:
                paged.append(b.cache, junk, junk, b.table, torch.tensor([i + 2], dtype=torch.int32, device=DEV), torch.tensor([0, 2], dtype=torch.int32, device=DEV))
        paged.append(b.cache, k[i:i + 1], v[i:i + 1], b.table, torch.tensor([i + 1], dtype=torch.int32, device=DEV))
    for x, y in zip(paged.read(a.cache, n, a.table, a.lengths, a.cu), paged.read(b.cache, n, b.table, a.lengths, a.cu)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_numbers_at_the_borders_and_beyond_the_format():
    """Midpoints of both grids, their neighbours, the smallest and the largest scales; NaN and infinities are tamed and reported."""
    b = Batch([64], [64], 1, 64, 64, torch.float16)
    x = torch.zeros(64, 1, 64, dtype=torch.float16, device=DEV)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    for i in range(48):
        s = (8 + i % 8) * 2.0 ** (i // 8 - 6)                 # an e4m3 number
        for j in range(4):
            x[i, 0, 16 * j] = 6 * s
            x[i, 0, 16 * j + 1:16 * j + 8] = mids * s * (1 + (j - 1) * 2.0 ** -10) if j < 3 else -mids * s
    for i in range(8):                                        # amax / 6 next to a midpoint of the scales
        t = torch.tensor(6 * (8.5 + i) / 8 * 2.0 ** -3, device=DEV).half()
        x[48 + i, 0, ::16] = torch.stack([t, torch.nextafter(t, t * 2), torch.nextafter(t, t * 0), -t])
    x[57, 0, :3] = torch.tensor([65504.0, 3000.0, -2688.0])
    x[58, 0, :3] = torch.tensor([2.0 ** -24, 2.0 ** -8, -(2.0 ** -9)])
    paged.append(b.cache, x, x, b.table, b.lengths, b.cu)
    b.cache.check()
    for got in paged.read(b.cache, 64, b.table, b.lengths, b.cu):
        assert torch.equal(got.double(), kv4(x))
    x[3, 0, 5], x[9, 0, 20], x[10, 0, 40] = math.nan, math.inf, -math.inf
    paged.append(b.cache, x, x, b.table, b.lengths, b.cu)
    with pytest.raises(native.NativeError, match="nonfinite"):
        b.cache.check()
    y = x.double()
    y[3, 0, 5], y[9, 0, 20], y[10, 0, 40] = 0.0, 1e30, -1e30
    for got in paged.read(b.cache, 64, b.table, b.lengths, b.cu):
        assert torch.equal(got.double(), kv4(y))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [745, 1023])
def test_many_heads_read_back(kv):
    """Rows enough for 32 of them a CTA, of numbers of heads whose blocks a bare multiplication does not count exactly; one page for all tokens."""
    b = Batch([16], [16], kv, 128, 16)
    cached = b.fill()
    n = 32 * 4 * 148
    table = b.table[:, :1].expand(1, n // 16).contiguous()
    for got, want in zip(paged.read(b.cache, n, table, torch.full_like(b.lengths, n), torch.tensor([0, n], dtype=torch.int32, device=DEV)), cached[0]):
        assert (got.view(-1, 16, kv, 128) == want.to(torch.bfloat16)).all()
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[3, 0, 2], [700], []])
def test_rows_of_no_sequence_read_back_as_zeros(rows):
    """A captured graph has as many rows as its largest batch; memory that held NaN before."""
    b = Batch(rows, [n + 20 for n in rows], 2, 64, 16) if rows else Batch([0], [0], 2, 64, 16)
    cached = b.fill()
    if not rows:
        b.table, b.lengths, b.cu = b.table[:0], b.lengths[:0], b.cu[:1]
    total = b.total + 5
    old = [torch.full((total, 2, 64), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    del old
    got = paged.read(b.cache, total, b.table, b.lengths, b.cu)
    b.cache.check()
    for i, x in enumerate(got):
        want = [c[i][20:] for c, n in zip(cached, rows)]
        assert torch.equal(x.double(), torch.cat(want + [torch.zeros(5, 2, 64, dtype=torch.float64, device=DEV)]))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [0.05, 0.01, 0.002, 100.0, 3000.0])
def test_numbers_far_from_one(size):
    """Blocks below the smallest scale and above the largest one; a caller's power of two on keys and values comes out of scale and output again."""
    b, c = (Batch([40], [40], 2, 128, 64, seed=7) for _ in range(2))
    k, v, q = (b.randn(40, n, 128) * size for n in (2, 2, 8))
    paged.append(b.cache, k, v, b.table, b.lengths, b.cu)
    b.cache.check()
    for got, x in zip(paged.read(b.cache, 40, b.table, b.lengths, b.cu), (k, v)):
        assert torch.equal(got.double(), kv4(x))
    check(b, [(kv4(k), kv4(v))], q, paged.attention(b.cache, q, b.table, b.lengths, b.cu))
    by = 2.0 ** -round(math.log2(size))
    paged.append(c.cache, k * by, v * by, c.table, c.lengths, c.cu)
    out = paged.attention(c.cache, q, c.table, c.lengths, c.cu, scale=128 ** -0.5 / by)
    check(c, [(kv4(k * by), kv4(v * by))], q, out, scale=128 ** -0.5 / by)
    for got, x in zip(paged.read(c.cache, 40, c.table, c.lengths, c.cu), (k, v)):
        off = (got.double() / by - x.double()).abs().view(40, 2, 8, 16)
        amax = x.double().abs().view(40, 2, 8, 16).amax(-1, keepdim=True)
        # half of the widest step (2 of 6) of a scale that is off by 2^-4 at most
        assert (off <= amax / 6 * (1 + 2.0 ** -4)).all()


@pytest.mark.gpu
def test_append_and_read_out_of_range_are_reported_and_stay_inside():
    for lens, rows, where in (([40], [3], "page of the table"), ([100], [2], "table's width"), ([1], [3], "before the first token")):
        b = Batch(rows, [min(lens[0], 40)], 2, 64, 16)
        b.lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
        if where == "page of the table":
            b.table[0, 2] = 1 << 20
        kb, vb = b.cache.k.clone(), b.cache.v.clone()
        k = b.randn(rows[0], 2, 64)
        q = paged.append(b.cache, k, k, b.table, b.lengths, b.cu, q=k)
        with pytest.raises(native.NativeError, match="bad_index"):
            b.cache.check()
        assert torch.equal(q, k)
        if where != "before the first token":
            assert torch.equal(b.cache.k, kb) and torch.equal(b.cache.v, vb)
        kk, vv = paged.read(b.cache, rows[0], b.table, b.lengths, b.cu)
        with pytest.raises(native.NativeError, match="bad_index"):
            b.cache.check()
        want = kv4(k)
        if where == "before the first token":
            want[:2] = 0
        else:
            want[:] = 0
        assert torch.equal(kk.double(), want) and torch.equal(vv.double(), want)
    b = Batch([2], [20], 2, 64, 16)                           # a position behind the table of angles
    k = b.randn(2, 2, 64)
    paged.append(b.cache, k, k, b.table, b.lengths, b.cu, rope=torch.zeros(19, 32, device=DEV))
    with pytest.raises(native.NativeError, match="bad_index"):
        b.cache.check()


# ------------------------------------------------------------------------------------------ attention
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,D,page,rows,lens", [
    (8, 1, 128, 64, [1], [1]),
    (8, 8, 64, 16, [1], [31]),
    (64, 8, 128, 64, [1], [300]),
    (16, 2, 128, 16, [1, 1, 1], [33, 1, 700]),
    (12, 4, 64, 32, [2, 0, 5, 1], [2, 0, 515, 97]),
    (16, 2, 128, 64, [4, 4], [2049, 130]),
    (24, 1, 64, 128, [1, 3], [5000, 3]),
    (5, 1, 128, 256, [3], [1000]),
    (32, 8, 128, 32, [9, 40], [9, 800]),
    (8, 2, 64, 16, [130], [130]),
    (16, 2, 128, 64, [257, 100], [1024, 100]),
    (4, 4, 128, 64, [300], [1300]),
])
def test_attention(dtype, heads, kv, D, page, rows, lens):
    b = Batch(rows, lens, kv, D, page, dtype, seed=heads + D + sum(lens))
    cached = b.fill()
    q = b.randn(b.total, heads, D) * torch.exp(torch.randn(heads, 1, generator=b.gen, device=DEV)).to(dtype)
    sink = torch.randn(heads, generator=b.gen, device=DEV)
    first = torch.tensor([(7 * i) % 40 for i in range(len(rows))], dtype=torch.int32, device=DEV)
    for more in (dict(), dict(window=1), dict(window=50, sink=sink), dict(first=first), dict(sink=sink, scale=0.3)):
        out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True, **more)
        b.cache.check()
        check(b, cached, q, out, lse, **more)
    again = paged.attention(b.cache, q, b.table, b.lengths, b.cu, sink=sink, scale=0.3)
    assert torch.equal(again, out)                            # the same bits every time


@pytest.mark.gpu
def test_rows_without_keys():
    """Sequences shorter than their rows, and keys that all lie before ``first``: zeros, and the sink's share alone."""
    b = Batch([5, 1, 40], [3, 70, 40], 2, 128, 16)
    b.lens = [3, 70, 40]
    cached = b.fill()
    q = b.randn(b.total, 4, 128)
    first = torch.tensor([0, 100, 39], dtype=torch.int32, device=DEV)
    for sink in (None, torch.randn(4, device=DEV)):
        out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, first=first, sink=sink, return_lse=True)
        check(b, cached, q, out, lse, first=first, sink=sink)
        empty = [0, 1, 5] + list(range(6, 6 + 39))
        assert not out[empty].any()
        if sink is None:
            assert torch.isneginf(lse[empty]).all()
        else:
            assert ((lse[empty] - sink).abs() <= 2.0 ** -22 * sink.abs()).all()
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_strides_rows_behind_the_last_sequence_and_pages_seen_twice(rows):
    b = Batch([rows, rows], [200, 200], 2, 128, 32)
    cached = b.fill()
    b.table[1] = b.table[0]                                   # two sequences over the same pages
    cached[1] = cached[0]
    wide = b.randn(2 * rows + 3, 6, 256)
    q = wide[:, 1:5, 64:192]
    out = torch.full((2 * rows + 3, 9, 128), 5.0, device=DEV, dtype=b.dtype)
    got = paged.attention(b.cache, q, b.table, b.lengths, b.cu, out=out[:, 2:6])
    assert got.data_ptr() == out[:, 2:6].data_ptr()
    check(b, cached, q[:2 * rows], out[:2 * rows, 2:6])
    out[:2 * rows, 2:6] = 5.0
    assert (out == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,length", [(1, 100), (1, 9000), (3, 9000), (40, 100), (40, 9000)])
def test_sinks_at_the_ends_of_the_numbers(rows, length):
    """Infinite ones and the type's ends, in every form of the kernels, for rows with keys and (the second sequence's) without."""
    b = Batch([rows, rows], [length, 0], 1, 64, 16)
    cached = b.fill()
    q = b.randn(2 * rows, 8, 64)
    top = torch.finfo(torch.float32)
    sink = torch.tensor([math.inf, top.max, 1000.0, -math.inf, top.min, -1000.0, 0.5, math.nan], device=DEV)
    plain, plse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True)
    out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, sink=sink, return_lse=True)
    b.cache.check()
    assert not out[:rows, :3].any() and torch.equal(lse[:rows, :2], sink[:2].expand(rows, 2))       # the sink takes all
    assert ((lse[:rows, 2] - 1000.0).abs() <= 2.0 ** -22 * 1000.0).all()
    assert torch.equal(out[:rows, 3:6], plain[:rows, 3:6]) and torch.equal(lse[:rows, 3:6], plse[:rows, 3:6])      # and nothing
    assert torch.isnan(out[:, 7]).all() and torch.isnan(lse[:, 7]).all()
    assert not out[rows:, :7].any() and torch.equal(lse[rows:, :7], sink[:7].expand(rows, 7))
    b.rows, b.lens = [rows, rows], [length, 0]
    check(b, cached, q[:, 6:7], out[:, 6:7], lse[:, 6:7], sink=sink[6:7])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 33])
def test_pages_that_cannot_be_read_count_as_zeros(rows):
    b = Batch([rows], [100], 1, 64, 16)
    cached = b.fill()
    b.table[0, 2] = -5
    b.table[0, 3] = b.cache.pages
    for x in cached[0]:
        x[32:64] = 0
    q = b.randn(rows, 8, 64)
    out = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    with pytest.raises(native.NativeError, match="bad_index"):
        b.cache.check()
    check(b, cached, q, out)
    # tokens that the table has no page for are not keys (every page of the table holds 16 stored tokens here)
    width = b.table.shape[1]
    b.table[0] = b.table[0, torch.tensor([0, 1, 4, 5], device=DEV).repeat(width)[:width]]
    kk, vv = paged.read(b.cache, 16 * width, b.table, torch.full_like(b.lengths, 16 * width), torch.tensor([0, 16 * width], dtype=torch.int32, device=DEV))
    b.lens = [1100]
    b.lengths[0] = 1100
    out = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    b.cache.check()
    check(b, [(kk.double(), vv.double())], q, out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 64])
def test_extreme_queries(rows):
    """Rows of zeros, of subnormal and of very large numbers; a NaN stays in its row."""
    b = Batch([rows, rows], [90, 65], 1, 128, 64)
    cached = b.fill()
    q = b.randn(2 * rows, 2, 128)
    q[0, 0] = 0
    q[0, 1] *= 2.0 ** -120
    out = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    check(b, cached, q, out)
    q[rows, 0] *= 2.0 ** 100                                  # one key takes all
    out = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    pos = 65 - rows
    s = (q[rows, 0].double() * cached[1][0][:pos + 1, 0]).sum(-1)
    assert (out[rows, 0].double() - cached[1][1][int(s.argmax()), 0]).abs().max() <= 2.0 ** -8 * 8
    q[rows, 0] = math.nan
    other = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    assert torch.isnan(other[rows, 0]).all()
    other[rows, 0] = out[rows, 0]
    assert torch.equal(other, out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 64])
def test_logits_below_all_numbers(rows):
    """Small queries times a small scale: the product of both scales is no fp32 number any more, the logits are zeros, and masked keys stay masked."""
    b = Batch([rows, rows], [300, rows], 1, 128, 64)
    cached = b.fill()
    q = b.randn(2 * rows, 2, 128) * 2.0 ** -60
    for more in (dict(), dict(window=7), dict(sink=torch.zeros(2, device=DEV))):
        out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, scale=1e-30, return_lse=True, **more)
        check(b, cached, q, out, lse, scale=1e-30, **more)
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,length,kernels", [(1, 300, 1), (1, 9000, 2), (40, 300, 1), (40, 9000, 2)])
def test_launches_are_counted(rows, length, kernels):
    """A call whose keys are cut joins the parts in a launch of its own."""
    b = Batch([rows], [length], 1, 64, 64)
    b.fill()
    q = b.randn(rows, 8, 64)
    paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    before = native.LAUNCHES[0]
    paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    assert native.LAUNCHES[0] - before == kernels


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pages at the end of pools of more than 4 GB."""
    D, kv, page, n = 128, 8, 256, 600
    pages = (1 << 32) // (kv * page * 72) + 8
    c = paged.PagedCache(*(torch.empty(pages, kv, page * 72, dtype=torch.uint8, device=DEV) for _ in range(2)), D, native.StatusWord(DEV))
    b = Batch([n], [n], kv, D, page)
    b.cache = c
    b.table[0, :3] = torch.tensor([pages - 1, pages - 3, pages - 2])
    cached = b.fill()
    kk, vv = paged.read(c, n, b.table, b.lengths, b.cu)
    assert torch.equal(kk.double(), cached[0][0]) and torch.equal(vv.double(), cached[0][1])
    for rows in (1, n):
        b.rows, b.total = [rows], rows
        b.cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
        q = b.randn(rows, 16, D)
        check(b, cached, q, paged.attention(c, q, b.table, b.lengths, b.cu))
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 48])
def test_captured_graphs_follow_their_inputs(rows):
    """Two graphs over one cache, replayed on two streams at a time; lengths, pages and rows change between the replays."""
    D, kv, S, page = 128, 2, 3, 32
    b = Batch([rows] * S, [300] * S, kv, D, page)
    cached = b.fill()
    table = paged.rope_table(400, oracle.rope_frequencies(64, 10000.0).to(DEV))
    k, v, q = b.randn(b.total, kv, D), b.randn(b.total, kv, D), b.randn(b.total, 8, D)
    q2 = b.randn(b.total, 8, D)

    def step():
        turned = paged.append(b.cache, k, v, b.table, b.lengths, b.cu, q=q, rope=table)
        return turned, paged.attention(b.cache, turned, b.table, b.lengths, b.cu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        paged.attention(b.cache, q2, b.table, b.lengths, b.cu)
    torch.cuda.current_stream().wait_stream(side)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        turned, out = step()
    with torch.cuda.graph(two):
        out2 = paged.attention(b.cache, q2, b.table, b.lengths, b.cu)
    for shift in (0, 7, 100):
        b.lens = [300 - shift - 10 * i for i in range(S)]
        b.lengths.copy_(torch.tensor(b.lens, dtype=torch.int32))
        cached = b.fill()
        q.copy_(b.randn(*q.shape))
        k.copy_(b.randn(*k.shape))
        one.replay()
        for i, length in enumerate(b.lens):
            pos = torch.arange(length - rows, length, device=DEV)
            mine = slice(i * rows, (i + 1) * rows)
            cached[i][0][length - rows:] = kv4(rotate(k[mine], table, pos, True))
            cached[i][1][length - rows:] = kv4(v[mine])
        check(b, cached, turned, out)
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            with torch.cuda.stream(side):
                two.replay()
            one.replay()
        torch.cuda.current_stream().wait_stream(side)
        check(b, cached, turned, out)
        check(b, cached, q2, out2)
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 70])
def test_a_block_in_four_bits(rows):
    """Projection, rotation, cache, attention and output projection, as a decode step and a prompt use them; each against the stage before it."""
    hid, heads, kv, D, S = 512, 8, 2, 64, 2
    b = Batch([rows] * S, [rows + 90, rows + 5], kv, D, 16)
    old = b.fill()
    gen = b.gen
    w1, w2 = (torch.randn(n, k, device=DEV, generator=gen) * k ** -0.5 for n, k in (((heads + 2 * kv) * D, hid), (hid, heads * D)))
    W1, W2 = fp4.quant_rows(w1), fp4.quant_rows(w2)
    rope = paged.rope_table(256, oracle.rope_frequencies(D, 10000.0).to(DEV))
    x = b.randn(b.total, hid)

    def product(x, W):
        return fp4.dequant_rows(fp4.quant_rows(x), torch.float32).double() @ fp4.dequant_rows(W, torch.float32).double().t()

    def near(y, want):
        # fp32 sums of up to 512 products and one rounding
        return ((y.double() - want).abs() <= torch.finfo(y.dtype).eps / 2 * want.abs() + 512 * 2.0 ** -23 * 512 ** 0.5 * want.abs().amax()).all()
    qkv = fp4.linear(x, W1)
    assert near(qkv, product(x, W1))
    q, k, v = (t.view(b.total, -1, D) for t in qkv.split([heads * D, kv * D, kv * D], -1))
    turned = paged.append(b.cache, k, v, b.table, b.lengths, b.cu, q=q, rope=rope, interleaved=False)
    o = paged.attention(b.cache, turned, b.table, b.lengths, b.cu)
    for i, length in enumerate(b.lens):
        mine = slice(i * rows, (i + 1) * rows)
        pos = torch.arange(length - rows, length, device=DEV)
        old[i][0][length - rows:] = kv4(rotate(k[mine], rope, pos, False))
        old[i][1][length - rows:] = kv4(v[mine])
    check(b, old, turned, o)
    y = fp4.linear(o.view(b.total, heads * D), W2)
    assert near(y, product(o.view(b.total, heads * D), W2))
    b.cache.check()


# ------------------------------------------------------------------------------------------ calls that the documentation allows
def test_refusals_of_tables_and_overlapping_rows():
    c, x, table, lengths, cu = cpu_batch()
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    wide = torch.zeros(2, 1, dtype=torch.int32).expand(2, (1 << 31) // 16)
    for call in (lambda t: paged.append(c, x, x, t, lengths, cu), lambda t: paged.read(c, 3, t, lengths, cu), lambda t: paged.attention(c, q, t, lengths, cu)):
        with pytest.raises(ValueError, match="without pages"):
            call(table[:, :0])
        with pytest.raises(ValueError, match="table"):        # (such a table is not contiguous here: one that is takes 1 GB)
            call(wide)
    both = torch.zeros(4, 8, 64, dtype=torch.float16)
    for out in (both[:3, :4].as_strided((3, 4, 64), (0, 64, 1)), both[:3, :4].as_strided((3, 4, 64), (256, 32, 1))):
        with pytest.raises(ValueError, match="rows of out overlap"):
            paged.attention(c, q, table, lengths, cu, out=out)
    for a, o in ((both[:3, :4], both[1:, :4]), (both[:3, :4], both[:3, 2:6]), (both[:3, :4], both.view(-1)[64:832].view(3, 4, 64))):
        with pytest.raises(ValueError, match="out overlaps q"):
            paged.attention(c, a, table, lengths, cu, out=o)
    for a, o in ((both[:3, :4], both[:3, :4]), (both[:3, :4], both[:3, 4:]), (both[1:, 4:], both[:3, :4])):
        with pytest.raises(ValueError, match="CUDA"):         # allowed: the same rows, or other columns of one buffer
            paged.attention(c, a, table, lengths, cu, out=o)
    flat = torch.zeros(2000, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q_out overlaps q"):
        paged.append(c, x, x, table, lengths, cu, q=flat[:384].view(3, 2, 64), q_out=flat[64:448].view(3, 2, 64))


def test_refusals_of_rotated_queries_over_their_neighbours():
    """``append`` reads queries, keys and values while it writes ``q_out``."""
    c, x, table, lengths, cu = cpu_batch()
    flat = torch.zeros(3 * 384 + 64, dtype=torch.bfloat16)
    a, b, d = (flat[i * 384:(i + 1) * 384].view(3, 2, 64) for i in range(3))
    late = flat[64:448].view(3, 2, 64)
    for k, v, q, out, what in ((a, b, d, a, "k"), (b, a, d, a, "v"), (b, d, a, a, "q"), (a, d, x, late, "k"), (d, b, x, late, "v"),
                               (x, a, x, flat[:3 * 128].view(3, 2, 64), "v")):
        with pytest.raises(ValueError, match="q_out overlaps " + what):
            paged.append(c, k, v, table, lengths, cu, q=q, q_out=out)
    # rows of a projection with a free block of its own between them, one too narrow, and one that begins inside the keys
    wide = torch.zeros(3, 1024, dtype=torch.bfloat16)
    k = wide[:, :128].view(3, 2, 64)
    for first, last, fits in ((128, 512, True), (640, 1024, True), (704, 1088, False), (64, 448, False)):
        with pytest.raises(ValueError, match="CUDA" if fits else "q_out overlaps k"):
            paged.append(c, k, x, table, lengths, cu, q=x, q_out=wide.view(-1)[first:last].view(3, 2, 64))


@pytest.mark.parametrize("total,heads,row,head", [(3, 4, 64, 64), (3, 4, 128, 64), (3, 4, 192, 64), (3, 4, 256, 64), (3, 4, 64, 192), (3, 4, 64, 128),
                                                  (3, 4, 128, 192), (3, 4, 192, 128), (2, 2, 192, 128), (2, 4, 512, 200), (4, 2, 200, 512), (2, 4, 584, 200),
                                                  (1, 4, 0, 64), (1, 4, 0, 56), (3, 4, 0, 64), (3, 4, 8192, 1024), (17, 12, 72, 1224), (18, 12, 72, 1224)])
def test_outputs_whose_rows_meet_are_refused(total, heads, row, head):
    """Strides of ``out`` that let a row's head lie over another row's, each stride by itself wide enough: by counting the numbers that they reach."""
    c, _, table, lengths, _ = cpu_batch()
    cu = torch.tensor([0, total, total], dtype=torch.int32)
    out = torch.zeros((total - 1) * row + (heads - 1) * head + 64, dtype=torch.float16).as_strided((total, heads, 64), (row, head, 1))
    at = torch.arange(out.untyped_storage().nbytes() // 2).as_strided(out.shape, out.stride())
    with pytest.raises(ValueError, match="CUDA" if at.unique().numel() == at.numel() else "rows of out overlap"):
        paged.attention(c, torch.zeros(total, heads, 64, dtype=torch.float16), table, lengths, cu, out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 7, 16])
def test_more_sequences_than_a_warp_looks_at_once(rows):
    """70 sequences, some of them without rows or tokens; append's search for a row's sequence and the walks of the attention's work."""
    gen = torch.Generator().manual_seed(rows)
    n = [int(x) if rows > 1 else 1 for x in torch.randint(0, rows + 1, (70,), generator=gen)]
    lens = [x + int(y) for x, y in zip(n, torch.randint(0, 200, (70,), generator=gen))]
    b = Batch(n, lens, 1, 64, 32, seed=rows)
    cached = b.fill()
    q = b.randn(b.total, 8, 64)
    k, v = b.randn(b.total, 1, 64), b.randn(b.total, 1, 64)
    paged.append(b.cache, k, v, b.table, b.lengths, b.cu)
    for i, (m, length) in enumerate(zip(n, lens)):
        at = slice(sum(n[:i]), sum(n[:i + 1]))
        cached[i][0][length - m:] = kv4(k[at])
        cached[i][1][length - m:] = kv4(v[at])
    out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True)
    b.cache.check()
    check(b, cached, q, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 255, 256, 257])
def test_blocks_that_end_anywhere(rows):
    """One kv head for all query heads: as many rows of a block as rows here, over enough keys to be cut, and over few."""
    for length in (rows, 1500):
        b = Batch([rows], [length], 1, 64, 64, seed=rows)
        cached = b.fill()
        q = b.randn(rows, 1, 64)
        out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True)
        b.cache.check()
        check(b, cached, q, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 7, 40])
def test_bounds_at_the_ends_of_the_numbers(rows):
    """The widest window is none, also where a sequence has more rows than tokens; a first key behind every key leaves none."""
    b = Batch([rows, rows], [200, max(rows - 2, 0)], 1, 64, 16)
    cached = b.fill()
    q = b.randn(2 * rows, 4, 64)
    out = paged.attention(b.cache, q, b.table, b.lengths, b.cu)
    check(b, cached, q, out)
    assert torch.equal(paged.attention(b.cache, q, b.table, b.lengths, b.cu, window=(1 << 31) - 1), out)
    for first in ((1 << 31) - 1, (1 << 31) - 32, (1 << 31) - 128, 4096, -(1 << 31)):
        f = torch.full((2,), first, dtype=torch.int32, device=DEV)
        got = paged.attention(b.cache, q, b.table, b.lengths, b.cu, first=f)
        assert torch.equal(got, out if first < 0 else torch.zeros_like(out))
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 40])
def test_offsets_outside_the_batch(rows):
    """Row offsets and lengths that no batch has: the rows inside are those of the clipped ranges, nothing else is touched, and the calls return."""
    b = Batch([rows, rows], [300, 300], 1, 64, 16)
    cached = b.fill()
    q = b.randn(2 * rows, 8, 64)
    for cu in ([0, rows, (1 << 31) - 1], [0, rows, 1 << 20], [-(1 << 30), rows, 2 * rows], [2 * rows, rows, 0]):
        bad = torch.tensor(cu, dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 5.0)
        paged.attention(b.cache, q, b.table, b.lengths, bad, out=out)
        paged.append(b.cache, q[:, :1], q[:, :1], torch.full_like(b.table, -1), b.lengths, bad)
        paged.read(b.cache, 2 * rows, torch.full_like(b.table, -1), b.lengths, bad)
        torch.cuda.synchronize()
        if cu[0] == 0:                                        # the first sequence is as it should be
            good = paged.attention(b.cache, q[:rows], b.table[:1].contiguous(), b.lengths[:1], b.cu[:2].contiguous())
            assert torch.equal(out[:rows], good)
        if cu[0] > 0:
            assert (out == 5.0).all()
    for lens in ([-(1 << 31), 300], [(1 << 31) - 1, 300]):
        paged.attention(b.cache, q, b.table, torch.tensor(lens, dtype=torch.int32, device=DEV), b.cu)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,S", [(1, 2), (50, 2), (400, 2), (2, 70), (9, 100)])
def test_offsets_outside_the_batch_are_reported(rows, S):
    """By append and by reading back, which touch nothing outside; offsets of a batch that is smaller than its rows are in order."""
    b = Batch([rows] * S, [rows + 20] * S, 1, 64, 16)
    b.fill()
    total = rows * S
    k = b.randn(total, 1, 64)
    cu = [rows * i for i in range(S + 1)]
    most, least = (1 << 31) - 1, -(1 << 31)
    for offsets, good in ((cu, True), (cu[:-1] + [cu[-1] - 1], True), (cu[:-1] + [cu[-2]], True), ([0] + cu[:-1], True),
                          (cu[:-1] + [total + 1], False), (cu[:-1] + [most], False), (cu[:-2] + [total + 1] * 2, False), ([-1] + cu[1:], False),
                          ([least] + cu[1:], False), (cu[:1] + [-1] + cu[2:], False), (cu[:-2] + [total, total - 1], False), (cu[::-1], False)):
        at = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        for call in (lambda: paged.append(b.cache, k, k, b.table, b.lengths, at, q=k), lambda: paged.read(b.cache, total, b.table, b.lengths, at)):
            call()
            code = b.cache.status.read()[0]
            b.cache.status.t.zero_()
            assert (code == 0) == good, (offsets, code)
    kb, vb = b.cache.k.clone(), b.cache.v.clone()
    paged.append(b.cache, k, k, b.table, b.lengths, torch.full_like(b.cu, total + 5))
    with pytest.raises(native.NativeError, match="bad_index"):
        b.cache.check()
    assert torch.equal(b.cache.k, kb) and torch.equal(b.cache.v, vb)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 4, 50])
def test_results_in_the_queries_place(rows):
    b = Batch([rows, rows], [2000, 700], 2, 128, 64)
    cached = b.fill()
    wide = b.randn(2 * rows, 16, 128)
    q = wide[:, 4:12]
    want = q.clone()
    out = paged.attention(b.cache, want, b.table, b.lengths, b.cu)
    side = wide[:, 12:]                                       # (columns of the same rows)
    kept = wide[:, :4].clone()
    paged.attention(b.cache, wide[:, 4:8], b.table, b.lengths, b.cu, out=side)
    paged.attention(b.cache, q, b.table, b.lengths, b.cu, out=q)
    assert torch.equal(wide[:, 4:12], out) and torch.equal(wide[:, :4], kept)
    check(b, cached, want, out)
    b.cache.check()


@pytest.mark.gpu
def test_a_cache_without_a_status_word():
    b = Batch([2], [40], 2, 64, 16)
    b.cache = paged.PagedCache(b.cache.k, b.cache.v, 64)
    cached = b.fill()
    b.table[0, 1] = 1 << 20                                   # reported nowhere, and still zeros
    for x in cached[0]:
        x[16:32] = 0
    q = b.randn(2, 4, 64)
    check(b, cached, q, paged.attention(b.cache, q, b.table, b.lengths, b.cu))
    b.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,group", [(1, 4), (1, 16), (4, 7)])
@pytest.mark.parametrize("longest", [1500, 3000])
def test_batches_of_many_sequences(rows, group, longest):
    """An item for every CTA: of middling keys (a CTA each) and with one long sequence among them (laid end to end and cut)."""
    S, kv = 40, 8
    gen = torch.Generator().manual_seed(longest + rows)
    lens = [int(x) for x in torch.randint(rows, 700, (S,), generator=gen)]
    lens[17] = longest
    b = Batch([rows] * S, lens, kv, 64, 64, torch.float16, seed=rows)
    cached = b.fill()
    q = b.randn(b.total, kv * group, 64)
    out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True)
    b.cache.check()
    check(b, cached, q, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 5, 40])
def test_one_head_over_a_long_sequence(rows, D):
    """The keys of one item in dozens of parts."""
    b = Batch([rows], [20011], 1, D, 128, seed=rows)
    cached = b.fill()
    q = b.randn(rows, 6, D)
    sink = torch.randn(6, generator=b.gen, device=DEV)
    out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, sink=sink, return_lse=True)
    b.cache.check()
    check(b, cached, q, out, lse, sink=sink)


@pytest.mark.gpu
@pytest.mark.parametrize("S,kv,group,longest", [(1, 1, 4, 300), (5, 2, 12, 3000), (40, 8, 4, 900), (40, 8, 20, 2500)])
def test_a_row_a_sequence_needs_no_offsets(S, kv, group, longest):
    """The same bits with offsets and without; fewer rows than sequences leave the later sequences alone."""
    gen = torch.Generator().manual_seed(S)
    lens = [int(x) for x in torch.randint(1, longest, (S,), generator=gen)]
    lens[0] = longest
    b = Batch([1] * S, lens, kv, 64, 32, seed=S)
    cached = b.fill()
    q = b.randn(S, kv * group, 64)
    out, lse = paged.attention(b.cache, q, b.table, b.lengths, b.cu, return_lse=True)
    check(b, cached, q, out, lse)
    for n in (S, (S + 1) // 2):
        got, lg = paged.attention(b.cache, q[:n], b.table, b.lengths, return_lse=True)
        if n == S:
            assert torch.equal(got, out) and torch.equal(lg, lse)
        b.rows = [1] * n
        check(b, cached, q[:n], got, lg)
    b.cache.check()
