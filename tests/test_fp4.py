"""MXFP4 rows and their product (``ops/fp4.py``) against their definition in 64 bits."""
import ctypes
import math

import pytest
import torch

from titanic_flash_41_b200.formats import codecs
from titanic_flash_41_b200.ops import fp4, native

DEV = "cuda"
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def reference(x):
    """Codes' values and scale bytes of x's MXFP4 form, 64 bits, blocks of 32 (zeros behind the last column)."""
    m, k = x.shape
    kb = -(-k // 32)
    b = torch.zeros(m, kb * 32, dtype=torch.float64, device=x.device)
    b[:, :k] = x.double()
    b = b.view(m, kb, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    powers = torch.tensor([6.0 * 2.0 ** e for e in range(-127, 121)], dtype=torch.float64, device=x.device)
    code = torch.bucketize(amax, powers).clamp(max=247)                 # smallest power with amax <= 6 times it
    s = torch.ldexp(torch.ones_like(amax), code - 127)[..., None]       # (pow is an ulp off some powers of two)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    a = (b / s).abs()
    lo, hi = torch.bucketize(a, mids), torch.bucketize(a, mids, right=True)
    idx = torch.where(lo % 2 == 0, lo, hi)                              # a tie goes to the even code
    v = VALUES.to(x.device)[idx] * s * torch.where(b < 0, -1.0, 1.0)
    v = torch.where(bad[..., None], torch.full_like(v, math.nan), v)
    code = torch.where(bad, torch.full_like(code, 255), code)
    return v.view(m, -1)[:, :k], code


def same(got, v):
    """Equal numbers, NaN at the same places (a block of f16 rows may hold an infinity)."""
    got = got.double()
    return torch.equal(torch.isnan(got), torch.isnan(v)) and torch.equal(got.nan_to_num(), v.nan_to_num())


def scale_bytes(r):
    kb, units, _ = r.sf.shape
    return r.sf.view(kb, units, 32, 4).permute(1, 2, 0, 3).reshape(units * 32, kb * 4)[:r.rows, :-(-r.K // 32)]


def weights(n, k, gen):
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=gen)
    scales = torch.randint(110, 126, (n, k // 32), dtype=torch.uint8, device=DEV, generator=gen)
    return packed, scales, codecs.mxfp4_dequant(packed, scales).double()


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def test_refusals():
    x = torch.zeros(4, 64)
    r = fp4.empty_rows(4, 64, "cpu")
    for bad, what in ((torch.zeros(4, 64, dtype=torch.float64), "f32, f16 or bf16"), (torch.zeros(64), "rows, K"), (torch.zeros(64, 4).t(), "contiguous"),
                      (torch.zeros(4, 0), "contiguous")):
        with pytest.raises(ValueError, match=what):
            fp4.quant_rows(bad)
    with pytest.raises(ValueError, match="another size"):
        fp4.quant_rows(torch.zeros(5, 64), out=r)
    with pytest.raises(ValueError, match="CUDA"):
        fp4.quant_rows(x)
    with pytest.raises(ValueError, match="K of the operands"):
        fp4.gemm(r, fp4.empty_rows(8, 96, "cpu"))
    with pytest.raises(ValueError, match="another size, type or device"):
        fp4.gemm(r, r, out=torch.zeros(4, 5))
    with pytest.raises(ValueError, match="overlap"):
        fp4.gemm(r, r, out=torch.zeros(1, 4).expand(4, 4))
    with pytest.raises(ValueError, match="f32, f16 or bf16"):
        fp4.gemm(r, r, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fp4.gemm(r, r)
    with pytest.raises(ValueError, match="q holds"):
        fp4.Fp4Rows(torch.zeros(4, 32, dtype=torch.uint8), r.sf, 4, 64)
    with pytest.raises(ValueError, match="sf is"):
        fp4.Fp4Rows(r.q, r.sf[:, :7].contiguous(), 4, 64)
    with pytest.raises(ValueError, match="32 divides"):
        fp4.rows_from_mxfp4(torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    with pytest.raises(ValueError, match="f32, f16 or bf16"):
        fp4.dequant_rows(r, torch.int8)


def test_library_refuses_what_the_kernels_cannot_take():
    lib, buf = native.lib(), torch.zeros(1 << 16, dtype=torch.uint8)
    at = (buf.data_ptr() + 63) & ~63
    assert lib.tf_gemm_fp4(at, at, 8, at, at, 8, at, 256, 2, 16, 256, 128, None, None) == -1          # K not padded
    assert lib.tf_gemm_fp4(at, at, 0, at, at, 8, at, 256, 2, 16, 256, 256, None, None) == -1          # scales of no rows
    assert lib.tf_gemm_fp4(at, at, 8, at, at, 7, at, 256, 2, 16, 256, 256, None, None) == -1          # part of a feature block's scales
    assert lib.tf_gemm_fp4(at + 8, at, 8, at, at, 8, at, 256, 2, 16, 256, 256, None, None) == -1      # operand off its boundary
    assert lib.tf_gemm_fp4(at, at, 8, at, at, 8, at, 255, 2, 16, 256, 256, None, None) == -1          # overlapping rows
    assert lib.tf_gemm_fp4(at, at, 8, at, at, 8, at, 256, 3, 16, 256, 256, None, None) == -1          # unknown type
    assert lib.tf_fp4_quant_rows(at, 3, 64, at, at, 8, 4, 64, None) == -1
    assert lib.tf_fp4_quant_rows(at, 2, 64, at, at, 0, 4, 64, None) == -1
    assert lib.tf_fp4_dequant_rows(at, at, 8, at, 2, 63, 4, 64, None) == -1


def test_stored_weights_take_the_operand_layout():
    gen = torch.Generator().manual_seed(3)
    for n, k in ((1, 32), (70, 96), (300, 256), (33, 544)):
        packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=gen)
        scales = torch.randint(0, 248, (n, k // 32), dtype=torch.uint8, generator=gen)
        r = fp4.rows_from_mxfp4(packed, scales)
        assert torch.equal(scale_bytes(r), scales) and torch.equal(r.q[:, :k // 2], packed) and not r.q[:, k // 2:].any()


def test_stored_weights_at_any_address():
    """A checkpoint's tensors may begin anywhere in its file; an operand's begin on 16-byte boundaries, or are refused where they are named."""
    gen = torch.Generator().manual_seed(4)
    for n, k in ((256, 128), (256, 256), (40, 512), (7, 96)):
        for shift in (1, 4, 8, 16):
            packed, scales = (torch.randint(0, 248, (n * w + shift,), dtype=torch.uint8, generator=gen)[shift:].view(n, w) for w in (k // 2, k // 32))
            r = fp4.rows_from_mxfp4(packed, scales)
            assert (r.q_at | r.sf_at) % 16 == 0 and r.q_at == r.q.data_ptr() and r.sf_at == r.sf.data_ptr()
            assert torch.equal(scale_bytes(r), scales) and torch.equal(r.q[:, :k // 2], packed)
    r, room = fp4.empty_rows(4, 256, "cpu"), torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(ValueError, match="boundar"):
        fp4.Fp4Rows(room[8:520].view(4, 128), r.sf, 4, 256)
    with pytest.raises(ValueError, match="boundar"):
        fp4.Fp4Rows(r.q, room[2:2050].view(2, 8, 128), 4, 256)
    odd = fp4.Fp4Rows(r.q, room[4:2052].view(2, 8, 128), 4, 256)          # scales that rows are written and read with, but not multiplied
    for a, w in ((odd, r), (r, odd)):
        with pytest.raises(ValueError, match="boundar"):
            fp4.gemm(a, w)


def test_a_wait_that_ran_out_is_seen(monkeypatch):
    """Products without a status word of the caller's report to the device's; the library's part is played here (code 2: a wait ran out)."""
    r, seen = fp4.empty_rows(4, 64, "cpu"), []

    def library(name, t, *args):
        if name == "tf_gemm_fp4":
            seen.append(args[-1])
            ctypes.memmove(args[-1], (ctypes.c_int32 * 4)(2, 184, 7, 0), 16)
    monkeypatch.setattr(native, "launch", library)
    fp4.check()
    for call in (lambda: fp4.gemm(r, r), lambda: fp4.linear(torch.zeros(4, 64), r)):
        for where in ((), ("cpu",), (torch.device("cpu"),)):
            call()
            with pytest.raises(native.NativeError, match="timeout"):
                fp4.check(*where)
            fp4.check(*where)
    own = native.StatusWord("cpu")
    seen.clear()
    fp4.gemm(r, r, status=own.t)
    assert seen == [own.t.data_ptr()]
    fp4.check()                                              # reported where the caller asked for it
    with pytest.raises(native.NativeError, match="timeout"):
        own.check()
    for bad in (own.t.to("meta"), own.t.long(), own.t[:3], torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="status"):
            fp4.gemm(r, r, status=bad)


def test_no_rows_have_bytes_and_scales_too():
    for K in (1, 75, 256, 4000):
        kp = fp4.padded(K, 256)
        for r in (fp4.empty_rows(0, K, "cpu"), fp4.quant_rows(torch.zeros(0, K))):
            assert r.q.shape == (0, kp // 2) and r.sf.shape == (kp // 128, 0, 128)
            again = fp4.Fp4Rows(r.q, r.sf, 0, K)
            assert (again.rows, again.K, again.units) == (0, K, 0)
    r = fp4.rows_from_mxfp4(torch.zeros(0, 48, dtype=torch.uint8), torch.zeros(0, 3, dtype=torch.uint8))
    assert r.q.shape == (0, 128) and r.sf.shape == (2, 0, 128)


# ------------------------------------------------------------------------------------------ rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 31), (3, 32), (33, 75), (257, 300), (16, 4096), (5, 8191)])
def test_rows_are_the_definitions(dtype, rows, K):
    gen = torch.Generator(device=DEV).manual_seed(rows * 7 + K)
    x = (torch.randn(rows, K, device=DEV, generator=gen) * torch.exp(3 * torch.randn(rows, K, device=DEV, generator=gen))).to(dtype)
    r = fp4.quant_rows(x)
    v, code = reference(x)
    assert torch.equal(scale_bytes(r).long(), code)
    assert same(fp4.dequant_rows(r, torch.float32), v)
    assert same(fp4.dequant_rows(r), v)                                  # two significant bits: exact in bf16
    assert not r.q[:, -(-K // 32) * 16:].any()


@pytest.mark.gpu
def test_rows_at_the_borders():
    """Every midpoint of the grid and its neighbours, at scales from the smallest to the largest."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    for e in (-127, -126, -100, -1, 0, 5, 119, 120):
        s = torch.tensor(2.0, dtype=torch.float64).pow(e).float().to(DEV)
        m = mids * s
        x = torch.zeros(3, 32, device=DEV)
        x[0, :7], x[1, :7], x[2, :7] = m, torch.nextafter(m, m * 2), torch.nextafter(m, m * 0)
        x[:, 8:15] = -x[:, :7]
        x[:, 31] = 6 * s
        r = fp4.quant_rows(x)
        v, code = reference(x)
        assert torch.equal(scale_bytes(r).long(), code) and int(code[0, 0]) == e + 127
        assert torch.equal(fp4.dequant_rows(r, torch.float32).double(), v)
    top = torch.zeros(4, 32, device=DEV)
    top[0, 0], top[1, 0], top[2, 0] = 6.0, torch.nextafter(torch.tensor(6.0), torch.tensor(7.0)), 3e38
    assert scale_bytes(fp4.quant_rows(top))[:, 0].tolist() == [127, 128, 247, 0]


@pytest.mark.gpu
def test_rows_of_nan_and_infinity_stay_their_blocks():
    x = torch.randn(4, 96, device=DEV)
    x[0, 5], x[1, 40], x[2, 95] = math.nan, math.inf, -math.inf
    v, code = reference(x)
    r = fp4.quant_rows(x)
    assert torch.equal(scale_bytes(r).long(), code)
    assert same(fp4.dequant_rows(r, torch.float32), v)
    w, s, wv = weights(40, 96, torch.Generator(device=DEV).manual_seed(1))
    y = fp4.gemm(r, fp4.rows_from_mxfp4(w, s))
    assert torch.isnan(y[:3]).all() and torch.isfinite(y[3]).all()


@pytest.mark.gpu
def test_rows_at_any_pitch_and_address():
    base = torch.randn(20, 1000, device=DEV).to(torch.bfloat16)
    for x in (base[:, 3:330], base[::2, :256], base[3:4].expand(9, 1000), base[:, 8:520], base[5:6, 999:]):
        v, code = reference(x)
        r = fp4.quant_rows(x)
        assert torch.equal(scale_bytes(r).long(), code) and torch.equal(fp4.dequant_rows(r).double(), v)
    assert fp4.dequant_rows(fp4.quant_rows(base[:0])).shape == (0, 1000)


# ------------------------------------------------------------------------------------------ product
def close(y, a, w, K):
    """fp32 sums of exact products: every one of the K additions is off by at most an ulp of a sum that stays below sum |a w|; then one rounding."""
    exact, size = a @ w.t(), a.abs() @ w.abs().t()
    bound = torch.finfo(y.dtype).eps / 2 * exact.abs() + K * 2.0 ** -23 * size + (6e-8 if y.dtype == torch.float16 else 0)
    worst = ((y.double() - exact).abs() - bound).max()
    assert worst <= 0, float(worst)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 256, 256), (3, 70, 96), (16, 4096, 2048), (31, 1000, 4096), (33, 300, 8192), (64, 512, 1280),
                                   (65, 257, 512), (130, 520, 2304), (257, 1027, 544), (1000, 640, 320)])
def test_product(dtype, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    x = torch.randn(M, K, device=DEV, generator=gen) * 0.5
    w, s, wv = weights(N, K, gen)
    r = fp4.quant_rows(x)
    st = native.StatusWord(DEV)
    y = fp4.gemm(r, fp4.rows_from_mxfp4(w, s), dtype=dtype, status=st.t)
    st.check()
    close(y, fp4.dequant_rows(r, torch.float32).double(), wv, K)
    assert torch.equal(y, fp4.gemm(r, fp4.rows_from_mxfp4(w, s), dtype=dtype))          # the same bits every time


@pytest.mark.gpu
def test_product_at_scales_far_apart():
    """Every scale byte of the form takes part: products from 2^-60 to 2^60."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(40, 512, device=DEV, generator=gen) * torch.exp2(torch.randint(-60, 61, (40, 1), device=DEV, generator=gen).float())
    w, _, _ = weights(300, 512, gen)
    s = torch.randint(67, 188, (300, 1), dtype=torch.uint8, device=DEV, generator=gen).expand(300, 16).contiguous()
    r = fp4.quant_rows(x)
    close(fp4.gemm(r, fp4.rows_from_mxfp4(w, s), dtype=torch.float32), fp4.dequant_rows(r, torch.float32).double(), codecs.mxfp4_dequant(w, s).double(), 512)


@pytest.mark.gpu
def test_product_writes_its_own_columns_only():
    gen = torch.Generator(device=DEV).manual_seed(6)
    w, s, wv = weights(301, 128, gen)
    W = fp4.rows_from_mxfp4(w, s)
    for M in (5, 40, 200):
        r = fp4.quant_rows(torch.randn(M, 128, device=DEV, generator=gen))
        big = torch.full((M + 2, 400), 7.0, device=DEV, dtype=torch.bfloat16)
        out = big[1:M + 1, 41:342]
        assert fp4.gemm(r, W, out=out).data_ptr() == out.data_ptr()
        close(out, fp4.dequant_rows(r, torch.float32).double(), wv, 128)
        big[1:M + 1, 41:342] = 7.0
        assert (big == 7.0).all()
    assert fp4.gemm(fp4.quant_rows(torch.zeros(0, 128, device=DEV)), W).shape == (0, 301)


@pytest.mark.gpu
def test_linear_in_a_captured_graph_and_on_another_stream():
    gen = torch.Generator(device=DEV).manual_seed(8)
    w, s, _ = weights(512, 512, gen)
    W = fp4.rows_from_mxfp4(w, s)
    x = torch.randn(24, 512, device=DEV, generator=gen).to(torch.bfloat16)
    fp4.linear(x, W)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = fp4.linear(x, W)
    for seed in (1, 2):
        x.copy_(torch.randn(24, 512, device=DEV, generator=gen))
        g.replay()
        assert torch.equal(y, fp4.linear(x, W))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = fp4.linear(x, W)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)


@pytest.mark.gpu
def test_the_device_has_one_status_word_that_graphs_share():
    r = fp4.quant_rows(torch.randn(8, 256, device=DEV))
    fp4._WORDS.clear()
    g, y = torch.cuda.CUDAGraph(), fp4.gemm(r, r, status=native.StatusWord(DEV).t)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        z = fp4.gemm(r, r)                                   # (a first call under capture makes none)
    assert not fp4._WORDS
    fp4.gemm(r, r)
    word, = fp4._WORDS.values()
    assert word.t.device == r.device and word.read() == [0, 0, 0, 0]
    fp4.gemm(r, r)
    assert list(fp4._WORDS.values()) == [word]
    g.replay()
    assert torch.equal(y, z)
    word.t[0] = 2
    with pytest.raises(native.NativeError, match="timeout"):
        fp4.check(DEV)
    fp4.check()


@pytest.mark.gpu
def test_product_with_stored_weights_off_their_boundary():
    gen = torch.Generator(device=DEV).manual_seed(9)
    w, s, wv = weights(256, 256, gen)
    r = fp4.quant_rows(torch.randn(16, 256, device=DEV, generator=gen))
    file = torch.zeros(3 + w.numel() + s.numel(), dtype=torch.uint8, device=DEV)
    packed, scales = file[3:3 + w.numel()].view_as(w), file[3 + w.numel():].view_as(s)
    packed.copy_(w)
    scales.copy_(s)
    y = fp4.gemm(r, fp4.rows_from_mxfp4(packed, scales))
    assert torch.equal(y, fp4.gemm(r, fp4.rows_from_mxfp4(w, s)))
    close(y, fp4.dequant_rows(r, torch.float32).double(), wv, 256)
