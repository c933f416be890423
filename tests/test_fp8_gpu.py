"""Block-scaled 8-bit operators on the GPU against float64 (fp8_reference).

Quantisation is compared bit for bit: x / scale is exact, so only the one
rounding to e4m3 remains.  The products of small integers are compared bit
for bit too: every partial sum is then exact in fp32, whatever the order."""

import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import forgetune_b200 as ft
from forgetune_b200 import _native, InvalidShapeError, Fp8Rows, Fp8Weight, fp8_linear, quantize_rows, quantize_weight, rms_norm

from . import fp8_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS32 = 2.0 ** -24  # half a step of fp32, relative


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def same(a, b):
    """Equal, NaN equal to NaN."""
    return np.array_equal(a, b, equal_nan=True)


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
def check_quantized(got, x, rows):
    v, s = ref.quantize(f64(x), rows)
    assert same(f64(got.scales), s)
    assert same(f64(got.data), v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 127), (2, 128), (3, 129), (5, 1000), (33, 784), (7, 4096), (300, 515),
                                 (1000, 128), (777, 384), (900, 64), (50, 8192), (3, 20000)])
def test_quantize_rows(m, k, dtype):
    x = randn(m, k, seed=m * 7 + k, dtype=dtype) * 3
    check_quantized(quantize_rows(x), x, 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (127, 129), (128, 128), (129, 64), (250, 784), (512, 1000), (10, 8192)])
def test_quantize_weight(n, k, dtype):
    w = randn(n, k, seed=n + k, dtype=dtype) / 16
    check_quantized(quantize_weight(w), w, 128)


def test_quantize_values_at_the_borders():
    """Every binade's border, zeros of both signs, the smallest and largest fp32 values."""
    rows = []
    for e in list(range(-149, -110)) + list(range(-12, 13)) + list(range(100, 128)):
        for f in (1.0, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), 1.9999999):
            r = np.zeros(200, np.float32)
            with np.errstate(over="ignore", under="ignore"):
                r[:8] = np.float32(np.ldexp(f, e)) * np.array([1, -1, .5, 1 / 3, -1 / 7, 2 ** -9, 2 ** -10, 0], np.float32)
            r[9] = -0.0
            r[130] = r[0]  # a second, ragged block
            rows.append(np.where(np.isfinite(r), r, 0))
    rows.append(np.zeros(200, np.float32))
    rows.append(np.full(200, np.finfo(np.float32).max, np.float32))
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    got = quantize_rows(x)
    check_quantized(got, x, 1)
    neg = f64(got.data)[0]
    assert np.signbit(neg[9]) and neg[9] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_keeps_what_is_not_finite_as_nan(dtype):
    x = randn(4, 300, dtype=dtype)
    x[0, 5] = float("inf")
    x[1, 130] = float("-inf")
    x[2, 299] = float("nan")
    x[3, :] = float("inf")
    check_quantized(quantize_rows(x), x, 1)
    check_quantized(quantize_weight(x), x, 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_and_offset_rows(dtype):
    base = randn(40, 700, dtype=dtype)
    for x in (base[:, 1:514], base[3::2, 4:516], base[5:6, 3:300], base.t()[:200, ::2], base[:1].expand(6, 700)):
        check_quantized(quantize_rows(x), x, 1)
        check_quantized(quantize_weight(x), x, 128)


def guarded(m, k):
    """An Fp8Rows inside larger buffers, and a check that nothing around it changed."""
    data = torch.full((m + 2, (k + 15) // 16 * 16 + 32), 0x55, dtype=torch.uint8, device="cuda")
    kb = -(-k // 128)
    scales = torch.full((m + 2, (kb + 3) // 4 * 4 + 4), 0x55, dtype=torch.uint8, device="cuda")
    out = Fp8Rows(data.view(torch.float8_e4m3fn)[1:m + 1, :k], scales.view(torch.float8_e8m0fnu)[1:m + 1, :kb])

    def check():
        for t, c in ((data, k), (scales, kb)):
            rest = t.clone()
            rest[1:m + 1, :c] = 0x55
            assert bool((rest == 0x55).all())
    return out, check


@pytest.mark.parametrize("m,k", [(1, 77), (3, 128), (65, 1000), (40, 4096)])
def test_quantize_writes_its_rows_only(m, k):
    out, check = guarded(m, k)
    x = randn(m, k)
    assert quantize_rows(x, out=out) is out
    check()
    check_quantized(out, x, 1)
    out, check = guarded(m, k)
    y, h = rms_norm(x, residual=x, quantize=True, out=out)
    check()


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------
def norm_bound(k):
    """Relative error of the fp32 norm.  The sum of k squares in partial sums
    of at most k/128 + 16 terms in a row: each addition half a step, each
    square and h half a step more; the root halves it.  Division by k, eps,
    rsqrt (2 steps) and the two products: 8 half steps."""
    return (0.5 * (k / 128 + 20) + 8) * EPS32


def check_plain(got, want, dtype, rel, absolute=0.0):
    tol = np.abs(want) * (torch.finfo(dtype).eps / 2 * (1 + rel) + rel) + absolute
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half the smallest fp16 step
    assert np.all(np.abs(f64(got) - want) <= tol), float(np.max(np.abs(f64(got) - want) / np.maximum(tol, 1e-300)))


def check_block(got, want, err, rows=1):
    """Quantised rows whose values are known up to +- err: the scale fits the largest value, the values are
    rounded once (2^-4 relative; 2^-10 of the scale below the normal range)."""
    s = f64(got.scales)
    amax, slack = ref._block_max(want, rows), ref._block_max(err, rows)
    assert np.all((amax - slack <= 448 * s) & ((amax + slack > 224 * s) | ((amax <= slack) & (s == 1))
                                                | (s == 2.0 ** -127)))
    sm = ref.spread(s, rows, want.shape)
    tol = np.maximum((np.abs(want) + err) * 2.0 ** -4, sm * 2.0 ** -10) + err
    assert np.all(np.abs(f64(got.data) * sm - want) <= tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 127), (2, 1111), (300, 512), (4, 4096), (2, 8192), (3, 8200), (2, 20001),
                                 (700, 64), (1001, 200), (900, 4096), (400, 1000), (2, 33000)])
def test_rms_norm(m, k, quantize, residual, dtype):
    x = randn(m, k, seed=k, dtype=dtype) * 2
    r = randn(m, k, seed=k + 1, dtype=dtype) if residual else None
    w = randn(k, seed=k + 2) + 1
    want, h = ref.rms_norm(f64(x), f64(w), 1e-5, None if r is None else f64(r))
    got = rms_norm(x, w, eps=1e-5, residual=r, quantize=quantize)
    if residual:
        got, hg = got
        assert hg.dtype == dtype
        check_plain(hg, h, dtype, EPS32)
    # h is rounded to fp32 once before it is used: that error is absolute where x and r cancel
    absolute = (np.abs(f64(x)) + (np.abs(f64(r)) if residual else 0)) * EPS32 * np.abs(want) / np.maximum(np.abs(h), 1e-30)
    if quantize:
        check_block(got, want, np.abs(want) * norm_bound(k) + absolute)
    else:
        assert got.dtype == dtype
        check_plain(got, want, dtype, norm_bound(k), absolute)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 384), (2, 1536), (300, 384), (301, 768), (299, 1280), (300, 1288), (333, 2560),
                                 (300, 4104), (297, 5120), (300, 7168), (300, 11008), (2, 8320), (300, 16384),
                                 (300, 136), (299, 264), (5, 640)])
def test_rms_norm_rows_of_any_number_of_warps(m, k, dtype):
    x, r, w = randn(m, k, seed=k, dtype=dtype) * 2, randn(m, k, seed=k + 1, dtype=dtype), randn(k, seed=k + 2) + 1
    want, h = ref.rms_norm(f64(x), f64(w), 1e-5, f64(r))
    absolute = (np.abs(f64(x)) + np.abs(f64(r))) * EPS32 * np.abs(want) / np.maximum(np.abs(h), 1e-30)
    y, hg = rms_norm(x, w, eps=1e-5, residual=r)
    check_plain(y, want, dtype, norm_bound(k), absolute)
    check_plain(hg, h, dtype, EPS32)
    check_block(rms_norm(x, w, eps=1e-5, residual=r, quantize=True)[0], want,
                np.abs(want) * norm_bound(k) + absolute)
    plain, _ = ref.rms_norm(f64(x), None, 1e-5)
    check_plain(rms_norm(x, eps=1e-5), plain, dtype, norm_bound(k))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 129), (2, 255), (700, 129), (301, 257), (300, 385), (299, 1111), (300, 4097),
                                 (2, 4097), (2, 7001), (400, 512), (300, 8192), (299, 8193), (300, 16384), (2, 16384), (2, 16385),
                                 (1, 32769)])
def test_rms_norm_rows_off_16_byte_boundaries(m, k, dtype):
    """Rows that begin one element off a boundary, with columns before and behind that stay as they are; the
    same values in rows on boundaries give the reference."""
    bx, br = randn(m, k + 9, seed=k, dtype=dtype) * 2, randn(m, k + 9, seed=k + 1, dtype=dtype)
    bx[:, 0] = br[:, 0] = float("nan")
    bx[:, k + 1:] = br[:, k + 1:] = float("nan")
    x, r = bx[:, 1:k + 1], br[:, 1:k + 1]
    w = (randn(k + 1, seed=k + 2) + 1)[1:]
    want, h = ref.rms_norm(f64(x), f64(w), 1e-5, f64(r))
    absolute = (np.abs(f64(x)) + np.abs(f64(r))) * EPS32 * np.abs(want) / np.maximum(np.abs(h), 1e-30)
    by, bh = torch.full_like(bx, 7), torch.full_like(bx, 7)
    y, hg = rms_norm(x, w, eps=1e-5, residual=r, out=by[:, 1:k + 1], residual_out=bh[:, 1:k + 1])
    check_plain(y, want, dtype, norm_bound(k), absolute)
    check_plain(hg, h, dtype, EPS32)
    for b in (by, bh):
        assert bool((b[:, 0] == 7).all()) and bool((b[:, k + 1:] == 7).all())
    q, hq = rms_norm(x, w, eps=1e-5, residual=r, quantize=True)
    assert torch.equal(hq, hg)
    check_block(q, want, np.abs(want) * norm_bound(k) + absolute)
    plain, _ = ref.rms_norm(f64(x), None, 1e-5)
    check_plain(rms_norm(x, eps=1e-5), plain, dtype, norm_bound(k))


@pytest.mark.parametrize("k", [129, 1111])
def test_rms_norm_rows_off_16_byte_boundaries_and_what_is_not_finite(k):
    x = randn(5, k)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    y, q = f64(rms_norm(x)), rms_norm(x, quantize=True)
    d, s = f64(q.data), f64(q.scales)
    rest = np.arange(k) != 9
    for v in (y, d):
        assert np.all(v[1] == 0) and np.all(np.isnan(v[2]))
        assert np.isnan(v[3, 9]) and np.all(v[3, rest] == 0)  # x / inf
    assert np.all(s[[1, 2, 3]] == 1)
    want, _ = ref.rms_norm(f64(x[[0, 4]]), None, 1e-6)
    check_plain(torch.from_numpy(y[[0, 4]]), want, torch.float32, norm_bound(k))
    # one value that is not finite after the norm: its block's scale comes from the others
    w = torch.ones(k, device="cuda")
    w[3] = float("inf")
    q = rms_norm(x[:1], w, quantize=True)
    full, _ = ref.rms_norm(f64(x[:1]), None, 1e-6)
    d, s = f64(q.data), f64(q.scales)
    assert np.isnan(d[0, 3])
    full[0, 3] = d[0, 3] = 0
    top = np.abs(full[0, :128]).max()
    assert 224 * s[0, 0] * (1 - 1e-4) < top <= 448 * s[0, 0] * (1 + 1e-4)
    assert np.all(np.abs(d * ref.spread(s, 1, full.shape) - full)
                  <= np.abs(full) * (2.0 ** -4 + 1e-4) + ref.spread(s, 1, full.shape) * 2.0 ** -10)


@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm_in_place_strided_and_without_weight(dtype):
    base = randn(10, 900, dtype=dtype)
    x, r = base[:, 3:803], randn(10, 800, seed=1, dtype=dtype)
    want, h = ref.rms_norm(f64(x), None, 1e-6, f64(r))
    before = base.clone()
    y0, h0 = rms_norm(x, residual=r)
    r1 = r.clone()
    y1, h1 = rms_norm(x, residual=r1, residual_out=r1)
    assert h1 is r1 and torch.equal(y0, y1) and torch.equal(h0, h1)
    out = torch.empty(10, 1000, dtype=dtype, device="cuda").fill_(7)
    y2, h2 = rms_norm(x, residual=r, out=x, residual_out=out[:, 1:801])
    assert torch.equal(y0, base[:, 3:803]) and torch.equal(h0, out[:, 1:801])
    assert torch.equal(base[:, :3], before[:, :3]) and torch.equal(base[:, 803:], before[:, 803:])
    assert bool((out[:, :1] == 7).all()) and bool((out[:, 801:] == 7).all())
    check_plain(y0, want, dtype, norm_bound(800), np.abs(want) * 0 + 1e-6)


def test_rms_norm_zero_rows_and_what_is_not_finite():
    x = randn(5, 384)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    y = f64(rms_norm(x))
    assert np.all(y[1] == 0) and np.all(np.isnan(y[2]))
    assert np.isnan(y[3, 9]) and np.all(y[3, np.arange(384) != 9] == 0)  # x / inf
    want, _ = ref.rms_norm(f64(x[[0, 4]]), None, 1e-6)
    assert np.allclose(y[[0, 4]], want, rtol=norm_bound(384) + EPS32, atol=0)
    q = rms_norm(x, quantize=True)
    assert np.all(f64(q.scales)[1] == 1) and np.all(np.isnan(f64(q.data)[2]))


# ---------------------------------------------------------------------------
# the matrix product
# ---------------------------------------------------------------------------
def integers(rows, k, row_block, seed):
    """Quantised integers -4 .. 4 with scales 1/4 .. 4: every sum of up to 2^13
    products is a multiple of 1/16 below 2^13 2^4 2^4 = 2^21, so 25 bits at
    most; |sum| itself stays far below, and all partial sums are exact."""
    g = torch.Generator().manual_seed(seed)
    d = torch.randint(-4, 5, (rows, k), generator=g).float()
    s = 2.0 ** torch.randint(-2, 3, (-(-rows // row_block), -(-k // 128)), generator=g).float()
    cls = Fp8Rows if row_block == 1 else Fp8Weight
    q = cls.pack(d.to(torch.float8_e4m3fn).cuda(), s.to(torch.float8_e8m0fnu).cuda())
    return q, f64(d) * ref.spread(f64(s), row_block, (rows, k))


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 250, 784), (2, 10, 31), (3, 129, 129), (15, 64, 4096), (16, 384, 1000),
          (16, 128, 8192), (17, 127, 512), (31, 256, 513), (33, 300, 640), (64, 136, 96), (65, 512, 2048),
          (100, 1000, 1536), (128, 128, 128), (129, 260, 257), (200, 512, 4096), (255, 1, 384), (256, 256, 1024),
          (257, 384, 200), (300, 250, 784), (512, 768, 512), (700, 1100, 130), (1024, 520, 2000), (1, 4096, 4096),
          (2050, 1024, 320), (1, 40000, 64), (5000, 96, 100), (640, 2304, 1152), (1290, 2051, 200), (2100, 2304, 130),
          (1500, 4000, 2100), (4133, 1153, 900), (3000, 5000, 64)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_of_integers_is_exact(m, n, k):
    a, av = integers(m, k, 1, seed=m + k)
    w, wv = integers(n, k, 128, seed=n + k)
    want, _ = ref.linear(av, wv)
    y = fp8_linear(a, w)
    assert y.dtype == torch.float32 and tuple(y.shape) == (m, n)
    assert same(f64(y), want)
    again = fp8_linear(a, w)
    assert torch.equal(y, again)


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("res_dtype", [None] + TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 250, 784), (20, 384, 512), (140, 513, 300), (600, 640, 384), (1290, 2051, 200),
                                   (2100, 2304, 130)])
def test_linear_epilogue_and_types(m, n, k, res_dtype, out_dtype):
    """Integer sums, an integer bias and residual: exact in fp32, one rounding to the output's type."""
    a, av = integers(m, k, 1, seed=1)
    w, wv = integers(n, k, 128, seed=2)
    bias = torch.arange(n).float().cuda() % 13 - 6
    res = None if res_dtype is None else (torch.arange(m * n).reshape(m, n) % 19 - 9).to(res_dtype).cuda()
    for relu in (False, True):
        want, _ = ref.linear(av, wv, f64(bias), relu, None if res is None else f64(res))
        got = fp8_linear(a, w, bias=bias, relu=relu, residual=res, out_dtype=out_dtype)
        assert got.dtype == out_dtype
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(out_dtype))
        out = torch.full((m + 1, n + 5), 7.0, dtype=out_dtype, device="cuda")
        fp8_linear(a, w, bias=bias, relu=relu, residual=res, out_dtype=out_dtype, out=out[:m, 2:n + 2])
        assert torch.equal(out[:m, 2:n + 2], got)
        out[:m, 2:n + 2] = 7
        assert bool((out == 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 250, 784), (16, 512, 4096), (20, 384, 512), (140, 513, 300), (600, 1000, 384),
                                   (1030, 256, 128), (1290, 2051, 200), (2100, 2304, 130), (3000, 1984, 512)])
def test_linear_quantized_output(m, n, k):
    a, av = integers(m, k, 1, seed=3)
    w, wv = integers(n, k, 128, seed=4)
    bias = torch.arange(n).float().cuda() % 13 - 6
    want, _ = ref.linear(av, wv, f64(bias), True)
    v, s = ref.quantize(want)
    out, check = guarded(m, n)
    got = fp8_linear(a, w, bias=bias, relu=True, quantize=True, out=out)
    check()
    assert same(f64(got.scales), s) and same(f64(got.data), v)
    res = torch.randn(m, n, device="cuda")
    want, _ = ref.linear(av, wv, f64(bias), True, f64(res))
    got = fp8_linear(a, w, bias=bias, relu=True, residual=res, quantize=True)
    check_block(got, want, (np.abs(want) + np.abs(f64(res))) * EPS32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (40, 1000, 300), (300, 512, 512), (2100, 2304, 130), (1290, 2051, 200)])
def test_linear_adds_to_its_output_in_place(m, n, k, dtype):
    a, av = integers(m, k, 1, seed=5)
    w, wv = integers(n, k, 128, seed=6)
    x = (torch.arange(m * n).reshape(m, n) % 19 - 9).to(dtype).cuda()
    want, _ = ref.linear(av, wv, None, False, f64(x))
    y = fp8_linear(a, w, residual=x, out_dtype=dtype, out=x)
    assert y is x and torch.equal(y.cpu(), torch.from_numpy(want).float().to(dtype))


@pytest.mark.parametrize("m,n,k", [(3, 300, 200), (300, 512, 512), (2100, 2304, 130)])
def test_linear_infinities_in_a_quantized_output(m, n, k):
    """An infinite sum is stored as NaN and leaves its block's scale to the finite ones."""
    a, av = integers(m, k, 1, seed=7)
    w, wv = integers(n, k, 128, seed=8)
    bias = torch.zeros(n, device="cuda")
    bias[5], bias[n - 1] = float("inf"), float("-inf")
    want, _ = ref.linear(av, wv, f64(bias))
    v, s = ref.quantize(want)
    got = fp8_linear(a, w, bias=bias, quantize=True)
    assert same(f64(got.scales), s) and same(f64(got.data), v)


def linear_bound(k, mass):
    """fp32 accumulation of k exact products in any order, each step off by at
    most a whole unit (the tensor cores' alignment truncates): k 2^-23 of
    sum |a||w|."""
    return k * 2.0 ** -23 * mass


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (16, 300, 8192), (40, 512, 1000), (333, 250, 784), (600, 1024, 2048),
                                   (1500, 2304, 4096)])
def test_linear_of_quantized_normals(m, n, k):
    x, wt = randn(m, k, seed=5) * 3, randn(n, k, seed=6) / k ** 0.5
    a, w = quantize_rows(x), quantize_weight(wt)
    av, sa = ref.quantize(f64(x))
    wv, sw = ref.quantize(f64(wt), 128)
    want, mass = ref.linear(av * ref.spread(sa, 1, av.shape), wv * ref.spread(sw, 128, wv.shape))
    got = fp8_linear(a, w)
    assert np.all(np.abs(f64(got) - want) <= linear_bound(k, mass) + np.abs(want) * EPS32)
    rel = np.linalg.norm(f64(got) - want) / np.linalg.norm(want)
    assert rel < 1e-6  # errors of single steps are independent: far below the bound
    plain = fp8_linear(x, w)
    assert torch.equal(plain, got)


def test_linear_extreme_scales():
    """Scales near both ends whose products are ordinary numbers."""
    for e in (-100, -60, 60, 100):
        d = torch.ones(4, 256).to(torch.float8_e4m3fn).cuda()
        sa = torch.full((4, 2), 2.0 ** e).to(torch.float8_e8m0fnu).cuda()
        sw = torch.full((1, 2), 2.0 ** -e).to(torch.float8_e8m0fnu).cuda()
        y = fp8_linear(Fp8Rows.pack(d, sa), Fp8Weight.pack(d, sw))
        assert bool((y == 256).all())


@pytest.mark.parametrize("m", [3, 40, 200, 600, 20000])
def test_linear_nan_stays_in_its_row(m):
    x, wt = randn(m, 300), randn(140, 300, seed=1)
    w = quantize_weight(wt)
    clean = fp8_linear(quantize_rows(x), w, relu=True)
    x[1, 250] = float("nan")
    got = fp8_linear(quantize_rows(x), w, relu=True)
    assert bool(got[1].isnan().all())
    keep = torch.arange(m, device="cuda") != 1
    assert torch.equal(got[keep], clean[keep])
    q = fp8_linear(quantize_rows(x), w, quantize=True)
    assert bool(q.data.float()[1].isnan().all()) and not bool(q.data.float()[keep].isnan().any())


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (7, 512, 2048), (40, 512, 2048), (130, 512, 2048), (300, 512, 2048),
                                   (900, 512, 2048), (1900, 2304, 512)])
def test_linear_ignores_what_lies_around_its_operands(m, n, k):
    """Columns past k, scales past the last block and rows past the last hold NaN; k ends inside a block."""
    k -= 100
    a, av = integers(m, k, 1, seed=8)
    w, wv = integers(n, k, 128, seed=9)

    def surround(q, cls):
        rows, cols = q.data.shape
        d = torch.full((rows + 2, 2176), 0x7F, dtype=torch.uint8, device="cuda")
        s = torch.full((q.scales.shape[0] + 2, 24), 0xFF, dtype=torch.uint8, device="cuda")
        d[:rows, :cols] = q.data.view(torch.uint8)
        s[:q.scales.shape[0], :q.scales.shape[1]] = q.scales.view(torch.uint8)
        return cls(d.view(torch.float8_e4m3fn)[:rows, :cols],
                   s.view(torch.float8_e8m0fnu)[:q.scales.shape[0], :q.scales.shape[1]])
    want, _ = ref.linear(av, wv)
    assert same(f64(fp8_linear(surround(a, Fp8Rows), surround(w, Fp8Weight))), want)


# ---------------------------------------------------------------------------
# together, streams and graphs
# ---------------------------------------------------------------------------
def block(x, res, g, w1, b1, w2, b2):
    """A residual block as it would be used: norm, two quantised layers."""
    h, res = rms_norm(x, g, residual=res, quantize=True)
    h = fp8_linear(h, w1, bias=b1, relu=True, quantize=True)
    return fp8_linear(h, w2, bias=b2, residual=res, out_dtype=x.dtype), res


@pytest.fixture(scope="module")
def layers():
    k, n = 500, 1030
    w1, w2 = randn(n, k, seed=11) / k ** 0.5, randn(k, n, seed=12) / n ** 0.5
    return randn(k, seed=13) * 0.1 + 1, quantize_weight(w1), randn(n, seed=14), quantize_weight(w2), randn(k, seed=15)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 5, 16, 70, 400, 3000])
def test_block_of_operators(m, dtype, layers):
    """Each operator against float64 on the values its predecessor returned, then the chain's own error: three
    roundings to e4m3 (2^-4 each, of values whose errors average out) stay below a tenth of the result."""
    g, w1, b1, w2, b2 = layers
    x, res = randn(m, 500, seed=m, dtype=dtype), randn(m, 500, seed=m + 1, dtype=dtype)
    y, h = block(x, res, g, w1, b1, w2, b2)
    q, _ = rms_norm(x, g, residual=res, quantize=True)
    z = fp8_linear(q, w1, bias=b1, relu=True, quantize=True)
    v1, m1 = ref.linear(f64(q.dequantize()), f64(w1.dequantize()), f64(b1), True)
    check_block(z, v1, linear_bound(500, m1) + (np.abs(v1) + np.abs(f64(b1))) * 2 * EPS32)
    v2, m2 = ref.linear(f64(z.dequantize()), f64(w2.dequantize()), f64(b2), False, f64(h))
    check_plain(y, v2, dtype, 4 * EPS32, linear_bound(1030, m2) + (np.abs(f64(b2)) + np.abs(f64(h))) * 2 * EPS32)
    e, eh = ref.rms_norm(f64(x), f64(g), 1e-6, f64(res))
    e, _ = ref.linear(e, f64(w1.dequantize()), f64(b1), True)
    e, _ = ref.linear(e, f64(w2.dequantize()), f64(b2), False, eh)
    assert np.linalg.norm(f64(y) - e) < 0.1 * np.linalg.norm(e)


@pytest.mark.parametrize("m", [1, 70, 600, 3000])
def test_block_in_a_graph_and_on_two_streams(m, layers):
    x, res = randn(m, 500, seed=1), randn(m, 500, seed=2)
    x2, res2 = randn(m, 500, seed=3), randn(m, 500, seed=4)
    want, want2 = block(x, res, *layers)[0], block(x2, res2, *layers)[0]
    xs, rs = x.clone(), res.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = block(xs, rs, *layers)[0]
    for a, b, w in ((x, res, want), (x2, res2, want2), (x, res, want)):
        xs.copy_(a)
        rs.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s1):
            y1 = block(x, res, *layers)[0]
        with torch.cuda.stream(s2):
            y2 = block(x2, res2, *layers)[0]
        torch.cuda.synchronize()
        assert torch.equal(y1, want) and torch.equal(y2, want2)


def test_calls_from_several_threads(layers):
    """Four threads, a stream each, one and many tokens at once."""
    sizes = (1, 33, 700, 3000)
    want = [block(randn(m, 500, seed=m), randn(m, 500, seed=m + 1), *layers)[0] for m in sizes]
    torch.cuda.synchronize()
    got = [None] * len(sizes)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = block(randn(sizes[i], 500, seed=sizes[i]), randn(sizes[i], 500, seed=sizes[i] + 1), *layers)[0]
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_graphs_replayed_at_once(layers):
    """There is no workspace for them to share."""
    graphs = []
    for seed in (1, 2):
        x, res = randn(200, 500, seed=seed), randn(200, 500, seed=seed + 5)
        want = block(x, res, *layers)[0]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            y = block(x, res, *layers)[0]
        graphs.append((graph, torch.cuda.Stream(), y, want, x, res))
    for _ in range(20):
        for graph, stream, *_rest in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, _, y, want, _, _ in graphs)


def test_graph_with_branches(layers):
    """Captured on two streams that fork and join: operators with more than one predecessor."""
    xs = [randn(m, 500, seed=m) for m in (3, 900)]
    rs = [randn(m, 500, seed=m + 1) for m in (3, 900)]
    want = [block(x, r, *layers)[0] for x, r in zip(xs, rs)]
    want.append(rms_norm(want[0], residual=want[1][:3])[0])
    torch.cuda.synchronize()
    main, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        y0 = block(xs[0], rs[0], *layers)[0]
        with torch.cuda.stream(side):
            y1 = block(xs[1], rs[1], *layers)[0]
        main.wait_stream(side)
        y2 = rms_norm(y0, residual=y1[:3])[0]
    for _ in range(5):
        for y in (y0, y1, y2):
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((y0, y1, y2), want))


def test_first_call_inside_a_capture():
    """In a process of its own: set-up and code loading happen while a stream is being captured."""
    code = """
import torch
from forgetune_b200 import quantize_rows, quantize_weight, rms_norm, fp8_linear
x = torch.randn(700, 512, device="cuda")
w = torch.randn(2000, 512, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    h, r = rms_norm(x, residual=x, quantize=True)
    y = fp8_linear(h, quantize_weight(w))
    z = fp8_linear(quantize_rows(x[:2]), quantize_weight(w))
g.replay()
h, r = rms_norm(x, residual=x, quantize=True)
assert torch.equal(y, fp8_linear(h, quantize_weight(w)))
assert torch.equal(z, fp8_linear(quantize_rows(x[:2]), quantize_weight(w)))
print("captured")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_views_that_stand_for_other_values():
    """Negated views, requires_grad leaves, bias and weight as strided vectors."""
    z = torch.randn(4, 300, dtype=torch.complex64, device="cuda")
    x = z.conj().imag  # a view with the negative bit
    assert x.is_neg()
    check_quantized(quantize_rows(x), x.clone(), 1)
    assert torch.equal(rms_norm(x), rms_norm(x.clone()))
    w = torch.nn.Parameter(randn(140, 300))
    wq = quantize_weight(w)
    assert not wq.data.requires_grad
    b = randn(140, 2)[:, 0]
    got = fp8_linear(x, wq, bias=b)
    assert torch.equal(got, fp8_linear(x.clone(), wq, bias=b.contiguous())) and not got.requires_grad
    g = randn(1).expand(300)
    assert torch.equal(rms_norm(x, g), rms_norm(x, g.contiguous()))


def test_offsets_past_32_bits():
    """Rows that begin beyond 2^31 elements (and bytes) of their matrix."""
    m, k = 270000, 8192
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = randn(3, k, dtype=torch.bfloat16)
    check_quantized(Fp8Rows((q := quantize_rows(x)).data[-3:], q.scales[-3:]), x[-3:], 1)
    del q
    y, h = rms_norm(x, residual=x)
    want, _ = ref.rms_norm(f64(x[-3:]) * 2, None, 1e-6)
    check_plain(y[-3:], want, torch.bfloat16, norm_bound(k))
    del x, y, h
    m, n, k = 70000, 32768, 128
    a, av = integers(m, k, 1, seed=1)
    w, wv = integers(n, k, 128, seed=2)
    y = fp8_linear(a, w)
    want, _ = ref.linear(av[-2:], wv)
    assert same(f64(y[-2:]), want)
    want, _ = ref.linear(av[:2], wv)
    assert same(f64(y[:2]), want)


@pytest.mark.parametrize("m", [3, 3000])
def test_a_wait_that_runs_out_is_reported_and_recoverable(m, layers):
    """The hook makes the MMA warp wait for what nothing completes; the kernel leaves after its limit, the next
    call reports it, and the one after works."""
    x, res = randn(m, 500, seed=1), randn(m, 500, seed=2)
    want = block(x, res, *layers)[0]
    q = quantize_rows(x)
    _native.lib().ftb_fp8_set_fault_injection(1)
    try:
        fp8_linear(q, layers[1])
        torch.cuda.synchronize()
    finally:
        _native.lib().ftb_fp8_set_fault_injection(0)
    with pytest.raises(ft.ForgeTuneRuntimeError, match="exceeded its limit"):
        fp8_linear(q, layers[1])
    assert torch.equal(block(x, res, *layers)[0], want)


def test_empty_batch():
    w = quantize_weight(randn(130, 200))
    x = torch.empty(0, 200, device="cuda")
    q = quantize_rows(x)
    assert tuple(q.shape) == (0, 200) and tuple(q.scales.shape) == (0, 2)
    assert tuple(fp8_linear(q, w).shape) == (0, 130)
    assert tuple(fp8_linear(q, w, quantize=True).shape) == (0, 130)
    y, h = rms_norm(x, residual=x)
    assert tuple(y.shape) == tuple(h.shape) == (0, 200)


def test_refusals_on_device_tensors():
    x = randn(4, 256)
    q, w = quantize_rows(x), quantize_weight(randn(128, 256))
    with pytest.raises(InvalidShapeError):
        fp8_linear(quantize_rows(randn(4, 255)), w)
    with pytest.raises(InvalidShapeError):
        fp8_linear(q, w, bias=randn(127))
    with pytest.raises(InvalidShapeError):
        fp8_linear(q, w, residual=randn(4, 127))
    with pytest.raises(TypeError):
        fp8_linear(q, w, bias=randn(128).half())
    with pytest.raises(TypeError):
        fp8_linear(q, q)
    with pytest.raises(TypeError):
        fp8_linear(q, w, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        rms_norm(x.double())
    with pytest.raises(TypeError):
        rms_norm(x, residual=x.half())
    with pytest.raises(ValueError):
        rms_norm(x, residual_out=x)
    with pytest.raises(ValueError):
        fp8_linear(q, w, bias=torch.zeros(128))
    with pytest.raises(InvalidShapeError):
        fp8_linear(q, w, out=torch.empty(128, 4, device="cuda").t())
    with pytest.raises(InvalidShapeError):
        rms_norm(x, out=torch.empty(1, 256, device="cuda").expand(4, 256))
    odd = torch.empty(4, 265, dtype=torch.float8_e4m3fn, device="cuda")[:, 1:257]
    with pytest.raises(InvalidShapeError, match="pack"):
        fp8_linear(Fp8Rows(odd, q.scales), w)
    with pytest.raises(ft.ForgeTuneRuntimeError, match="eps"):
        rms_norm(x, eps=-1.0)
    with pytest.raises(ft.ForgeTuneRuntimeError, match="overlaps"):
        rms_norm(x, residual=x, out=x, residual_out=x)
    with pytest.raises(ft.ForgeTuneRuntimeError, match="overlaps"):
        fp8_linear(q, quantize_weight(randn(256, 256)), quantize=True, out=q)
    with pytest.raises(ValueError):
        fp8_linear(q, w, quantize=True, out_dtype=torch.float32)
