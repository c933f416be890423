"""Block-scaled 8-bit operators without a GPU: refusals of the C ABI and of
the Python entry points, and the format's container."""

import ctypes
import os
import struct
import subprocess

import numpy as np
import pytest
import torch

from forgetune_b200 import (Fp8Rows, Fp8Weight, InvalidShapeError, _native, fp8_linear, quantize_rows,
                            quantize_weight, rms_norm)

from . import fp8_reference as ref

P = 1 << 20  # a well aligned address that no refused call touches

# the argument structs of include/forgetune_b200.h, every field of eight bytes
QUANTIZE_ARGS = struct.Struct("=9q")  # x (data, ld, type), q (data, ld, scales, ld), m, k
RMS_NORM_ARGS = struct.Struct("=7qd12q")  # x, residual, weight, eps, h, y, q, m, k
LINEAR_ARGS = struct.Struct("=23q")  # a, w, bias, residual, y, q, m, n, k, flags


def rc(name, fmt, *args):
    return getattr(_native.lib(), name)(ctypes.c_char_p(fmt.pack(*args)), None)


@pytest.mark.parametrize("name", ["ftb_quantize_rows", "ftb_quantize_weight"])
def test_quantize_refusals(name):
    def call(x=P, x_ld=200, t=0, q=P, q_ld=208, s=P, s_ld=4, m=3, k=200):
        return rc(name, QUANTIZE_ARGS, x, x_ld, t, q, q_ld, s, s_ld, m, k)
    assert call(m=0) == 0
    assert getattr(_native.lib(), name)(None, None) == -1
    assert call(x=0) == call(q=0) == call(s=0) == -1
    for bad in (dict(m=-1), dict(k=0), dict(m=1 << 31), dict(k=1 << 31), dict(t=3), dict(t=-1), dict(x=P + 2),
                dict(x_ld=199), dict(q=P + 8), dict(q_ld=200), dict(q_ld=192), dict(s=P + 2), dict(s_ld=2),
                dict(s_ld=0), dict(s_ld=6)):
        assert call(**bad) == -2, bad
        assert name in _native.last_error()


def test_rms_norm_refusals():
    def call(x=P, x_ld=200, t=2, r=P, r_ld=200, rt=2, w=P, eps=1e-6, h=P, h_ld=200, ht=2, y=P, y_ld=208, yt=2, q=0,
             q_ld=208, s=0, s_ld=4, m=3, k=200):
        return rc("ftb_rms_norm", RMS_NORM_ARGS, x, x_ld, t, r, r_ld, rt, w, eps, h, h_ld, ht, y, y_ld, yt, q,
                  q_ld, s, s_ld, m, k)
    fp8_out = dict(y=0, q=P, s=P)
    assert call(m=0) == 0
    assert _native.lib().ftb_rms_norm(None, None) == -1
    assert call(x=0) == call(y=0) == call(y=0, q=P) == -1
    for bad in (dict(m=-1), dict(k=0), dict(t=3), dict(t=9), dict(yt=0), dict(rt=1), dict(ht=7), dict(r=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=P + 1), dict(x_ld=1), dict(r=P + 1), dict(r_ld=7),
                dict(w=P + 2), dict(h=P + 1), dict(h_ld=0), dict(y=P + 1), dict(y_ld=199), dict(q=P, s=P),
                dict(fp8_out, q=P + 8), dict(fp8_out, q_ld=200), dict(fp8_out, s=P + 3), dict(fp8_out, s_ld=1)):
        assert call(**bad) == -2, bad


def test_linear_refusals():
    def call(a=P, a_ld=208, sa=P, sa_ld=4, w=P, w_ld=208, sw=P, sw_ld=4, bias=P, res=P, r_ld=130, rt=0, y=P,
             y_ld=144, yt=0, q=0, q_ld=144, s=0, s_ld=4, m=3, n=130, k=200, flags=1):
        return rc("ftb_fp8_linear", LINEAR_ARGS, a, a_ld, sa, sa_ld, w, w_ld, sw, sw_ld, bias, res, r_ld, rt, y,
                  y_ld, yt, q, q_ld, s, s_ld, m, n, k, flags)
    fp8_out = dict(y=0, q=P, s=P)
    assert call(m=0) == 0
    assert _native.lib().ftb_fp8_linear(None, None) == -1
    for bad in ("a", "sa", "w", "sw", "y"):
        assert call(**{bad: 0}) == -1
    assert call(y=0, q=P) == -1
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(m=1 << 31), dict(flags=2), dict(yt=4), dict(rt=3),
                dict(a=P + 8), dict(a_ld=200), dict(sa=P + 1), dict(sa_ld=5), dict(w=P + 1), dict(w_ld=192),
                dict(sw=P + 2), dict(sw_ld=0), dict(bias=P + 2), dict(res=P + 2), dict(r_ld=129), dict(y=P + 2),
                dict(y_ld=129), dict(q=P, s=P), dict(fp8_out, q=P + 8), dict(fp8_out, q_ld=130),
                dict(fp8_out, s=P + 2), dict(fp8_out, s_ld=1)):
        assert call(**bad) == -2, bad


def test_scales_over_their_own_values_are_refused():
    B = 1 << 24  # far from P

    def calls(s, s_ld=512):
        yield rc("ftb_quantize_rows", QUANTIZE_ARGS, P, 512, 0, B, 512, s, s_ld, 4, 200)
        yield rc("ftb_quantize_weight", QUANTIZE_ARGS, P, 512, 0, B, 512, s, s_ld, 4, 200)
        yield rc("ftb_rms_norm", RMS_NORM_ARGS, P, 512, 0, 0, 0, 0, 0, 1e-6, 0, 0, 0, 0, 0, 0, B, 512, s, s_ld, 4, 200)
        yield rc("ftb_fp8_linear", LINEAR_ARGS, P, 512, 2 * B, 4, 3 * B, 512, 4 * B, 4, 0, 0, 0, 0, 0, 0, 0, B, 512, s,
                 s_ld, 4, 200, 200, 0)
    for s, s_ld in ((B, 512), (B + 196, 512), (B + 512, 4), (B + 3 * 512 + 8, 4)):
        for got in calls(s, s_ld):
            assert got == -2 and "overlap" in _native.last_error(), (s - B, s_ld)
    if _native.device_count() == 0:  # the scales behind each row's values, or behind them all
        for s, s_ld in ((B + 208, 512), (B + 4 * 512, 4)):
            for got in calls(s, s_ld):
                assert got == -5, _native.last_error()


def test_outputs_over_operands_are_refused():
    """Overlaps other than in place; side by side in one buffer's rows is none."""
    B = 1 << 24  # far from P

    def quantize(x, q, s):
        return rc("ftb_quantize_rows", QUANTIZE_ARGS, x, 512, 0, q, 2048, s, 2048, 4, 200)
    assert quantize(P, P, B) == -2 and "overlaps" in _native.last_error()
    assert quantize(P, P + 784, B) == -2  # x's rows have 800 bytes each 2048
    assert quantize(P, B, P + 2048) == -2

    def norm(**over):
        a = dict(x=P, r=2 * B, w=3 * B, h=4 * B, y=5 * B, q=0, s=0, ld=256)
        a.update(over)
        ld = a["ld"]
        return rc("ftb_rms_norm", RMS_NORM_ARGS, a["x"], ld, 0, a["r"], ld, 0, a["w"], 1e-6, a["h"], ld, 0, a["y"], ld,
                  0, a["q"], 256, a["s"], 4, 4, 200)
    for bad in (dict(h=P + 4), dict(y=P + 16), dict(h=5 * B), dict(h=P, y=P), dict(y=3 * B), dict(h=3 * B + 400),
                dict(y=0, q=P, s=B), dict(y=0, q=B, s=P + 800 - 4), dict(y=0, q=4 * B + 16, s=B)):
        assert norm(**bad) == -2 and "overlaps" in _native.last_error(), bad

    def linear(**over):
        a = dict(y=B, res=2 * B, bias=3 * B, a=4 * B, sa=5 * B, w=6 * B, sw=7 * B, q=0, s=0, yt=0, rt=0)
        a.update(over)
        return rc("ftb_fp8_linear", LINEAR_ARGS, a["a"], 256, a["sa"], 4, a["w"], 256, a["sw"], 4, a["bias"], a["res"],
                  130, a["rt"], a["y"], 130, a["yt"], a["q"], 144, a["s"], 4, 3, 130, 200, 0)
    for bad in (dict(y=2 * B + 4), dict(y=2 * B, yt=1), dict(y=3 * B), dict(y=4 * B), dict(y=5 * B), dict(y=6 * B),
                dict(y=7 * B), dict(y=0, q=4 * B, s=B), dict(y=0, q=B, s=5 * B), dict(y=0, q=2 * B, s=B)):
        assert linear(**bad) == -2 and "overlaps" in _native.last_error(), bad
    # allowed as far as the checks go: without a GPU the next step is the device
    if _native.device_count() == 0:
        for good in (norm(), norm(h=P), norm(y=P), norm(h=2 * B), norm(h=P, y=2 * B), norm(ld=512, h=P + 800),
                     linear(), linear(y=2 * B), quantize(P, P + 800, B)):
            assert good == -5, _native.last_error()


def test_one_row_outputs_over_operands_are_refused():
    """The same for one row, where both spans may be without a stride (a norm weight, a bias)."""
    B = 1 << 24  # far from P

    def quantize(name, x, q, s):
        return rc(name, QUANTIZE_ARGS, x, 256, 0, q, 256, s, 4, 1, 200)
    for name in ("ftb_quantize_rows", "ftb_quantize_weight"):
        for x, q, s in ((P, P, B), (P, P + 784, B), (P, B, P + 400), (P, B, B), (P, B, B + 196)):
            assert quantize(name, x, q, s) == -2 and "overlap" in _native.last_error(), (name, x - P, q - P, s - P)

    def norm(**over):
        a = dict(x=P, r=2 * B, w=3 * B, h=4 * B, y=5 * B, q=0, s=0)
        a.update(over)
        return rc("ftb_rms_norm", RMS_NORM_ARGS, a["x"], 256, 0, a["r"], 256, 0, a["w"], 1e-6, a["h"], 256, 0, a["y"],
                  256, 0, a["q"], 256, a["s"], 4, 1, 200)
    for bad in (dict(h=P + 4), dict(y=P + 16), dict(h=5 * B), dict(h=P, y=P), dict(y=3 * B), dict(y=3 * B + 796),
                dict(y=3 * B - 796), dict(h=3 * B), dict(h=3 * B + 400), dict(y=0, q=P, s=B), dict(y=0, q=B, s=P + 796),
                dict(y=0, q=4 * B + 16, s=B), dict(y=0, q=3 * B, s=B), dict(y=0, q=3 * B + 784, s=B),
                dict(y=0, q=B, s=3 * B), dict(y=0, q=B, s=3 * B + 796)):
        assert norm(**bad) == -2 and "overlaps" in _native.last_error(), bad

    def linear(**over):
        a = dict(y=B, res=2 * B, bias=3 * B, a=4 * B, sa=5 * B, w=6 * B, sw=7 * B, q=0, s=0, yt=0, rt=0)
        a.update(over)
        return rc("ftb_fp8_linear", LINEAR_ARGS, a["a"], 256, a["sa"], 4, a["w"], 256, a["sw"], 4, a["bias"], a["res"],
                  130, a["rt"], a["y"], 130, a["yt"], a["q"], 144, a["s"], 4, 1, 130, 200, 0)
    for bad in (dict(y=2 * B + 4), dict(y=2 * B, yt=1), dict(y=3 * B), dict(y=3 * B + 516), dict(y=3 * B - 516),
                dict(y=4 * B), dict(y=5 * B), dict(y=6 * B), dict(y=7 * B), dict(y=0, q=4 * B, s=B),
                dict(y=0, q=B, s=5 * B), dict(y=0, q=2 * B, s=B), dict(y=0, q=3 * B, s=B), dict(y=0, q=3 * B + 512, s=B),
                dict(y=0, q=B, s=3 * B), dict(y=0, q=B, s=3 * B + 516)):
        assert linear(**bad) == -2 and "overlaps" in _native.last_error(), bad
    # allowed as far as the checks go: in place, or right behind the operand
    if _native.device_count() == 0:
        for good in (norm(), norm(h=P), norm(y=P), norm(h=2 * B), norm(h=P, y=2 * B), norm(y=3 * B + 800),
                     norm(y=3 * B - 800), norm(y=0, q=3 * B + 800, s=3 * B + 1008), linear(), linear(y=2 * B),
                     linear(y=3 * B + 520), linear(y=3 * B - 520), quantize("ftb_quantize_rows", P, P + 800, P + 1008)):
            assert good == -5, _native.last_error()


def test_kernel_hook_refuses_kernels_that_do_not_exist():
    hook = _native.lib().ftb_fp8_set_kernel
    try:
        for nt in (16, 32, 64, 128):
            for split in (1, 2, 4, 8):
                assert hook(nt, split) == 0
        assert hook(0, 1) == 0 and hook(-1, 0) == 0
        for nt, split in ((48, 1), (256, 1), (16, 0), (16, 3), (16, 16), (0, 0), (0, 2), (-2, 1), (128, -1), (1 << 30, 1)):
            assert hook(nt, split) == -2 and "ftb_fp8_set_kernel" in _native.last_error(), (nt, split)
    finally:
        assert hook(-1, 0) == 0


def fp8(*shape):
    return torch.zeros(*shape).to(torch.float8_e4m3fn)


def scale(*shape):
    return torch.ones(*shape).to(torch.float8_e8m0fnu)


def test_containers_check_their_parts():
    Fp8Rows(fp8(3, 200), scale(3, 2))
    Fp8Weight(fp8(130, 200), scale(2, 2))
    with pytest.raises(TypeError):
        Fp8Rows(torch.zeros(3, 200), scale(3, 2))
    with pytest.raises(TypeError):
        Fp8Rows(fp8(3, 200), torch.ones(3, 2))
    for cls, d, s in ((Fp8Rows, fp8(3, 200), scale(3, 1)), (Fp8Weight, fp8(130, 200), scale(130, 2)),
                      (Fp8Rows, fp8(200), scale(2)), (Fp8Rows, fp8(3, 0), scale(3, 0))):
        with pytest.raises(InvalidShapeError):
            cls(d, s)


def test_pack_lays_rows_out_and_keeps_the_values():
    g = torch.Generator().manual_seed(0)
    d = torch.randn(5, 77, generator=g).to(torch.float8_e4m3fn)
    s = (2.0 ** torch.randint(-3, 3, (5, 1), generator=g).float()).to(torch.float8_e8m0fnu)
    q = Fp8Rows.pack(d, s)
    assert q.data.stride() == (80, 1) and q.scales.stride() == (4, 1)
    assert np.array_equal(q.dequantize().numpy(), d.float().numpy() * s.float().numpy())
    again = Fp8Rows.pack(q.data, q.scales)
    assert again.data.data_ptr() == q.data.data_ptr() and again.scales.data_ptr() == q.scales.data_ptr()
    t = Fp8Weight.pack(fp8(77, 5).t(), scale(1, 1))  # columns in place of rows
    assert t.data.stride() == (80, 1)


def test_entry_points_refuse_host_tensors():
    x = torch.zeros(2, 128)
    q, w = Fp8Rows.pack(fp8(2, 128), scale(2, 1)), Fp8Weight.pack(fp8(128, 128), scale(1, 1))
    for call in (lambda: quantize_rows(x), lambda: quantize_weight(x), lambda: rms_norm(x), lambda: fp8_linear(x, w),
                 lambda: fp8_linear(q, w), lambda: quantize_rows(None), lambda: fp8_linear(q, x)):
        with pytest.raises(TypeError):
            call()


def test_reference_rounds_to_the_nearest_e4m3_value():
    """The reference's rounding against torch's conversion on every border between two e4m3 values."""
    bits = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    mid = (bits[1:] + bits[:-1]) / 2
    v = np.concatenate([bits, mid, np.nextafter(mid.astype(np.float32), np.float32(0)).astype(np.float64),
                        np.nextafter(mid.astype(np.float32), np.float32(999)).astype(np.float64)])
    v = np.concatenate([v, -v])
    want = torch.from_numpy(v).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.e4m3(v), want)
    assert ref.scale_exponent(np.array([0.0, 448.0, 448.1, 1.0, 1e-45, 3.4e38])).tolist() == [0, 0, 1, -8, -127, 120]


def test_argument_structs_match_the_header(tmp_path):
    """The packed arguments have the header's sizes and constants, as a C compiler sees them."""
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "forgetune_b200.h"\nint main(void) { printf("%d %d %d %d %d %d %d\\n", '
                   "(int)sizeof(ftb_quantize_args), (int)sizeof(ftb_rms_norm_args), (int)sizeof(ftb_fp8_linear_args), "
                   "FTB_F32, FTB_F16, FTB_BF16, FTB_FP8_RELU); return 0; }\n")
    include = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "t")], check=True)
    got = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [QUANTIZE_ARGS.size, RMS_NORM_ARGS.size, LINEAR_ARGS.size, 0, 1, 2, 1]


def test_containers_refuse_negated_views():
    """A view that stands for the negated values has the values' own bytes."""
    d, s = fp8(3, 200), scale(3, 2)
    for cls, dd, ss in ((Fp8Rows, torch._neg_view(d), s), (Fp8Rows, d, torch._neg_view(s)),
                        (Fp8Weight, torch._neg_view(d), scale(1, 2))):
        for make in (cls, cls.pack):
            with pytest.raises(TypeError, match="negat"):
                make(dd, ss)
