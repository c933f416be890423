"""The matrix product's kernels one by one: every tile size, depth split and
output path against float64, exact by integers (see integers)."""

import contextlib
import threading

import numpy as np
import pytest
import torch

from forgetune_b200 import ForgeTuneRuntimeError, _native, fp8_linear, quantize_rows, quantize_weight

from . import fp8_reference as ref
from .test_fp8_gpu import TYPES, f64, guarded, integers, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,offset", [(4000, 2320, 0), (4000, 2304, 1), (2600, 4112, 0)])
def test_residual_boxes_after_boxes_stored_by_rows(m, n, offset, dtype):
    """Residual rows on 16-byte boundaries come in by TMA through the box that the output leaves by rows: at the
    right edge, or everywhere where the output is off the boundaries.  Several tiles per pair."""
    a, av = integers(m, 128, 1, seed=1)
    w, wv = integers(n, 128, 128, seed=2)
    res = (torch.arange(m * n).reshape(m, n) % 19 - 9).to(dtype).cuda()
    want, _ = ref.linear(av, wv, None, True, f64(res))
    out = torch.full((m, n + 8), 7.0, dtype=dtype, device="cuda")
    for _ in range(3):
        fp8_linear(a, w, relu=True, residual=res, out_dtype=dtype, out=out[:, offset:n + offset])
        assert torch.equal(out[:, offset:n + offset].cpu(), torch.from_numpy(want).float().to(dtype))
    assert bool((out[:, :offset] == 7).all()) and bool((out[:, n + offset:] == 7).all())


# tokens per tile and CTAs that share a tile's depth; (0, 1): SM pairs
KERNELS = [(nt, split) for nt in (16, 32, 64, 128) for split in (1, 2, 4, 8)] + [(0, 1)]


@contextlib.contextmanager
def kernel(nt, split):
    assert _native.lib().ftb_fp8_set_kernel(nt, split) == 0
    try:
        yield
    finally:
        assert _native.lib().ftb_fp8_set_kernel(-1, 0) == 0


def shapes(nt):
    """Tokens that end inside a tile, outputs that end inside a block (and off four columns), and depths of one
    block, of two groups of four (CTAs 2 .. 7 of a cluster have none), of nine (CTAs 5 .. 7 of eight have none,
    and the rest two, the last one of them one) and of sixteen."""
    tile = nt or 256
    yield 2 * tile + 3, 517, 100
    yield 1, 300, 1000
    yield tile, 512, 4196
    yield tile + 9, 645, 700
    yield tile - 1, 127, 8192


@pytest.mark.parametrize("nt,split", KERNELS)
def test_every_kernel_with_every_output(nt, split):
    for m, n, k in shapes(nt):
        a, av = integers(m, k, 1, seed=m + k)
        w, wv = integers(n, k, 128, seed=n + k)
        bias = torch.arange(n).float().cuda() % 13 - 6
        ints = torch.arange(m * n).reshape(m, n) % 19 - 9
        plain, _ = ref.linear(av, wv)
        with kernel(nt, split):
            assert same(f64(fp8_linear(a, w)), plain)
            for dtype, res_dtype in zip(TYPES, TYPES[1:] + TYPES[:1]):
                res = ints.to(res_dtype).cuda()
                want, _ = ref.linear(av, wv, f64(bias), True, f64(res))
                want = torch.from_numpy(want).float().to(dtype)
                out = torch.full((m + 1, (n + 31) // 8 * 8), 7.0, dtype=dtype, device="cuda")
                for at in (0, 8, 3):  # rows on 16-byte boundaries and off them
                    fp8_linear(a, w, bias=bias, relu=True, residual=res, out_dtype=dtype, out=out[:m, at:n + at])
                    assert torch.equal(out[:m, at:n + at].cpu(), want), (m, n, k, dtype, at)
                    out[:m, at:n + at] = 7
                assert bool((out == 7).all())
                want, _ = ref.linear(av, wv, None, False, f64(res))
                fp8_linear(a, w, residual=res, out_dtype=res_dtype, out=res)  # in place
                assert torch.equal(res.cpu(), torch.from_numpy(want).float().to(res_dtype)), (m, n, k, res_dtype)
            for res in (None, ints.half().cuda(), ints.float().cuda()):
                want, _ = ref.linear(av, wv, f64(bias), True, None if res is None else f64(res))
                v, s = ref.quantize(want)
                out, check = guarded(m, n)
                fp8_linear(a, w, bias=bias, relu=True, residual=res, quantize=True, out=out)
                check()
                assert same(f64(out.scales), s) and same(f64(out.data), v), (m, n, k)


@pytest.mark.parametrize("nt,split", KERNELS)
def test_every_kernel_with_what_is_not_finite(nt, split):
    """NaN in one row of the operand, infinities in the bias: NaN where the formula has them, scales from the rest."""
    tile = nt or 256
    m, n, k = tile + 5, 389, 1100
    a, av = integers(m, k, 1, seed=3)
    w, wv = integers(n, k, 128, seed=4)
    a.data.view(torch.uint8)[tile, k - 1] = 0x7F
    av[tile, k - 1] = np.nan
    bias = torch.zeros(n, device="cuda")
    bias[5], bias[n - 1] = float("inf"), float("-inf")
    with np.errstate(invalid="ignore"):
        want, _ = ref.linear(av, wv, f64(bias))
    with kernel(nt, split):
        assert same(f64(fp8_linear(a, w, bias=bias)), want)
        got = fp8_linear(a, w, bias=bias, quantize=True)
    v, s = ref.quantize(want)
    assert same(f64(got.scales), s) and same(f64(got.data), v)


@pytest.mark.parametrize("nt,split", KERNELS)
def test_every_kernel_on_inputs_written_right_before(nt, split):
    """Operands, bias and residual change on the stream before each call and nothing is waited for: every result
    is that of its own inputs, bit for bit."""
    m, n, k = (nt or 256) + 40, 900, 1500
    sets = []
    for seed in range(3):
        a, w = integers(m, k, 1, seed=seed)[0], integers(n, k, 128, seed=seed + 50)[0]
        g = torch.Generator(device="cuda").manual_seed(seed)
        sets.append([a.data.view(torch.uint8), a.scales.view(torch.uint8), w.data.view(torch.uint8),
                     w.scales.view(torch.uint8), torch.randn(n, device="cuda", generator=g),
                     torch.randn(m, n, device="cuda", generator=g)])
    live_a, live_w = integers(m, k, 1, seed=9)[0], integers(n, k, 128, seed=9)[0]
    live = [live_a.data.view(torch.uint8), live_a.scales.view(torch.uint8), live_w.data.view(torch.uint8),
            live_w.scales.view(torch.uint8), torch.empty(n, device="cuda"), torch.empty(m, n, device="cuda")]

    def call(i):
        for t, v in zip(live, sets[i]):
            t.copy_(v)
        q = fp8_linear(live_a, live_w, bias=live[4], relu=True, residual=live[5], quantize=True)
        return fp8_linear(live_a, live_w, bias=live[4], residual=live[5]), q.data.view(torch.uint8), q.scales.view(torch.uint8)
    with kernel(nt, split):
        want = []
        for i in range(3):
            want.append(call(i))
            torch.cuda.synchronize()
        got = [call(i % 3) for i in range(12)]
    for i, g in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(g, want[i % 3])), i


def test_a_wait_that_ran_out_is_reported_to_one_of_many_threads():
    """Eight threads call at once after it: one is told, the others' calls run."""
    a, w = integers(5, 256, 1, seed=1)[0], integers(130, 256, 128, seed=2)[0]
    x = torch.randn(5, 256, device="cuda")
    want = quantize_rows(x)
    fp8_linear(a, w)
    torch.cuda.synchronize()
    _native.lib().ftb_fp8_set_fault_injection(1)
    try:
        fp8_linear(a, w)
        torch.cuda.synchronize()
    finally:
        _native.lib().ftb_fp8_set_fault_injection(0)
    told, right, start = [], [], threading.Barrier(8)

    def work():
        start.wait()
        try:
            q = quantize_rows(x)
            torch.cuda.current_stream().synchronize()
            right.append(torch.equal(q.data.view(torch.uint8), want.data.view(torch.uint8)))
        except ForgeTuneRuntimeError as e:
            told.append(str(e))
    threads = [threading.Thread(target=work) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(told) == 1 and "exceeded its limit" in told[0]
    assert len(right) == 7 and all(right)


@pytest.mark.parametrize("nt,split", KERNELS)
def test_every_kernel_right_behind_what_writes_its_operands(nt, split):
    """Weights and activations quantised into memory of the ones before, the product launched early behind them
    (its first weights are sent for before they are written)."""
    m, n, k = (nt or 256) + 40, 900, 1500
    xs = [torch.randn(m, k, device="cuda") for _ in range(3)]
    ws = [torch.randn(n, k, device="cuda") for _ in range(3)]
    with kernel(nt, split):
        want = []
        for x, w in zip(xs, ws):
            a, b = quantize_rows(x), quantize_weight(w)
            torch.cuda.synchronize()
            want.append(fp8_linear(a, b))
            torch.cuda.synchronize()
        del a, b
        places, got = set(), []
        for i in range(12):
            a, b = quantize_rows(xs[i % 3]), quantize_weight(ws[i % 3])
            places.add(b.data.data_ptr())
            got.append(fp8_linear(a, b))
            del a, b
    assert len(places) < 12  # memory is taken again
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 3]), i
