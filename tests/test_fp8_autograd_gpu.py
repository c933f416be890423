"""The 8-bit operators and autograd: they have no backward pass, and say so where it would matter."""

import pytest
import torch

from forgetune_b200 import fp8_linear, quantize_rows, quantize_weight, rms_norm

pytestmark = pytest.mark.gpu


def calls():
    """(call with `out`, the tensors it writes) for every output a caller can pass."""
    x, r = torch.randn(4, 256, device="cuda"), torch.randn(4, 256, device="cuda")
    w = quantize_weight(torch.randn(128, 256, device="cuda"))
    y, h, z = torch.empty_like(x), torch.empty_like(x), torch.empty(4, 128, device="cuda")
    q, q2 = quantize_rows(x), quantize_rows(z)
    yield lambda: quantize_rows(x, out=q), [q.data, q.scales]
    yield lambda: rms_norm(x, out=y), [y]
    yield lambda: rms_norm(x, residual=r, out=y, residual_out=h), [y, h]
    yield lambda: rms_norm(x, residual=r, residual_out=r), [r]
    yield lambda: rms_norm(x, residual=r, quantize=True, out=q, residual_out=x), [q.data, q.scales, x]
    yield lambda: fp8_linear(x, w, out=z), [z]
    yield lambda: fp8_linear(x, w, residual=z, out=z), [z]
    yield lambda: fp8_linear(x, w, quantize=True, out=q2), [q2.data, q2.scales]


def test_written_outputs_count_as_changed_in_place():
    for call, outs in calls():
        before = [t._version for t in outs]
        call()
        assert all(t._version > v for t, v in zip(outs, before))


def test_a_backward_pass_refuses_values_that_an_operator_wrote_over():
    x = torch.randn(4, 256, device="cuda", requires_grad=True)
    y = x * 2
    z = (y * y).sum()  # saves y
    rms_norm(torch.randn(4, 256, device="cuda"), out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_outputs_that_require_grad_are_refused():
    for call, outs in calls():
        outs[0].requires_grad_()
        before = outs[0].detach().clone().view(torch.uint8)
        with pytest.raises(ValueError, match="requires grad"):
            call()
        assert torch.equal(outs[0].detach().view(torch.uint8), before)
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()


def test_tensors_made_in_inference_mode_are_outputs_anywhere():
    with torch.inference_mode():
        made = list(calls())
        for call, _ in made:
            call()
    for call, _ in made:
        call()


def test_forward_mode_tangents_are_refused():
    x, r, b = torch.randn(4, 256, device="cuda"), torch.randn(4, 128, device="cuda"), torch.randn(128, device="cuda")
    g = torch.randn(256, device="cuda")
    w = quantize_weight(torch.randn(128, 256, device="cuda"))
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: quantize_rows(dual(x)), lambda: quantize_weight(dual(x)), lambda: rms_norm(dual(x)),
                     lambda: rms_norm(x, dual(g)), lambda: rms_norm(x, residual=dual(x)),
                     lambda: rms_norm(x, out=dual(x)), lambda: fp8_linear(dual(x), w),
                     lambda: fp8_linear(x, w, bias=dual(b)), lambda: fp8_linear(x, w, residual=dual(r)),
                     lambda: fp8_linear(x, w, out=dual(r))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        fp8_linear(torch.autograd.forward_ad.unpack_dual(dual(x)).primal, w)
    fp8_linear(x, w, bias=b, residual=r)
