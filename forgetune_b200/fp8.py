"""Block-scaled 8-bit operators on CUDA tensors.

A dense layer in 8 bits is a chain of three operators, each one call of the
engine library's C ABI (``ftb_quantize_rows``, ``ftb_quantize_weight``,
``ftb_rms_norm``, ``ftb_fp8_linear``; include/forgetune_b200.h) on the current
torch stream, made by the extension ``lib/_torch_ops.so`` (csrc/torch_ops.cpp),
which checks the arguments and allocates the results::

    w1 = quantize_weight(layer1.weight)                 # once, [n, k]
    h, res = rms_norm(x, norm.weight, residual=res, quantize=True)
    h = fp8_linear(h, w1, bias=layer1.bias, relu=True, quantize=True)
    x = fp8_linear(h, w2, bias=layer2.bias)

The format is e4m3 values with one power-of-two scale (ue8m0, the format the
tensor cores take) for each block of 128 along a row of activations and for
each 128 x 128 block of a weight: the smallest power of two with
``max|x| / scale <= 448``, 1 for a block of zeros.  Values that are not finite
are stored as NaN.  Products are accumulated in fp32 by the tensor cores, which
truncate where they add: relative error 5e-7 at depth 8192 for values of both
signs, 4e-6 for sums of one sign.

Inputs are 2-D; a plain input whose rows are not contiguous is copied first,
as ``CompiledModel.run_device`` does.  The operators are for inference: they
return tensors without gradients.  An
output that requires grad is refused outside ``torch.no_grad()``; writing into
a caller's tensor counts as a change in place, which a backward pass that
saved it reports.  They need no workspace, so calls may run
on several streams at once and be captured into CUDA graphs.  The reference
has no counterpart (its models are float32 only).
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native

__all__ = ["Fp8Rows", "Fp8Weight", "quantize_rows", "quantize_weight", "rms_norm", "fp8_linear"]

BLOCK = 128
_ops = None


def _load():
    global _ops
    _ops = _native.torch_ops()
    return _ops


def _laid_out(t: torch.Tensor, unit: int) -> torch.Tensor:
    """A copy in rows that start on multiples of ``unit`` elements."""
    m, k = t.shape
    return torch.empty_strided((m, k), ((k + unit - 1) // unit * unit, 1), dtype=t.dtype, device=t.device).copy_(t)


class _Fp8:
    """8-bit values [rows, k] with their block scales."""

    __slots__ = ("data", "scales")
    _row_block = 1

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        (_ops or _load()).check(data, scales, self._row_block, type(self).__name__)
        self.data = data
        self.scales = scales

    @classmethod
    def pack(cls, data: torch.Tensor, scales: torch.Tensor):
        """The same values in rows laid out as the operators need them (copied where they are not)."""
        if not (_ops or _load()).check(data, scales, cls._row_block, cls.__name__):
            data, scales = _laid_out(data, 16), _laid_out(scales, 4)
        return cls(data, scales)

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the blocks stand for."""
        rows, k = self.data.shape
        f = self.scales.float().repeat_interleave(BLOCK, 1)[:, :k]
        if self._row_block > 1:
            f = f.repeat_interleave(self._row_block, 0)[:rows]
        return (self.data.float() * f).to(dtype)


class Fp8Rows(_Fp8):
    """Quantised activations [m, k]: e4m3 ``data`` and ue8m0 ``scales`` [m, ceil(k / 128)].

    Rows of ``data`` start on 16-byte and rows of ``scales`` on 4-byte
    boundaries; :meth:`pack` lays out tensors that do not."""

    __slots__ = ()


class Fp8Weight(_Fp8):
    """A quantised weight [n, k]: e4m3 ``data`` and ue8m0 ``scales`` [ceil(n / 128), ceil(k / 128)],
    laid out like :class:`Fp8Rows`."""

    __slots__ = ()
    _row_block = BLOCK


def _new(cls, data, scales):
    """An instance of tensors that are right by construction."""
    r = cls.__new__(cls)
    r.data = data
    r.scales = scales
    return r


def _parts(out, what: str):
    """Data and scales of a caller's quantised output."""
    if not isinstance(out, Fp8Rows):
        raise TypeError("%s must be an Fp8Rows" % what)
    return out.data, out.scales


def quantize_rows(x: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """Activations [m, k] (float32, float16, bfloat16) to 8 bits with a scale for each 128 along a row."""
    ops = _ops or _load()
    if out is None:
        return _new(Fp8Rows, *ops.quantize_rows(x, None, None))
    ops.quantize_rows(x, *_parts(out, "quantize_rows: out"))
    return out


def quantize_weight(w: torch.Tensor) -> Fp8Weight:
    """A weight [n, k] (``nn.Linear``'s layout; float32, float16, bfloat16) to 8 bits with a scale for each
    128 x 128 block.  Done once, where a model is loaded."""
    return _new(Fp8Weight, *(_ops or _load()).quantize_weight(w))


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None, quantize: bool = False,
             out: Union[torch.Tensor, Fp8Rows, None] = None, residual_out: Optional[torch.Tensor] = None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the rows of ``h = x + residual``.

    ``x`` and ``residual`` are [m, k] of one type (float32, float16,
    bfloat16), ``weight`` float32 [k] or None.  The sum, the mean and the norm
    are computed in fp32 and ``y`` is rounded once: to ``x``'s type, or to an
    :class:`Fp8Rows` with ``quantize``.  Without a residual returns ``y``; with
    one returns ``(y, h)``, ``h`` in ``x``'s type.  ``out`` and
    ``residual_out`` receive them in place of new tensors; ``residual_out``
    may be ``x`` or ``residual``, ``out`` may be ``x``.
    """
    ops = _ops or _load()
    if not quantize or out is None:
        y, scales, h = ops.rms_norm(x, weight, eps, residual, quantize, out, None, residual_out)
        if quantize:
            y = _new(Fp8Rows, y, scales)
    else:
        data, scales = _parts(out, "rms_norm: out")
        h = ops.rms_norm(x, weight, eps, residual, True, data, scales, residual_out)[2]
        y = out
    return y if residual is None else (y, h)


def fp8_linear(x: Union[Fp8Rows, torch.Tensor], weight: Fp8Weight, bias: Optional[torch.Tensor] = None,
               relu: bool = False, residual: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, quantize: bool = False,
               out: Union[torch.Tensor, Fp8Rows, None] = None) -> Union[torch.Tensor, Fp8Rows]:
    """``relu(x @ weight.T + bias) + residual`` with 8-bit operands: [m, k] and [n, k] to [m, n].

    ``x`` is an :class:`Fp8Rows`, or a plain tensor that is quantised first.
    ``bias`` is float32 [n]; ``relu`` keeps NaN; ``residual`` is [m, n] of any
    plain type.  The result has ``out_dtype`` (default: the plain ``x``'s type,
    else the residual's, else float32), or is an :class:`Fp8Rows` with
    ``quantize``.  ``out`` receives it in place of a new tensor and may be
    ``residual``.
    """
    if not isinstance(weight, Fp8Weight):
        raise TypeError("fp8_linear: weight must be an Fp8Weight (see quantize_weight)")
    x, x_scales = (x.data, x.scales) if isinstance(x, Fp8Rows) else (x, None)
    ops = _ops or _load()
    if not quantize:
        return ops.linear(x, x_scales, weight.data, weight.scales, bias, relu, residual, out_dtype, False, out,
                          None)[0]
    data, scales = (None, None) if out is None else _parts(out, "fp8_linear: out")
    r = ops.linear(x, x_scales, weight.data, weight.scales, bias, relu, residual, out_dtype, True, data, scales)
    return _new(Fp8Rows, *r) if out is None else out
