"""Block-scaled 8-bit operators on CUDA tensors.

A dense layer in 8 bits is a chain of three operators, each one call of the
engine library's C ABI (``ftb_quantize_rows``, ``ftb_quantize_weight``,
``ftb_rms_norm``, ``ftb_fp8_linear``; include/forgetune_b200.h) on the current
torch stream::

    w1 = quantize_weight(layer1.weight)                 # once, [n, k]
    h, res = rms_norm(x, norm.weight, residual=res, quantize=True)
    h = fp8_linear(h, w1, bias=layer1.bias, relu=True, quantize=True)
    x = fp8_linear(h, w2, bias=layer2.bias)

The format is e4m3 values with one power-of-two scale (ue8m0, the format the
tensor cores take) for each block of 128 along a row of activations and for
each 128 x 128 block of a weight: the smallest power of two with
``max|x| / scale <= 448``, 1 for a block of zeros.  Values that are not finite
are stored as NaN.  Products are accumulated in fp32.

Inputs are 2-D; a plain input whose rows are not contiguous is copied first,
as ``CompiledModel.run_device`` does.  The operators are for inference: they
return tensors without gradients.  The first call on a device sets it up, so
make it before capturing a CUDA graph.  The reference has no counterpart (its
models are float32 only).
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple, Union

import torch

from . import _native
from .errors import ForgeTuneRuntimeError, InvalidShapeError

__all__ = ["Fp8Rows", "Fp8Weight", "quantize_rows", "quantize_weight", "rms_norm", "fp8_linear"]

BLOCK = 128
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # FTB_F32, FTB_F16, FTB_BF16
_FP8_RELU = 1

# The argument structs of include/forgetune_b200.h: every field has eight
# bytes.  A matrix is (pointer, stride, type), a quantised one (pointer,
# stride, scales pointer, stride).
_QUANTIZE_ARGS = struct.Struct("=9q")  # x, q, m, k
_RMS_NORM_ARGS = struct.Struct("=7qd12q")  # x, residual, weight, eps, h, y, q, m, k
_LINEAR_ARGS = struct.Struct("=23q")  # a, w, bias, residual, y, q, m, n, k, flags
_NO_MATRIX = (0, 0, 0)
_NO_FP8 = (0, 0, 0, 0)


def _rows(m: int, k: int, unit: int, dtype, device) -> torch.Tensor:
    """An uninitialised matrix whose rows start on multiples of ``unit`` elements."""
    return torch.empty_strided((m, k), ((k + unit - 1) // unit * unit, 1), dtype=dtype, device=device)


class _Fp8:
    """8-bit values [rows, k] with their block scales."""

    __slots__ = ("_data", "_scales", "_m", "_k", "_ld", "_scales_ld")
    _row_block = 1

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        name = type(self).__name__
        if not isinstance(data, torch.Tensor) or data.dtype is not _E4M3:
            raise TypeError("%s: data must be a torch.float8_e4m3fn tensor" % name)
        if not isinstance(scales, torch.Tensor) or scales.dtype is not _E8M0:
            raise TypeError("%s: scales must be a torch.float8_e8m0fnu tensor" % name)
        shape, s_shape = data.shape, scales.shape
        if len(shape) != 2 or shape[1] < 1:
            raise InvalidShapeError("%s: data must be [rows, k] with k >= 1, got %s" % (name, tuple(shape)))
        m, k = shape
        b = self._row_block
        rows, kb = (m + b - 1) // b, (k + BLOCK - 1) // BLOCK
        if s_shape != (rows, kb):
            raise InvalidShapeError("%s: scales of data %s must be %s, got %s"
                                    % (name, (m, k), (rows, kb), tuple(s_shape)))
        if data.get_device() != scales.get_device():
            raise ValueError("%s: data and scales are on different devices" % name)
        self._data = data
        self._scales = scales
        self._m = m
        self._k = k
        self._ld = _ld8(m, k, data.stride(), 16)  # None: not laid out as the operators need it
        self._scales_ld = _ld8(rows, kb, scales.stride(), 4)

    @classmethod
    def pack(cls, data: torch.Tensor, scales: torch.Tensor):
        """The same values in rows laid out as the operators need them (copied where they are not)."""
        r = cls(data, scales)
        if r._ld is None or data.data_ptr() % 16:
            data = _rows(*data.shape, 16, _E4M3, data.device).copy_(data)
        if r._scales_ld is None or scales.data_ptr() % 4:
            scales = _rows(*scales.shape, 4, _E8M0, scales.device).copy_(scales)
        return cls(data, scales)

    @classmethod
    def _empty(cls, m: int, k: int, device):
        """Uninitialised values, laid out as the operators need them."""
        kb = (k + BLOCK - 1) // BLOCK
        r = cls.__new__(cls)
        r._m = m
        r._k = k
        r._ld = ld = (k + 15) // 16 * 16
        r._scales_ld = s_ld = (kb + 3) // 4 * 4
        r._data = torch.empty_strided((m, k), (ld, 1), dtype=_E4M3, device=device)
        r._scales = torch.empty_strided(((m + cls._row_block - 1) // cls._row_block, kb), (s_ld, 1), dtype=_E8M0,
                                        device=device)
        return r

    def _args(self, what: str) -> Tuple[int, int, int, int]:
        """The matrix as the C ABI takes it."""
        p, s = self._data.data_ptr(), self._scales.data_ptr()
        if self._ld is None or self._scales_ld is None or p % 16 or s % 4:
            raise InvalidShapeError("%s: rows of data must start on 16-byte and rows of scales on 4-byte boundaries "
                                    "(see %s.pack)" % (what, type(self).__name__))
        return p, self._ld, s, self._scales_ld

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @property
    def shape(self) -> torch.Size:
        return self._data.shape

    @property
    def device(self) -> torch.device:
        return self._data.device

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


def _ld8(rows: int, cols: int, stride, unit: int) -> Optional[int]:
    """Row stride of an 8-bit matrix, or None where its rows are not laid out in units of ``unit`` bytes."""
    ld, step = stride
    if step != 1 and cols > 1:
        return None
    if rows <= 1:
        return (cols + unit - 1) // unit * unit
    return ld if ld >= cols and ld % unit == 0 else None


def _ld(t: torch.Tensor) -> Optional[int]:
    """Row stride of a plain matrix, or None where its rows are not contiguous or overlap."""
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        return None
    if rows <= 1:
        return cols
    return ld if ld >= cols else None


def _input(t, what: str) -> Tuple[torch.Tensor, int, int, int, int]:
    """A plain 2-D CUDA input (copied where its rows are not contiguous), its sizes, row stride and type."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _TYPES):
        raise TypeError("%s must be a float32, float16 or bfloat16 CUDA tensor" % what)
    if t.dim() != 2 or t.shape[1] < 1:
        raise InvalidShapeError("%s must be 2-D with at least one column, got %s" % (what, tuple(t.shape)))
    rows, cols = t.shape
    ld = _ld(t)
    if ld is None:
        t, ld = t.contiguous(), cols
    return t, rows, cols, ld, _TYPES[t.dtype]


def _check(t: torch.Tensor, what: str, shape, device) -> None:
    if t.shape != shape:
        raise InvalidShapeError("%s must be %s, got %s" % (what, tuple(shape), tuple(t.shape)))
    if t.device != device:
        raise ValueError("%s is on %s, the input on %s" % (what, t.device, device))


def _output(out, what: str, shape, dtype: torch.dtype, device) -> Tuple[torch.Tensor, Tuple[int, int, int]]:
    """A new plain output, or the caller's, and the matrix the C ABI takes."""
    if out is None:
        out = torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
        return out, (out.data_ptr(), shape[1], _TYPES[dtype])
    if not (isinstance(out, torch.Tensor) and out.dtype == dtype):
        raise TypeError("%s must be a %s tensor" % (what, dtype))
    _check(out, what, shape, device)
    ld = _ld(out)
    if ld is None:
        raise InvalidShapeError("%s: rows must be contiguous and must not overlap" % what)
    return out, (out.data_ptr(), ld, _TYPES[dtype])


def _fp8_output(out, what: str, m: int, k: int, device) -> Fp8Rows:
    """A new quantised output, or the caller's."""
    if out is None:
        return Fp8Rows._empty(m, k, device)
    if not isinstance(out, Fp8Rows):
        raise TypeError("%s must be an Fp8Rows" % what)
    _check(out, what, (m, k), device)
    return out


def _vector(t, what: str, n: int, device) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.float32):
        raise TypeError("%s must be a float32 tensor" % what)
    _check(t, what, (n,), device)
    return t if n == 1 or t.stride(0) == 1 else t.contiguous()


def _call(name: str, device: torch.device, args: bytes) -> None:
    """One C call on the current stream of ``device``."""
    fn = getattr(_native.lib(), name)
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(args, stream)
    if rc != 0:
        raise ForgeTuneRuntimeError("%s failed (%d): %s" % (name, rc, _native.last_error()))


def quantize_rows(x: torch.Tensor, out: Optional[Fp8Rows] = None) -> Fp8Rows:
    """Activations [m, k] (float32, float16, bfloat16) to 8 bits with a scale for each 128 along a row."""
    x, m, k, ld, t = _input(x, "quantize_rows: x")
    dev = x.device
    r = _fp8_output(out, "quantize_rows: out", m, k, dev)
    _call("ftb_quantize_rows", dev, _QUANTIZE_ARGS.pack(x.data_ptr(), ld, t, *r._args("quantize_rows: out"), m, k))
    return r


def quantize_weight(w: torch.Tensor) -> Fp8Weight:
    """A weight [n, k] (``nn.Linear``'s layout; float32, float16, bfloat16) to 8 bits with a scale for each
    128 x 128 block.  Done once, where a model is loaded."""
    w, n, k, ld, t = _input(w, "quantize_weight: w")
    if n < 1:
        raise InvalidShapeError("quantize_weight: w must have at least one row")
    r = Fp8Weight._empty(n, k, w.device)
    _call("ftb_quantize_weight", w.device,
          _QUANTIZE_ARGS.pack(w.data_ptr(), ld, t, *r._args("quantize_weight"), n, k))
    return r


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
    x, m, k, ld, t = _input(x, "rms_norm: x")
    dtype, dev = x.dtype, x.device
    weight = _vector(weight, "rms_norm: weight", k, dev)
    r_arg = h_arg = y_arg = _NO_MATRIX
    q_arg = _NO_FP8
    if residual is not None:
        residual, rm, rk, r_ld, rt = _input(residual, "rms_norm: residual")
        if rt != t:
            raise TypeError("rms_norm: residual must be %s, got %s" % (dtype, residual.dtype))
        if rm != m or rk != k or residual.device != dev:
            _check(residual, "rms_norm: residual", (m, k), dev)
        r_arg = (residual.data_ptr(), r_ld, t)
        h, h_arg = _output(residual_out, "rms_norm: residual_out", (m, k), dtype, dev)
    elif residual_out is not None:
        raise ValueError("rms_norm: residual_out needs a residual")
    if quantize:
        y = _fp8_output(out, "rms_norm: out", m, k, dev)
        q_arg = y._args("rms_norm: out")
    else:
        y, y_arg = _output(out, "rms_norm: out", (m, k), dtype, dev)
    _call("ftb_rms_norm", dev, _RMS_NORM_ARGS.pack(
        x.data_ptr(), ld, t, *r_arg, 0 if weight is None else weight.data_ptr(), eps, *h_arg, *y_arg, *q_arg, m, k))
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
    if quantize and out_dtype is not None:
        raise ValueError("fp8_linear: a quantised result has no out_dtype")
    if not isinstance(x, Fp8Rows):
        x = _input(x, "fp8_linear: x")[0]
        out_dtype = out_dtype or x.dtype
        x = quantize_rows(x)
    elif not x._data.is_cuda:
        raise TypeError("fp8_linear: x must be on a CUDA device")
    m, k, n, dev = x._m, x._k, weight._m, x._data.device
    if weight._k != k:
        raise InvalidShapeError("fp8_linear: x is %s, weight %s: their depths differ" % ((m, k), (n, weight._k)))
    if weight._data.device != dev:
        raise ValueError("fp8_linear: weight is on %s, the input on %s" % (weight._data.device, dev))
    bias = _vector(bias, "fp8_linear: bias", n, dev)
    r_arg = y_arg = _NO_MATRIX
    q_arg = _NO_FP8
    if residual is not None:
        residual, rm, rn, r_ld, rt = _input(residual, "fp8_linear: residual")
        if rm != m or rn != n or residual.device != dev:
            _check(residual, "fp8_linear: residual", (m, n), dev)
        r_arg = (residual.data_ptr(), r_ld, rt)
    if quantize:
        y = _fp8_output(out, "fp8_linear: out", m, n, dev)
        q_arg = y._args("fp8_linear: out")
    else:
        if out_dtype is None:
            out_dtype = torch.float32 if residual is None else residual.dtype
        elif out_dtype not in _TYPES:
            raise TypeError("fp8_linear: out_dtype must be float32, float16 or bfloat16, got %s" % (out_dtype,))
        y, y_arg = _output(out, "fp8_linear: out", (m, n), out_dtype, dev)
    _call("ftb_fp8_linear", dev, _LINEAR_ARGS.pack(
        *x._args("fp8_linear: x"), *weight._args("fp8_linear: weight"), 0 if bias is None else bias.data_ptr(),
        *r_arg, *y_arg, *q_arg, m, n, k, _FP8_RELU if relu else 0))
    return y
