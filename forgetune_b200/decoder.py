"""Operators on CUDA tensors around a decoder layer's attention and behind its logits.

Between the products of :mod:`forgetune_b200.fp8` a decoder layer turns its
queries and keys by their positions, keeps keys and values in a cache, and
attends over it; behind the last product the logits are scored::

    qkv = fp8_linear(h, w_qkv, out_dtype=torch.bfloat16).unflatten(1, (-1, 128))
    q, k, v = qkv.split((32, 8, 8), 1)                                       # [tokens, heads, dim]
    q = append_heads(q, k, v, keys, values, page_table, starts, lengths, frequencies)
    o = paged_attention(q, keys, values, page_table, starts, lengths)        # as q
    ...
    logprobs, entropy, top, top_tokens = token_logprobs(logits, tokens, top=5)

Each is one call of the engine library's C ABI (``ftb_rotate_heads``,
``ftb_append_heads``, ``ftb_paged_attention``, ``ftb_token_logprobs``;
include/forgetune_b200.h) on the current torch stream, made by the extension
``lib/_torch_ops.so`` (csrc/torch_ops.cpp).

**The cache** is a pool of pages for keys and one for values, ``[pages,
page_size, kv_heads, dim]`` each, with any strides but that the values of a
head lie side by side (a transposed view of ``[pages, kv_heads, page_size,
dim]`` is one).  **A batch** is three int32 tensors, read on the device when
the kernels run, so that a captured graph follows their contents: rows
``starts[b]`` to ``starts[b + 1]`` of the heads are the new tokens of sequence
``b``, which has ``lengths[b]`` tokens with them; its token at position ``j``
lies in page ``page_table[b, j // page_size]``.  Any mix of single tokens and
prompts goes.  Rows in no sequence (behind the last one, as in a padded batch)
are left as they were, and undefined in a new output.

The operators are for inference: they return tensors without gradients, refuse
inputs with a forward-mode tangent, and outputs that require grad outside
``torch.no_grad()``.  Results are the same bits every time.  The reference has
no counterpart.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native

__all__ = ["rope_frequencies", "rotate_heads", "append_heads", "paged_attention", "token_logprobs"]

_ops = None


def _load():
    global _ops
    _ops = _native.torch_ops()
    return _ops


def rope_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None, scale: float = 1.0,
                     original: int = 8192, fast: float = 32.0, slow: float = 1.0, device="cuda") -> torch.Tensor:
    """Frequencies of rotary positions over ``dim`` elements, float64 [dim / 2]: ``base ** (-2 i / dim)``.

    ``scaling`` changes them for contexts ``scale`` times as long as the ``original`` one a model was trained on:
    ``"linear"`` divides all by ``scale``; ``"base"`` raises the base so that the slowest is divided by it and the
    fastest is kept; ``"parts"`` keeps those that turn at least ``fast`` times in the original context, divides those
    that turn at most ``slow`` times, and goes over between them in proportion to their turns.  Frequencies of any
    other rule are a tensor of the caller's.
    """
    if dim < 2 or dim % 2:
        raise ValueError("rope_frequencies: dim must be even and positive")
    if not (base > 0 and scale > 0):
        raise ValueError("rope_frequencies: base and scale must be positive")
    if scaling == "base" and dim > 2:
        base *= scale ** (dim / (dim - 2))
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        f = f / scale
    elif scaling == "parts":
        if not fast > slow:
            raise ValueError("rope_frequencies: fast must be above slow")
        keep = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / scale * (1 - keep)
    elif scaling not in (None, "base"):
        raise ValueError("rope_frequencies: scaling must be None, 'linear', 'base' or 'parts'")
    return f.to(device)


def rotate_heads(x: torch.Tensor, positions: torch.Tensor, frequencies: Optional[torch.Tensor],
                 weight: Optional[torch.Tensor] = None, eps: float = 1e-6, norm: bool = False,
                 interleaved: bool = False, amplitude: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Heads [tokens, heads, dim] turned by their tokens' ``positions`` (int32 or int64 [tokens]).

    Pair ``i`` of a head turns by ``positions * frequencies[i]``, formed in 64
    bits (see :func:`rope_frequencies`), and is multiplied by ``amplitude``.
    Pairs are elements ``(i, i + pairs)``, or ``(2 i, 2 i + 1)`` where
    ``interleaved``; elements from ``2 * pairs`` on stay.  With ``norm`` each
    head is first divided by ``sqrt(mean(x^2) + eps)`` and multiplied by
    ``weight`` (float32 [dim] or None).  ``dim`` is at most 512.  The result
    has ``x``'s type; ``out`` receives it in place of a new tensor and may be
    ``x``.
    """
    return (_ops or _load()).rotate_heads(x, positions, frequencies, weight, eps, norm, interleaved, amplitude, out)


def append_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                 page_table: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor,
                 frequencies: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, norm: bool = False,
                 interleaved: bool = False, amplitude: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """New tokens' heads into a paged cache: ``k`` normalised and turned as by :func:`rotate_heads`, ``v`` as it is.

    Returns the queries, normalised and turned alike, in the cache's type.
    ``q`` is [tokens, heads, dim], ``k`` and ``v`` [tokens, kv_heads, dim], of
    the cache's type or float32; positions are the batch's.  ``frequencies``
    None: no rotation.  A token whose position has no page in the pool is not
    stored.  ``out`` receives the queries in place of a new tensor and may be
    ``q`` where their types are alike.
    """
    return (_ops or _load()).append_heads(q, k, v, keys, values, page_table, starts, lengths, frequencies, q_weight,
                                          k_weight, eps, norm, interleaved, amplitude, out)


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, page_table: torch.Tensor,
                    starts: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                    window: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a batch's new tokens over the cache that holds them and what came before.

    ``q`` is [tokens, heads, dim] of the cache's type, ``heads`` a multiple of
    the cache's ``kv_heads``.  A token sees the tokens of its sequence up to
    its own position, and with ``window`` the last ``window`` of them only;
    ``scale`` (default ``dim ** -0.5``) multiplies the scores.  A token at a
    negative position (a length below its number of new tokens) sees nothing
    and gets zeros.  What a token does not see does not change its output,
    whatever it holds (infinities and NaN too).  A token that sees one whose page
    number is outside of the pool, or whose own position is beyond the table, gets
    NaN.  ``out`` receives the result in place of a new tensor; it may not be ``q``.

    Softmax statistics and sums are float32; a weight is rounded to the
    cache's type where the tensor cores multiply it by the values.
    """
    return (_ops or _load()).paged_attention(q, keys, values, page_table, starts, lengths, scale, window, out)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0):
    """Scores of ``tokens`` (int32 or int64 [m]) against rows of ``logits`` [m, n] (float32, float16, bfloat16).

    Returns ``(logprobs, entropy)``, float32 [m]: the natural logarithm of the
    softmax at the token (NaN for one outside of the row) and the entropy of
    the distribution; with ``top`` (at most 64) also the ``top`` largest log
    probabilities, float32 [m, top], and their tokens, int64 [m, top], largest
    first, equal ones by the lower token, NaN last.
    """
    return (_ops or _load()).token_logprobs(logits, tokens, top)
