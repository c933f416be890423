"""Attention over the paged cache at its edges: far tails in float16."""

import pytest
import torch

from forgetune_b200 import paged_attention

from . import decoder_reference as ref
from .test_decoder_gpu import BF16, F16, randn, within

pytestmark = pytest.mark.gpu

# ---------------------------------------------------------------------------
# float16 weights
# ---------------------------------------------------------------------------
def tail(new, length, strong, nats, group=1, dim=64):
    """A key of score 0 and value 0 at position `strong`, all others `nats` below it with values of 1."""
    b = ref.Batch([new], [length], 128, 1, dim, F16)
    page, col = b.slots(0, torch.arange(length, device="cuda"))
    b.keys[:], b.values[:] = 0, 1
    b.keys[page, col, 0, 0] = -nats
    page, col = b.slots(0, torch.tensor([strong], device="cuda"))
    b.keys[page, col], b.values[page, col] = 0, 0
    q = torch.zeros(new, group, dim, dtype=F16, device="cuda")
    q[..., 0] = 1
    return q, b


@pytest.mark.parametrize("nats", [9.0, 12.5, 17.0, 17.25, 17.5, 19.0])
@pytest.mark.parametrize("new,length,strong,group,dim", [(1, 4097, 0, 1, 64), (1, 131072, 0, 1, 64), (1, 131072, 70000, 4, 128),
                                                         (1, 9000, 8999, 7, 128), (200, 6000, 3, 1, 128), (3, 700, 600, 2, 80)])
def test_the_tail_of_a_long_context_in_float16(nats, new, length, strong, group, dim):
    """Together the others weigh length e^-nats, most of which lies below float16's smallest number.

    The weights' step: with the row's reference at 2^7, a weight is off by at most 2^-25 / 2^7 of the reference's."""
    q, b = tail(new, length, strong, nats, group, dim)
    want, tol, _ = ref.attention(q, b, 1.0, least=2.0 ** -32)
    within(paged_attention(q, *b.args(), scale=1.0), want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_equal_values_come_out_as_they_are(dtype):
    """A mean of equal values is the value, whatever the weights: within the weights' roundings and the output's."""
    for new, length, spread in ((1, 50000, 3.0), (300, 2000, 3.0), (1, 131072, 0.1)):
        b = ref.Batch([new], [length], 64, 2, 128, dtype)
        b.values[:] = 1
        q = (spread * randn(new, 8, 128)).to(dtype)
        want, tol, _ = ref.attention(q, b, least=2.0 ** -32)
        within(paged_attention(q, *b.args()), want, tol)
