"""Attention over the paged cache at its edges: far tails in float16, pages outside of the pool, lengths beyond the
table, infinities that are seen, scores whose steps are large."""

import math

import pytest
import torch

from forgetune_b200 import append_heads, paged_attention

from . import decoder_reference as ref
from .test_decoder_gpu import BF16, F16, F32, randn, within

pytestmark = pytest.mark.gpu

# kernel by type and head size: tensor cores, tensor cores, a key at a time, a key at a time
KINDS = [(BF16, 128), (F16, 80), (F32, 64), (BF16, 136)]


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


# ---------------------------------------------------------------------------
# pages outside of the pool, lengths beyond the table
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", KINDS, ids=str)
@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("new,length,window,group", [(300, 300, 0, 1), (300, 1000, 0, 2), (100, 700, 0, 4), (40, 90, 20, 2),
                                                     (700, 700, 130, 1), (1, 500, 60, 4), (1, 3000, 0, 4), (5, 5, 0, 1)])
def test_only_rows_that_see_a_bad_page_are_nan(dtype, dim, page, new, length, window, group):
    b = ref.Batch([3, new, 2], [40, length, 9], page, 2, dim, dtype)
    q = randn(b.tokens, 2 * group, dim, dtype=dtype)
    clean = paged_attention(q, *b.args(), window=window)
    position = torch.arange(length - new, length, device="cuda")
    pages = -(-length // page)
    for bad in sorted({0, pages // 2, max(0, pages - 2), pages - 1}):
        for number in (-1, b.keys.shape[0], 2 ** 31 - 1):
            kept = int(b.page_table[1, bad])
            b.page_table[1, bad] = number
            got = paged_attention(q, *b.args(), window=window)
            b.page_table[1, bad] = kept
            sees = position >= bad * page
            if window:
                sees &= position - window < (bad + 1) * page - 1
            assert got[3:3 + new][sees].isnan().all()
            assert torch.equal(got[3:3 + new][~sees], clean[3:3 + new][~sees])
            assert torch.equal(got[:3], clean[:3]) and torch.equal(got[3 + new:], clean[3 + new:])
    for bad in (slice(0, pages), slice(pages // 2, pages)):  # several
        kept = b.page_table[1, bad].clone()
        b.page_table[1, bad] = -5
        got = paged_attention(q, *b.args(), window=window)[3:3 + new]
        b.page_table[1, bad] = kept
        sees = position >= (bad.start or 0) * page
        assert got[sees].isnan().all() and torch.equal(got[~sees], clean[3:3 + new][~sees])


@pytest.mark.parametrize("dtype,dim", KINDS, ids=str)
@pytest.mark.parametrize("new,length,places,window", [(200, 300, 160, 0), (200, 300, 112, 0), (300, 300, 16, 0), (600, 1500, 1008, 100),
                                                      (1, 300, 160, 0), (2, 161, 160, 0), (200, 300, 160, 30), (500, 900, 128, 0)])
def test_rows_beyond_the_table_are_nan_and_others_are_not(dtype, dim, new, length, places, window):
    b = ref.Batch([new, 2], [length, 9], 16, 2, dim, dtype)
    q = randn(b.tokens, 4, dim, dtype=dtype)
    want, tol, _ = ref.attention(q, b, window=window)
    b.page_table = b.page_table[:, :places // 16].contiguous()
    got = paged_attention(q, *b.args(), window=window)
    beyond = torch.arange(length - new, length, device="cuda") >= places
    assert got[:new][beyond].isnan().all()
    within(got[:new][~beyond], want[:new][~beyond], tol[:new][~beyond])
    within(got[new:], want[new:], tol[new:])


@pytest.mark.parametrize("dtype,dim", KINDS, ids=str)
def test_bad_rows_are_the_same_every_time(dtype, dim):
    """The halves of a block come to a bad page at different times; a full machine makes them differ more."""
    b = ref.Batch([400] * 20, [500 + 7 * i for i in range(20)], 16, 2, dim, dtype)
    q = randn(b.tokens, 2, dim, dtype=dtype)
    b.page_table[torch.arange(20), torch.arange(20) + 10] = -1
    first = paged_attention(q, *b.args())
    for _ in range(20):
        assert torch.equal(paged_attention(q, *b.args()).nan_to_num(123.0), first.nan_to_num(123.0))


def test_tokens_before_the_end_of_the_table_are_stored():
    b = ref.Batch([40], [60], 16, 1, 64, BF16)
    b.page_table = b.page_table[:, :2].contiguous()
    q, k, v = randn(40, 3, 64, dtype=BF16).split((1, 1, 1), 1)
    append_heads(q, k, v, *b.args())
    page, col = b.slots(0, torch.arange(20, 32, device="cuda"))
    assert torch.equal(b.keys[page, col], k[:12]) and torch.equal(b.values[page, col], v[:12])


# ---------------------------------------------------------------------------
# infinities that are seen
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", KINDS, ids=str)
@pytest.mark.parametrize("new,length,window", [(1, 100, 0), (20, 400, 0), (300, 300, 0), (300, 700, 140), (1, 5000, 0)])
def test_an_infinite_value_makes_an_infinite_output(dtype, dim, new, length, window):
    """In tiles that all rows see and in those that some see in part; two of unlike signs, and NaN, give NaN."""
    b = ref.Batch([new], [length], 16, 1, dim, dtype)
    q = (0.1 * randn(new, 4, dim)).to(dtype)
    clean = paged_attention(q, *b.args(), window=window)
    p = torch.arange(length - new, length, device="cuda")
    for position in {length - 1, max(0, length - new - 3), length // 2}:
        page, col = b.slots(0, torch.tensor([position], device="cuda"))
        kept = b.values[page, col].clone()
        b.values[page, col, 0, 0] = math.inf
        b.values[page, col, 0, 1] = -math.inf
        b.values[page, col, 0, dim - 1] = math.nan
        got = paged_attention(q, *b.args(), window=window)
        sees = p >= position
        if window:
            sees &= p - window < position
        assert torch.equal(got[~sees], clean[~sees]) and torch.equal(got[..., 2:dim - 1], clean[..., 2:dim - 1])
        assert (got[sees][..., 0] == math.inf).all() and (got[sees][..., 1] == -math.inf).all()
        assert got[sees][..., dim - 1].isnan().all()
        b.values[page, col] = kept
    if length > 1:
        at = torch.tensor([max(0, length - new - 1), length - 1], device="cuda")
        page, col = b.slots(0, at)
        b.values[page, col, 0, 5] = torch.tensor([math.inf, -math.inf], device="cuda", dtype=dtype)
        got = paged_attention(q, *b.args(), window=window)
        first = (p >= at[0]) & (not window or p - window < at[0])
        both = first & (p >= at[1])
        assert (got[first & ~both][..., 5] == math.inf).all() and got[both][..., 5].isnan().all()


# ---------------------------------------------------------------------------
# scores of every size
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim,step", [(F16, 128, 4.0), (F16, 64, 4.0), (BF16, 128, 2.0 ** 13), (BF16, 64, 2.0 ** 40),
                                            (F32, 64, 2.0 ** 13), (BF16, 136, 2.0 ** 13)], ids=str)
@pytest.mark.parametrize("new,length", [(1, 100), (100, 100), (120, 120), (3, 1000)])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_whose_steps_are_larger_than_one(dtype, dim, step, new, length, falling):
    """Of keys so far apart each row takes the largest that it sees alone, though no float32 near the scores is exact."""
    b = ref.Batch([new], [length], 16, 1, dim, dtype)
    n = min(length, 120)  # the last ones; those before score 0
    at = torch.arange(n, device="cuda")
    page, col = b.slots(0, length - n + at)
    base = 1250 if dtype == F16 else 128
    b.keys[:] = 0
    b.keys[page, col] = ((base + (n - 1 - at if falling else at)) * step).to(dtype)[:, None, None]
    q = torch.full((new, 2, dim), base * step, dtype=dtype, device="cuda")
    p = torch.arange(length - new, length, device="cuda")
    page, col = b.slots(0, torch.full_like(p, length - n) if falling else p)
    for scale, sign in ((None, 1), (-1.0, -1)):
        got = paged_attention(sign * q, *b.args(), scale=scale)
        assert torch.equal(got, b.values[page, col].expand(new, 2, dim))
