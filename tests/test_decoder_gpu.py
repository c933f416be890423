"""Head rotation, cache append, attention over the paged cache and token log probabilities against float64."""

import math

import pytest
import torch

from forgetune_b200 import (append_heads, fp8_linear, paged_attention, quantize_weight, rms_norm, rope_frequencies,
                            rotate_heads, token_logprobs)

from . import decoder_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), "%d of %d off, worst %.3g times the tolerance" % (
        bad.sum(), bad.numel(), ((got.double() - want).abs() / tol).nan_to_num(math.inf).max())


# ---------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 32), (257, 8, 128, 64),
                                                  (7, 3, 80, 80), (5, 2, 256, 256), (2, 3, 512, 128), (4, 9, 130, 62),
                                                  (6, 1, 5, 2), (2, 67, 8, 8), (1000, 16, 128, 128), (3, 2, 96, 0)])
@pytest.mark.parametrize("interleaved,norm", [(False, False), (True, False), (False, True), (True, True)])
def test_rotation(dtype, tokens, heads, dim, rot, interleaved, norm):
    x = randn(tokens, heads, dim, dtype=dtype, seed=tokens + dim)
    positions = torch.randint(-5, 1 << 20, (tokens,), generator=gen(1), device="cuda")
    f = rope_frequencies(rot) if rot else None
    weight = 1 + 0.3 * randn(dim, seed=2) if norm else None
    kw = dict(norm=norm, interleaved=interleaved, amplitude=1.25, eps=1e-5)
    y = rotate_heads(x, positions, f, weight=weight, **kw)
    want, size = ref.rotate(x, positions, f, weight, **kw)
    assert y.dtype == dtype and y.shape == x.shape
    within(y, want, ref.rotate_tolerance(want, size, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rotation_of_views_and_in_place(dtype):
    """Heads inside of a product's rows, heads before tokens, bases off any boundary; int32 positions; in place."""
    f = rope_frequencies(64, scaling="parts", scale=8.0)
    positions = torch.arange(37, dtype=torch.int32, device="cuda") * 1000
    wide = randn(37, 12 * 64 + 1, dtype=dtype)
    for x in (wide[:, 64:64 * 6].unflatten(1, (5, 64)), wide[:, 1:321].unflatten(1, (5, 64)),
              randn(5, 37, 64, dtype=dtype).transpose(0, 1), wide[:, :64].unflatten(1, (1, 64)).expand(37, 5, 64)):
        want, size = ref.rotate(x, positions, f)
        before = x.clone()
        y = rotate_heads(x, positions, f)
        assert torch.equal(x, before)
        within(y, want, ref.rotate_tolerance(want, size, dtype))
        out = torch.full((37, 7, 64), 3.0, dtype=dtype, device="cuda")
        assert rotate_heads(x, positions, f, out=out[:, 1:6]) is not None
        assert torch.equal(out[:, 1:6], y) and (out[:, 0] == 3).all() and (out[:, 6] == 3).all()
        if x.stride(1) != 0:
            rest = wide.clone()
            rotate_heads(x, positions, f, out=x)
            assert torch.equal(x, y)
            x.copy_(before)
            assert torch.equal(wide, rest)
    assert rotate_heads(randn(0, 5, 64, dtype=dtype), positions[:0], f).shape == (0, 5, 64)


def test_far_positions_are_as_exact_as_near_ones():
    f = rope_frequencies(128, base=1e6)
    x = randn(64, 2, 128)
    positions = torch.full((64,), 2 ** 31 - 1, device="cuda", dtype=torch.int64) - torch.arange(64, device="cuda")
    want, size = ref.rotate(x, positions, f)
    # 2^31 radians are 3.4e8 turns, which 64 bits hold to 2^-25 of a turn
    within(rotate_heads(x, positions, f), want, ref.rotate_tolerance(want, size, F32) + 2.0 ** -22 * size)


def test_frequencies():
    f = rope_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** (-torch.arange(32).double() / 32))
    assert torch.allclose(rope_frequencies(64, scaling="linear", scale=4.0, device="cpu"), f / 4)
    b = rope_frequencies(64, scaling="base", scale=4.0, device="cpu")
    assert b[0] == 1 and torch.allclose(b[-1], f[-1] / 4)
    p = rope_frequencies(64, scaling="parts", scale=4.0, device="cpu")
    assert torch.allclose(p[:4], f[:4]) and torch.allclose(p[-4:], f[-4:] / 4) and (p.diff() < 0).all()


def test_norm_of_zeros_and_of_values_that_are_not_finite():
    x = randn(4, 2, 128)
    x[0] = 0
    x[1, 0, 5] = math.nan
    x[2, 1, 7] = math.inf
    y = rotate_heads(x, torch.zeros(4, dtype=torch.int64, device="cuda"), rope_frequencies(128), norm=True)
    assert (y[0] == 0).all() and y[1, 0].isnan().all() and not y[1, 1].isnan().any()
    assert y[2, 1].isnan().any() and not y[2, 0].isnan().any() and not y[3].isnan().any()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,held", [(F32, F32), (F32, BF16), (F32, F16), (F16, F16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("new,lengths,page,heads,kv,dim,rot,layout", [
    ([1], [1], 16, 1, 1, 128, 128, "tokens"),
    ([1] * 33, [3 * i + 1 for i in range(33)], 16, 8, 2, 128, 128, "tokens"),
    ([0, 17, 0, 1, 300, 0], [5, 17, 0, 40, 301, 0], 64, 6, 3, 64, 32, "heads"),
    ([5, 9], [5, 21], 7, 4, 1, 80, 80, "tokens"),
    ([2, 40], [70, 40], 3, 2, 2, 50, 50, "odd"),
    ([70], [200], 128, 3, 1, 512, 512, "tokens"),
])
@pytest.mark.parametrize("interleaved,norm", [(False, True), (True, False)])
def test_append(dtype, held, new, lengths, page, heads, kv, dim, rot, layout, interleaved, norm):
    b = ref.Batch(new, lengths, page, kv, dim, held, layout=layout, behind=3)
    qkv = randn(b.tokens, heads + 2 * kv, dim, dtype=dtype, seed=5)
    q, k, v = qkv.split((heads, kv, kv), 1)
    f = rope_frequencies(rot)
    wq, wk = (1 + 0.2 * randn(dim, seed=6), 1 + 0.2 * randn(dim, seed=7)) if norm else (None, None)
    how = dict(norm=norm, interleaved=interleaved, amplitude=0.9)
    keys, values = b.keys.clone(), b.values.clone()
    out = torch.full((b.tokens, heads, dim), 9.0, dtype=held, device="cuda")
    got = append_heads(q, k, v, *b.args(), frequencies=f, q_weight=wq, k_weight=wk, out=out, **how)
    n = sum(new)
    positions = b.positions().cuda()
    want, size = ref.rotate(q[:n], positions, f, wq, **how)
    within(got[:n], want, ref.rotate_tolerance(want, size, held))
    assert (got[n:] == 9).all()  # rows behind the last sequence
    want, size = ref.rotate(k[:n], positions, f, wk, **how)
    tol = ref.rotate_tolerance(want, size, held)
    at = 0
    for s, m in enumerate(new):
        page_of, col = b.slots(s, positions[at:at + m])
        within(b.keys[page_of, col], want[at:at + m], tol[at:at + m])
        assert torch.equal(b.values[page_of, col], v[at:at + m].to(held))
        keys[page_of, col], values[page_of, col] = b.keys[page_of, col], b.values[page_of, col]
        at += m
    assert torch.equal(b.keys, keys) and torch.equal(b.values, values)  # nothing else changed
    assert torch.equal(append_heads(q, k, v, *b.args(), frequencies=f, q_weight=wq, k_weight=wk, **how)[:n], got[:n])


def test_append_in_place_and_without_rotation():
    b = ref.Batch([4, 5], [4, 9], 16, 2, 64, BF16)
    q, k, v = randn(9, 8, 64, dtype=BF16).split((4, 2, 2), 1)
    want = q.clone()
    assert append_heads(q, k, v, *b.args(), out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, want)
    page, col = b.slots(1, torch.arange(4, 9, device="cuda"))
    assert torch.equal(b.keys[page, col], k[4:]) and torch.equal(b.values[page, col], v[4:])


def test_keys_and_values_of_one_pool():
    """Side by side by pages, by tokens and by heads."""
    for shape, at in (((4, 2, 16, 3, 64), 1), ((4, 16, 2, 3, 64), 2), ((4, 16, 3, 2, 64), 3)):
        pool = torch.zeros(shape, dtype=BF16, device="cuda")
        b = ref.Batch([20], [30], 16, 3, 64, BF16)
        b.keys, b.values = pool.select(at, 0), pool.select(at, 1)
        q, k, v = randn(20, 9, 64, dtype=BF16).split((3, 3, 3), 1)
        append_heads(q, k, v, *b.args())
        page, col = b.slots(0, torch.arange(10, 30, device="cuda"))
        assert torch.equal(b.keys[page, col], k) and torch.equal(b.values[page, col], v)
        assert pool.count_nonzero() == k.count_nonzero() + v.count_nonzero()
        want, tol, _ = ref.attention(q[10:], _rest(b), window=12)
        within(paged_attention(q[10:], *_rest(b).args(), window=12), want, tol)


def _rest(b):
    """The same cache with half of the new tokens."""
    r = ref.Batch([10], [30], 16, 3, 64, BF16)
    r.keys, r.values, r.page_table = b.keys, b.values, b.page_table
    return r


def test_tokens_without_a_place_are_not_stored():
    """Pages outside of the pool, positions behind the table and below zero."""
    b = ref.Batch([8, 8, 8, 8], [8, 8, 8, 8], 4, 1, 64, F16)
    b.page_table[0, 1] = -1
    b.page_table[1, 0] = b.keys.shape[0]
    b.page_table[2, 0] = 2 ** 31 - 1
    b.lengths[2] = 100  # 92 .. 99: the table ends at 8
    b.lengths[3] = 5    # -3 .. 4
    keys = b.keys.clone()
    q, k, v = randn(32, 3, 64, dtype=F16).split((1, 1, 1), 1)
    append_heads(q, k, v, *b.args())
    table = b.page_table.cpu()
    for s, i, position in [(0, i, i) for i in range(4)] + [(1, i, i) for i in range(4, 8)] + [(3, i, i - 3) for i in range(3, 8)]:
        page = int(table[s, position // 4])
        assert torch.equal(b.keys[page, position % 4], k[8 * s + i])
        keys[page, position % 4] = k[8 * s + i]
    assert torch.equal(b.keys, keys)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def check_attention(new, lengths, page, heads, kv, dim, dtype, window=0, layout="tokens", scale=None, behind=0, seed=0,
                    spread=1.5):
    b = ref.Batch(new, lengths, page, kv, dim, dtype, layout=layout, behind=behind, seed=seed)
    q = (spread * randn(b.tokens, heads, dim, seed=seed + 9)).to(dtype)
    out = torch.full_like(q, 7.0)
    got = paged_attention(q, *b.args(), scale=scale, window=window, out=out)
    want, tol, inside = ref.attention(q, b, scale, window)
    within(got[inside.cuda()], want[inside.cuda()], tol[inside.cuda()])
    assert (got[~inside.cuda()] == 7).all()
    assert torch.equal(paged_attention(q, *b.args(), scale=scale, window=window)[inside.cuda()], got[inside.cuda()])
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [128, 64, 80, 8, 120, 20, 130, 256, 512])
def test_attention_head_sizes(dtype, dim):
    check_attention([1, 37, 0, 150], [1, 40, 7, 333], 16, 6, 2, dim, dtype)


@pytest.mark.parametrize("page", [1, 5, 16, 32, 48, 64, 80, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["tokens", "heads", "odd"])
def test_attention_pages(page, layout):
    check_attention([1, 33, 129], [700, 200, 129], page, 8, 2, 128, BF16, layout=layout)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 383, 511, 512, 640, 1023, 4097])
@pytest.mark.parametrize("group", [1, 4, 7])
def test_attention_of_one_token(length, group):
    check_attention([1], [length], 16, 2 * group, 2, 128, BF16)
    check_attention([1, 1, 1], [length, 1, length + 3], 64, group, 1, 64, F16)


@pytest.mark.parametrize("new", [1, 2, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1000])
@pytest.mark.parametrize("group,before", [(1, 0), (2, 77), (3, 1000), (8, 0), (130, 3)])
def test_attention_of_prompts(new, group, before):
    if new * group > 20000:
        new = 160
    check_attention([new], [new + before], 32, group, 1, 128, BF16)
    check_attention([new, 1], [new + before, new], 16, 2 * group, 2, 64, F16)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 127, 128, 129, 256, 300, 5000])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 72), (F32, 64)], ids=str)
def test_attention_windows(window, dtype, dim):
    check_attention([1, 3, 200, 130], [600, 129, 200, 900], 16, 4, 2, dim, dtype, window=window)


def test_attention_of_many_sequences():
    lengths = [(37 * i) % 900 + 1 for i in range(300)]
    check_attention([1] * 300, lengths, 16, 8, 2, 128, BF16)
    new = [(i * 13) % 29 if i % 3 else 0 for i in range(200)]
    check_attention(new, [n + (i * 71) % 500 for i, n in enumerate(new)], 32, 4, 4, 64, F16)


def test_attention_of_long_caches():
    check_attention([1], [40000], 128, 8, 1, 128, BF16)
    check_attention([1, 20, 1], [17, 30011, 9000], 64, 16, 2, 128, F16)
    check_attention([300], [20000], 64, 2, 2, 128, BF16)


def test_attention_of_a_long_prompt():
    check_attention([3000], [3000], 64, 4, 2, 128, BF16)
    check_attention([1500, 2000], [1500, 4100], 16, 4, 1, 128, F16)


def test_rows_that_see_nothing_are_zero_and_rows_of_no_sequence_stay():
    b = ref.Batch([6, 0, 3, 5], [2, 9, 0, 5], 16, 1, 64, BF16, behind=4)
    q = randn(b.tokens, 2, 64, dtype=BF16)
    out = torch.full_like(q, 5.0)
    paged_attention(q, *b.args(), out=out)
    assert (out[:4] == 0).all() and (out[6:9] == 0).all() and (out[14:] == 5).all()
    assert torch.equal(out[4], b.values[b.page_table[0, 0], 0].expand(2, 64))  # one key: its value
    assert torch.equal(out[9], b.values[b.page_table[3, 0], 0].expand(2, 64))


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("new,length,window,group", [(1, 100, 0, 4), (1, 130, 50, 4), (20, 150, 0, 4), (20, 400, 33, 4),
                                                     (300, 300, 0, 1), (300, 700, 140, 2), (140, 141, 5, 8)])
def test_what_a_token_does_not_see_does_not_matter(dtype, new, length, window, group):
    """NaN and infinities behind the length, in other pages, in later tokens and before the window."""
    b = ref.Batch([new], [length], 16, 2, 128, dtype)
    q = randn(new, 2 * group, 128, dtype=dtype)
    clean = paged_attention(q, *b.args(), window=window)
    used = torch.zeros(b.keys.shape[:2], dtype=torch.bool, device="cuda")
    first = max(0, length - new - window + 1) if window else 0
    page, col = b.slots(0, torch.arange(first, length, device="cuda"))
    used[page, col] = True
    for bad in (math.nan, math.inf, -math.inf):
        b.keys[~used], b.values[~used] = bad, bad
        assert torch.equal(paged_attention(q, *b.args(), window=window), clean)
    if new > 1:  # the last token's key and value, then the first one's that some rows see
        page, col = b.slots(0, torch.tensor([length - 1], device="cuda"))
        kept = b.keys[page, col].clone(), b.values[page, col].clone()
        b.values[page, col, 1, 3] = math.inf
        got = paged_attention(q, *b.args(), window=window)
        assert torch.equal(got[:-1], clean[:-1]) and torch.equal(got[-1, :group], clean[-1, :group])
        assert not got[-1, group:, 3].isfinite().any() and torch.equal(got[-1, group:, 4:], clean[-1, group:, 4:])
        b.values[page, col] = kept[1]
        b.keys[page, col, 0, 0] = math.nan
        got = paged_attention(q, *b.args(), window=window)
        assert torch.equal(got[:-1], clean[:-1]) and got[-1, :group].isnan().all()
        b.keys[page, col] = kept[0]
    if window:
        position = max(0, length - new - 3)
        page, col = b.slots(0, torch.tensor([position], device="cuda"))
        b.values[page, col] = math.nan
        got = paged_attention(q, *b.args(), window=window)
        p = torch.arange(length - new, length, device="cuda")
        sees = (p >= position) & (p - position < window)
        assert torch.equal(got[~sees], clean[~sees]) and not got[sees].isfinite().any()


def test_scores_of_every_size():
    """Scores up to thousands, all alike, and all -inf but one."""
    check_attention([1, 140], [300, 300], 16, 4, 2, 128, BF16, scale=3.0, spread=8.0)
    check_attention([1, 140], [300, 300], 16, 4, 2, 128, F16, scale=0.0)
    check_attention([1, 140], [300, 300], 16, 4, 2, 128, F16, scale=-0.2)
    b = ref.Batch([1, 130], [200, 130], 16, 1, 64, BF16)
    b.keys[:] = 0
    b.keys[..., 0] = -math.inf
    page, col = b.slots(0, torch.tensor([150], device="cuda"))
    b.keys[page, col] = 0
    q = torch.ones(131, 1, 64, dtype=BF16, device="cuda")
    got = paged_attention(q, *b.args())
    assert torch.equal(got[0, 0], b.values[page, col][0, 0])
    assert got[1:].isnan().all()  # every key that they see scores -inf: 0 / 0, as a softmax has it
    rising = ref.Batch([1], [1000], 16, 1, 64, F16)  # the maximum moves with every key
    page, col = rising.slots(0, torch.arange(1000, device="cuda"))
    rising.keys[:] = 0
    rising.keys[page, col, 0, 0] = torch.arange(1000, device="cuda").half()
    q = torch.ones(1, 1, 64, dtype=F16, device="cuda")
    want, tol, _ = ref.attention(q, rising, 1.0)
    within(paged_attention(q, *rising.args(), scale=1.0), want, tol)


def test_bad_pages_and_lengths_make_nan_and_no_fault():
    b = ref.Batch([1, 1, 1, 40, 1], [100, 100, 90, 200, 50], 16, 2, 128, BF16)
    q = randn(b.tokens, 4, 128, dtype=BF16)
    clean = paged_attention(q, *b.args())
    b.page_table[0, 2] = b.keys.shape[0]
    b.page_table[1, 0] = -7
    b.lengths[2] = 2 ** 31 - 1
    b.page_table[3, 0] = 2 ** 31 - 1
    got = paged_attention(q, *b.args())
    assert got[:43].isnan().all() and torch.equal(got[43], clean[43])


def test_a_long_cache_beyond_32_bit_offsets():
    """A pool of more than 2^32 bytes and 2^31 elements, the pages used at its end."""
    pages, page, kv, dim = 1100, 1024, 16, 128
    keys = torch.empty(pages, page, kv, dim, dtype=F16, device="cuda")
    values = torch.empty_like(keys)
    b = ref.Batch([3, 1], [2000, 50], page, kv, dim, F16)
    n = b.keys.shape[0]
    keys[-n:], values[-n:] = b.keys, b.values
    q = randn(4, 16, dim, dtype=F16)
    want = paged_attention(q, *b.args())
    b.page_table = torch.where(b.page_table >= 0, b.page_table + (pages - n), b.page_table)
    assert torch.equal(paged_attention(q, keys, values, *b.args()[2:]), want)
    k = randn(4, kv, dim, dtype=F16, seed=3)
    append_heads(q, k, k, keys, values, *b.args()[2:])
    at, col = b.slots(0, torch.arange(1997, 2000, device="cuda"))
    assert torch.equal(keys[at, col], k[:3]) and torch.equal(values[at, col], k[:3])


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def check_logprobs(x, tokens, top):
    got = token_logprobs(x, tokens, top=top)
    want = ref.logprobs(x, tokens, top)
    n = x.shape[1]
    high = x.double().amax(1)
    logs = torch.logsumexp(x.double() - high[:, None], 1)
    # x - max, its logarithm of the sum and their difference in fp32; sums of n / 512 terms, a tree of 12 levels and
    # exponentials of 2^-21
    sums = (n / 512 + 16) * 2.0 ** -24 + 2.0 ** -21

    def tol(values):
        return 2.0 ** -23 * ((values + logs).abs() + logs.abs() + values.abs()) + sums
    within(got[0], want[0], tol(want[0]))
    lp = torch.log_softmax(x.double(), 1)
    spread = torch.where(lp > -1e30, lp.exp() * (x.double() - high[:, None]).clamp(min=-1e30).abs(), torch.zeros_like(lp)).sum(1)
    within(got[1], want[1], (2 * sums + 2.0 ** -21 * (1 + spread)) * (1 + spread) + 2.0 ** -22 * logs.abs())
    if top:
        assert torch.equal(got[3], want[3])
        within(got[2], want[2], tol(want[2].T).T if top == 1 else torch.stack([tol(c) for c in want[2].T], 1))
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 64, 64), (1, 1000, 20), (5, 4096, 64), (1, 32768, 5),
                                     (2, 32001, 0), (37, 50001, 20), (1, 200003, 64), (300, 513, 8), (700, 3001, 3)])
def test_logprobs(dtype, m, n, top):
    x = (3 * randn(m, n, seed=n)).to(dtype)
    tokens = torch.randint(n, (m,), generator=gen(3), device="cuda")
    check_logprobs(x, tokens, top)
    check_logprobs(x, tokens.int(), top)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_of_views(dtype):
    wide = randn(9, 5003, dtype=dtype)
    tokens = torch.randint(4000, (9,), generator=gen(3), device="cuda")
    for x in (wide[:, 1:4502], wide[:, 3:4003], wide[2:9:2, :4001], randn(4001, 9, dtype=dtype).T, wide[:1, 5:]):
        check_logprobs(x, tokens[:x.shape[0]], 7)
    strided = torch.stack([tokens, tokens + 1], 1)[:, 0]
    check_logprobs(wide, strided, 3)
    assert [t.shape for t in token_logprobs(wide[:0], tokens[:0], top=3)] == [(0,), (0,), (0, 3), (0, 3)]


@pytest.mark.parametrize("m,n", [(1, 40000), (400, 5000), (2, 900)])
def test_equal_logits_go_by_the_lowest_token(m, n):
    tokens = torch.zeros(m, dtype=torch.int64, device="cuda")
    check_logprobs(torch.zeros(m, n, device="cuda"), tokens, 64)
    check_logprobs((randn(m, n) * 0.7).round().half(), tokens, 64)  # a few values, thousands of each
    x = torch.zeros(m, n, device="cuda")
    x[:, 1::2] = -0.0  # zeros alike
    check_logprobs(x, tokens, 33)
    x[:, n - 40:] = 1.0
    check_logprobs(x, tokens, 50)
    check_logprobs(torch.arange(n, device="cuda").float().expand(m, n) / 100, tokens + n - 1, 20)  # rising
    check_logprobs(torch.arange(n, 0, -1, device="cuda").float().expand(m, n) / 100, tokens, 20)  # falling
    x = randn(m, n)
    x[:, 100:400] += 100  # all of the top in one place
    check_logprobs(x, tokens + 150, 64)


@pytest.mark.parametrize("n", [70, 3000, 100000])
def test_logits_that_are_not_finite(n):
    tokens = torch.tensor([0, 1, 2, 3, -1, n, 2], device="cuda")
    x = randn(7, n)
    x[0, 5:] = -math.inf          # masked vocabulary: five left
    x[1, 1] = -math.inf
    x[2] = -math.inf
    x[3, 7] = math.nan
    x[6, 3] = math.inf
    lp, entropy, top, ids = token_logprobs(x, tokens, top=8)
    want = ref.logprobs(x, tokens, 8)
    assert torch.equal(ids, want[3])
    for got, exact in ((lp, want[0]), (entropy, want[1]), (top, want[2])):
        assert torch.equal(got.isnan(), exact.isnan()) and torch.equal(got == -math.inf, exact == -math.inf)
        keep = exact.isfinite()
        assert torch.allclose(got[keep].double(), exact[keep], rtol=1e-5, atol=1e-5)
    assert lp[1] == -math.inf and lp[4].isnan() and lp[5].isnan() and lp[2].isnan() and entropy[2].isnan()
    assert entropy[3].isnan() and (ids[2] == torch.arange(8, device="cuda")).all()
    x = torch.full((2, n), math.nan, device="cuda")
    x[1, 2] = 1.0
    assert torch.equal(token_logprobs(x, tokens[:2], top=3)[3].cpu(), torch.tensor([[0, 1, 2], [2, 0, 1]]))


def test_large_logits_and_many_rows():
    x = 1e4 * randn(3, 9000)
    check_logprobs(x, torch.tensor([0, 5, 8999], device="cuda"), 4)
    x = torch.full((2, 5000), -3e38, device="cuda")
    x[:, 77] = 3e38
    lp, entropy, top, ids = token_logprobs(x, torch.tensor([77, 0], device="cuda"), top=2)
    assert lp[0] == 0 and lp[1] == -math.inf and (entropy == 0).all() and ids.tolist() == [[77, 0], [77, 0]]
    big = torch.zeros(70000, 33, dtype=F16, device="cuda")
    big[:, 3] = 1
    assert (token_logprobs(big, torch.zeros(70000, dtype=torch.int32, device="cuda"), top=1)[3] == 3).all()


# ---------------------------------------------------------------------------
# together, on streams and in graphs
# ---------------------------------------------------------------------------
class Layer:
    """A decoder layer's attention half and a vocabulary, in 8-bit products."""

    def __init__(self, heads=8, kv=2, dim=64, width=256, vocabulary=1000):
        self.heads, self.kv, self.dim = heads, kv, dim
        self.qkv = quantize_weight(randn((heads + 2 * kv) * dim, width, seed=1) / width ** 0.5)
        self.out = quantize_weight(randn(width, heads * dim, seed=2) / (heads * dim) ** 0.5)
        self.words = quantize_weight(4 * randn(vocabulary, width, seed=3) / width ** 0.5)
        self.norm = 1 + 0.1 * randn(width, seed=4)
        self.head_norm = 1 + 0.1 * randn(dim, seed=5)
        self.frequencies = rope_frequencies(dim)

    def __call__(self, x, batch, tokens):
        h = rms_norm(x, self.norm, quantize=True)
        qkv = fp8_linear(h, self.qkv, out_dtype=BF16).unflatten(1, (-1, self.dim))
        q, k, v = qkv.split((self.heads, self.kv, self.kv), 1)
        q = append_heads(q, k, v, *batch.args(), frequencies=self.frequencies, q_weight=self.head_norm,
                         k_weight=self.head_norm, norm=True)
        o = paged_attention(q, *batch.args())
        x = fp8_linear(o.flatten(1), self.out, residual=x, out_dtype=BF16)
        h = rms_norm(x, self.norm, quantize=True)
        return token_logprobs(fp8_linear(h, self.words), tokens, top=4)


def test_a_prompt_at_once_and_token_by_token_agree():
    """Scores of a prompt's tokens, in one pass, in chunks and one by one through the cache."""
    layer, n = Layer(), 70
    x = randn(n, 256, dtype=BF16)
    tokens = torch.randint(1000, (n,), generator=gen(8), device="cuda")
    whole = layer(x, ref.Batch([n], [n], 16, 2, 64, BF16), tokens)
    # the products sum in another order for another number of rows: single roundings of bf16 and 8-bit values differ,
    # a step of an 8-bit value is 2^-3 of it, of which a logit of norm 4 averages 256
    for step in (1, 33):
        cache = ref.Batch([n], [n], 16, 2, 64, BF16, seed=4)
        done = 0
        while done < n:
            k = min(step, n - done)
            cache.starts = torch.tensor([0, k], dtype=torch.int32, device="cuda")
            cache.lengths = torch.tensor([done + k], dtype=torch.int32, device="cuda")
            got = layer(x[done:done + k], cache, tokens[done:done + k])
            for g, w in zip(got[:3], whole[:3]):
                assert (g - w[done:done + k]).abs().max() < 0.5
            done += k
    assert whole[0].isfinite().all() and (whole[1] > 0).all() and (whole[2].diff(dim=1) <= 0).all()


def test_a_captured_step_follows_its_batch():
    """A decoding step replayed with other lengths, pages, inputs: the same bits as calls of their own."""
    layer = Layer()
    lengths = [[3, 40, 100], [4, 41, 101], [64, 1, 17]]
    batches = [ref.Batch([1, 1, 1], n, 16, 2, 64, BF16, seed=2) for n in lengths]
    xs = [randn(3, 256, dtype=BF16, seed=20 + i) for i in range(3)]
    tokens = torch.tensor([5, 999, 0], device="cuda")
    held = ref.Batch([1, 1, 1], [112, 112, 112], 16, 2, 64, BF16, seed=3)
    x = xs[0].clone()
    layer(x, held, tokens)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        out = layer(x, held, tokens)
    for i in range(3):
        b = batches[i]
        held.keys[:len(b.keys)], held.values[:len(b.values)] = b.keys, b.values
        held.page_table.fill_(-1)
        held.page_table[:, :b.page_table.shape[1]] = b.page_table
        held.lengths.copy_(b.lengths)
        x.copy_(xs[i])
        graph.replay()
        for got, want in zip(out, layer(xs[i], b, tokens)):
            assert torch.equal(got, want)


def test_calls_on_streams_at_once():
    """Streams and two graphs side by side give what one after the other gives."""
    cases = []
    for i, (new, lengths) in enumerate((([1] * 8, [3000] * 8), ([500, 1], [700, 9000]), ([1], [20000]), ([40] * 3, [60] * 3))):
        b = ref.Batch(new, lengths, 16, 2, 128, BF16, seed=i)
        cases.append((randn(b.tokens, 8, 128, dtype=BF16, seed=30 + i), b.args()))
    want = [paged_attention(q, *args) for q, args in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for s, g, (q, args) in zip(streams, got, cases):
            with torch.cuda.stream(s):
                g.append(paged_attention(q, *args))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
    graphs, outs = [], []
    for q, args in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, *args))
        graphs.append(graph)
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_outputs_count_as_changed():
    b = ref.Batch([2], [2], 16, 1, 64, BF16)
    q, k, v = randn(2, 3, 64, dtype=BF16).split((1, 1, 1), 1)
    before = b.keys._version, b.values._version
    append_heads(q, k, v, *b.args())
    assert b.keys._version > before[0] and b.values._version > before[1]
    w = torch.ones(2, 1, 64, dtype=BF16, device="cuda", requires_grad=True)
    saved = w * 2
    y = (saved * saved).sum()
    paged_attention(q, *b.args(), out=saved.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_a_wait_that_runs_out_is_reported_once():
    """The failure-detection hook: a kernel whose products never come leaves, the next call says so, later ones work."""
    from forgetune_b200 import ForgeTuneRuntimeError, _native
    b = ref.Batch([1, 300], [500, 300], 16, 2, 128, BF16)
    q = randn(b.tokens, 8, 128, dtype=BF16)
    want = paged_attention(q, *b.args())
    torch.cuda.synchronize()
    try:
        _native.lib().ftb_fp8_set_fault_injection(1)
        paged_attention(q, *b.args())
        torch.cuda.synchronize()
    finally:
        _native.lib().ftb_fp8_set_fault_injection(0)
    with pytest.raises(ForgeTuneRuntimeError, match="gave up"):
        rotate_heads(q, torch.zeros(b.tokens, dtype=torch.int32, device="cuda"), rope_frequencies(128))
    assert torch.equal(paged_attention(q, *b.args()), want)


def test_pools_with_strides_of_their_own():
    """A pool that repeats one page, one of rows apart, and one whose pages lie backwards in memory order."""
    b = ref.Batch([3, 20], [64, 40], 16, 2, 64, F16)
    q = randn(b.tokens, 4, 64, dtype=F16)
    for change in (lambda x: x[:1].expand(x.shape), lambda x: torch.cat([x, x], 3)[..., :64],
                   lambda x: x.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)):
        b.keys, b.values = change(b.keys), change(b.values)
        want, tol, inside = ref.attention(q, b)
        within(paged_attention(q, *b.args()), want, tol)


def test_python_refusals():
    b = ref.Batch([2, 3], [4, 9], 16, 2, 64, BF16)
    q, k, v = randn(5, 8, 64, dtype=BF16).split((4, 2, 2), 1)
    f, positions = rope_frequencies(64), torch.arange(5, device="cuda")
    keys, values, table, starts, lengths = b.args()
    from forgetune_b200 import InvalidShapeError
    x = randn(5, 4, 64)

    def attend(**over):
        a = dict(q=q, keys=keys, values=values, page_table=table, starts=starts, lengths=lengths)
        a.update(over)
        return lambda: paged_attention(**a)

    def append(**over):
        a = dict(q=q, k=k, v=v, keys=keys, values=values, page_table=table, starts=starts, lengths=lengths, frequencies=f)
        a.update(over)
        return lambda: append_heads(**a)
    logits, tokens = randn(3, 100), torch.zeros(3, dtype=torch.int64, device="cuda")
    grad = torch.zeros(5, 4, 64, device="cuda", requires_grad=True)
    cases = [
        (TypeError, lambda: rotate_heads(x.double(), positions, f)), (TypeError, lambda: rotate_heads(x, positions.float(), f)),
        (TypeError, lambda: rotate_heads(x, positions, f.float())), (InvalidShapeError, lambda: rotate_heads(x[0], positions, f)),
        (InvalidShapeError, lambda: rotate_heads(x, positions[:4], f)), (InvalidShapeError, lambda: rotate_heads(x, positions, rope_frequencies(66))),
        (ValueError, lambda: rotate_heads(x, positions, f, weight=torch.ones(64, device="cuda"))),
        (InvalidShapeError, lambda: rotate_heads(x, positions, f, weight=torch.ones(32, device="cuda"), norm=True)),
        (TypeError, lambda: rotate_heads(x, positions, f, out=torch.empty_like(x).half())),
        (InvalidShapeError, lambda: rotate_heads(x, positions, f, out=torch.empty(5, 4, 128, device="cuda")[..., ::2])),
        (ValueError, lambda: rotate_heads(x, positions.cpu(), f)), (ValueError, lambda: rotate_heads(x, positions, f, out=grad)),
        (TypeError, append(k=k.float())), (TypeError, append(q=q.half(), k=k.half(), v=v.half())), (InvalidShapeError, append(k=q)),
        (InvalidShapeError, append(q=q[:4])), (TypeError, append(values=values.half())), (InvalidShapeError, append(values=values[:1])),
        (InvalidShapeError, append(keys=torch.empty(3, 16, 2, 128, dtype=BF16, device="cuda")[..., ::2])),
        (TypeError, append(lengths=lengths.long())), (InvalidShapeError, append(starts=starts[1:])), (ValueError, append(page_table=table.cpu())),
        (TypeError, attend(q=q.float())), (InvalidShapeError, attend(q=q[:, :3])), (InvalidShapeError, attend(q=q[..., :32])),
        (ValueError, attend(window=-1)), (InvalidShapeError, attend(lengths=lengths[:1])), (TypeError, attend(page_table=table.float())),
        (TypeError, attend(window="all")), (InvalidShapeError, attend(out=torch.empty(5, 4, 32, dtype=BF16, device="cuda"))),
        (TypeError, lambda: token_logprobs(logits.double(), tokens)), (InvalidShapeError, lambda: token_logprobs(logits, tokens[:2])),
        (ValueError, lambda: token_logprobs(logits, tokens, top=65)), (ValueError, lambda: token_logprobs(logits[:, :5], tokens, top=6)),
        (TypeError, lambda: token_logprobs(logits, tokens.float())), (ValueError, lambda: token_logprobs(logits, tokens, top=-1)),
    ]
    for i, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail("case %d was taken" % i)
    from forgetune_b200 import ForgeTuneRuntimeError
    inside = keys[0, :5]  # heads that lie in the pool that is written
    for call in (attend(out=q), append(k=inside, q=torch.cat([q, q], 1)), append(values=keys)):
        with pytest.raises(ForgeTuneRuntimeError, match="overlap"):
            call()


def test_no_gradients_and_no_tangents():
    import torch.autograd.forward_ad as ad
    x = torch.randn(3, 2, 64, device="cuda", requires_grad=True)
    positions, f = torch.arange(3, device="cuda"), rope_frequencies(64)
    assert not rotate_heads(x, positions, f).requires_grad
    with ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            rotate_heads(ad.make_dual(x.detach(), torch.ones_like(x)), positions, f)
    with torch.no_grad():
        assert rotate_heads(x, positions, f, out=x) is not None


def test_a_negated_view_is_taken_as_what_it_stands_for():
    x = torch.randn(3, 2, 64, dtype=torch.complex64, device="cuda")
    neg = x.conj().imag
    assert neg.is_neg()
    positions, f = torch.arange(3, device="cuda"), rope_frequencies(64)
    assert torch.equal(rotate_heads(neg, positions, f), rotate_heads(neg.resolve_neg(), positions, f))
