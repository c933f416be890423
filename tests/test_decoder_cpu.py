"""The operators around a decoder layer's attention without a GPU: refusals of the C ABI and of the Python entry
points, and the reference they are tested against."""

import ctypes
import math
import struct

import pytest
import torch

from forgetune_b200 import (InvalidShapeError, _native, append_heads, paged_attention, rope_frequencies, rotate_heads,
                            token_logprobs)

from . import decoder_reference as ref

B = 1 << 28  # well aligned addresses far apart that no refused call touches


class Fields:
    """An argument struct of include/forgetune_b200.h: fields of eight bytes, by name."""

    def __init__(self, **fields):
        self.fields = fields

    def call(self, name, **over):
        unknown = set(over) - set(self.fields)
        assert not unknown, unknown
        values = [over.get(k, v) for k, v in self.fields.items()]
        raw = b"".join(struct.pack("=d" if isinstance(v, float) else "=q", v) for v in values)
        fn = getattr(_native.lib(), name)
        return fn(ctypes.c_char_p(raw)) if name.endswith("workspace") else fn(ctypes.c_char_p(raw), None)


def heads(n, at, token, head, type=2):
    return {n: at, n + "_token": token, n + "_head": head, n + "_type": type}


ROTATION = dict(f=90 * B, pairs=32, interleaved=0, amplitude=1.0, norm=0, eps=1e-6)
CACHE = dict(keys=20 * B, values=30 * B, kp=16 * 2 * 64, kt=2 * 64, kh=64, vp=16 * 2 * 64, vt=2 * 64, vh=64, type=2, pages=9,
             page_size=16, kv=2, dim=64)
BATCH = dict(table=40 * B, table_ld=4, most=4, seqs=3, starts=41 * B, lengths=42 * B)
ROTATE = Fields(**heads("x", B, 256, 64), **heads("y", 2 * B, 256, 64), tokens=5, heads=4, dim=64, positions=3 * B,
                positions64=1, **ROTATION, weight=0)
APPEND = Fields(**heads("q", B, 256, 64), **heads("k", 2 * B, 128, 64), **heads("v", 3 * B, 128, 64),
                **heads("o", 4 * B, 256, 64), tokens=5, heads=4, **CACHE, **BATCH, **ROTATION, wq=0, wk=0)
ATTENTION = Fields(**heads("q", B, 256, 64), **heads("o", 4 * B, 256, 64), tokens=5, heads=4, **CACHE, **BATCH, scale=0.1,
                   window=0, work=50 * B, work_bytes=1 << 27)
LOGPROBS = Fields(x=B, ld=1000, type=0, m=7, n=1000, tokens=2 * B, tokens64=1, stride=1, lp=3 * B, entropy=4 * B, top=5,
                  top_lp=5 * B, top_tokens=6 * B)


def refused(args, name, **over):
    rc = args.call(name, **over)
    assert rc == -2, (over, rc, _native.last_error())
    assert name in _native.last_error()


def reaches_the_device(args, name, **over):
    """Allowed as far as the checks go: without a GPU the next step is the device."""
    if _native.device_count() == 0:
        rc = args.call(name, **over)
        assert rc == -5, (over, rc, _native.last_error())


def test_rotate_refusals():
    name = "ftb_rotate_heads"
    assert ROTATE.call(name, tokens=0) == 0 and getattr(_native.lib(), name)(None, None) == -1
    for null in ("x", "y", "positions"):
        assert ROTATE.call(name, **{null: 0}) == -1
    for over in (dict(tokens=-1), dict(tokens=1 << 31), dict(heads=0), dict(dim=0), dict(dim=513), dict(x_type=3), dict(y_type=0),
                 dict(x=B + 1), dict(x_head=63), dict(x_token=255), dict(x_token=-256), dict(y_token=10), dict(y_head=1 << 41),
                 dict(pairs=33), dict(pairs=-1), dict(f=0), dict(f=90 * B + 4), dict(eps=-1.0), dict(eps=math.nan),
                 dict(positions=3 * B + 4), dict(weight=7), dict(y=B + 2), dict(y=B + 128), dict(y=B, y_token=512),
                 dict(y=3 * B), dict(y=90 * B), dict(weight=2 * B)):
        refused(ROTATE, name, **over)
    for over in (dict(), dict(y=B), dict(pairs=0, f=0), dict(positions=3 * B + 4, positions64=0), dict(x_token=64, x_head=320),
                 dict(x_token=512, y=B + 512, y_token=512)):
        reaches_the_device(ROTATE, name, **over)


def test_append_refusals():
    name = "ftb_append_heads"
    assert APPEND.call(name, tokens=0) == 0 and getattr(_native.lib(), name)(None, None) == -1
    for null in ("q", "k", "v", "o", "keys", "values", "table", "starts", "lengths"):
        assert APPEND.call(name, **{null: 0}) == -1
    for over in (dict(tokens=-1), dict(heads=0), dict(heads=5000), dict(type=1), dict(type=7), dict(k_type=1), dict(v_type=0),
                 dict(o_type=0), dict(q_type=1, k_type=1, v_type=1), dict(pages=0), dict(page_size=0), dict(kv=0), dict(dim=600),
                 dict(keys=20 * B + 1), dict(kt=-1), dict(seqs=0), dict(most=0), dict(table_ld=3), dict(table=40 * B + 2),
                 dict(starts=41 * B + 1), dict(lengths=42 * B + 2), dict(pairs=40), dict(wq=2), dict(wk=B + 2), dict(eps=-0.5),
                 dict(kt=63), dict(kp=16), dict(vh=0), dict(vp=100), dict(o=2 * B), dict(o=3 * B + 4), dict(o=B + 2),
                 dict(o=20 * B), dict(o=30 * B + 8), dict(keys=B), dict(values=2 * B), dict(values=41 * B), dict(keys=40 * B),
                 dict(keys=90 * B), dict(values=20 * B), dict(values=20 * B + 64), dict(values=20 * B + 128),
                 dict(q_type=0, k_type=0, v_type=0, o=B)):
        refused(APPEND, name, **over)
    side = dict(kp=16 * 4 * 64, vp=16 * 4 * 64)
    for over in (dict(), dict(o=B), dict(q_type=0, k_type=0, v_type=0), dict(type=0, q_type=0, k_type=0, v_type=0, o_type=0),
                 dict(pairs=0, f=0), dict(norm=1, wq=70 * B, wk=71 * B),
                 dict(side, values=20 * B + 16 * 2 * 64 * 2),                         # halves of each page
                 dict(side, kt=256, vt=256, values=20 * B + 2 * 64 * 2),              # of each token
                 dict(side, kt=256, vt=256, kh=128, vh=128, values=20 * B + 64 * 2),  # of each head
                 dict(kt=64, kh=16 * 64, vt=64, vh=16 * 64)):
        reaches_the_device(APPEND, name, **over)


def test_attention_refusals():
    for name in ("ftb_paged_attention", "ftb_paged_attention_workspace"):
        assert ATTENTION.call(name, tokens=0) == 0
        for null in ("q", "o", "keys", "values", "table", "starts", "lengths"):
            assert ATTENTION.call(name, **{null: 0}) == -1
        for over in (dict(tokens=-1), dict(heads=0), dict(heads=3), dict(type=1), dict(q_type=0), dict(o_type=1), dict(o=B),
                     dict(o=20 * B), dict(o=30 * B + 64), dict(o=40 * B), dict(o=41 * B), dict(o=42 * B), dict(window=-1),
                     dict(scale=math.nan), dict(scale=math.inf), dict(q_head=60), dict(o_token=0), dict(dim=513), dict(seqs=0),
                     dict(lengths=3), dict(keys=20 * B + 1), dict(window=1 << 31), dict(tokens=1 << 28), dict(scale=1e300),
                     dict(scale=-2.9e38)):
            refused(ATTENTION, name, **over)
    assert ATTENTION.call("ftb_paged_attention_workspace") >= 0
    assert _native.lib().ftb_paged_attention(None, None) == -1 and _native.lib().ftb_paged_attention_workspace(None) == -1
    for over in (dict(), dict(values=20 * B), dict(q_token=64, q_head=5 * 64), dict(window=5, scale=0.0)):
        reaches_the_device(ATTENTION, "ftb_paged_attention", **over)


def test_logprobs_refusals():
    name = "ftb_token_logprobs"
    assert LOGPROBS.call(name, m=0) == 0 and getattr(_native.lib(), name)(None, None) == -1
    for null in ("x", "tokens", "lp", "entropy", "top_lp", "top_tokens"):
        assert LOGPROBS.call(name, **{null: 0}) == -1
    for over in (dict(m=-1), dict(n=0), dict(n=1 << 28), dict(type=3), dict(x=B + 2), dict(ld=999), dict(top=-1), dict(top=65),
                 dict(n=4), dict(tokens=2 * B + 4), dict(stride=-1), dict(lp=3 * B + 2), dict(entropy=4 * B + 1),
                 dict(top_tokens=6 * B + 4), dict(top_lp=5 * B + 2), dict(lp=B), dict(entropy=B + 400), dict(top_lp=2 * B),
                 dict(entropy=3 * B), dict(top_tokens=5 * B), dict(top_tokens=3 * B)):
        refused(LOGPROBS, name, **over)
    for over in (dict(), dict(top=0, top_lp=0, top_tokens=0), dict(tokens=2 * B + 4, tokens64=0), dict(type=2)):
        reaches_the_device(LOGPROBS, name, **over)


def test_python_entry_points_refuse_cpu_tensors_and_other_types():
    q = torch.zeros(2, 4, 64)
    cache = torch.zeros(3, 16, 2, 64)
    table, starts, lengths = (torch.zeros(s, dtype=torch.int32) for s in ((1, 2), (2,), (1,)))
    f = rope_frequencies(64, device="cpu")
    for call in (lambda: rotate_heads(q, torch.zeros(2, dtype=torch.int64), f),
                 lambda: append_heads(q, q[:, :2], q[:, :2], cache, cache.clone(), table, starts, lengths),
                 lambda: paged_attention(q, cache, cache, table, starts, lengths),
                 lambda: token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)),
                 lambda: rotate_heads(q.int(), None, f), lambda: paged_attention(None, cache, cache, table, starts, lengths)):
        with pytest.raises(TypeError, match="must be a float32, float16 or bfloat16 CUDA tensor"):
            call()


def test_frequency_refusals():
    for bad in (dict(dim=0), dict(dim=7), dict(dim=64, base=0.0), dict(dim=64, scale=-1.0), dict(dim=64, scaling="other"),
                dict(dim=64, scaling="parts", fast=1.0, slow=2.0)):
        with pytest.raises(ValueError, match="rope_frequencies"):
            rope_frequencies(device="cpu", **bad)


def test_the_reference_attends_as_torch_does():
    """One sequence without a window: torch's own attention in float64 says the same."""
    b = ref.Batch([9], [30], 16, 2, 32, torch.float16, device="cpu")
    q = torch.randn(9, 6, 32).half()
    got, tol, inside = ref.attention(q, b)
    page, col = b.slots(0, torch.arange(30))
    k, v = (x[page, col].double().transpose(0, 1).repeat_interleave(3, 0) for x in (b.keys, b.values))
    mask = torch.arange(30) <= torch.arange(21, 30)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask).transpose(0, 1)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12) and inside.all() and (tol > 0).all()


def test_the_reference_rotates_as_complex_numbers_do():
    x = torch.randn(5, 3, 16, dtype=torch.float64)
    f = rope_frequencies(16, device="cpu")
    positions = torch.tensor([0, 1, 7, -3, 100000])
    y, _ = ref.rotate(x, positions, f, interleaved=True)
    turn = torch.polar(torch.ones(5, 1, 8, dtype=torch.float64), positions.double()[:, None, None] * f)
    want = torch.view_as_real(torch.view_as_complex(x.unflatten(2, (8, 2))) * turn).flatten(2)
    assert torch.allclose(y, want, atol=1e-12)
    order = torch.cat([torch.arange(0, 16, 2), torch.arange(1, 16, 2)])
    assert torch.allclose(ref.rotate(x[..., order], positions, f)[0], want[..., order], atol=1e-12)


def test_the_reference_scores_as_torch_does():
    x = torch.randn(4, 50)
    x[1, 7] = x[1, 3]
    tokens = torch.tensor([0, 3, 49, 50])
    lp, entropy, top, ids = ref.logprobs(x, tokens, 6)
    d = torch.distributions.Categorical(logits=x.double())
    assert torch.allclose(entropy, d.entropy()) and torch.allclose(lp[:3], d.log_prob(tokens.clamp(max=49))[:3]) and lp[3].isnan()
    assert torch.allclose(top, x.double().log_softmax(1).topk(6).values)
    assert (ids[1] == 3).nonzero()[0] + 1 == (ids[1] == 7).nonzero()[0] if (ids[1] == 3).any() else True
