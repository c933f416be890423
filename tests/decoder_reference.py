"""The operators of forgetune_b200.decoder in float64, from their formulas, and batches to try them on."""

import math

import torch

# a rounding to the type is off by at most this, relative to the value
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
assert all(HALF_STEP[t] == torch.finfo(t).eps / 2 for t in HALF_STEP)


def rotate(x, positions, frequencies, weight=None, eps=1e-6, norm=False, interleaved=False, amplitude=1.0):
    """Returns the result and, of each element, the magnitude that its fp32 error is relative to."""
    x = x.double()
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        x = x if weight is None else x * weight.double()
    y, size = x.clone(), x.abs()
    if frequencies is not None:
        r = frequencies.shape[0]
        angle = (positions.double()[:, None] * frequencies)[:, None]
        i = torch.arange(r, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
        y[..., a] = amplitude * (x[..., a] * angle.cos() - x[..., b] * angle.sin())
        y[..., b] = amplitude * (x[..., b] * angle.cos() + x[..., a] * angle.sin())
        size[..., a] = size[..., b] = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return y, size


def rotate_tolerance(y, size, dtype):
    """One rounding of the result; before it fp32: the sum of squares (dim terms, half of its relative error in the
    root), division, root, weight, cosine and sine (2^-22 with the rounding of their angle), products and sum."""
    return HALF_STEP[dtype] * y.abs() + (y.shape[-1] / 2 + 16) * 2.0 ** -24 * size + (2.0 ** -24 if dtype == torch.float16 else 1e-37)


class Batch:
    """Sequences of `new` new tokens and `lengths` tokens with them over a pool of pages in random order."""

    def __init__(self, new, lengths, page, kv, dim, dtype, device="cuda", seed=0, behind=0, layout="tokens", spare=2):
        g = torch.Generator().manual_seed(seed)
        self.new, self.whole, self.page = list(new), list(lengths), page
        need = [max(0, -(-n // page)) for n in self.whole]
        most = max(1, max(need))
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(need), most), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.tokens = sum(self.new) + behind
        self.page_table = table.to(device)
        self.starts = torch.tensor([0] + self.new).cumsum(0).int().to(device)
        self.lengths = torch.tensor(self.whole).int().to(device)

        def pool():
            if layout == "heads":
                return torch.randn(pages, kv, page, dim, generator=g).to(dtype).to(device).transpose(1, 2)
            if layout == "odd":  # no 16-byte boundary anywhere
                wide = torch.randn(pages, page, kv, dim + 3, generator=g).to(dtype).to(device)
                return wide[..., 1:dim + 1]
            return torch.randn(pages, page, kv, dim, generator=g).to(dtype).to(device)
        self.keys, self.values = pool(), pool()

    def args(self):
        return self.keys, self.values, self.page_table, self.starts, self.lengths

    def positions(self):
        """Of each new token; int64 on the CPU."""
        return torch.cat([torch.arange(n - k, n) for k, n in zip(self.new, self.whole)] + [torch.zeros(0, dtype=torch.int64)])

    def slots(self, b, positions):
        return self.page_table[b].long()[positions // self.page], positions % self.page


def attention(q, batch, scale=None, window=0, least=2.0 ** -25):
    """float64 result, its tolerance, and which rows belong to a sequence.  float16: a weight below the smallest normal
    number is off by at most `least`, relative to the row's largest."""
    tokens, heads, dim = q.shape
    kv = batch.keys.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    inside = torch.zeros(tokens, dtype=torch.bool)
    half = HALF_STEP[q.dtype]
    at = 0
    for b, (n, whole) in enumerate(zip(batch.new, batch.whole)):
        if n == 0:
            continue
        inside[at:at + n] = True
        if whole > 0:
            page, col = batch.slots(b, torch.arange(whole, device=q.device))
            k = batch.keys[page, col].double().repeat_interleave(heads // kv, 1)
            v = batch.values[page, col].double().repeat_interleave(heads // kv, 1)
            x = q[at:at + n].double() * scale
            p = torch.arange(whole - n, whole, device=q.device)[:, None]
            j = torch.arange(whole, device=q.device)
            seen = j <= p
            if window:
                seen &= j > p - window
            s = torch.einsum("thd,jhd->htj", x, k).masked_fill(~seen, -math.inf)
            # fp32 sums of dim products; 2^-20 for the exponent's argument and the exponential
            size = torch.einsum("thd,jhd->htj", x.abs(), k.abs()).masked_fill(~seen, 0)
            off = (dim + 8) * 2.0 ** -24 * size.amax(2).T[..., None] + 2.0 ** -20
            w = torch.softmax(s, 2)
            w = torch.where(seen.any(1)[None, :, None], w, torch.zeros_like(w))
            o = torch.einsum("htj,jhd->thd", w, v)
            mean = torch.einsum("htj,jhd->thd", w, v.abs())
            # the result's rounding; each weight's rounding and error; sums of `whole` terms in fp32 (which the tensor
            # cores truncate); weights below the smallest normal fp16 number
            out[at:at + n] = o
            tol[at:at + n] = half * o.abs() + (half + 2 * off + whole * 2.0 ** -23) * mean
            if q.dtype == torch.float16:
                # and of the result below the smallest normal number: half of float16's smallest step, 2^-25
                tol[at:at + n] += (whole * least + 2.0 ** -25) * max(1.0, float(v.abs().max()))
        at += n
    return out, tol + 1e-30, inside


def logprobs(x, tokens, top):
    x = x.double()
    lp = torch.log_softmax(x, 1)
    token = tokens.long().clamp(0, x.shape[1] - 1)
    of_token = lp.gather(1, token[:, None])[:, 0]
    of_token = torch.where((tokens >= 0) & (tokens < x.shape[1]), of_token, torch.full_like(of_token, math.nan))
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    entropy = torch.where(lp.isnan().any(1), torch.full_like(entropy, math.nan), entropy)
    order = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    # NaN behind -inf, equal values by index
    rank = torch.argsort(x.isnan().double(), dim=1, stable=True)
    first = torch.argsort(order.gather(1, rank), dim=1, descending=True, stable=True)
    ids = rank.gather(1, first)[:, :top]
    return of_token, entropy, lp.gather(1, ids), ids
