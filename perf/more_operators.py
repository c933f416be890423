"""The operators around a decoder layer's attention and behind its logits as they are measured.

``rotate_heads`` turns the heads of queries or keys by their positions, with an
optional norm of each head; ``append_heads`` does this for a batch's new tokens
and stores keys and values into a paged cache; ``paged_attention`` attends from
the new tokens over the cache; ``token_logprobs`` scores given tokens against
the logits.  They are used in this order around the framework's 8-bit products.

Cases with ``own`` false run the operators' plain forms in elementary torch
operations; with ``own`` true they make the framework's calls on the same
tensors.
"""

import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token's queries between two layers: latency alone counts
        {"name": "rotate_row", "op": "rotate", "t": 1, "heads": 32, "dim": 128, "type": "bf16", "rot": 128,
         "interleaved": False, "norm": False, "far": 4096, "scale": 1.0},
        # a long document in fp32: part of each head, neighbouring pairs, far positions, stretched frequencies
        {"name": "rotate_far_f32", "op": "rotate", "t": 16384, "heads": 16, "dim": 128, "type": "f32", "rot": 64,
         "interleaved": True, "norm": True, "far": 1000000, "scale": 32.0},
        # sixteen sequences decoding: one token each into the cache, heads normalised
        {"name": "append_tokens", "op": "append", "b": 16, "new": 1, "ctx": 1500, "heads": 32, "kv": 8, "dim": 128,
         "page": 16, "type": "bf16", "rot": 128, "interleaved": False, "norm": True},
        # prompts of unlike length written to the cache, queries, keys and values side by side in the product's rows
        {"name": "append_prompts", "op": "append", "b": 5, "new": 4001, "ctx": 0, "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "type": "bf16", "rot": 128, "interleaved": False, "norm": True},
        # the first token after a short prompt: latency
        {"name": "attend_token", "op": "attend", "b": 1, "new": 1, "ctx": 777, "heads": 32, "kv": 8, "dim": 128,
         "page": 16, "type": "bf16", "window": 0},
        # many sequences decoding side by side, contexts of unlike length: the cache's bytes bound it
        {"name": "attend_tokens", "op": "attend", "b": 64, "new": 1, "ctx": 8192, "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "type": "bf16", "window": 0},
        # one sequence decoding at the end of a very long context: one row of work over all SMs
        {"name": "attend_far_token", "op": "attend", "b": 1, "new": 1, "ctx": 131072, "heads": 32, "kv": 4, "dim": 128,
         "page": 128, "type": "f16", "window": 0},
        # chunks of unlike length over a window, an odd head size, seven queries to a key
        {"name": "attend_chunks", "op": "attend", "b": 7, "new": 1000, "ctx": 4099, "heads": 14, "kv": 2, "dim": 80,
         "page": 16, "type": "f16", "window": 1024},
        # a whole prompt at once: the tensor cores bound it
        {"name": "attend_prompt", "op": "attend", "b": 1, "new": 8192, "ctx": 0, "heads": 32, "kv": 8, "dim": 128,
         "page": 64, "type": "bf16", "window": 0},
        # the next token's distribution of one sequence, with alternatives
        {"name": "logprobs_row", "op": "logprobs", "m": 1, "n": 32768, "type": "f32", "top": 5},
        # the tokens of a short prompt over an odd vocabulary
        {"name": "logprobs_ragged", "op": "logprobs", "m": 333, "n": 50001, "type": "f16", "top": 20},
        # a batch of long answers scored: the logits' bytes bound it
        {"name": "logprobs_large", "op": "logprobs", "m": 4096, "n": 131072, "type": "bf16", "top": 8},
    ]


def _spread(rng, low, high):
    """A size spread over its logarithm, odd ones among them."""
    v = int(round(low * (high / low) ** rng.random()))
    if v > 64 and rng.random() < 0.5:  # half of the longer ones as real layers have them
        v = max(64, v // 64 * 64)
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend", "attend", "logprobs"])
    if op == "logprobs":
        while True:
            m, n = _spread(rng, 1, 4096), _spread(rng, 512, 131072)
            if m * n <= 1 << 28:
                break
        return {"op": op, "m": m, "n": n, "type": rng.choice(sorted(TYPES)), "top": rng.choice([0, 1, 5, 8, 20])}
    dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 16)])
    rot = rng.choice([dim, dim, dim // 4 * 2])
    if op == "rotate":
        while True:
            t, heads = _spread(rng, 1, 16384), rng.randint(1, 64)
            if t * heads * dim <= 16384 * 16 * 128:
                break
        return {"op": op, "t": t, "heads": heads, "dim": dim, "type": rng.choice(sorted(TYPES)), "rot": rot,
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5, "far": _spread(rng, 1024, 1000000),
                "scale": rng.choice([1.0, 8.0, 32.0])}
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    case = {"op": op, "heads": kv * group, "kv": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        while True:
            b, new = _spread(rng, 1, 64), rng.choice([1, _spread(rng, 1, 4096)])
            ctx = _spread(rng, 1, 4096)
            if b * new * (kv * group + 2 * kv) * dim <= 5 * 4001 * 48 * 128 and b * (ctx + new) <= 1 << 16:
                break
        return {**case, "b": b, "new": new, "ctx": ctx, "type": rng.choice(sorted(TYPES)), "rot": rot,
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5}
    while True:
        b, new, ctx = _spread(rng, 1, 64), rng.choice([1, 1, _spread(rng, 2, 8192)]), _spread(rng, 1, 131072)
        tokens = b * (ctx + new)
        if new * tokens * kv * group <= 1 << 30 and tokens * kv <= 1 << 21:
            break
    return {**case, "b": b, "new": new, "ctx": ctx, "type": rng.choice(["bf16", "f16"]),
            "window": rng.choice([0, 0, 0, _spread(rng, 16, 4096)])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sequences(case):
    """New tokens and length (with them) of each sequence: the longest first, the others spread below it."""
    golden = 0.6180339887498949
    new, length = [], []
    for b in range(case["b"]):
        part = 1.0 if b == 0 else (b * golden) % 1.0
        n = max(1, int(round(case["new"] * part)))
        new.append(n)
        length.append(n + int(round(case["ctx"] * (1.0 if b == 0 else (0.3 + b * golden) % 1.0))))
    return new, length


def _frequencies(rot, scale):
    """Rotary frequencies; `scale` > 1 stretches the slow ones, which turn less than once in 8192 tokens, and keeps
    the fast ones, in between by a ramp."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    if scale == 1.0:
        return f
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return f * keep + f / scale * (1 - keep)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], TYPES[case["type"]]
    state = {"op": op, "dtype": dtype}
    if op == "logprobs":
        m, n = case["m"], case["n"]
        x = 2.5 * torch.randn(m, n, generator=g, device="cuda")  # a few tokens hold most of the probability
        state["logits"] = x.to(dtype)
        likely = x.topk(4, 1).indices.gather(1, torch.randint(4, (m, 1), generator=g, device="cuda"))[:, 0]
        other = torch.randint(n, (m,), generator=g, device="cuda")
        state["tokens"] = torch.where(torch.rand(m, generator=g, device="cuda") < 0.7, likely, other)
        state["top"] = case["top"]
        return state
    d = case["dim"]
    if op in ("rotate", "append"):
        state["frequencies"] = _frequencies(case["rot"], case.get("scale", 1.0))
        state["interleaved"], state["norm"] = case["interleaved"], case["norm"]
        state["amplitude"] = 0.1 * math.log(case.get("scale", 1.0)) + 1.0
    if op == "rotate":
        state["x"] = _randn(g, case["t"], case["heads"], d, dtype=dtype)
        state["positions"] = torch.randint(case["far"], (case["t"],), generator=g, device="cuda")
        state["weight"] = 1 + 0.1 * _randn(g, d) if case["norm"] else None
        return state
    heads, kv, page = case["heads"], case["kv"], case["page"]
    new, length = _sequences(case)
    t, b = sum(new), case["b"]
    most = max(-(-n // page) for n in length)
    pages = sum(-(-n // page) for n in length) + 3  # a few that belong to nobody
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, most, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(length):
        k = -(-n // page)
        table[i, :k] = order[at:at + k]
        at += k
    starts = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    state.update(page_table=table, starts=starts, lengths=torch.tensor(length, dtype=torch.int32).cuda(), most=max(new),
                 pairs=[new, length])
    held = dtype if dtype != torch.float32 else torch.bfloat16
    state["keys"] = _randn(g, pages, page, kv, d, dtype=held)
    state["values"] = _randn(g, pages, page, kv, d, dtype=held)
    if op == "append":
        qkv = _randn(g, t, (heads + 2 * kv) * d, dtype=dtype)  # as one product leaves them
        state["q"] = qkv[:, :heads * d].unflatten(1, (heads, d))
        state["k"] = qkv[:, heads * d:(heads + kv) * d].unflatten(1, (kv, d))
        state["v"] = qkv[:, (heads + kv) * d:].unflatten(1, (kv, d))
        state["q_weight"] = 1 + 0.1 * _randn(g, d) if case["norm"] else None
        state["k_weight"] = 1 + 0.1 * _randn(g, d) if case["norm"] else None
    else:
        state["q"] = 1.5 * _randn(g, t, heads, d, dtype=dtype)  # scores of some spread: a few keys matter most
        state["window"] = case["window"]
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_rotate(x, positions, frequencies, weight, norm, interleaved, amplitude):
    x = x.float()
    if norm:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * weight
    angle = positions.double()[:, None] * frequencies  # 64 bits: far positions turn many times
    c, s = (amplitude * angle.cos()).float()[:, None], (amplitude * angle.sin()).float()[:, None]
    half = frequencies.shape[0]
    y = x.clone()
    if interleaved:
        x1, x2 = x[:, :, 0:2 * half:2], x[:, :, 1:2 * half:2]
        y[:, :, 0:2 * half:2], y[:, :, 1:2 * half:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[:, :, :half], x[:, :, half:2 * half]
        y[:, :, :half], y[:, :, half:2 * half] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def _places(state):
    """Of each new token: its sequence, its number among the sequence's new tokens, its position."""
    t = torch.arange(state["q"].shape[0], device="cuda")
    b = torch.searchsorted(state["starts"].long(), t, right=True) - 1
    i = t - state["starts"][b]
    new = state["starts"][1:] - state["starts"][:-1]
    return b, i, state["lengths"][b] - new[b] + i


def _plain_append(state):
    b, _, position = _places(state)
    page = state["keys"].shape[1]
    row, col = state["page_table"][b, position // page].long(), (position % page).long()
    with_positions = (position, state["frequencies"])
    how = (state["norm"], state["interleaved"], state["amplitude"])
    held = state["keys"].dtype
    q = _plain_rotate(state["q"], *with_positions, state["q_weight"], *how).to(held)
    state["keys"][row, col] = _plain_rotate(state["k"], *with_positions, state["k_weight"], *how).to(held)
    state["values"][row, col] = state["v"].to(held)
    return q, state["keys"], state["values"]


def _plain_attend(state):
    """Every sequence padded to the longest."""
    q, table = state["q"], state["page_table"]
    heads, d = q.shape[1:]
    kv = state["keys"].shape[2]
    seqs = table.shape[0]
    k = state["keys"][table.long()].flatten(1, 2).float()  # [b, keys, kv, d]
    v = state["values"][table.long()].flatten(1, 2).float()
    new = state["starts"][1:] - state["starts"][:-1]
    i = torch.arange(state["most"], device="cuda")
    rows = (state["starts"][:-1, None] + i).clamp(max=q.shape[0] - 1)
    p = state["lengths"][:, None] - new[:, None] + i  # [b, new]
    j = torch.arange(k.shape[1], device="cuda")
    seen = (j <= p[:, :, None]) & (j < state["lengths"][:, None, None])
    if state["window"]:
        seen &= j > p[:, :, None] - state["window"]
    x = q[rows].float().view(seqs, state["most"], kv, heads // kv, d).permute(0, 2, 3, 1, 4)  # [b, kv, group, new, d]
    s = (x.flatten(2, 3) @ k.permute(0, 2, 3, 1)).mul_(d ** -0.5)  # [b, kv, group * new, keys]
    s = s.view(seqs, kv, heads // kv, state["most"], -1).masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(4, keepdim=True).clamp(min=-1e30)).exp_()
    total = s.sum(4, keepdim=True)
    o = (s.flatten(2, 3) @ v.permute(0, 2, 1, 3)).view(x.shape) / total.clamp(min=1e-30)
    b, i, _ = _places(state)
    return o.permute(0, 3, 1, 2, 4)[b, i].reshape(q.shape).to(q.dtype)


def _plain_logprobs(state):
    x = state["logits"].float()
    top_x = x.amax(1, keepdim=True)
    e = (x - top_x).exp()
    total = e.sum(1, keepdim=True)
    of_token = (x.gather(1, state["tokens"][:, None]) - top_x - total.log())[:, 0]
    entropy = (total.log() - (e * (x - top_x)).sum(1, keepdim=True) / total)[:, 0]
    if not state["top"]:
        return of_token, entropy
    # one whole number for a value and its place, so that equal values go by the lowest index
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    order += x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device)
    tokens = x.shape[1] - 1 - (order.topk(state["top"], 1).values & 0xFFFFFFFF)
    return of_token, entropy, x.gather(1, tokens) - top_x - total.log(), tokens


def _run_plain(state):
    if state["op"] == "rotate":
        return _plain_rotate(state["x"], state["positions"], state["frequencies"], state["weight"], state["norm"],
                             state["interleaved"], state["amplitude"]).to(state["dtype"])
    if state["op"] == "append":
        return _plain_append(state)
    if state["op"] == "attend":
        return _plain_attend(state)
    return _plain_logprobs(state)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(state):
    from forgetune_b200 import append_heads, paged_attention, rotate_heads, token_logprobs
    if state["op"] == "rotate":
        return rotate_heads(state["x"], state["positions"], state["frequencies"], weight=state["weight"], eps=EPS,
                            norm=state["norm"], interleaved=state["interleaved"], amplitude=state["amplitude"])
    if state["op"] == "append":
        q = append_heads(state["q"], state["k"], state["v"], state["keys"], state["values"], state["page_table"],
                         state["starts"], state["lengths"], frequencies=state["frequencies"],
                         q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS, norm=state["norm"],
                         interleaved=state["interleaved"], amplitude=state["amplitude"])
        return q, state["keys"], state["values"]
    if state["op"] == "attend":
        return paged_attention(state["q"], state["keys"], state["values"], state["page_table"], state["starts"],
                               state["lengths"], window=state["window"])
    return token_logprobs(state["logits"], state["tokens"], top=state["top"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its value in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    size = TYPES[case["type"]].itemsize
    if case["op"] == "logprobs":
        m, n = case["m"], case["n"]
        return {"bytes": m * (n * size + 8 + 8 + 12 * case["top"]), "flops": 6 * m * n}
    d = case["dim"]
    if case["op"] == "rotate":
        n = case["t"] * case["heads"] * d
        return {"bytes": 2 * n * size + 8 * case["t"], "flops": n * (7 if case["norm"] else 3)}
    new, length = _sequences(case)
    heads, kv = case["heads"], case["kv"]
    if case["op"] == "append":
        n = sum(new) * (heads + 2 * kv) * d
        return {"bytes": n * (size + 2), "flops": n * (7 if case["norm"] else 3)}
    pairs = keys = 0
    for n, whole in zip(new, length):
        w = case["window"] or whole
        first = whole - n  # position of the first new token
        grow = max(0, min(n, w - first))  # rows that see all before them: first + 1 ... first + grow keys
        pairs += grow * first + grow * (grow + 1) // 2 + (n - grow) * w
        keys += whole - max(0, first + 1 - w)
    return {"bytes": 2 * sum(new) * heads * d * size + 2 * keys * kv * d * size, "flops": 4 * d * heads * pairs}


def _exact_rotate(x, positions, state, weight):
    x = x.double()
    if state["norm"]:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    f = state["frequencies"]
    turn = torch.polar(torch.full((x.shape[0], 1, f.shape[0]), state["amplitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), f)[:, None])
    r = f.shape[0] * 2
    part = x[..., :r]
    if state["interleaved"]:
        z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * turn
        done = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * turn
        done = torch.cat([z.real, z.imag], -1)
    return torch.cat([done, x[..., r:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s["x"], s["positions"], s, s["weight"])
    if case["op"] == "logprobs":
        of_token, entropy, values = [], [], []
        for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
            lp = torch.log_softmax(x.double(), 1)
            of_token.append(lp[torch.arange(len(t), device="cuda"), t])
            entropy.append(-(lp.exp() * lp).sum(1))
            if case["top"]:
                values.append(lp.sort(1, descending=True).values[:, :case["top"]])
        out = [torch.cat(of_token), torch.cat(entropy)]
        return tuple(out + [torch.cat(values), None]) if case["top"] else tuple(out)
    new, length = s["pairs"]
    page = case["page"]
    if case["op"] == "append":
        keys, values = s["keys"].double(), s["values"].double()
        position = torch.cat([torch.arange(n - k, n) for k, n in zip(new, length)]).cuda()
        q = _exact_rotate(s["q"], position, s, s["q_weight"])
        k = _exact_rotate(s["k"], position, s, s["k_weight"])
        at = 0
        for b, n in enumerate(new):
            slots = position[at:at + n]
            where = s["page_table"][b].long()[slots // page] * page + slots % page
            keys.view(-1, *keys.shape[2:])[where] = k[at:at + n]
            values.view(-1, *values.shape[2:])[where] = s["v"][at:at + n].double()
            at += n
        return q, keys, values
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv"]
    at = 0
    for b, (n, whole) in enumerate(zip(new, length)):
        own_pages = s["page_table"][b, :-(-whole // page)].long()
        position = torch.arange(whole - n, whole, device="cuda")
        for r0 in range(0, n, 1024):  # rows by the thousand: the scores of long prompts are large
            p = position[r0:r0 + 1024, None]
            last = int(whole - n + min(n, r0 + 1024))
            j = torch.arange(last, device="cuda")
            hidden = j > p
            if case["window"]:
                hidden = hidden | (j <= p - case["window"])
            for h in range(case["kv"]):
                k = s["keys"][own_pages, :, h].flatten(0, 1)[:last].double()
                v = s["values"][own_pages, :, h].flatten(0, 1)[:last].double()
                x = s["q"][at + r0:at + min(n, r0 + 1024), h * group:(h + 1) * group].double()
                score = torch.einsum("tgd,jd->gtj", x, k) / math.sqrt(case["dim"])
                prob = torch.softmax(score.masked_fill(hidden, -math.inf), 2)
                out[at + r0:at + min(n, r0 + 1024), h * group:(h + 1) * group] = torch.einsum("gtj,jd->tgd", prob, v)
        at += n
    return out
