"""The block-scaled 8-bit operators as they are measured: quantisation, RMS norm and the matrix product.

All three meet in one chain: a layer's activations are normalised (with the
residual's addition) and quantised, multiplied by quantised weights, passed
through bias and ReLU, quantised again and multiplied by the next layer's
weights.  8-bit values are e4m3 with one power-of-two scale for each block of
128 along a row (activations) or of 128 x 128 (weights).

Cases with ``own`` false run the operators' plain forms in elementary torch
operations; with ``own`` true they make the framework's calls on the same
tensors.
"""

import torch

own = False

BLOCK = 128
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token's activations before a quantised layer: latency alone counts
        {"name": "quantize_row", "op": "quantize", "m": 1, "k": 4096, "type": "f32"},
        # a ragged batch of the small MLP's input width, blocks that end inside the row
        {"name": "quantize_ragged", "op": "quantize", "m": 777, "k": 784, "type": "f16"},
        # a long prompt's worth of activations as wide as the wide MLP's hidden layer
        {"name": "quantize_wide", "op": "quantize", "m": 16384, "k": 8192, "type": "bf16"},
        # one token between two layers: residual, norm and quantised output in one call
        {"name": "norm_row", "op": "norm", "m": 1, "k": 4096, "type": "bf16", "residual": True, "quantize": True},
        # an odd width without a residual, the output in the input's type
        {"name": "norm_odd", "op": "norm", "m": 333, "k": 1111, "type": "f32", "residual": False, "quantize": False},
        # a large batch in the framework's own type: residual and plain output
        {"name": "norm_large_f32", "op": "norm", "m": 8192, "k": 4096, "type": "f32", "residual": True,
         "quantize": False},
        # the same between two quantised layers of the wide MLP
        {"name": "norm_wide_fp8", "op": "norm", "m": 16384, "k": 8192, "type": "bf16", "residual": True,
         "quantize": True},
        # one token through a square layer: the weights' bytes bound it
        {"name": "linear_row", "op": "linear", "m": 1, "k": 4096, "n": 4096, "type": "f32", "bias": True,
         "relu": True, "residual": False, "quantize": False},
        # sixteen sequences decoding through the wide MLP's last layer, residual added
        {"name": "linear_few", "op": "linear", "m": 16, "k": 8192, "n": 4096, "type": "bf16", "bias": True,
         "relu": False, "residual": True, "quantize": False},
        # the small MLP's first layer on a ragged batch; a width that ends inside a block
        {"name": "linear_ragged", "op": "linear", "m": 333, "k": 784, "n": 250, "type": "f32", "bias": True,
         "relu": True, "residual": False, "quantize": False},
        # a medium batch through the wide MLP's first layer, output ready for the next quantised one
        {"name": "linear_fp8_out", "op": "linear", "m": 1024, "k": 4096, "n": 8192, "type": "bf16", "bias": True,
         "relu": True, "residual": False, "quantize": True},
        # a large batch through the wide MLP's square layer: the tensor cores bound it
        {"name": "linear_large", "op": "linear", "m": 8192, "k": 8192, "n": 8192, "type": "bf16", "bias": True,
         "relu": True, "residual": False, "quantize": False},
    ]


def _spread(rng, low, high):
    """A size spread over its logarithm, odd ones among them."""
    v = int(round(low * (high / low) ** rng.random()))
    if v > 64 and rng.random() < 0.5:  # half of the longer ones as real layers have them
        v = max(64, v // 64 * 64)
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear", "linear"])
    case = {"op": op, "type": rng.choice(sorted(TYPES))}
    if op == "linear":
        while True:
            m, k, n = _spread(rng, 1, 8192), _spread(rng, 64, 8192), _spread(rng, 64, 8192)
            if m * k * n >= 1 << 18:
                break
        quantize = rng.random() < 0.3
        case.update(m=m, k=k, n=n, bias=rng.random() < 0.7, relu=rng.random() < 0.5,
                    residual=rng.random() < 0.4, quantize=quantize)
    else:
        case.update(m=_spread(rng, 1, 16384), k=_spread(rng, 64, 8192))
        if op == "norm":
            case.update(residual=rng.random() < 0.6, quantize=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, m, k, dtype):
    """Activations as a network has them: unit normal, a few channels ten times as large, rows of unlike size."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x = x * (1 + 9 * (torch.rand(k, generator=g, device="cuda") < 0.01).float())
    return (x * torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))).to(dtype)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _aligned(t, unit):
    """The same values in rows that start on multiples of `unit` elements."""
    wide = torch.zeros(t.shape[0], (t.shape[1] + unit - 1) // unit * unit, dtype=torch.uint8, device=t.device)
    wide[:, :t.shape[1]] = t.view(torch.uint8)
    return wide.view(t.dtype)[:, :t.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, k, dtype = case["m"], case["k"], TYPES[case["type"]]
    state = {"op": case["op"], "dtype": dtype}
    if case["op"] == "quantize":
        state["x"] = _activations(g, m, k, dtype)
    elif case["op"] == "norm":
        state["x"] = _activations(g, m, k, dtype)
        state["weight"] = 1 + 0.1 * torch.randn(k, generator=g, device="cuda")
        state["residual"] = _activations(g, m, k, dtype) if case["residual"] else None
        state["quantize"] = case["quantize"]
    else:
        n = case["n"]
        q, s = _plain_quantize(_activations(g, m, k, torch.float32))
        state["x"], state["x_scales"] = _aligned(q, 16), _aligned(s, 4)
        w = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
        q, s = _plain_quantize_weight(w)
        state["w"], state["w_scales"] = _aligned(q, 16), _aligned(s, 4)
        state["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        state["residual"] = torch.randn(m, n, generator=g, device="cuda").to(dtype) if case["residual"] else None
        state["relu"], state["quantize"] = case["relu"], case["quantize"]
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _power(amax):
    """The exponent of the smallest power of two s with amax / s <= 448, from fp32 bits; 0 for a block of zeros."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).int()
    return torch.where(amax == 0, torch.zeros_like(e), e.clamp(-127, 127))


def _plain_quantize(x):
    """fp32 [m, k] -> e4m3 [m, k] and a power-of-two scale for each 128 along a row."""
    m, k = x.shape
    kb = _blocks(k)
    b = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    e = _power(b.abs().amax(2))
    q = (b * torch.ldexp(torch.ones_like(e, dtype=torch.float32), -e)[:, :, None]).to(torch.float8_e4m3fn)
    s = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e).to(torch.float8_e8m0fnu)
    return q.view(m, kb * BLOCK)[:, :k], s


def _plain_quantize_weight(w):
    """fp32 [n, k] -> e4m3 [n, k] and a power-of-two scale for each 128 x 128."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    b = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    e = _power(b.abs().amax(3).amax(1))
    q = (b * torch.ldexp(torch.ones_like(e, dtype=torch.float32), -e)[:, None, :, None]).to(torch.float8_e4m3fn)
    s = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e).to(torch.float8_e8m0fnu)
    return q.view(nb * BLOCK, kb * BLOCK)[:n, :k], s


def _values(q, s, dtype):
    """What quantised rows stand for; the scales are of 1 x 128 or, where they have fewer rows, of 128 x 128."""
    f = s.to(dtype).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    if s.shape[0] != q.shape[0]:
        f = f.repeat_interleave(BLOCK, 0)[:q.shape[0]]
    return q.to(dtype) * f


def _run_plain(state):
    if state["op"] == "quantize":
        return _plain_quantize(state["x"].float())
    if state["op"] == "norm":
        h = state["x"].float()
        if state["residual"] is not None:
            h = h + state["residual"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * state["weight"]
        y = _plain_quantize(y) if state["quantize"] else y.to(state["dtype"])
        return (y, h.to(state["dtype"])) if state["residual"] is not None else y
    y = _values(state["x"], state["x_scales"], torch.float32) @ _values(state["w"], state["w_scales"], torch.float32).T
    if state["bias"] is not None:
        y = y + state["bias"]
    if state["relu"]:
        y = torch.where(y < 0, torch.zeros_like(y), y)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return _plain_quantize(y) if state["quantize"] else y.to(state["dtype"])


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(state):
    from forgetune_b200 import Fp8Rows, Fp8Weight, fp8_linear, quantize_rows, rms_norm
    if state["op"] == "quantize":
        r = quantize_rows(state["x"])
        return r.data, r.scales
    if state["op"] == "norm":
        r = rms_norm(state["x"], state["weight"], eps=EPS, residual=state["residual"], quantize=state["quantize"])
        y, h = r if state["residual"] is not None else (r, None)
        y = (y.data, y.scales) if state["quantize"] else y
        return (y, h) if h is not None else y
    y = fp8_linear(Fp8Rows(state["x"], state["x_scales"]), Fp8Weight(state["w"], state["w_scales"]),
                   bias=state["bias"], relu=state["relu"], residual=state["residual"],
                   out_dtype=None if state["quantize"] else state["dtype"], quantize=state["quantize"])
    return (y.data, y.scales) if state["quantize"] else y


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its value in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    m, k = case["m"], case["k"]
    size = TYPES[case["type"]].itemsize
    if case["op"] == "quantize":
        return {"bytes": m * k * (size + 1) + m * _blocks(k), "flops": 2 * m * k}
    if case["op"] == "norm":
        out = m * k + m * _blocks(k) if case["quantize"] else m * k * size
        return {"bytes": m * k * size * (3 if case["residual"] else 1) + 4 * k + out,
                "flops": m * k * (5 if case["residual"] else 4)}
    n = case["n"]
    out = m * n + m * _blocks(n) if case["quantize"] else m * n * size
    ops = m * k + m * _blocks(k) + n * k + _blocks(n) * _blocks(k)
    return {"bytes": ops + out + (4 * n if case["bias"] else 0) + (m * n * size if case["residual"] else 0),
            "flops": 2 * m * n * k}


def _exact_quantize(y):
    """float64 [m, k] -> the values over their block's scale, unrounded, and the scales."""
    m, k = y.shape
    kb = _blocks(k)
    parts = [y[:, i * BLOCK:(i + 1) * BLOCK] for i in range(kb)]
    amax = torch.stack([p.abs().max(1).values for p in parts], 1)
    mantissa, power = torch.frexp(amax)  # amax = mantissa 2^power, 0.5 <= mantissa < 1; 448 = 0.875 2^9
    power = torch.where(mantissa > 0.875, power - 8, power - 9)
    s = torch.where(amax > 0, 2.0 ** power.clamp(-127, 127).double(), torch.ones_like(amax))
    return torch.cat([p / s[:, i:i + 1] for i, p in enumerate(parts)], 1), s


def exact(case, seed):
    own_inputs = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(own_inputs["x"].double())
    if op == "norm":
        h = own_inputs["x"].double()
        if case["residual"]:
            h = h + own_inputs["residual"].double()
        y = h / torch.sqrt(torch.einsum("mk,mk->m", h, h) / case["k"] + EPS)[:, None]
        y = torch.einsum("mk,k->mk", y, own_inputs["weight"].double())
        y = _exact_quantize(y) if case["quantize"] else y
        return (y, h) if case["residual"] else y
    a, w = own_inputs["x"].double(), own_inputs["w"].double()
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for b in range(_blocks(case["k"])):  # block by block of k: the scales leave the sum
        cols = slice(b * BLOCK, (b + 1) * BLOCK)
        ws = own_inputs["w_scales"][:, b].double()[torch.arange(case["n"], device="cuda") // BLOCK]
        y += (a[:, cols] @ w[:, cols].T) * own_inputs["x_scales"][:, b].double()[:, None] * ws
    if case["bias"]:
        y = y + own_inputs["bias"].double()
    if case["relu"]:
        y = y.clamp(min=0)
    if case["residual"]:
        y = y + own_inputs["residual"].double()
    return _exact_quantize(y) if case["quantize"] else y
