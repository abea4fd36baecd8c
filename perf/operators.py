"""Cases of the 8-bit serving operators (``pi05_pytorch_fast_b200.w8a8``) for timing and comparison.

Four operators, each in a plain form (elementary torch operations in 32 bits, rounded once at the end) and
as a user calls it:

* ``norm``    residual addition + (adaptive) RMSNorm with the result in 8 bits, one scale for each token;
* ``linear``  matrix product in 8-bit integers with a scale for each token and each output channel, with the
              quantisation of its input (plain, or of gelu(gate) * up) where the input is not in 8 bits yet;
* ``append``  writing new keys and values into the 8-bit cache (a scale for each block of 16 tokens and
              key/value head), padded tokens left out;
* ``attend``  attention of new queries over that cache.

Sizes are those of this repository's models (Gemma-2B prefix language model: hidden 2048, MLP 16384, 8 query
heads and 1 key/value head of width 256, prefixes of 776 tokens; the action expert: hidden 1024, MLP 4096,
chunks of 50 tokens, 8 observations; SigLIP: hidden 1152, MLP 4304, 256 tokens a camera), and generic ones.
What an operator holds in 8 bits is returned as the values that it stands for.
"""

import math

import torch

own = False

BLOCK = 16  # tokens of the cache that share a scale
INV127 = 1.0 / 127.0


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one token of the prefix language model between two sublayers
        dict(name="norm_token", op="norm", batch=1, tokens=1, hidden=2048, dtype="float16", delta=True, gate=False, shift=False),
        # the action expert's adaptive norm with gated residual, 64 observations of 50 action tokens
        dict(name="norm_expert", op="norm", batch=64, tokens=50, hidden=1024, dtype="bfloat16", delta=True, gate=True, shift=True),
        # q, k and v of one token of the prefix language model (one product for the three)
        dict(name="linear_token", op="linear", rows=1, k=2048, n=2560, dtype="float16", source="values", bias=False),
        # the expert's down projection at 8 observations, its input gelu(gate) * up
        dict(name="linear_expert_down", op="linear", rows=400, k=4096, n=1024, dtype="bfloat16", source="geglu", bias=False),
        # SigLIP's second MLP product for two cameras: a ragged inner size and a bias
        dict(name="linear_vision", op="linear", rows=512, k=4304, n=1152, dtype="bfloat16", source="values", bias=True),
        # one of the prefix language model's MLP products at 8 observations, its input from the norm
        dict(name="linear_prefix", op="linear", rows=6208, k=2048, n=16384, dtype="float16", source="codes", bias=False),
        # one more token for each of 8 sequences of different lengths
        dict(name="append_token", op="append", batch=8, tokens=1, kv_heads=1, width=256, capacity=1024, start=676, dtype="bfloat16", real=1.0),
        # a prefix of 776 tokens at 8 observations, 148 of them padding
        dict(name="append_prefix", op="append", batch=8, tokens=776, kv_heads=1, width=256, capacity=832, start=0, dtype="float16", real=0.81),
        # a single token over one prefix
        dict(name="attend_token", op="attend", batch=1, tokens=1, heads=8, kv_heads=1, width=256, length=776, dtype="bfloat16", causal=False),
        # the action chunk over the prefix and itself, 8 observations
        dict(name="attend_expert", op="attend", batch=8, tokens=50, heads=8, kv_heads=1, width=256, length=678, dtype="bfloat16", causal=False),
        # single tokens over long caches, grouped heads
        dict(name="attend_long", op="attend", batch=4, tokens=1, heads=16, kv_heads=2, width=128, length=65536, dtype="float16", causal=True),
        # a chunk of a prompt over a long cache
        dict(name="attend_chunk", op="attend", batch=1, tokens=512, heads=8, kv_heads=1, width=256, length=16384, dtype="bfloat16", causal=True),
    ]


def _size(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    v = min(high, max(low, v))
    for top in (1536, 3072):
        if top - 16 < v <= top:
            v = top - 16
    return v


def draw(rng):
    op = rng.choice(("norm", "linear", "append", "attend"))
    dtype = rng.choice(("float16", "bfloat16"))
    if op == "norm":
        hidden = _size(rng, 64, 8192)
        batch = _size(rng, 1, 64)
        tokens = _size(rng, 1, max(1, min(776, (1 << 24) // (hidden * batch))))
        delta = rng.random() < 0.8
        return dict(op=op, batch=batch, tokens=tokens, hidden=hidden, dtype=dtype, delta=delta,
                    gate=delta and rng.random() < 0.5, shift=rng.random() < 0.5)
    if op == "linear":
        k, n = _size(rng, 64, 16384), _size(rng, 64, 16384)
        rows = _size(rng, 1, min(6208, 6208 * 2048 * 16384 // (k * n)))
        if rng.random() < 0.7:
            k = (k + 15) // 16 * 16
        return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, source=rng.choice(("values", "geglu", "codes")), bias=rng.random() < 0.5)
    width, kv_heads = rng.choice((64, 128, 256)), rng.choice((1, 1, 2, 4, 8))
    if op == "append":
        batch = _size(rng, 1, 32)
        tokens = _size(rng, 1, max(1, min(1024, (1 << 22) // (batch * kv_heads * width))))
        start = rng.choice((0, _size(rng, 1, 1024)))
        capacity = (start + tokens + 15) // 16 * 16 + 16 * rng.randrange(4)
        return dict(op=op, batch=batch, tokens=tokens, kv_heads=kv_heads, width=width, capacity=capacity, start=start, dtype=dtype,
                    real=rng.choice((1.0, round(rng.uniform(0.3, 1.0), 2))))
    heads = kv_heads * rng.choice((1, 2, 4, 8))
    batch = _size(rng, 1, 16)
    tokens = rng.choice((1, 1, _size(rng, 2, 512)))
    longest = min(131072, 134217728 // (batch * kv_heads * width * 2), 67108864 // (batch * heads * tokens))
    length = max(tokens, _size(rng, 1, max(1, longest)))
    return dict(op=op, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, width=width, length=length, dtype=dtype, causal=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _activations(g, rows, cols, dtype):
    """Normal values with a few channels that are much larger, as a residual stream has them."""
    loud = torch.exp(0.6 * torch.randn(cols, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * loud).to(dtype)


def _codes(g, *shape):
    return (torch.randn(*shape, generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)


def _rows_of_codes(g, rows, cols):
    """int8 [rows, cols] in rows that begin at multiples of 16 bytes."""
    return _codes(g, rows, (cols + 15) // 16 * 16)[:, :cols]


def _scales(g, *shape):
    return torch.exp(0.3 * torch.randn(*shape, generator=g, device="cuda")) / 32


def _cache(g, batch, capacity, kv_heads, width):
    """Keys and values int8 [batch, capacity, kv_heads, width], scales fp32 [batch, kv_heads, capacity / 16]."""
    shape = (batch, capacity, kv_heads, width)
    keys, values = _codes(g, *shape), _codes(g, *shape)
    return keys, values, _scales(g, batch, kv_heads, capacity // BLOCK), _scales(g, batch, kv_heads, capacity // BLOCK)


def prepare(case, seed):
    g = _gen(seed)
    dtype = getattr(torch, case["dtype"])
    op = case["op"]
    if op == "norm":
        b, t, h = case["batch"], case["tokens"], case["hidden"]
        state = dict(x=_activations(g, b * t, h, dtype).view(b, t, h), eps=1e-6)
        # one gain for all tokens, or one for each observation (the adaptive norm's)
        state["gain"] = 1.0 + 0.1 * torch.randn(*((b, h) if case["shift"] else (h,)), generator=g, device="cuda")
        state["delta"] = _activations(g, b * t, h, dtype).view(b, t, h) if case["delta"] else None
        state["gate"] = torch.randn(b, h, generator=g, device="cuda").to(dtype) if case["gate"] else None
        state["shift"] = 0.1 * torch.randn(b, h, generator=g, device="cuda") if case["shift"] else None
    elif op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        state = dict(weight=_rows_of_codes(g, n, k), weight_scale=_scales(g, n) * 0.02,
                     bias=torch.randn(n, generator=g, device="cuda").to(dtype) if case["bias"] else None)
        if case["source"] == "codes":
            state.update(codes=_rows_of_codes(g, m, k), scale=_scales(g, m))
        elif case["source"] == "geglu":
            both = _activations(g, m, 2 * k, dtype)  # gate and up as one product gives them
            state.update(x=both[:, :k], up=both[:, k:])
        else:
            state.update(x=_activations(g, m, k, dtype))
    elif op == "append":
        b, t, h, w = case["batch"], case["tokens"], case["kv_heads"], case["width"]
        state = dict(cache=_cache(g, b, case["capacity"], h, w))
        loud = torch.exp(0.5 * torch.randn(h, w, generator=g, device="cuda"))
        state["k"] = (torch.randn(b, t, h, w, generator=g, device="cuda") * loud).to(dtype)
        state["v"] = torch.randn(b, t, h, w, generator=g, device="cuda").to(dtype)
        state["start"] = torch.randint(case["start"] // 2, case["start"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        state["valid"] = torch.rand(b, t, generator=g, device="cuda") < case["real"] if case["real"] < 1 else None
    else:
        b, t, length = case["batch"], case["tokens"], case["length"]
        capacity = (length + BLOCK - 1) // BLOCK * BLOCK
        state = dict(cache=_cache(g, b, capacity, case["kv_heads"], case["width"]))
        state["q"] = (2 * torch.randn(b, t, case["heads"], case["width"], generator=g, device="cuda")).to(dtype)
        low = max(t, length - length // 8)
        state["lengths"] = torch.randint(low, length + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    state["case"], state["dtype"] = case, dtype
    return state


# ---------------------------------------------------------------- the plain forms
def _over_tokens(p):
    """[B, h] -> [B, 1, h]; [h] and None stay."""
    return p if p is None or p.dim() == 1 else p[:, None]


def _to_codes(y):
    """Codes and scale of each row: scale = amax / 127, codes = round(y / scale)."""
    scale = y.abs().amax(-1, keepdim=True) * INV127
    codes = torch.where(scale > 0, y / scale, 0.0).round().clamp(-127, 127)
    return codes, scale


def _plain_norm(s):
    total = s["x"].float()
    if s["delta"] is not None:
        delta = s["delta"].float()
        total = total + (delta if s["gate"] is None else delta * _over_tokens(s["gate"]).float())
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + s["eps"]) * _over_tokens(s["gain"])
    if s["shift"] is not None:
        y = y + _over_tokens(s["shift"])
    codes, scale = _to_codes(y)
    return dict(values=(codes * scale).to(s["dtype"]), scale=scale[..., 0], total=total.to(s["dtype"]))


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_linear(s):
    if "codes" in s:
        codes, scale = s["codes"].float(), s["scale"][:, None]
    else:
        x = s["x"].float()
        codes, scale = _to_codes(x if "up" not in s else _gelu(x) * s["up"].float())
    y = torch.matmul(codes, s["weight"].float().t()) * scale * s["weight_scale"]
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["dtype"])


def _spread(scale):
    """Block scales [B, H, C / 16] -> [B, C, H, 1]."""
    return scale.repeat_interleave(BLOCK, 2).transpose(1, 2)[..., None]


def _plain_append_one(codes, scale, x, slot, old, touched):
    """One of keys and values: x [B, T, H, W] into codes [B, C, H, W] and scale [B, H, C / 16], in place. slot [B, T]: where each token
    goes (C: nowhere); old [B, C / 16]: tokens that a block keeps; touched [B, C / 16]: whether it gets new ones."""
    b, c, h, w = codes.shape
    new = torch.zeros(b, c + 1, h, w, device=x.device).scatter_(1, slot[..., None, None].expand(-1, -1, h, w), x.float())[:, :c]
    amax = new.abs().view(b, c // BLOCK, BLOCK, h, w).amax((2, 4)).transpose(1, 2)
    was = torch.where((old > 0)[:, None], scale, 0.0)
    now = torch.where(touched[:, None], torch.maximum(was, amax * INV127), scale)
    ratio = torch.where(now > 0, was / now, 0.0)
    at = torch.arange(c, device=x.device)
    keeps = (at % BLOCK < old.repeat_interleave(BLOCK, 1)) & touched.repeat_interleave(BLOCK, 1)
    takes = torch.zeros(b, c + 1, dtype=torch.bool, device=x.device).scatter_(1, slot, True)[:, :c]
    step = _spread(now)
    kept = (codes.float() * _spread(ratio)).round()
    fresh = torch.where(step > 0, new / step, 0.0).round().clamp(-127, 127)
    codes.copy_(torch.where(takes[..., None, None], fresh, torch.where(keeps[..., None, None], kept, codes.float())).to(torch.int8))
    scale.copy_(now)


def _plain_append(s):
    keys, values, key_scale, value_scale = s["cache"]
    b, c = keys.shape[:2]
    start = s["start"].long()
    real = torch.ones(s["k"].shape[:2], dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"]
    slot = start[:, None] + real.long().cumsum(1) - 1
    slot = torch.where(real & (slot < c), slot, c)
    end = start + real.sum(1)
    first = torch.arange(0, c, BLOCK, device="cuda")
    old = (start[:, None] - first).clamp(0, BLOCK)
    touched = (first < end[:, None]) & (first + BLOCK > start[:, None]) & (end > start)[:, None]
    _plain_append_one(keys, key_scale, s["k"], slot, old, touched)
    _plain_append_one(values, value_scale, s["v"], slot, old, touched)
    lengths = end.clamp(max=c).to(torch.int32)
    within = (torch.arange(c, device="cuda") < lengths[:, None])[..., None, None]
    return dict(lengths=lengths, keys=torch.where(within, keys.float() * _spread(key_scale), 0.0).to(s["dtype"]),
                values=torch.where(within, values.float() * _spread(value_scale), 0.0).to(s["dtype"]))


def _plain_attend(s):
    keys, values, key_scale, value_scale = s["cache"]
    q = s["q"].float()
    b, t, heads, w = q.shape
    c, kv_heads = keys.shape[1:3]
    k = (keys.float() * _spread(key_scale)).permute(0, 2, 3, 1)
    v = (values.float() * _spread(value_scale)).transpose(1, 2)
    rows = q.view(b, t, kv_heads, heads // kv_heads, w).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, w)
    scores = (torch.matmul(rows, k) * w ** -0.5).view(b, kv_heads, -1, t, c)
    sees = s["lengths"].long()[:, None].expand(b, t)
    if s["case"]["causal"]:
        sees = sees - t + 1 + torch.arange(t, device="cuda")
    hidden = torch.arange(c, device="cuda") >= sees[:, None, None, :, None]
    scores = scores.masked_fill(hidden, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -torch.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0).view(b, kv_heads, -1, c)
    out = torch.matmul(p, v).view(b, kv_heads, heads // kv_heads, t, w).permute(0, 3, 1, 2, 4)
    return out.reshape(b, t, heads, w).to(s["dtype"])


# ---------------------------------------------------------------- one pass
def _own_norm(ops, s):
    codes, scale, total = ops.rms_norm_quant(s["x"], s["gain"], s["eps"], delta=s["delta"], gate=s["gate"], shift=s["shift"])
    return dict(values=ops.dequantize(codes, scale, s["dtype"]), scale=scale, total=total)


def _own_linear(ops, s):
    codes, scale = (s["codes"], s["scale"]) if "codes" in s else ops.quantize(s["x"], up=s.get("up"))
    return ops.linear(codes, scale, ops.Int8Weight(s["weight"], s["weight_scale"]), bias=s["bias"], dtype=s["dtype"])


def _own_append(ops, s):
    cache = ops.KVCache8(*s["cache"])
    lengths = ops.kv_append(cache, s["k"], s["v"], s["start"], valid=s["valid"])
    keys, values = ops.kv_values(cache, lengths, s["dtype"])
    return dict(lengths=lengths, keys=keys, values=values)


def _own_attend(ops, s):
    return ops.kv_attention(s["q"], ops.KVCache8(*s["cache"]), s["lengths"], causal=s["case"]["causal"])


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[op](state)
    from pi05_pytorch_fast_b200 import w8a8

    return {"norm": _own_norm, "linear": _own_linear, "append": _own_append, "attend": _own_attend}[op](w8a8, state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        rows, h = case["batch"] * case["tokens"], case["hidden"]
        params = h * 4 * (case["batch"] if case["shift"] else 1)
        params += case["batch"] * h * (2 * case["gate"] + 4 * case["shift"])
        # x and delta in, the sum and the normalised values out, a scale for each row
        return dict(bytes=rows * h * 2 * (3 + case["delta"]) + rows * 4 + params, flops=rows * h * 10)
    if op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        read = {"codes": m * k + 4 * m, "values": 2 * m * k, "geglu": 4 * m * k}[case["source"]]
        return dict(bytes=read + n * k + 4 * n + 2 * n * case["bias"] + 2 * m * n, flops=2 * m * k * n)
    if op == "append":
        rows = case["batch"] * case["kv_heads"] * case["width"]
        # new keys and values in and into the cache; the cache's values out
        return dict(bytes=2 * rows * (3 * case["tokens"] + 3 * (case["start"] + case["tokens"])), flops=2 * rows * (4 * case["tokens"] + case["start"] + case["tokens"]))
    q = case["batch"] * case["tokens"] * case["heads"] * case["width"]
    kv = case["batch"] * case["length"] * case["kv_heads"] * case["width"]
    seen = case["length"] - (case["tokens"] - 1) / 2 * case["causal"]
    return dict(bytes=4 * q + 2 * kv + kv // (2 * case["width"]), flops=4 * q * seen)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_codes(y):
    """Rows of y, rounded to 255 levels of their own largest value: (values, scale)."""
    step = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127
    return torch.nan_to_num(torch.round(y / step)) * step, step.squeeze(-1)


def _exact_norm(s):
    b, t, h = s["x"].shape
    wide = lambda p: p.double().reshape(-1, 1, h)  # noqa: E731
    z = s["x"].double()
    if s["delta"] is not None:
        z = torch.addcmul(z, s["delta"].double(), wide(s["gate"])) if s["gate"] is not None else z + s["delta"].double()
    length = torch.sqrt((z * z).sum(-1, keepdim=True) / h + s["eps"])
    y = z / length * wide(s["gain"])
    values, step = _exact_codes(y if s["shift"] is None else y + wide(s["shift"]))
    return dict(values=values, scale=step, total=z)


def _exact_linear(s):
    if "codes" in s:
        a = s["codes"].double() * s["scale"].double().unsqueeze(1)
    else:
        h = s["x"].double()
        if "up" in s:
            # gelu(x) by its tanh formula, tanh(u) = 1 - 2 / (exp(2 u) + 1)
            u = 0.7978845608028654 * (h + 0.044715 * h.pow(3))
            h = h * (1 - 1 / (torch.exp(2 * u) + 1)) * s["up"].double()
        a = _exact_codes(h)[0]
    w = s["weight"].double() * s["weight_scale"].double().unsqueeze(1)
    y = a @ w.T
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_append_one(codes, scale, x, start, real):
    """The cache's values after the append, by sequence and block; zero past the end."""
    b, c, h, w = codes.shape
    values = torch.zeros(b, c, h, w, dtype=torch.float64, device=x.device)
    for i in range(b):
        s0 = int(start[i])
        new = x[i][real[i]].double()[: c - s0]
        end = s0 + new.shape[0]
        old = (codes[i].double().view(c // BLOCK, BLOCK, h, w) * scale[i].double().T[:, None, :, None]).view(c, h, w)
        values[i, :s0] = old[:s0]
        if end == s0:
            continue
        values[i, s0:end] = new
        for j in range(s0 // BLOCK, (end - 1) // BLOCK + 1):
            lo, hi = j * BLOCK, min((j + 1) * BLOCK, end)
            part = values[i, max(lo, s0):hi]
            step = part.abs().amax((0, 2)) / 127
            if lo < s0:
                step = torch.maximum(step, scale[i, :, j].double())
            step = step[None, :, None]
            values[i, lo:hi] = torch.round(values[i, lo:hi] / step) * step
    return values


def _exact_append(s):
    keys, values, key_scale, value_scale = s["cache"]
    real = torch.ones(s["k"].shape[:2], dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"]
    ends = torch.minimum(s["start"].long() + real.sum(1), torch.tensor(keys.shape[1], device="cuda"))
    return dict(lengths=ends, keys=_exact_append_one(keys, key_scale, s["k"], s["start"], real),
                values=_exact_append_one(values, value_scale, s["v"], s["start"], real))


def _exact_attend(s):
    keys, values, key_scale, value_scale = s["cache"]
    q = s["q"].double()
    b, t, heads, w = q.shape
    group = heads // keys.shape[2]
    out = torch.zeros_like(q)
    for i in range(b):
        n = int(s["lengths"][i])
        for h in range(keys.shape[2]):
            ks = key_scale[i, h].double().repeat_interleave(BLOCK)[:n, None]
            vs = value_scale[i, h].double().repeat_interleave(BLOCK)[:n, None]
            k, v = keys[i, :n, h].double() * ks, values[i, :n, h].double() * vs
            for j in range(h * group, (h + 1) * group):
                scores = q[i, :, j] @ k.T / math.sqrt(w)
                if s["case"]["causal"]:
                    scores += torch.full_like(scores, -math.inf).triu(n - t + 1)
                out[i, :, j] = torch.softmax(scores, -1) @ v
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](prepare(case, seed))
