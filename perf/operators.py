"""Timed cases of the serving operators: rotary positions in every layout, the
key/value cache held in 4 bits, attention over that cache, and drawing the next
token from filtered logits.

Each case has a plain form in elementary torch operations (`own = False`) and
the call a program makes of the framework (`own = True`); both take what
`prepare` returns. `exact` computes the same outputs in 64 bits.

Layouts are the framework's: activations [s, b, heads, head_dim]; position_ids
[b, s]; one uniform number per drawn token.
"""

import math

import torch

own = False

GROUP = 32  # values of one head that share a scale and a zero point
HELD_MAX = 57344.0  # larger magnitudes are held as this
DTYPES = {
    "bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# cases

def listed():
    return [
        # the projection of a whole training micro-batch, forward and backward
        dict(name="rotary-train", op="rotary", s=4096, b=4, n=32, nkv=32,
             h=128, rot=128, interleaved=True, dtype="bf16", first=0,
             backward=True, scaling="linear", factor=1.0, theta=10000.0,
             native=4096),
        # a part of an uncommon head, odd lengths, full precision
        dict(name="rotary-part-odd", op="rotary", s=1533, b=3, n=16, nkv=16,
             h=80, rot=20, interleaved=True, dtype="fp32", first=77,
             backward=True, scaling="ntk", factor=4.0, theta=10000.0,
             native=2048),
        # one token for each of 16 sequences, far beyond the trained length
        dict(name="rotary-step-far", op="rotary", s=1, b=16, n=32, nkv=8,
             h=128, rot=128, interleaved=False, dtype="fp16", first=30000,
             backward=False, scaling="yarn", factor=8.0, theta=10000.0,
             native=4096),
        # one decode step: rotate q and k, write k and v into the cache
        dict(name="append-step", op="append", s=1, b=16, n=32, nkv=8, h=128,
             dtype="bf16", capacity=4096, rotate=True, interleaved=True),
        # a prompt's keys and values go into the cache at once
        dict(name="append-prompt", op="append", s=2047, b=4, n=32, nkv=8,
             h=128, dtype="bf16", capacity=4096, rotate=False,
             interleaved=True),
        # the smallest call: one stream shortly after its prompt
        dict(name="attend-short", op="attend", s=1, b=1, n=32, nkv=32, h=128,
             dtype="bf16", capacity=128, longest=61, window=0, sinks=0),
        # a served batch whose requests have any age
        dict(name="attend-ragged", op="attend", s=1, b=32, n=32, nkv=8, h=128,
             dtype="bf16", capacity=8192, longest=8192, window=0, sinks=0),
        # few long streams with eight query heads to a key head
        dict(name="attend-long", op="attend", s=1, b=4, n=64, nkv=8, h=128,
             dtype="bf16", capacity=32768, longest=32768, window=0, sinks=0),
        # several new tokens at a time, one key head, window and sinks
        dict(name="attend-window", op="attend", s=5, b=8, n=71, nkv=1, h=64,
             dtype="fp16", capacity=6016, longest=6001, window=2048, sinks=4),
        # a single stream with top-k
        dict(name="sample-one", op="sample", b=1, v=32000, pad=0,
             dtype="fp32", temperature=0.8, top_k=40, top_p=0.0, min_p=0.0,
             per_row=False),
        # a served batch in which each request has settings of its own
        dict(name="sample-mixed", op="sample", b=64, v=65024, pad=0,
             dtype="bf16", temperature=0.9, top_k=200, top_p=0.95, min_p=0.02,
             per_row=True),
        # a large batch, temperature only, a vocabulary padded in its rows
        dict(name="sample-all", op="sample", b=256, v=50257, pad=47,
             dtype="fp32", temperature=0.7, top_k=0, top_p=0.0, min_p=0.0,
             per_row=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "sample"])
    heads = [(32, 32), (32, 8), (64, 8), (16, 2), (71, 1), (12, 12), (5, 5)]
    if op == "rotary":
        n, nkv = rng.choice(heads)
        h = rng.choice([64, 80, 96, 128])
        rot = rng.choice([h, h, h // 2, 2 * rng.randint(1, h // 2)])
        s = 1 if rng.random() < 0.3 else _log(rng, 2, 4096)
        b = max(1, min(_log(rng, 1, 32), 4096 * 4 * 64 // (s * (n + nkv))))
        return dict(op=op, s=s, b=b, n=n, nkv=nkv, h=h, rot=rot,
                    interleaved=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    first=rng.choice([0, rng.randint(1, 60000)]),
                    backward=s > 1 and rng.random() < 0.7,
                    scaling=rng.choice(["linear", "ntk", "yarn"]),
                    factor=rng.choice([1.0, 2.0, 4.0, 8.0]),
                    theta=rng.choice([10000.0, 1000000.0]), native=4096)
    if op == "append":
        n, nkv = rng.choice(heads)
        h = rng.choice([32, 64, 128, 256])
        rotate = rng.random() < 0.5
        s = rng.randint(1, 4) if rotate else _log(rng, 1, 4096)
        b = max(1, min(_log(rng, 1, 64), 4 * 2047 * 8 * 128 // (s * nkv * h)))
        return dict(op=op, s=s, b=b, n=n, nkv=nkv, h=h,
                    dtype=rng.choice(["bf16", "fp16"]),
                    capacity=s + _log(rng, 1, 4000), rotate=rotate,
                    interleaved=rng.random() < 0.5)
    if op == "attend":
        n, nkv = rng.choice(heads)
        h = rng.choice([32, 64, 128, 128, 256])
        s = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 2, 64)])
        longest = s + _log(rng, 1, 32768)
        limit = 4 * 8 * 32768 * 128
        b = max(1, min(_log(rng, 1, 64), limit // (longest * nkv * h),
                       limit // (longest * n * h * s) * 8))
        while b * longest * n * s * h > 8 * limit and s > 1:
            s = max(1, s // 2)
        longest = max(s, min(longest, limit // (b * nkv * h),
                             8 * limit // (b * n * s * h)))
        window = rng.choice([0, 0, _log(rng, 1, longest)])
        return dict(op=op, s=s, b=b, n=n, nkv=nkv, h=h,
                    dtype=rng.choice(["bf16", "fp16"]),
                    capacity=longest + rng.choice([0, 1, 100]),
                    longest=longest, window=window,
                    sinks=rng.choice([0, rng.randint(1, 8)]) if window else 0)
    b = _log(rng, 1, 256)
    v = min(_log(rng, 100, 131072), 256 * 50257 // b)
    kind = rng.choice(["none", "k", "p", "min", "all"])
    return dict(op=op, b=b, v=v, pad=rng.choice([0, 0, rng.randint(1, 100)]),
                dtype=rng.choice(["fp32", "bf16", "fp16"]),
                temperature=round(rng.uniform(0.3, 1.5), 3),
                top_k=min(v, _log(rng, 1, 1000)) if kind in ("k", "all")
                else 0,
                top_p=round(rng.uniform(0.3, 0.99), 3) if kind in ("p", "all")
                else 0.0,
                min_p=round(rng.uniform(0.01, 0.3), 3)
                if kind in ("min", "all") else 0.0,
                per_row=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _inverse_frequencies(rot, theta, scaling, factor, native):
    """Inverse frequencies in 64 bits and the factor on cos and sin."""
    if scaling == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    exponent = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    inv = theta ** -exponent
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "ntk" or factor == 1.0:
        return inv, 1.0
    # yarn: frequencies that turn fewer than once over the trained length are
    # interpolated, those that turn more than 32 times are kept, and a linear
    # ramp over the pairs' numbers lies between

    def pair(turns):
        return (rot * math.log(native / (turns * 2 * math.pi))
                / (2 * math.log(theta)))

    low = max(math.floor(pair(32.0)), 0)
    high = min(math.ceil(pair(1.0)), rot - 1)
    ramp = (torch.arange(rot // 2, dtype=torch.float64) - low) / max(
        high - low, 0.001)
    ramp = ramp.clamp(0.0, 1.0)
    return inv / factor * ramp + inv * (1 - ramp), (
        0.1 * math.log(factor) + 1.0)


def _tables(end, rot, theta, scaling, factor, native):
    """cos and sin, [end, rot / 2] in 32 bits, from angles in 64 bits."""
    if own:
        from megatron_amd.models.rope import precompute_rotary_tables

        return precompute_rotary_tables(
            rot, end, theta=theta, scaling_type=scaling, scaling_factor=factor,
            original_max_position=native, device="cuda")
    inv, scale = _inverse_frequencies(rot, theta, scaling, factor, native)
    angles = torch.outer(
        torch.arange(end, dtype=torch.float64, device="cuda"), inv.cuda())
    return (angles.cos() * scale).float(), (angles.sin() * scale).float()


def _rotary_inputs(case, seed):
    g = _gen(seed)
    t = DTYPES[case["dtype"]]
    s, b, n, nkv, h = (case[x] for x in ("s", "b", "n", "nkv", "h"))
    q = _randn(g, s, b, n, h, dtype=t)
    # keys are a slice of the fused projection's output
    k = _randn(g, s, b, nkv, 3 * h, dtype=t)[..., h:2 * h]
    positions = None
    if case["first"]:
        shift = torch.randint(0, 1000, (b, 1), generator=g, device="cuda")
        positions = (case["first"] + shift
                     + torch.arange(s, device="cuda")[None, :])
    grads = None
    if case["backward"]:
        grads = (_randn(g, s, b, n, h, dtype=t),
                 _randn(g, s, b, nkv, h, dtype=t))
    return q, k, positions, grads


def _append_inputs(case, seed):
    g = _gen(seed)
    t = DTYPES[case["dtype"]]
    s, b, n, nkv, h = (case[x] for x in ("s", "b", "n", "nkv", "h"))
    bias = 2.0 * _randn(g, nkv, h)
    mixed = _randn(g, s, b, nkv, 2 * h)
    mixed[..., :h] += bias  # keys have channels far from zero
    mixed = mixed.to(t)
    q = _randn(g, s, b, n, h, dtype=t)
    start = torch.randint(0, case["capacity"] - s + 1, (b,), generator=g,
                          device="cuda")
    return q, mixed[..., :h], mixed[..., h:], start


def _attend_inputs(case, seed):
    g = _gen(seed)
    t = DTYPES[case["dtype"]]
    s, b, n, nkv, h = (case[x] for x in ("s", "b", "n", "nkv", "h"))
    q = _randn(g, s, b, n, h, dtype=t)
    # some heads look more sharply than others
    q = q * (1.0 + 0.5 * torch.rand(s, b, n, 1, generator=g, device="cuda")
             ).to(t)
    start = torch.randint(0, case["longest"] - s + 1, (b,), generator=g,
                          device="cuda")
    start[0] = case["longest"] - s
    return q, start, g


def _attend_rows(case, g, low, high):
    """Keys and values of the positions low..high of every sequence."""
    t = DTYPES[case["dtype"]]
    shape = (high - low, case["b"], case["nkv"], case["h"])
    return _randn(g, *shape, dtype=t), _randn(g, *shape, dtype=t)


def _attend_steps(case):
    step = max(1, (1 << 25) // (case["b"] * case["nkv"] * case["h"]))
    for low in range(0, case["longest"], step):
        yield low, min(case["longest"], low + step)


def _sample_inputs(case, seed):
    g = _gen(seed)
    b, v = case["b"], case["v"]
    logits = 2.0 * _randn(g, b, v + case["pad"])
    # some tokens stand out, as they do after a trained model's last layer
    for lift in (8.0, 6.0, 6.0, 5.0, 5.0, 5.0, 4.0, 4.0, 4.0, 4.0):
        at = torch.randint(0, v, (b, 1), generator=g, device="cuda")
        logits.scatter_add_(
            1, at, lift * torch.rand(b, 1, generator=g, device="cuda"))
    logits = logits.to(DTYPES[case["dtype"]])[:, :v]
    uniform = torch.rand(b, generator=g, device="cuda")
    setting = [case["temperature"], case["top_k"], case["top_p"],
               case["min_p"]]
    if case["per_row"]:
        part = torch.rand(3, b, generator=g, device="cuda")
        setting[0] = setting[0] * (0.5 + part[0])
        setting[1] = ((setting[1] * part[1]).long() + 1
                      if setting[1] else torch.zeros(
                          b, dtype=torch.long, device="cuda"))
        setting[2] = torch.full((b,), setting[2], device="cuda")
        setting[3] = setting[3] * part[2]
    return logits, uniform, setting


def prepare(case, seed):
    op = case["op"]
    state = dict(case=case)
    if op == "rotary":
        q, k, positions, grads = _rotary_inputs(case, seed)
        end = case["s"] if positions is None else (
            case["first"] + 1000 + case["s"])
        cos, sin = _tables(end, case["rot"], case["theta"], case["scaling"],
                           case["factor"], case["native"])
        if own and grads is not None:
            q, k = q.requires_grad_(), k.detach().requires_grad_()
        state.update(q=q, k=k, positions=positions, grads=grads, cos=cos,
                     sin=sin)
    elif op == "append":
        q, k, v, start = _append_inputs(case, seed)
        state.update(q=q, k=k, v=v, start=start, cache=_new_cache(case))
        if case["rotate"]:
            state["cos"], state["sin"] = _tables(
                case["capacity"], case["h"], 10000.0, "linear", 1.0, 4096)
    elif op == "attend":
        q, start, g = _attend_inputs(case, seed)
        cache = _new_cache(case)
        for low, high in _attend_steps(case):
            k, v = _attend_rows(case, g, low, high)
            if own:
                cache.append(k, v, low)
            else:
                at = torch.full((case["b"],), low, device="cuda")
                _plain_store(cache, k, v, at)
        state.update(q=q, start=start, cache=cache)
    else:
        logits, uniform, setting = _sample_inputs(case, seed)
        state.update(logits=logits, uniform=uniform, setting=setting)
    return state


def _new_cache(case):
    b, nkv, h = case["b"], case["nkv"], case["h"]
    if own:
        from megatron_amd.ops import QuantKVCache

        return QuantKVCache(case["capacity"], b, nkv, h,
                            dtype=DTYPES[case["dtype"]], device="cuda")
    rows = (b, case["capacity"], nkv)
    return {
        x: (torch.zeros(*rows, h // 2, dtype=torch.uint8, device="cuda"),
            torch.zeros(*rows, h // GROUP, dtype=torch.half, device="cuda"),
            torch.zeros(*rows, h // GROUP, dtype=torch.half, device="cuda"))
        for x in "kv"
    }


# ---------------------------------------------------------------------------
# plain forms

def _rotate(x, cos, sin, interleaved, dtype=torch.float32):
    """x [s, b, n, h] by cos, sin [s, b or 1, rot / 2]."""
    half = cos.shape[-1]
    c, s = cos.unsqueeze(2).to(dtype), sin.unsqueeze(2).to(dtype)
    turned, rest = x[..., :2 * half].to(dtype), x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        out = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([out.to(x.dtype), rest], -1)


def _rows_of(table, positions, s):
    if positions is None:
        return table[:s].unsqueeze(1)
    return table[positions].transpose(0, 1)


def _run_rotary(state):
    case = state["case"]
    q, k, grads = state["q"], state["k"], state["grads"]
    inter = case["interleaved"]
    if own:
        from megatron_amd.ops import rotary_embedding

        yq, yk = rotary_embedding(q, k, state["cos"], state["sin"],
                                  positions=state["positions"],
                                  interleaved=inter)
        if grads is None:
            return yq, yk
        dq, dk = torch.autograd.grad((yq, yk), (q, k), grads)
        return yq.detach(), yk.detach(), dq, dk
    cos = _rows_of(state["cos"], state["positions"], case["s"])
    sin = _rows_of(state["sin"], state["positions"], case["s"])
    out = tuple(_rotate(x, cos, sin, inter) for x in (q, k))
    if grads is not None:  # the transpose of a rotation turns back
        out += tuple(_rotate(x, cos, -sin, inter) for x in grads)
    return out


def _quantize(x):
    """Codes 0..15, scale and zero point of groups of 32 values.

    A group's zero point is its least value and its scale a fifteenth of its
    range, both held in 16 bits; a code is the nearest whole number of scales
    above the zero point, a tie going to the even one. In 64 bits, since the
    codes are decided at borders."""
    x = x.double().clamp(-HELD_MAX, HELD_MAX)
    x = x.unflatten(-1, (-1, GROUP))
    zero = x.amin(-1).half()
    scale = ((x.amax(-1) - zero.double()) / 15.0).half()
    steps = (x - zero.double().unsqueeze(-1)) / scale.double().unsqueeze(-1)
    code = torch.where(scale.unsqueeze(-1) > 0, steps.round(),
                       torch.zeros_like(steps)).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), scale, zero


def _plain_store(cache, k, v, start):
    s, b = k.shape[:2]
    rows = torch.arange(b, device="cuda")[:, None]
    at = start[:, None] + torch.arange(s, device="cuda")[None, :]
    for name, x in (("k", k), ("v", v)):
        code, scale, zero = _quantize(x.transpose(0, 1))
        codes, scales, zeros = cache[name]
        codes[rows, at] = code[..., 0::2] | (code[..., 1::2] << 4)
        scales[rows, at] = scale
        zeros[rows, at] = zero


def _plain_values(held):
    """What packed codes stand for, in 32 bits."""
    codes, scales, zeros = held
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    code = code.unflatten(-1, (-1, GROUP))
    return (code * scales.float().unsqueeze(-1)
            + zeros.float().unsqueeze(-1)).flatten(-2)


def _run_append(state):
    case = state["case"]
    q, k, v, start = (state[x] for x in ("q", "k", "v", "start"))
    cache, s = state["cache"], case["s"]
    out = ()
    if own:
        if case["rotate"]:
            out = (cache.append(k, v, start, query=q, cos=state["cos"],
                                sin=state["sin"],
                                interleaved=case["interleaved"]),)
        else:
            cache.append(k, v, start)
        return out + tuple(cache.dequantize(start, s))
    at = start[:, None] + torch.arange(s, device="cuda")[None, :]
    if case["rotate"]:
        # in 64 bits: the codes hang on the rounded keys
        cos = _rows_of(state["cos"], at, s)
        sin = _rows_of(state["sin"], at, s)
        q, k = (_rotate(x, cos, sin, case["interleaved"], torch.float64)
                for x in (q, k))
        out = (q,)
    _plain_store(cache, k, v, start)
    rows = torch.arange(case["b"], device="cuda")[:, None]
    for name in "kv":
        held = tuple(x[rows, at] for x in cache[name])
        out += (_plain_values(held).transpose(0, 1).to(k.dtype),)
    return out


def _run_attend(state):
    case = state["case"]
    q, start, cache = state["q"], state["start"], state["cache"]
    if own:
        return cache.attention(q, start, window_size=case["window"] or None,
                               sink_size=case["sinks"])
    s, b, n, h = q.shape
    nkv, longest = case["nkv"], case["longest"]
    rep = n // nkv
    # [b, nkv, rep * s, h] against [b, nkv, longest, h]
    rows = q.float().reshape(s, b, nkv, rep, h).permute(1, 2, 3, 0, 4)
    rows = rows.reshape(b, nkv, rep * s, h)
    keys = _plain_values(tuple(x[:, :longest] for x in cache["k"]))
    score = torch.matmul(rows, keys.permute(0, 2, 3, 1)) / math.sqrt(h)
    del keys
    at = start[:, None] + torch.arange(s, device="cuda")[None, :]
    key = torch.arange(longest, device="cuda")
    seen = key <= at[..., None]
    if case["window"]:
        seen &= (key > at[..., None] - case["window"]) | (
            key < case["sinks"])
    score = score.unflatten(2, (rep, s)).masked_fill(
        ~seen[:, None, None], float("-inf"))
    score = (score - score.amax(-1, keepdim=True)).exp()
    total = score.sum(-1, keepdim=True)
    values = _plain_values(tuple(x[:, :longest] for x in cache["v"]))
    out = torch.matmul(score.flatten(2, 3),
                       values.permute(0, 2, 1, 3)).unflatten(2, (rep, s))
    out = out / total
    return out.permute(3, 0, 1, 2, 4).reshape(s, b, n * h).to(q.dtype)


def _filtered_weights(x, temperature, top_k, top_p, min_p):
    """Weights exp((x - max) / temperature) of the tokens that every filter
    keeps, 0 for the others; x in 64 bits, settings [b, 1]. Tokens are ordered
    by their logit, equal ones by their index."""
    weight = ((x - x.amax(-1, keepdim=True)) / temperature).exp()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ranked = weight.gather(-1, order)
    rank = torch.arange(x.shape[-1], device=x.device)[None, :]
    keep = (rank < top_k) | (top_k <= 0)
    ranked = ranked * keep
    before = ranked.cumsum(-1) - ranked
    within = before <= top_p * ranked.sum(-1, keepdim=True)
    keep &= within | (top_p <= 0.0) | (top_p >= 1.0)
    keep &= ranked >= min_p
    kept = torch.zeros_like(keep).scatter(-1, order, keep)
    return weight * kept


def _run_sample(state):
    case = state["case"]
    logits, uniform = state["logits"], state["uniform"]
    temperature, top_k, top_p, min_p = state["setting"]
    if own:
        from megatron_amd.ops import sample_tokens

        return sample_tokens(logits, uniform, temperature=temperature,
                             top_k=top_k, top_p=top_p, min_p=min_p)
    if not case["per_row"]:
        like = torch.ones(case["b"], device="cuda", dtype=torch.float64)
        temperature, top_k, top_p, min_p = (
            x * like for x in (temperature, top_k, top_p, min_p))
    weight = _filtered_weights(
        logits.double(), temperature.double()[:, None], top_k[:, None],
        top_p.double()[:, None], min_p.double()[:, None])
    upto = weight.cumsum(-1)
    target = uniform.double()[:, None] * upto[:, -1:]
    return (upto <= target).sum(-1)


def run(state):
    return {"rotary": _run_rotary, "append": _run_append,
            "attend": _run_attend, "sample": _run_sample}[
                state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op = case["op"]
    size = BYTES[case["dtype"]]
    if op == "rotary":
        values = case["s"] * case["b"] * (case["n"] + case["nkv"])
        turns = 2 if case["backward"] else 1
        rows = case["s"] * (1 if not case["first"] else case["b"])
        return {"bytes": turns * values * case["h"] * size * 2
                + rows * case["rot"] * 4,
                "flops": turns * values * case["rot"] * 3}
    if op == "append":
        tokens = case["s"] * case["b"]
        values = tokens * 2 * case["nkv"] * case["h"]
        moved = values * size * 2 + values // 2 + values // GROUP * 4
        flops = values * 6
        if case["rotate"]:
            moved += tokens * (case["n"] * case["h"] * size * 2
                               + case["h"] * 4)
            flops += tokens * (case["n"] + case["nkv"]) * case["h"] * 3
        return {"bytes": moved, "flops": flops}
    if op == "attend":
        s, b, n, nkv, h = (case[x] for x in ("s", "b", "n", "nkv", "h"))
        # sequences end anywhere up to the longest: half of it on average
        ends = [case["longest"]] + [(case["longest"] + s) // 2] * (b - 1)
        if case["window"]:
            ends = [min(e, case["window"] + s - 1 + case["sinks"])
                    for e in ends]
        row = 2 * nkv * (h // 2 + h // GROUP * 4)
        return {"bytes": sum(ends) * row + 2 * s * b * n * h * size,
                "flops": 4 * sum(ends) * s * n * h}
    cells = case["b"] * case["v"]
    return {"bytes": cells * size + 12 * case["b"], "flops": 4 * cells}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions

def _exact_turn(x, positions, case, back=False):
    """Pairs as complex numbers, multiplied by a unit number each."""
    rot = case.get("rot", case["h"])
    inv, scale = _inverse_frequencies(
        rot, case.get("theta", 10000.0), case.get("scaling", "linear"),
        case.get("factor", 1.0), case.get("native", 4096))
    angle = positions.double()[..., None] * inv.cuda()  # [s, b, rot / 2]
    unit = torch.polar(torch.full_like(angle, scale),
                       -angle if back else angle)[:, :, None]
    out = x.double().clone()
    if case["interleaved"]:
        first, second = slice(0, rot, 2), slice(1, rot, 2)
    else:
        first, second = slice(0, rot // 2), slice(rot // 2, rot)
    turned = torch.complex(out[..., first], out[..., second]) * unit
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _exact_held(x):
    """Values that a row of x is held as, [..., h] in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for low in range(0, x.shape[-1], GROUP):
        part = x[..., low:low + GROUP].double()
        part = part.clamp(min=-HELD_MAX, max=HELD_MAX)
        zero = part.min(-1, keepdim=True)[0].half().double()
        scale = ((part.max(-1, keepdim=True)[0] - zero) / 15).half().double()
        code = torch.round((part - zero) / scale.clamp(min=1e-300))
        out[..., low:low + GROUP] = zero + scale * code.clamp(0, 15)
    return out


def exact(case, seed):
    op = case["op"]
    s, b = case.get("s"), case["b"]
    if op == "rotary":
        q, k, positions, grads = _rotary_inputs(case, seed)
        if positions is None:
            positions = torch.arange(s, device="cuda")[None].expand(b, s)
        at = positions.t()
        out = [_exact_turn(x, at, case) for x in (q, k)]
        if grads is not None:
            out += [_exact_turn(x, at, case, back=True) for x in grads]
        return tuple(out)
    if op == "append":
        q, k, v, start = _append_inputs(case, seed)
        out = ()
        if case["rotate"]:
            # rotated keys are rounded to the model's type before their codes
            # are chosen, so there is no value of theirs in 64 bits
            out = (_exact_turn(q, start[None] + torch.arange(
                s, device="cuda")[:, None], case),)
            return out + (None, _exact_held(v))
        return out + (_exact_held(k), _exact_held(v))
    if op == "attend":
        q, start, g = _attend_inputs(case, seed)
        n, nkv, h = case["n"], case["nkv"], case["h"]
        rep = n // nkv
        parts = [_attend_rows(case, g, low, high)
                 for low, high in _attend_steps(case)]
        keys, values = (torch.cat(x) for x in zip(*parts))
        del parts
        out = torch.zeros(s, b, n, h, dtype=torch.float64, device="cuda")
        for i, first in enumerate(start.tolist()):
            for head in range(nkv):
                mine = slice(head * rep, (head + 1) * rep)
                end = first + s
                key = _exact_held(keys[:end, i, head])
                value = _exact_held(values[:end, i, head])
                for j in range(s):
                    stop = first + j + 1
                    low = max(0, stop - case["window"]) if case["window"] \
                        else 0
                    at = torch.arange(low, stop, device="cuda")
                    if case["sinks"]:
                        early = torch.arange(min(low, case["sinks"]),
                                             device="cuda")
                        at = torch.cat([early, at])
                    score = q[j, i, mine].double() @ key[at].t() / h ** 0.5
                    out[j, i, mine] = torch.softmax(score, -1) @ value[at]
        return out.reshape(s, b, n * h)
    logits, uniform, setting = _sample_inputs(case, seed)
    logits, uniform = logits.double().cpu(), uniform.double().cpu().tolist()
    setting = [x.tolist() if torch.is_tensor(x) else [x] * b for x in setting]
    out = []
    for row, u, t, k, p, least in zip(logits, uniform, *setting):
        # walk down from the likeliest token; indices stay in order
        value, index = torch.sort(row, descending=True, stable=True)
        if k > 0:
            value, index = value[:k], index[:k]
        chance = torch.exp((value - value[0]) / t)
        count = len(chance)
        if 0.0 < p < 1.0:
            before = torch.cat([chance.new_zeros(1), chance.cumsum(0)[:-1]])
            count = int((before <= p * chance.sum()).sum())
        count = min(count, int((chance >= least).sum()))
        index, order = torch.sort(index[:count])
        mass = chance[:count][order].cumsum(0)
        at = int((mass <= u * mass[-1]).sum())
        out.append(int(index[min(at, count - 1)]))
    return torch.tensor(out)
