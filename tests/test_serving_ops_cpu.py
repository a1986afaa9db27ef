"""Serving operators on the CPU: what they refuse, their plain paths, and the
rotary tables."""

import math

import pytest
import torch

from megatron_amd.models.rope import (
    precompute_freqs,
    precompute_rotary_tables,
)
from megatron_amd.ops import (
    QuantKVCache,
    rotary_embedding,
    sample_tokens,
)

BF16 = torch.bfloat16


# ---------------------------------------------------------------------------
# tables

def test_tables_near_positions_as_before():
    """Unscaled tables agree with the 32-bit ones where those are good: an
    angle of up to 100 is off by 100 * 2^-24 from each of three roundings."""
    for theta in (10000.0, 500000.0):
        old = precompute_freqs(128, 100, theta=theta)
        new = precompute_rotary_tables(128, 100, theta=theta)
        for a, b in zip(old, new):
            assert b.dtype == torch.float32
            assert (a - b).abs().max() < 3 * 100 * 2.0 ** -24


def test_tables_far_positions():
    dim, theta, at = 64, 10000.0, 200001
    cos, sin = precompute_rotary_tables(dim, at + 1, theta=theta)
    for j in (0, 1, 7, 31):
        angle = at * theta ** (-2 * j / dim)
        # an angle in 64 bits is off by a few 2^-53 of itself
        assert abs(float(cos[at, j]) - math.cos(angle)) < 2.0 ** -23
        assert abs(float(sin[at, j]) - math.sin(angle)) < 2.0 ** -23


def test_tables_linear_and_ntk():
    cos, _ = precompute_rotary_tables(32, 80, scaling_factor=4.0)
    plain, _ = precompute_rotary_tables(32, 20)
    assert (cos[::4] - plain).abs().max() < 2.0 ** -23
    # ntk: the slowest pair as under linear scaling, the fastest one kept
    ntk = precompute_rotary_tables(32, 80, scaling_type="ntk",
                                   scaling_factor=4.0)
    assert (ntk[0][:20, 0] - plain[:, 0]).abs().max() < 2.0 ** -23
    assert (ntk[0][:, -1] - cos[:, -1]).abs().max() < 2.0 ** -23


def test_tables_yarn():
    dim, native, factor, theta = 128, 4096, 8.0, 10000.0
    got = precompute_rotary_tables(dim, 50, theta=theta, scaling_type="yarn",
                                   scaling_factor=factor,
                                   original_max_position=native)
    magnitude = 0.1 * math.log(factor) + 1
    for j in range(dim // 2):
        inv = theta ** (-2 * j / dim)

        def border(turns):
            return dim * math.log(native / (turns * 2 * math.pi)) / (
                2 * math.log(theta))

        low, high = math.floor(border(32)), math.ceil(border(1))
        part = min(1.0, max(0.0, (j - low) / (high - low)))
        inv = inv * (1 - part) + inv / factor * part
        for t in (1, 49):
            assert abs(float(got[0][t, j])
                       - magnitude * math.cos(t * inv)) < 2.0 ** -22
            assert abs(float(got[1][t, j])
                       - magnitude * math.sin(t * inv)) < 2.0 ** -22
    same = precompute_rotary_tables(dim, 50, scaling_type="yarn")
    assert torch.equal(same[0], precompute_rotary_tables(dim, 50)[0])


@pytest.mark.parametrize("bad", [
    dict(dim=0), dict(dim=7), dict(scaling_type="other"),
    dict(scaling_factor=0.0), dict(scaling_type="ntk", scaling_factor=0.5),
    dict(theta=1.0), dict(end=0),
])
def test_tables_refuse(bad):
    with pytest.raises(ValueError):
        precompute_rotary_tables(**{**dict(dim=64, end=10), **bad})


# ---------------------------------------------------------------------------
# rotary positions

def test_rotary_interleaved_as_apply_rope():
    from megatron_amd.ops import apply_rope

    torch.manual_seed(0)
    q, k = torch.randn(6, 2, 4, 32), torch.randn(6, 2, 1, 32)
    cos, sin = precompute_freqs(32, 10)
    yq, yk = rotary_embedding(q, k, cos, sin)
    assert torch.equal(yq, apply_rope(q, cos[:6], sin[:6]))
    assert torch.equal(yk, apply_rope(k, cos[:6], sin[:6]))


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_gradient_and_second_order(interleaved):
    torch.manual_seed(1)
    q = torch.randn(3, 2, 2, 12, requires_grad=True)
    k = torch.randn(3, 2, 1, 12, requires_grad=True)
    cos, sin = precompute_rotary_tables(8, 9)
    positions = torch.randint(0, 9, (2, 3))
    yq, yk = rotary_embedding(q, k, cos, sin, positions, interleaved)
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    gq.requires_grad_()
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk),
                                 create_graph=True)
    # turning forth and back changes nothing: three roundings each way
    back, _ = rotary_embedding(dq, None, cos, sin, positions, interleaved)
    assert (back - gq).abs().max() < 2.0 ** -20
    # the gradient is linear in gq, and its own transpose turns forth
    u = torch.randn_like(dq)
    second, = torch.autograd.grad(dq, gq, u)
    forth, _ = rotary_embedding(u, None, cos, sin, positions, interleaved)
    assert (second - forth).abs().max() < 2.0 ** -20


def test_rotary_refuses():
    cos, sin = precompute_rotary_tables(32, 8)
    q = torch.randn(4, 2, 3, 32)
    bad = [
        dict(query=q[0]), dict(query=q.double()), dict(key=q.bfloat16()),
        dict(key=q[:3]), dict(key=q[..., :16]), dict(cos=cos[:, :4]),
        dict(cos=cos.double(), sin=sin.double()), dict(cos=cos[:3],
                                                       sin=sin[:3]),
        dict(cos=torch.ones(8, 17), sin=torch.ones(8, 17)),
        dict(positions=torch.zeros(4, 2, dtype=torch.int64)),
        dict(positions=torch.zeros(2, 4, dtype=torch.int32)),
        dict(positions=torch.full((2, 4), 8)),
        dict(positions=torch.full((2, 4), -1)),
        dict(cos=cos.clone().requires_grad_()),
    ]
    good = dict(query=q, key=q, cos=cos, sin=sin, positions=None)
    rotary_embedding(**good)
    for change in bad:
        with pytest.raises(ValueError):
            rotary_embedding(**{**good, **change})


# ---------------------------------------------------------------------------
# 4-bit cache

@pytest.mark.parametrize("h", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_cache_holds_nearest_codes(h, dtype):
    torch.manual_seed(h)
    cache = QuantKVCache(70, 3, 2, h, dtype=dtype)
    k, v = (torch.randn(9, 3, 2, h).to(dtype) * 5 for _ in range(2))
    start = torch.tensor([0, 33, 61])
    cache.append(k, v, start)
    for held, x in zip(cache.dequantize(start, 9), (k, v)):
        part, got = (t.double().unflatten(-1, (-1, 32)) for t in (x, held))
        low, high = part.amin(-1, True), part.amax(-1, True)
        # half a step; 15 scales and the zero point in fp16; the rounding
        limit = (high - low) / 30 + (high - low) * 2.0 ** -11 + (
            part.abs().amax(-1, True) * (2.0 ** -11 + torch.finfo(
                dtype).eps))
        assert ((part - got).abs() <= limit).all()
    assert cache.nbytes() == (128 * 3 * 2 * (
        h // 2 + 2 * max(16, h // 4) + 2 * h // 8))


@pytest.mark.parametrize("window,sinks", [(None, 0), (5, 0), (5, 2)])
def test_cache_attention_plain(window, sinks):
    torch.manual_seed(2)
    b, n, nkv, h, s = 3, 4, 2, 32, 2
    cache = QuantKVCache(30, b, nkv, h)
    k, v = (torch.randn(30, b, nkv, h).to(BF16) for _ in range(2))
    cache.append(k, v, 0)
    hk, hv = cache._held(torch.arange(30).expand(b, 30))
    q = torch.randn(s, b, n, h).to(BF16)
    start = [28, 3, -1]
    got = cache.attention(q, torch.tensor(start), window_size=window,
                          sink_size=sinks).view(s, b, n, h)
    assert (got[:, 2] == 0).all()
    for i in range(s):
        for j in range(2):
            pos = start[j] + i
            at = [t for t in range(pos + 1) if window is None
                  or t > pos - window or t < sinks]
            for head in range(n):
                key, value = (x[j, at, head // 2].double() for x in (hk, hv))
                p = torch.softmax(
                    key @ q[i, j, head].double() / math.sqrt(h), 0)
                want = p @ value
                # one rounding to bf16, and sums in 32 bits
                off = (got[i, j, head].double() - want).abs()
                assert (off <= want.abs() * 2.0 ** -8 + 1e-5).all()


def test_cache_nan_reaches_only_who_sees_it():
    torch.manual_seed(3)
    cache = QuantKVCache(8, 1, 1, 32)
    k, v = (torch.randn(8, 1, 1, 32).to(BF16) for _ in range(2))
    v[4, 0, 0, 3] = math.nan
    cache.append(k, v, 0)
    out = cache.attention(torch.randn(8, 1, 2, 32).to(BF16), 0)
    assert not out[:4].isnan().any() and out[4:].isnan().all()


def test_cache_idle_start_is_bounded_too():
    """An idle sequence's tokens may reach the capacity, not pass it."""
    cache = QuantKVCache(8, 1, 1, 32)
    x = torch.randn(9, 1, 1, 32).to(BF16)
    cache.append(x, x, -1)
    assert not cache.attention(x, -1).any()
    key, _ = cache.dequantize(-1, 9)
    assert key[0].isnan().all() and not key[1:].any()
    more = torch.randn(90, 1, 1, 32).to(BF16)
    for call in (lambda: cache.append(more, more, -1),
                 lambda: cache.attention(more, -1),
                 lambda: cache.dequantize(-1, 90)):
        with pytest.raises(ValueError):
            call()


def test_cache_refuses():
    for bad in (dict(head_dim=96), dict(head_dim=48),
                dict(dtype=torch.float32), dict(batch_size=0),
                dict(max_sequence_len=0), dict(num_heads_kv=0)):
        with pytest.raises(ValueError):
            QuantKVCache(**{**dict(max_sequence_len=8, batch_size=2,
                                   num_heads_kv=2, head_dim=64), **bad})
    cache = QuantKVCache(8, 2, 2, 64)
    x = torch.randn(3, 2, 2, 64).to(BF16)
    cos, sin = precompute_rotary_tables(64, 8)
    cache.append(x, x, 5)
    cache.append(x, x, torch.tensor([5, -1]))
    for args, kw in [
        ((x, x, 6), {}), ((x, x, torch.tensor([6, 0])), {}),
        ((x, x[:2], 0), {}), ((x.float(), x, 0), {}),
        ((x, x.half(), 0), {}), ((x[:, :1], x[:, :1], 0), {}),
        ((x[:, :, :1], x[:, :, :1], 0), {}), ((x[..., :32], x, 0), {}),
        ((x, x, torch.tensor([0, 1, 2])), {}),
        ((x, x, torch.tensor([0], dtype=torch.int32)), {}),
        ((x, x, torch.tensor(0)), {}),
        ((x, x, 0), dict(query=x)), ((x, x, 0), dict(cos=cos, sin=sin)),
        ((x, x, 0), dict(query=x[:2], cos=cos, sin=sin)),
        ((x, x, 0), dict(query=x, cos=cos.double(), sin=sin)),
        ((x, x, 5), dict(query=x, cos=cos[:7].contiguous(),
                         sin=sin[:7].contiguous())),
        ((x.clone().requires_grad_(), x, 0), {}),
    ]:
        with pytest.raises(ValueError):
            cache.append(*args, **kw)
    q = torch.randn(1, 2, 4, 64).to(BF16)
    cache.attention(q, 7)
    for args, kw in [
        ((q, 8), {}), ((q[:, :, :3], 0), {}), ((q.half(), 0), {}),
        ((q, 0), dict(window_size=0)), ((q, 0), dict(sink_size=1)),
        ((q, 0), dict(window_size=3, sink_size=-1)),
        ((q, 0), dict(softmax_scale=math.inf)),
        ((q.clone().requires_grad_(), 0), {}),
    ]:
        with pytest.raises(ValueError):
            cache.attention(*args, **kw)
    for args in ((0, 9), (7, 2), (torch.tensor([0]),), (0, -1)):
        with pytest.raises(ValueError):
            cache.dequantize(*args)
    with pytest.raises(ValueError):
        cache.reorder(torch.tensor([0]))


# ---------------------------------------------------------------------------
# sampling

def test_sample_plain_filters():
    logits = torch.tensor([[0.0, 2.0, 1.0, 2.0, -1.0]])
    weight = torch.tensor([math.exp(-2), 1, math.exp(-1), 1, math.exp(-3)],
                          dtype=torch.float64)

    def drawn(u, **kw):
        return int(sample_tokens(logits, torch.tensor([u]), **kw))

    upto = (weight.cumsum(0) / weight.sum()).tolist()
    for i in range(5):
        assert drawn(upto[i] - 1e-4) == i
        if i < 4:
            assert drawn(upto[i] + 1e-4) == i + 1
    assert drawn(0.99, top_k=1) == 1 and drawn(0.0, temperature=0.0) == 1
    assert [drawn(u, top_k=2) for u in (0.0, 0.49, 0.51)] == [1, 1, 3]
    # before the third token lie 2 / 2.52 of the weight
    assert drawn(0.9999, top_p=0.5) == 3
    assert drawn(0.9999, top_p=0.81) == 3 and drawn(0.5, top_p=0.81) == 2
    assert drawn(0.9999, min_p=0.3) == 3 and drawn(0.55, min_p=0.3) == 2
    assert drawn(0.55, min_p=1.0) == 3


def test_sample_plain_per_row_and_void_rows():
    logits = torch.zeros(4, 10)
    logits[2] = -math.inf
    logits[3, 4] = math.nan
    got = sample_tokens(logits, torch.tensor([0.95, 0.95, 0.5, 0.5]),
                        top_k=torch.tensor([0, 2, 0, 0]),
                        temperature=torch.tensor([1.0, 0.0, 1.0, 1.0]))
    assert got.tolist() == [9, 0, -1, -1]
    assert sample_tokens(logits[:0], torch.empty(0)).shape == (0,)


def test_sample_follows_the_distribution():
    """Evenly spaced uniform numbers meet each token as often as its weight
    says, to one."""
    torch.manual_seed(4)
    logits = torch.randn(1, 20)
    n = 5000
    u = (torch.arange(n) + 0.5) / n
    got = sample_tokens(logits.expand(n, -1), u, temperature=0.8)
    count = torch.bincount(got, minlength=20)
    want = torch.softmax(logits[0].double() / 0.8, 0) * n
    assert (count - want).abs().max() <= 1.0


def test_sample_refuses():
    logits, u = torch.zeros(3, 10), torch.zeros(3)
    for bad in (
        dict(logits=logits[0]), dict(logits=logits[:, :0]),
        dict(logits=logits.double()), dict(logits=logits.long()),
        dict(uniform=u[:2]), dict(uniform=u.double()), dict(uniform=0.5),
        dict(temperature=-1.0), dict(temperature=math.inf),
        dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.5),
        dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan),
        dict(top_k=torch.zeros(3)), dict(top_p=torch.zeros(2)),
        dict(min_p=torch.zeros(3, dtype=torch.float64)),
        dict(logits=torch.empty(1, 1).expand(3, (1 << 20) + 1)),
    ):
        with pytest.raises(ValueError):
            sample_tokens(**{**dict(logits=logits, uniform=u), **bad})
