"""Serving operators on the GPU against plain implementations in 64 bits:
rotary positions, the 4-bit key/value cache, attention over it, sampling."""

import math

import pytest
import torch

from megatron_amd.models.rope import precompute_rotary_tables
from megatron_amd.ops import (
    QuantKVCache,
    rotary_embedding,
    sample_tokens,
)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def generator(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def randn(g, *shape, dtype=FP32):
    return torch.randn(*shape, generator=g).to(dtype)


# ---------------------------------------------------------------------------
# rotary positions

def rotate_exact(x, cos, sin, interleaved):
    """x [s, b, n, h], tables [s, b, r], all in 64 bits."""
    r = cos.shape[-1]
    y = x.double().clone()
    first = slice(0, 2 * r, 2) if interleaved else slice(0, r)
    second = slice(1, 2 * r, 2) if interleaved else slice(r, 2 * r)
    c, s = cos.double()[:, :, None], sin.double()[:, :, None]
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def rotary_bound(x, cos, sin, dtype):
    """Two products, one sum and the rounding at the end: the sums' terms are
    at most (|a| + |b|) max(|c|, |s|), off by 2^-24 three times."""
    r = cos.shape[-1]
    big = 2 * x.double().abs().amax() * max(cos.abs().max(), sin.abs().max())
    return 3 * 2.0 ** -24 * float(big) if r else 0.0


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("s,b,n,nkv,h,r", [
    (1, 1, 1, 1, 64, 32), (7, 2, 4, 2, 128, 64), (5, 3, 3, 1, 80, 10),
    (3, 2, 2, 2, 64, 1), (130, 1, 71, 1, 64, 32), (2, 5, 5, 5, 96, 24),
    (9, 2, 2, 1, 50, 21), (4, 2, 16, 8, 128, 48), (3, 2, 8, 8, 256, 128),
])
def test_rotary_matches(dtype, interleaved, s, b, n, nkv, h, r):
    g = generator(s * 1000 + r)
    q = randn(g, s, b, n, h, dtype=dtype)
    k = randn(g, s, b, nkv, 3 * h, dtype=dtype)[..., h:2 * h]
    gq, gk = randn(g, s, b, n, h, dtype=dtype), randn(g, s, b, nkv, h,
                                                      dtype=dtype)
    cos, sin = precompute_rotary_tables(2 * r, 500, scaling_type="yarn",
                                        scaling_factor=4.0)
    for positions in (None, torch.randint(0, 500, (b, s), generator=g)):
        dq = q.cuda().requires_grad_()
        dk = k.cuda().requires_grad_()
        if k.shape[-1] != k.stride(2):  # keep the slice's strides
            dk = torch.empty(s, b, nkv, 3 * h, dtype=dtype, device="cuda")[
                ..., h:2 * h].copy_(k).requires_grad_()
        yq, yk = rotary_embedding(
            dq, dk, cos.cuda(), sin.cuda(),
            positions=None if positions is None else positions.cuda(),
            interleaved=interleaved)
        grads = torch.autograd.grad((yq, yk), (dq, dk), (gq.cuda(), gk.cuda()))
        at = (torch.arange(s)[:, None].expand(s, b) if positions is None
              else positions.t())
        c, sn = cos[at], sin[at]
        for got, x, back in ((yq, q, False), (yk, k, False),
                             (grads[0], gq, True), (grads[1], gk, True)):
            want = rotate_exact(x, c, -sn if back else sn, interleaved)
            slack = rotary_bound(x, c, sn, dtype)
            off = (got.detach().double().cpu() - want).abs()
            limit = want.abs() * half_step(dtype) + slack + 2.0 ** -25
            assert got.dtype == dtype and got.shape == want.shape
            assert (off <= limit).all()


def test_rotary_gradient_against_differences():
    """The loss is linear in x, so a central difference is exact but for
    roundings: y is off by 3 * 2^-24 of at most 2 * 4.5 * 1.21 a value (that
    many values of a normal sample stay under 4.5, 1.21 the tables'
    magnitude), over 2 * step = 2 and a product with g."""
    g = generator(3)
    s, b, n, h = 4, 2, 3, 32
    q = randn(g, s, b, n, h).cuda().requires_grad_()
    weight = randn(g, s, b, n, h).cuda()
    cos, sin = (t.cuda() for t in precompute_rotary_tables(
        16, 64, scaling_type="yarn", scaling_factor=8.0))
    positions = torch.randint(0, 64, (b, s), generator=g).cuda()

    def loss(x):
        y, none = rotary_embedding(x, None, cos, sin, positions, False)
        assert none is None
        return (y.double() * weight.double()).sum()

    grad, = torch.autograd.grad(loss(q), q)
    for place in range(0, q.numel(), 37):
        step = torch.zeros(q.numel(), device="cuda")
        step[place] = 1.0
        step = step.view_as(q)
        slope = (loss(q.detach() + step) - loss(q.detach() - step)) / 2
        assert abs(float(slope) - float(grad.view(-1)[place])) < 1e-4


def test_rotary_one_gradient_and_expanded_one():
    g = generator(4)
    cos, sin = (t.cuda() for t in precompute_rotary_tables(64, 16))
    q = randn(g, 5, 2, 4, 64).cuda().requires_grad_()
    k = randn(g, 5, 2, 2, 64).cuda().requires_grad_()
    yq, yk = rotary_embedding(q, k, cos, sin)
    yk.sum().backward()  # an expanded gradient, and none for the query
    assert q.grad is None
    at = torch.arange(5)[:, None].expand(5, 2)
    want = rotate_exact(torch.ones(5, 2, 2, 64), cos.cpu()[at],
                        -sin.cpu()[at], True)
    assert (k.grad.double().cpu() - want).abs().max() < 2.0 ** -20


def test_rotary_position_outside_is_nan():
    cos, sin = (t.cuda() for t in precompute_rotary_tables(32, 8))
    q = torch.ones(3, 1, 2, 64, device="cuda", dtype=BF16)
    y, _ = rotary_embedding(q, None, cos, sin,
                            torch.tensor([[7, 8, -1]], device="cuda"))
    assert not y[0].isnan().any()
    assert y[1:, ..., :32].isnan().all() and (y[1:, ..., 32:] == 1).all()


def test_rotary_empty():
    cos, sin = (t.cuda() for t in precompute_rotary_tables(32, 8))
    q = torch.ones(0, 3, 2, 64, device="cuda", dtype=BF16)
    y, k = rotary_embedding(q, q, cos, sin)
    assert y.shape == q.shape and k.shape == q.shape


# ---------------------------------------------------------------------------
# 4-bit cache

def caches(length, b, nkv, h, dtype):
    return (QuantKVCache(length, b, nkv, h, dtype=dtype),
            QuantKVCache(length, b, nkv, h, dtype=dtype, device="cuda"))


def assert_same_buffers(cpu, gpu):
    for a, b in zip(cpu.buffers, gpu.buffers):
        b = b.cpu()
        if a.dtype == torch.float16:
            same = (a == b) | (a.isnan() & b.isnan())
        else:
            same = a == b
        assert same.all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("h", [32, 64, 128, 256])
@pytest.mark.parametrize("s,b,nkv,length", [
    (1, 1, 1, 1), (1, 3, 2, 65), (5, 2, 3, 70), (130, 2, 1, 200),
    (64, 1, 8, 64),
])
def test_append_same_as_plain(dtype, h, s, b, nkv, length):
    g = generator(h + s)
    cpu, gpu = caches(length, b, nkv, h, dtype)
    mixed = randn(g, s, b, nkv, 2 * h) * 3.0 + randn(g, nkv, 2 * h)
    mixed = mixed.to(dtype)
    start = torch.randint(0, length - s + 1, (b,), generator=g)
    for cache, m, at in ((cpu, mixed, start),
                         (gpu, mixed.cuda(), start.cuda())):
        cache.append(m[..., :h], m[..., h:], at)
    assert_same_buffers(cpu, gpu)
    for a, x in zip(cpu.dequantize(start, s), gpu.dequantize(start.cuda(),
                                                            s)):
        assert torch.equal(a, x.cpu())


def special_rows(dtype, h):
    g = generator(11)
    rows = [torch.zeros(h), torch.full((h,), 3.25), torch.full((h,), -0.0),
            randn(g, h) * 1e-6, randn(g, h) * 3e4, randn(g, h) * 1e-3 + 500,
            torch.arange(h).float(), torch.arange(h).float() / 2,
            torch.arange(h).float() % 16 * 0.5 - 4.25]
    for bad in (math.inf, -math.inf, math.nan, torch.finfo(dtype).max):
        row = randn(g, h)
        row[h // 2 + 3] = bad
        rows.append(row)
    # ties: halves of a whole scale
    row = torch.arange(h).float() % 31 / 2
    row[0::32], row[1::32] = 0, 15
    rows.append(row)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("h", [32, 64, 128, 256])
def test_append_special_values(dtype, h):
    rows = special_rows(dtype, h)
    t = rows.shape[0]
    cpu, gpu = caches(t, 2, 1, h, dtype)
    key = torch.stack([rows, rows.flip(0)], 1)[:, :, None]
    value = key.flip(1)
    cpu.append(key, value, 0)
    gpu.append(key.cuda(), value.cuda(), 0)
    assert_same_buffers(cpu, gpu)
    # a NaN in the key or the value of a token makes its key NaN
    fine = ~(key.isnan() | value.isnan()).any(-1)
    for held, x in zip(gpu.dequantize(), (key, value)):
        x, held = x.double(), held.double().cpu()
        x, held = x[fine].clamp(-57344, 57344), held[fine]
        part, got = x.unflatten(-1, (-1, 32)), held.unflatten(-1, (-1, 32))
        span = part.amax(-1, keepdim=True) - part.amin(-1, keepdim=True)
        peak = part.abs().amax(-1, keepdim=True)
        # half a step of span / 15, 15 steps whose scale is off by 2^-11 of
        # itself (or 2^-25), a zero point off by 2^-11 (or 2^-25), and the
        # value's rounding
        limit = (span / 30 * (1 + 2.0 ** -11) + span * 2.0 ** -11
                 + 16 * 2.0 ** -25 + peak * 2.0 ** -11
                 + 2 * peak * half_step(dtype))
        assert ((part - got).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("h,r", [(64, 32), (128, 64), (128, 16), (32, 5),
                                 (256, 128)])
def test_append_rotated(dtype, interleaved, h, r):
    g = generator(h + r)
    s, b, n, nkv, length = 3, 4, 6, 2, 40
    cpu, gpu = caches(length, b, nkv, h, dtype)
    cos, sin = precompute_rotary_tables(2 * r, length, theta=500.0)
    q, k, v = (randn(g, s, b, x, h, dtype=dtype) for x in (n, nkv, nkv))
    start = torch.tensor([0, 37, -1, 12])
    want = cpu.append(k, v, start, query=q, cos=cos, sin=sin,
                      interleaved=interleaved)
    got = gpu.append(k.cuda(), v.cuda(), start.cuda(), query=q.cuda(),
                     cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved)
    assert torch.equal(want, got.cpu())
    assert (got[:, 2] == 0).all()
    assert_same_buffers(cpu, gpu)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_append_many_groups_of_any_scale(dtype):
    """Scales and codes near a border are decided as exactly as the others:
    32768 groups whose middles and spans lie anywhere."""
    g = generator(52)
    s, b, nkv, h = 1024, 2, 2, 128
    cpu, gpu = caches(s, b, nkv, h, dtype)
    rows = [randn(g, s, b, nkv, 4, 32)
            * 2.0 ** torch.randint(-9, 10, (s, b, nkv, 4, 1), generator=g)
            + randn(g, s, b, nkv, 4, 1)
            * 2.0 ** torch.randint(-9, 10, (s, b, nkv, 4, 1), generator=g)
            for _ in range(2)]
    k, v = (x.reshape(s, b, nkv, h).to(dtype) for x in rows)
    cpu.append(k, v, 0)
    gpu.append(k.cuda(), v.cuda(), 0)
    assert_same_buffers(cpu, gpu)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("h", [32, 64, 128, 256])
def test_rows_at_odd_places_as_at_even_ones(dtype, h):
    """Rows that begin anywhere, one value off among them, give the same
    bits as rows at multiples of 16 bytes."""
    g = generator(53 + h)
    s, b, n, nkv, length = 5, 2, 6, 2, 50
    packed = randn(g, s, b, n + 2 * nkv, h + 3, dtype=dtype).cuda()
    odd = packed[..., 1:h + 1].split([n, nkv, nkv], dim=2)
    even = [x.contiguous() for x in odd]
    cos, sin = (t.cuda() for t in precompute_rotary_tables(h, length))
    at = torch.tensor([3, 40], device="cuda")
    got = []
    for q, k, v in (odd, even):
        cache = QuantKVCache(length, b, nkv, h, dtype=dtype, device="cuda")
        cache.append(k, v, at - 3)
        rows = [x.clone() for x in cache.buffers]
        turned = cache.append(k, v, at, query=q, cos=cos, sin=sin)
        got.append(rows + cache.buffers
                   + [turned, cache.attention(q, at),
                      cache.attention(q[:1], at)])
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_append_leaves_other_rows():
    """Idle sequences and rows behind the capacity stay as they were."""
    g = generator(5)
    cache = QuantKVCache(10, 3, 2, 64, dtype=BF16, device="cuda")
    fill = randn(g, 10, 3, 2, 64, dtype=BF16).cuda()
    cache.append(fill, fill, 0)
    before = [t.clone() for t in cache.buffers]
    more = randn(g, 4, 3, 2, 64, dtype=BF16).cuda()
    cache.append(more, more, torch.tensor([-1, 8, -5], device="cuda"))
    kd, _ = cache.dequantize()
    old = QuantKVCache(10, 3, 2, 64, dtype=BF16, device="cuda")
    for t, x in zip(old.buffers, before):
        t.copy_(x)
    kb, _ = old.dequantize()
    assert torch.equal(kd[:8], kb[:8])
    assert torch.equal(kd[:, [0, 2]], kb[:, [0, 2]])
    assert not torch.equal(kd[8:, 1], kb[8:, 1])
    # nothing was written behind the ten tokens either
    assert torch.equal(cache.k_codes[:, :, 10:], before[0][:, :, 10:])
    assert cache.dequantize(torch.tensor([9], device="cuda"), 2)[0][
        1].isnan().all()


@pytest.mark.parametrize("start", [2 ** 63 - 1, 2 ** 63 - 4, 2 ** 62])
def test_positions_at_the_end_of_64_bits(start):
    """A position to which a token's number cannot be added is behind the
    capacity like any other: nothing is written, what is read is NaN."""
    g = generator(51)
    cache = QuantKVCache(70, 2, 2, 64, dtype=BF16, device="cuda")
    fill = randn(g, 70, 2, 2, 64, dtype=BF16).cuda()
    cache.append(fill, fill, 0)
    before = [t.clone() for t in cache.buffers]
    at = torch.tensor([start, -start - 1], device="cuda")
    more = randn(g, 9, 2, 2, 64, dtype=BF16).cuda()
    cos, sin = (t.cuda() for t in precompute_rotary_tables(64, 70))
    cache.append(more, more, at)
    q = cache.append(more, more, at, query=more, cos=cos, sin=sin)
    assert q[:, 0].isnan().all() and not q[:, 1].any()
    for a, b in zip(cache.buffers, before):
        assert torch.equal(a, b)
    for x in cache.dequantize(at, 9):
        assert x.isnan().all()
    out = cache.attention(more, at)
    assert out[:, 0].isnan().all() and not out[:, 1].any()


def test_append_empty():
    cache = QuantKVCache(4, 2, 1, 64, dtype=BF16, device="cuda")
    none = torch.empty(0, 2, 1, 64, dtype=BF16, device="cuda")
    cache.append(none, none, 4)
    k, v = cache.dequantize(2, 0)
    assert k.shape == (0, 2, 1, 64) and v.shape == k.shape
    assert all((t == 0).all() for t in cache.buffers)


def attention_exact(cache, q, start, scale, window, sinks):
    """In 64 bits from what the cache holds, and a bound on the error: keys
    and values are rounded to fp16 (2^-11), so a score is off by 2^-11 of its
    absolute terms, a weight by twice the largest such, by fp16 (2^-11) and by
    2^-20 for exponentials and sums in 32 bits; the output is rounded once."""
    s, b, n, h = q.shape
    nkv = cache.num_heads_kv
    held = QuantKVCache(cache.max_sequence_len, b, nkv, h, dtype=cache.dtype)
    for t, x in zip(held.buffers, cache.buffers):
        t.copy_(x)
    everything = torch.arange(cache.max_sequence_len)
    key, value = (x.double().permute(0, 2, 1, 3).repeat_interleave(
        n // nkv, dim=1) for x in held._held(everything.expand(b, -1)))
    out = torch.zeros(s, b, n, h, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(s):
        for j, first in enumerate(start):
            if first < 0:
                continue
            pos = first + i
            seen = everything <= pos
            if window:
                seen &= (everything > pos - window) | (everything < sinks)
            at = everything[seen]
            x = q[i, j].double()[:, None]  # [n, 1, h]
            k, v = key[j][:, at], value[j][:, at]
            p = torch.softmax((x * k).sum(-1) * scale, -1)[:, None]
            out[i, j] = (p @ v)[:, 0]
            off = 2.0 ** -11 * scale * (x * k).abs().sum(-1).amax(-1)
            wide = 2 * torch.expm1(off) + 2 * 2.0 ** -11 + 2.0 ** -20
            bound[i, j] = (p @ v.abs())[:, 0] * wide[:, None]
            # weights below fp16's normal range are off by 2^-25 of the peak
            bound[i, j] += 2.0 ** -25 * v.abs().sum(1)
    limit = out.abs() * half_step(q.dtype) + bound + 1e-9
    return out.reshape(s, b, n * h), limit.reshape(s, b, n * h)


def filled_cache(g, length, b, nkv, h, dtype):
    cache = QuantKVCache(length, b, nkv, h, dtype=dtype, device="cuda")
    bias = randn(g, nkv, h)
    cache.append((randn(g, length, b, nkv, h) + bias).to(dtype).cuda(),
                 randn(g, length, b, nkv, h, dtype=dtype).cuda(), 0)
    return cache


def check_attention(cache, q, start, scale=None, window=None, sinks=0):
    h = q.shape[-1]
    got = cache.attention(q.cuda(), torch.tensor(start, device="cuda"),
                          softmax_scale=scale, window_size=window,
                          sink_size=sinks)
    want, limit = attention_exact(cache, q, start, scale or h ** -0.5,
                                  window, sinks)
    assert got.dtype == q.dtype
    off = (got.double().cpu() - want).abs()
    assert (off <= limit).all(), float((off / limit).max())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("h", [32, 64, 128, 256])
@pytest.mark.parametrize("s,n,nkv,length,start", [
    (1, 1, 1, 1, [0, -1]), (1, 4, 4, 63, [62, 0]), (1, 8, 2, 65, [64, 63]),
    (1, 8, 1, 200, [15, 16]), (3, 6, 3, 130, [127, 0]),
    (17, 4, 2, 100, [83, 31]), (1, 71, 1, 90, [89, 3]),
    (5, 71, 1, 90, [85, 3]), (1, 2, 2, 1500, [1499, 1024]),
])
def test_attention_matches(dtype, h, s, n, nkv, length, start):
    g = generator(h + length)
    cache = filled_cache(g, length, 2, nkv, h, dtype)
    check_attention(cache, randn(g, s, 2, n, h, dtype=dtype), start)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4),
                                          (100, 130), (500, 2), (33, 64)])
@pytest.mark.parametrize("s,start", [(1, [299, 5, 40]), (6, [0, 294, 131])])
def test_attention_window_and_sinks(window, sinks, s, start):
    g = generator(window + s)
    cache = filled_cache(g, 300, 3, 2, 64, BF16)
    check_attention(cache, randn(g, s, 3, 8, 64, dtype=BF16), start,
                    window=window, sinks=sinks)


def test_attention_long_and_sharp():
    """A key far back outweighs the rest, which the running maximum meets
    late or early."""
    g = generator(9)
    length, h = 5000, 128
    key = randn(g, length, 2, 1, h, dtype=BF16)
    q = randn(g, 1, 2, 4, h, dtype=BF16)
    key[10, 0, 0] = 6 * q[0, 0, 1]
    key[4990, 1, 0] = 6 * q[0, 1, 2]
    cache = QuantKVCache(length, 2, 1, h, dtype=BF16, device="cuda")
    cache.append(key.cuda(), randn(g, length, 2, 1, h, dtype=BF16).cuda(), 0)
    check_attention(cache, q, [4999, 4995])


def test_attention_scale_and_strides():
    g = generator(10)
    cache = filled_cache(g, 80, 2, 2, 64, FP16)
    wide = randn(g, 2, 2, 4, 3 * 64, dtype=FP16)
    q = wide.cuda()[..., 64:128]
    at = torch.tensor([70, 9, 5, 9], device="cuda")[::2]  # strided start
    got = cache.attention(q, at, softmax_scale=0.3)
    want, limit = attention_exact(cache, wide[..., 64:128], [70, 5], 0.3,
                                  None, 0)
    assert ((got.double().cpu() - want).abs() <= limit).all()
    one = cache.attention(q, torch.tensor([5], device="cuda"))
    assert torch.equal(one, cache.attention(q, 5))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 4.0])
def test_attention_unusual_scales(scale):
    g = generator(15)
    cache = filled_cache(g, 300, 2, 2, 64, BF16)
    q = randn(g, 1, 2, 4, 64, dtype=BF16)
    got = cache.attention(q.cuda(), torch.tensor([299, 40], device="cuda"),
                          softmax_scale=scale)
    want, _ = attention_exact(cache, q, [299, 40], scale, None, 0)
    bound = attention_exact(cache, q, [299, 40], abs(scale), None, 0)[1]
    # a bound for |scale| holds its sums with other weights: the largest value
    # takes their place
    most = bound.max() + 4.5 * 2.0 ** -8
    assert ((got.double().cpu() - want).abs() <= most).all()


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4, 1e30])
def test_attention_queries_of_any_size(size):
    """The scale undoes the query's size: the same output, to its roundings
    (a power of two changes nothing in bf16)."""
    g = generator(16)
    cache = filled_cache(g, 100, 1, 1, 128, BF16)
    q = randn(g, 2, 1, 3, 128, dtype=BF16).cuda()
    power = 2.0 ** round(math.log2(size))
    want = cache.attention(q, 98, softmax_scale=0.1)
    got = cache.attention(q * power, 98, softmax_scale=0.1 / power)
    assert torch.equal(got, want)


@pytest.mark.parametrize("b,length", [(65, 700), (150, 300), (3, 9000)])
def test_attention_many_ragged_sequences(b, length):
    """Shares of the tokens are settled over all sequences, by waves of 64."""
    g = generator(b)
    cache = QuantKVCache(length, b, 2, 64, dtype=BF16, device="cuda")
    gpu = torch.Generator(device="cuda").manual_seed(b)
    k, v = (torch.randn(length, b, 2, 64, generator=gpu, device="cuda")
            .to(BF16) for _ in range(2))
    cache.append(k, v, 0)
    q = randn(g, 1, b, 4, 64, dtype=BF16)
    start = torch.randint(0, length, (b,), generator=g)
    start[torch.rand(b, generator=g) < 0.2] = -1
    start[-1] = length - 1
    out = cache.attention(q.cuda(), start.cuda())
    for j in range(b):  # one sequence at a time, alone in a cache
        one = QuantKVCache(length, 1, 2, 64, dtype=BF16, device="cuda")
        for t, x in zip(one.buffers, cache.buffers):
            t.copy_(x[j:j + 1])
        alone = one.attention(q[:, j:j + 1].cuda(), int(start[j]))
        # shares differ, and so do the sums' roundings in 32 bits: one step
        # of bf16, or 2^-16 of values up to 5 where terms cancel
        off = (out[:, j].float() - alone[:, 0].float()).abs()
        assert (off <= alone[:, 0].float().abs() * 2.0 ** -7
                + 5 * 2.0 ** -16).all()
    assert (out[:, start < 0] == 0).all()
    some = [0, b // 2, b - 1]
    part = QuantKVCache(length, 3, 2, 64, dtype=BF16)
    for t, x in zip(part.buffers, cache.buffers):
        t.copy_(x[some])
    want, limit = attention_exact(part, q[:, some],
                                  [int(start[j]) for j in some], 0.125, None,
                                  0)
    assert ((out[:, some].double().cpu() - want).abs() <= limit).all()


def test_attention_over_a_prompt():
    """Many query tokens: more rows than shares of the tokens pay for."""
    g = generator(17)
    cache = filled_cache(g, 400, 2, 1, 64, FP16)
    q = randn(g, 300, 2, 3, 64, dtype=FP16)
    check_attention(cache, q, [100, 17], window=90, sinks=3)


def test_attention_window_beyond_everything():
    g = generator(18)
    cache = filled_cache(g, 100, 2, 1, 64, BF16)
    q = randn(g, 1, 2, 3, 64, dtype=BF16).cuda()
    at = torch.tensor([99, 7], device="cuda")
    want = cache.attention(q, at)
    assert torch.equal(want, cache.attention(q, at, window_size=1 << 62,
                                             sink_size=1 << 62))


def test_cache_past_32_bit_offsets():
    """A head's codes take more than 2^31 bytes."""
    g = generator(19)
    length = (1 << 24) + 5000
    cache = QuantKVCache(length, 1, 1, 256, dtype=BF16, device="cuda")
    assert cache.k_codes.numel() > 1 << 31
    x = randn(g, 200, 1, 1, 256, dtype=BF16)
    small = QuantKVCache(200, 1, 1, 256, dtype=BF16, device="cuda")
    q = randn(g, 1, 1, 4, 256, dtype=BF16).cuda()
    small.append(x.cuda(), x.cuda(), 0)
    for at in (0, length - 200):
        cache.append(x.cuda(), x.cuda(), at)
        for a, b in zip(cache.dequantize(at, 200), small.dequantize()):
            assert torch.equal(a, b)
        got = cache.attention(q, at + 199, window_size=200)
        want = small.attention(q, 199)
        # other shares, other roundings of sums in 32 bits
        off = (got.float() - want.float()).abs()
        assert (off <= want.float().abs() * 2.0 ** -7 + 5 * 2.0 ** -16).all()


@pytest.mark.parametrize("h", [64, 128])
def test_attention_nan_stays_where_it_is_seen(h):
    """NaN in a value or a key reaches the queries that see it and no other;
    rows behind the end and outside the window may hold anything."""
    g = generator(12)
    b, nkv, n, length = 2, 2, 4, 150
    key = randn(g, length, b, nkv, h, dtype=BF16)
    value = randn(g, length, b, nkv, h, dtype=BF16)
    value[100, 0, 1, 5] = math.nan
    key[20, 1, 0, 7] = math.nan
    value[140:] = math.nan
    key[140:] = math.nan
    cache = QuantKVCache(length, b, nkv, h, dtype=BF16, device="cuda")
    cache.append(key.cuda(), value.cuda(), 0)
    q = randn(g, 8, b, n, h, dtype=BF16).cuda()
    out = cache.attention(q, torch.tensor([96, 24], device="cuda"))
    out = out.view(8, b, n, h)
    seen = torch.zeros(8, b, n, dtype=torch.bool)
    seen[4:, 0, 2:] = True  # positions 100.. of the second key head
    seen[:, 1, :2] = True
    assert torch.equal(out.isnan().any(-1).cpu(), seen)
    assert torch.equal(out.isnan().all(-1).cpu(), seen)
    out = cache.attention(q[:1], torch.tensor([130, 139], device="cuda"),
                          window_size=30, sink_size=2)
    out = out.view(1, b, n, h)
    assert not out.isnan()[:, 1].any()
    out = cache.attention(q[:1], torch.tensor([129, 50], device="cuda"),
                          window_size=29, sink_size=2)
    assert not out.isnan().any()


def test_attention_values_at_the_limit():
    """Saturated values stay finite: the largest code stands for 57344."""
    cache = QuantKVCache(4, 1, 1, 64, dtype=BF16, device="cuda")
    x = torch.full((4, 1, 1, 64), math.inf)
    x[..., 0::2] = -math.inf
    x = x.to(BF16).cuda()
    cache.append(x * 0 + 1, x * 0 + 1, 0)  # NaN: inf * 0
    assert cache.dequantize()[0].isnan().all()
    cache.append(torch.ones_like(x), x, 0)
    out = cache.attention(torch.ones(1, 1, 2, 64, dtype=BF16, device="cuda"),
                          3)
    assert (out.abs().float() - 57344).abs().max() <= 57344 * 2.0 ** -8


def test_attention_outside_capacity_is_nan():
    g = generator(13)
    cache = filled_cache(g, 20, 2, 1, 64, BF16)
    q = randn(g, 2, 2, 2, 64, dtype=BF16).cuda()
    out = cache.attention(q, torch.tensor([19, 500], device="cuda"))
    assert not out[0, 0].isnan().any()
    assert out[1, 0].isnan().all() and out[:, 1].isnan().all()


def test_reorder():
    g = generator(14)
    cache = filled_cache(g, 33, 3, 2, 64, BF16)
    k, v = cache.dequantize()
    cache.reorder(torch.tensor([2, 0, 2], device="cuda"))
    k2, v2 = cache.dequantize()
    assert torch.equal(k2, k[:, [2, 0, 2]])
    assert torch.equal(v2, v[:, [2, 0, 2]])


# ---------------------------------------------------------------------------
# sampling

def sample_exact(logits, u, temperature, top_k, top_p, min_p):
    """One row in 64 bits, walking down the sorted tokens."""
    row = logits.double()
    if bool(row.isnan().any()) or float(row.max()) == -math.inf:
        return -1
    value, index = torch.sort(row, descending=True, stable=True)
    if temperature == 0:
        return int(index[0])
    if top_k:
        value, index = value[:top_k], index[:top_k]
    weight = ((value - value[0]) / temperature).exp()
    weight[value == value[0]] = 1.0
    if 0 < top_p < 1:
        before = weight.cumsum(0) - weight
        keep = before <= top_p * weight.sum()
        weight, index = weight[keep], index[keep]
    keep = weight >= min_p
    weight, index = weight[keep], index[keep]
    order = index.argsort()
    upto = weight[order].cumsum(0)
    return int(index[order][(upto <= u * upto[-1]).sum()])


FILTERS = [(0, 0.0, 0.0), (1, 0.0, 0.0), (40, 0.0, 0.0), (0, 0.9, 0.0),
           (0, 0.0, 0.1), (50, 0.8, 0.05), (7, 0.3, 0.0), (0, 1.0, 1.0),
           (1000, 0.999, 0.001)]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("vocab", [1, 2, 65, 1000, 32000, 50257])
@pytest.mark.parametrize("spread", [0.01, 2.5])
def test_sample_matches(dtype, vocab, spread):
    """Tokens are whole numbers and have to be equal. The kernel's weights are
    off by 2^-40 of the largest at most, so a uniform number would have to
    fall within about 1e-11 of a border to be told apart."""
    g = generator(vocab)
    b = 6
    logits = (randn(g, b, vocab + 3) * spread).to(dtype)[:, :vocab]
    u = torch.rand(b, generator=g)
    u[0] = 0.0
    dev = torch.empty(b, vocab + 3, dtype=dtype, device="cuda")[:, :vocab]
    dev.copy_(logits)
    for top_k, top_p, min_p in FILTERS:
        for temperature in (0.0, 0.7, 1.3):
            got = sample_tokens(dev, u.cuda(), temperature=temperature,
                                top_k=top_k, top_p=top_p, min_p=min_p)
            want = [sample_exact(logits[i], float(u[i]), temperature, top_k,
                                 top_p, min_p) for i in range(b)]
            assert got.tolist() == want, (top_k, top_p, min_p, temperature)


def test_sample_settings_per_row():
    g = generator(21)
    b, vocab = 9, 5000
    logits = randn(g, b, vocab) * 2
    u = torch.rand(b, generator=g)
    temperature = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 0.9, 0.8, 0.7, 1.0])
    top_k = torch.tensor([f[0] for f in FILTERS])
    top_p = torch.tensor([f[1] for f in FILTERS])
    min_p = torch.tensor([f[2] for f in FILTERS])
    got = sample_tokens(logits.cuda(), u.cuda(), temperature.cuda(),
                        top_k.cuda(), top_p.cuda(), min_p.cuda())
    want = [sample_exact(logits[i], float(u[i]), float(temperature[i]),
                         int(top_k[i]), float(top_p[i]), float(min_p[i]))
            for i in range(b)]
    assert got.tolist() == want


@pytest.mark.parametrize("vocab", [300, 70001])
def test_sample_equal_logits(vocab):
    """All alike: the order is the index's, top-k and top-p cut at exact
    counts, the draw is the uniform number's share."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.99])
    logits = torch.full((4, vocab), -3.5, device="cuda")
    for top_k, top_p, kept in ((0, 0.0, vocab), (64, 0.0, 64),
                               (64, 0.5, 33), (128, 0.25, 33)):
        got = sample_tokens(logits, u.cuda(), top_k=top_k, top_p=top_p)
        assert got.tolist() == [int(float(x) * kept) for x in u]
    assert sample_tokens(logits, u.cuda(), temperature=0.0).tolist() == [0] * 4


def test_sample_ties_at_the_border():
    """Two heavy tokens, then many equal ones of which a part is kept."""
    logits = torch.full((1, 2000), 0.0)
    logits[0, 700], logits[0, 1500] = 2.0, 2.0
    u = torch.rand(1, 64, generator=generator(22))
    rows = logits.expand(64, -1)
    for top_k, top_p in ((10, 0.0), (0, 0.6), (500, 0.9), (2, 0.0),
                         (3, 0.95)):
        got = sample_tokens(rows.cuda(), u[0].cuda(), top_k=top_k,
                            top_p=top_p)
        want = [sample_exact(logits[0], float(x), 1.0, top_k, top_p, 0.0)
                for x in u[0]]
        assert got.tolist() == want


def test_sample_infinities_and_nan():
    g = generator(23)
    logits = randn(g, 6, 400)
    logits[0] = -math.inf
    logits[1, 7] = math.nan
    logits[2, 100:] = -math.inf
    logits[3, [5, 9]] = math.inf
    logits[4] = -math.inf
    logits[4, 399] = -1e30
    logits[5] = torch.finfo(FP32).min
    u = torch.tensor([0.5, 0.5, 0.99, 0.6, 0.0, 0.5])
    got = sample_tokens(logits.cuda(), u.cuda())
    assert got.tolist() == [-1, -1,
                            sample_exact(logits[2], float(u[2]), 1, 0, 0, 0),
                            9, 399, 200]
    got = sample_tokens(logits.cuda(), u.cuda(), top_k=150, top_p=0.9,
                        min_p=0.01)
    assert got[:2].tolist() == [-1, -1]
    assert int(got[2]) < 100 and int(got[3]) in (5, 9) and int(got[4]) == 399


@pytest.mark.parametrize("kind", ["floor", "masked", "offset", "tiny", "two",
                                  "steps", "wide"])
def test_sample_ranges_that_are_hard_to_share_out(kind):
    """Logits of which most are far from the others, or next to each other."""
    g = generator(25)
    b, vocab = 5, 3001
    logits = randn(g, b, vocab)
    if kind == "floor":  # masked by the type's lowest value
        logits[:, 500:] = torch.finfo(FP32).min
    elif kind == "masked":
        logits[torch.rand(b, vocab, generator=g) < 0.5] = -1e4
    elif kind == "offset":
        logits = 1000 + logits * 1e-3
    elif kind == "tiny":  # all within the subnormal numbers
        logits = logits * 1e-40
    elif kind == "two":
        logits = (logits > 0).float() * 1e-30
    elif kind == "steps":
        logits = (logits * 4).round() / 4
    else:
        logits = logits * 1e38
    u = torch.rand(b, generator=g)
    for top_k, top_p, min_p in FILTERS + [(400, 0.0, 0.0), (2000, 0.7, 0.0)]:
        got = sample_tokens(logits.cuda(), u.cuda(), top_k=top_k,
                            top_p=top_p, min_p=min_p)
        want = [sample_exact(logits[i], float(u[i]), 1.0, top_k, top_p,
                             min_p) for i in range(b)]
        assert got.tolist() == want, (top_k, top_p, min_p)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_sample_rows_that_begin_anywhere(dtype, offset):
    g = generator(26)
    b, vocab = 4, 4999
    wide = (randn(g, b, vocab + 11) * 2).to(dtype)
    u = torch.rand(b, generator=g)
    rows = wide.cuda()[:, offset:offset + vocab]
    for top_k, top_p, min_p in ((0, 0.0, 0.0), (33, 0.0, 0.0),
                                (0, 0.9, 0.0), (600, 0.9, 0.02),
                                (1, 0.0, 0.0)):
        got = sample_tokens(rows, u.cuda(), 0.8, top_k, top_p, min_p)
        want = [sample_exact(wide[i, offset:offset + vocab], float(u[i]),
                             0.8, top_k, top_p, min_p) for i in range(b)]
        assert got.tolist() == want


def test_sample_largest_vocabulary():
    g = generator(27)
    vocab = 1 << 20
    logits = randn(g, 2, vocab) * 2
    u = torch.rand(2, generator=g)
    for top_k, top_p in ((0, 0.0), (0, 0.95), (5000, 0.9), (20, 0.0)):
        got = sample_tokens(logits.cuda(), u.cuda(), top_k=top_k,
                            top_p=top_p)
        want = [sample_exact(logits[i], float(u[i]), 1.0, top_k, top_p, 0.0)
                for i in range(2)]
        assert got.tolist() == want


def test_sample_uniform_outside_still_falls_on_a_kept_token():
    logits = torch.zeros(4, 100)
    logits[:, 20:30] = 5.0
    u = torch.tensor([1.0, 7.0, -1.0, math.nan])
    got = sample_tokens(logits.cuda(), u.cuda(), top_k=10).tolist()
    assert got == [29, 29, 20, 20]


def test_sample_rows_agree_with_themselves_and_empty():
    g = generator(24)
    logits = (randn(g, 1, 40000) * 3).to(BF16).cuda().expand(32, -1)
    u = torch.full((32,), 0.613).cuda()
    for k, p, m in FILTERS:
        got = sample_tokens(logits, u, top_k=k, top_p=p, min_p=m)
        assert (got == got[0]).all()
        again = sample_tokens(logits, u, top_k=k, top_p=p, min_p=m)
        assert torch.equal(got, again)
    assert sample_tokens(logits[:0], u[:0]).shape == (0,)


# ---------------------------------------------------------------------------
# captured, on other streams, together

def decode_step(cache, mixed, cos, sin, start, u, weight, heads, nkv, h):
    q, k, v = mixed.split([heads * h, nkv * h, nkv * h], dim=-1)
    s, b = mixed.shape[:2]
    q = q.view(s, b, heads, h)
    k, v = k.view(s, b, nkv, h), v.view(s, b, nkv, h)
    q = cache.append(k, v, start, query=q, cos=cos, sin=sin,
                     interleaved=False)
    out = cache.attention(q, start, window_size=48, sink_size=2)
    return out, sample_tokens(out[-1] @ weight, u, top_k=30, top_p=0.9,
                              min_p=0.01)


def test_decode_step_captured_replays_as_eager():
    g = generator(31)
    b, heads, nkv, h, length, vocab = 3, 8, 2, 64, 200, 1024
    cos, sin = (t.cuda() for t in precompute_rotary_tables(h, length))
    weight = randn(g, heads * h, vocab, dtype=BF16).cuda()
    prompt = randn(g, 90, b, nkv, h, dtype=BF16).cuda()
    caches = [QuantKVCache(length, b, nkv, h, dtype=BF16, device="cuda")
              for _ in range(2)]
    for c in caches:
        c.append(prompt, prompt, 0)
    steps = [(randn(g, 1, b, (heads + 2 * nkv) * h, dtype=BF16).cuda(),
              torch.rand(b, generator=g).cuda()) for _ in range(6)]
    mixed, u = steps[0][0].clone(), steps[0][1].clone()
    start = torch.tensor([90, 40, 89], device="cuda")
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_step(caches[0], mixed, cos, sin, start, u, weight, heads,
                        nkv, h)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            out, token = decode_step(caches[0], mixed, cos, sin, start, u,
                                     weight, heads, nkv, h)
        at = start.clone()
        for x, y in steps:
            mixed.copy_(x)
            u.copy_(y)
            graph.replay()
            want, drawn = decode_step(caches[1], x, cos, sin, at, y, weight,
                                      heads, nkv, h)
            assert torch.equal(out, want) and torch.equal(token, drawn)
            start.add_(1)
            at.add_(1)
            torch.cuda.synchronize()
    for a, c in zip(caches[0].buffers, caches[1].buffers):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))


def test_two_streams_at_once():
    g = generator(32)
    cache = filled_cache(g, 3000, 2, 2, 128, BF16)
    qs = [randn(g, 1, 2, 8, 128, dtype=BF16).cuda() for _ in range(2)]
    starts = [torch.tensor([2999, 77], device="cuda"),
              torch.tensor([5, 1500], device="cuda")]
    want = [cache.attention(q, s) for q, s in zip(qs, starts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(cache.attention(qs[i], starts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("by", ["top_k", "top_p"])
def test_sample_cuts_at_any_place_of_a_bin(by):
    """Filters that keep more tokens than are listed, with the cut at each of a
    bin's few logits in turn, its largest among them. All tokens weigh the same
    (the temperature is 1e30), so that the last kept index is the one drawn and
    tells the number of kept tokens; each row draws the same in every run."""
    g = generator(40)
    rows, vocab = 700, 4096
    place = torch.stack([torch.randperm(vocab, generator=g)
                         for _ in range(rows)])
    logits = torch.empty(rows, vocab).scatter_(
        1, place, torch.linspace(9.0, -9.0, vocab).expand(rows, vocab))
    kept = 257 + torch.arange(rows)
    if by == "top_k":
        setting = kept
    else:  # before the last kept token lie kept - 1
        setting = (kept - 0.5).float() / vocab
    uniform = torch.full((rows,), 1.0 - 2.0 ** -24)
    among = torch.arange(vocab)[None] < kept[:, None]
    want = place.masked_fill(~among, -1).amax(1)
    for _ in range(5):
        got = sample_tokens(logits.cuda(), uniform.cuda(), temperature=1e30,
                            **{by: setting.cuda()})
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("gap", [16, 22, 26, 30, 33])
def test_attention_small_weights_count(dtype, gap):
    """A token whose value is 0 weighs 2^gap times each other one, whose value
    is 1, all read by one wave: the output is what the others weigh, also where
    a weight is under fp16's least against the largest. A weight is held to
    2^-32 of the wave's largest."""
    h, tokens = 64, 32
    cache = QuantKVCache(tokens, 1, 1, h, dtype=dtype, device="cuda")
    key = torch.zeros(tokens, 1, 1, h, dtype=dtype, device="cuda")
    value = torch.ones_like(key)
    key[5], value[5] = 1.0, 0.0
    cache.append(key, value, 0)
    q = torch.ones(1, 1, 1, h, dtype=dtype, device="cuda")
    got = cache.attention(q, tokens - 1,
                          softmax_scale=gap * math.log(2.0) / h).double()
    least = 31 * 2.0 ** -gap
    want = least / (1 + least)
    # the output's rounding (fp16: its subnormals' too), and each weight's:
    # 2^-11 of itself (2^-22 in two parts), a 32-bit score's of up to 33
    limit = (want * (half_step(dtype) + 2.0 ** -11 + 33 * 2.0 ** -22)
             + 31 * 2.0 ** -32 + (2.0 ** -25 if dtype == FP16 else 0.0))
    assert ((got - want).abs() <= limit).all(), (got.flatten()[0], want)
