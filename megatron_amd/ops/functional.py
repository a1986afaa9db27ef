"""Autograd wrappers over the HIP ops extension, with plain-PyTorch reference
paths for CPU (unit tests / gloo runs).

Dispatch rule: on CUDA (= ROCm/HIP) tensors the extension is REQUIRED — if
_C.so is missing the op raises OpsExtensionMissing rather than silently running
an eager fallback (the round-end harness checks that the native code actually
loads). On CPU tensors the reference implementation runs.

Reference ops replaced (epfLLM/Megatron-LLM):
  fused_softmax.py:9-99, fused_layer_norm.py:26-139, fused_bias_gelu.py:14-43,
  glu_activations.py:8-49, positional_embeddings.py:7-51,
  transformer.py:596-609 (bias_dropout_add), flash-attn (transformer.py:369).
"""

from __future__ import annotations

import math
import torch
from torch.autograd import forward_ad

from . import ext as _ext


def _C(t: torch.Tensor):
    if t.is_cuda:
        return _ext.load(required=True)
    return None


# ---------------------------------------------------------------------------
# RMSNorm

class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ext = _C(x)
        shape = x.shape
        x2d = x.contiguous().view(-1, shape[-1])
        if ext is not None:
            y, invrms = ext.rmsnorm_fwd(x2d, weight, eps)
        else:
            xf = x2d.float()
            invrms = torch.rsqrt(xf.pow(2).mean(-1) + eps)
            y = (xf * invrms.unsqueeze(-1) * weight.float()).to(x.dtype)
        ctx.save_for_backward(x2d, weight, invrms)
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x2d, weight, invrms = ctx.saved_tensors
        shape = dy.shape
        dy2d = dy.contiguous().view(-1, shape[-1])
        ext = _C(dy)
        if ext is not None:
            dx, dw = ext.rmsnorm_bwd(dy2d, x2d, weight, invrms)
        else:
            H = x2d.shape[-1]
            xf = x2d.float()
            gyf = dy2d.float() * weight.float()
            r = invrms.unsqueeze(-1)
            dot = (gyf * xf).sum(-1, keepdim=True)
            dx = (gyf * r - xf * (r ** 3) * dot / H).to(x2d.dtype)
            dw = (dy2d.float() * xf * r).sum(0).to(weight.dtype)
        return dx.view(shape), dw, None


def rmsnorm(x, weight, eps: float = 1e-5):
    return RMSNormFunction.apply(x, weight, eps)


class RMSNormResFunction(torch.autograd.Function):
    """rmsnorm that also passes x through as a second output so the residual
    branch's gradient arrives HERE (instead of an autograd fan-in add) and is
    folded into the norm-backward dx epilogue in-kernel. Replaces the
    2-per-layer eager grad-accumulate adds (reference transformer.py:596-609
    residual stream; measured ~8-12 ms/step at Llama-7B mbs8)."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        ext = _C(x)
        shape = x.shape
        x2d = x.contiguous().view(-1, shape[-1])
        if ext is not None:
            y, invrms = ext.rmsnorm_fwd(x2d, weight, eps)
        else:
            xf = x2d.float()
            invrms = torch.rsqrt(xf.pow(2).mean(-1) + eps)
            y = (xf * invrms.unsqueeze(-1) * weight.float()).to(x.dtype)
        ctx.save_for_backward(x2d, weight, invrms)
        return y.view(shape), x

    @staticmethod
    def backward(ctx, dy, dres):
        x2d, weight, invrms = ctx.saved_tensors
        shape = dy.shape
        dy2d = dy.contiguous().view(-1, shape[-1])
        ext = _C(dy)
        if ext is not None:
            dx, dw = ext.rmsnorm_bwd(dy2d, x2d, weight, invrms,
                                     dres if dres is not None else None)
        else:
            H = x2d.shape[-1]
            xf = x2d.float()
            gyf = dy2d.float() * weight.float()
            r = invrms.unsqueeze(-1)
            dot = (gyf * xf).sum(-1, keepdim=True)
            dx = (gyf * r - xf * (r ** 3) * dot / H).to(x2d.dtype)
            dw = (dy2d.float() * xf * r).sum(0).to(weight.dtype)
            if dres is not None:
                dx = dx + dres.contiguous().view_as(dx)
        return dx.view(shape), dw, None


def rmsnorm_res(x, weight, eps: float = 1e-5):
    return RMSNormResFunction.apply(x, weight, eps)


# ---------------------------------------------------------------------------
# LayerNorm (affine)

class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ext = _C(x)
        shape = x.shape
        x2d = x.contiguous().view(-1, shape[-1])
        if ext is not None:
            y, mean, invvar = ext.layernorm_fwd(x2d, weight, bias, eps)
        else:
            xf = x2d.float()
            mean = xf.mean(-1)
            var = xf.var(-1, unbiased=False)
            invvar = torch.rsqrt(var + eps)
            y = ((xf - mean.unsqueeze(-1)) * invvar.unsqueeze(-1)
                 * weight.float() + bias.float()).to(x.dtype)
        ctx.save_for_backward(x2d, weight, mean, invvar)
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x2d, weight, mean, invvar = ctx.saved_tensors
        shape = dy.shape
        dy2d = dy.contiguous().view(-1, shape[-1])
        ext = _C(dy)
        if ext is not None:
            dx, dw, db = ext.layernorm_bwd(dy2d, x2d, weight, mean, invvar)
        else:
            H = x2d.shape[-1]
            xf = x2d.float()
            xhat = (xf - mean.unsqueeze(-1)) * invvar.unsqueeze(-1)
            g = dy2d.float() * weight.float()
            dx = (g - g.mean(-1, keepdim=True)
                  - xhat * (g * xhat).mean(-1, keepdim=True)) * invvar.unsqueeze(-1)
            dx = dx.to(x2d.dtype)
            dw = (dy2d.float() * xhat).sum(0).to(weight.dtype)
            db = dy2d.float().sum(0).to(weight.dtype)
        return dx.view(shape), dw, db, None


def layernorm(x, weight, bias, eps: float = 1e-5):
    return LayerNormFunction.apply(x, weight, bias, eps)


class LayerNormResFunction(torch.autograd.Function):
    """layernorm twin of RMSNormResFunction (pass-through residual output,
    dres folded into the backward dx epilogue in-kernel)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ext = _C(x)
        shape = x.shape
        x2d = x.contiguous().view(-1, shape[-1])
        if ext is not None:
            y, mean, invvar = ext.layernorm_fwd(x2d, weight, bias, eps)
        else:
            xf = x2d.float()
            mean = xf.mean(-1)
            var = xf.var(-1, unbiased=False)
            invvar = torch.rsqrt(var + eps)
            y = ((xf - mean.unsqueeze(-1)) * invvar.unsqueeze(-1)
                 * weight.float() + bias.float()).to(x.dtype)
        ctx.save_for_backward(x2d, weight, mean, invvar)
        return y.view(shape), x

    @staticmethod
    def backward(ctx, dy, dres):
        x2d, weight, mean, invvar = ctx.saved_tensors
        shape = dy.shape
        dy2d = dy.contiguous().view(-1, shape[-1])
        ext = _C(dy)
        if ext is not None:
            dx, dw, db = ext.layernorm_bwd(dy2d, x2d, weight, mean, invvar,
                                           dres if dres is not None else None)
        else:
            H = x2d.shape[-1]
            xf = x2d.float()
            xhat = (xf - mean.unsqueeze(-1)) * invvar.unsqueeze(-1)
            g = dy2d.float() * weight.float()
            dx = (g - g.mean(-1, keepdim=True)
                  - xhat * (g * xhat).mean(-1, keepdim=True)) * invvar.unsqueeze(-1)
            dx = dx.to(x2d.dtype)
            dw = (dy2d.float() * xhat).sum(0).to(weight.dtype)
            db = dy2d.float().sum(0).to(weight.dtype)
            if dres is not None:
                dx = dx + dres.contiguous().view_as(dx)
        return dx.view(shape), dw, db, None


def layernorm_res(x, weight, bias, eps: float = 1e-5):
    return LayerNormResFunction.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------
# Fused scale + (causal-)mask + softmax, computed in fp32, stored in x.dtype.
# Input (b, np, sq, sk). mask, if given, is additive-style boolean
# (True = masked out), broadcastable (b, 1, sq, sk).

class ScaledMaskedSoftmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mask, scale, causal):
        ext = _C(x)
        if ext is not None:
            y = ext.scaled_masked_softmax_fwd(
                x.contiguous(),
                mask.contiguous() if mask is not None else None,
                float(scale), bool(causal),
            )
        else:
            xf = x.float() * scale
            sq, sk = x.shape[-2], x.shape[-1]
            if causal:
                cm = torch.ones(sq, sk, dtype=torch.bool, device=x.device).triu(
                    sk - sq + 1
                )
                xf = xf.masked_fill(cm, -10000.0)
            if mask is not None:
                xf = xf.masked_fill(mask, -10000.0)
            y = torch.softmax(xf, dim=-1).to(x.dtype)
        ctx.save_for_backward(y)
        ctx.scale = scale
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        ext = _C(dy)
        if ext is not None:
            dx = ext.scaled_masked_softmax_bwd(dy.contiguous(), y, float(ctx.scale))
        else:
            yf = y.float()
            g = dy.float() * yf
            dx = ((g - yf * g.sum(-1, keepdim=True)) * ctx.scale).to(dy.dtype)
        return dx, None, None, None


def scaled_masked_softmax(x, mask=None, scale: float = 1.0, causal: bool = False):
    return ScaledMaskedSoftmax.apply(x, mask, scale, causal)


# ---------------------------------------------------------------------------
# GLU family: y = x1 * act(x2)  with [x1, x2] = chunk(x, 2, dim=-1)
# (reference glu_activations.py:13-15; dense_h_to_4h packs [up; gate] so
#  x1 = up-projection, x2 = gate — y = up * silu(gate) for swiglu)
# act mode: 0 identity (liglu), 1 gelu (geglu), 2 relu (reglu), 3 silu (swiglu)

_ACT_MODES = {"liglu": 0, "geglu": 1, "reglu": 2, "swiglu": 3}


def _act(mode, t):
    if mode == 0:
        return t
    if mode == 1:
        return torch.nn.functional.gelu(t)
    if mode == 2:
        return torch.relu(t)
    return torch.nn.functional.silu(t)


class GLUFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mode):
        ctx.mode = mode
        ctx.save_for_backward(x)
        ext = _C(x)
        if ext is not None:
            shape = x.shape
            x2d = x.contiguous().view(-1, shape[-1])
            y = ext.glu_fwd(x2d, mode)
            return y.view(*shape[:-1], shape[-1] // 2)
        x1, x2 = x.chunk(2, dim=-1)
        return x1 * _act(mode, x2)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        mode = ctx.mode
        ext = _C(dy)
        if ext is not None:
            shape = x.shape
            dx = ext.glu_bwd(dy.contiguous().view(-1, dy.shape[-1]),
                             x.contiguous().view(-1, shape[-1]), mode)
            return dx.view(shape), None
        x1, x2 = x.chunk(2, dim=-1)
        x2d = x2.detach().requires_grad_(True)
        with torch.enable_grad():
            a = _act(mode, x2d)
        dx1 = dy * a
        da = dy * x1
        if mode == 0:
            dx2 = da
        else:
            (dx2,) = torch.autograd.grad(a, x2d, grad_outputs=da)
        return torch.cat([dx1, dx2], dim=-1), None


def glu_activation(x, kind: str = "swiglu"):
    return GLUFunction.apply(x, _ACT_MODES[kind])


def swiglu(x):
    return GLUFunction.apply(x, 3)


# ---------------------------------------------------------------------------
# Rotary embedding (interleaved complex pairs, fp32 math — reference
# positional_embeddings.py:27-51). x: (s, b, np, hn); freqs_cis given as
# cos/sin (s, hn/2) fp32 (already position-selected/scaled).

class RoPEFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        ctx.save_for_backward(cos, sin)
        ext = _C(x)
        if ext is not None:
            # kernel reads strided views (dense head_dim) directly
            if x.stride(-1) != 1:
                x = x.contiguous()
            return ext.rope_fwd(x, cos, sin)
        xf = x.float()
        x1 = xf[..., 0::2]
        x2 = xf[..., 1::2]
        c = cos.view(cos.shape[0], 1, 1, -1)
        s = sin.view(sin.shape[0], 1, 1, -1)
        o1 = x1 * c - x2 * s
        o2 = x2 * c + x1 * s
        out = torch.stack([o1, o2], dim=-1).flatten(-2)
        return out.to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        cos, sin = ctx.saved_tensors
        ext = _C(dy)
        if ext is not None:
            if dy.stride(-1) != 1:
                dy = dy.contiguous()
            return ext.rope_bwd(dy, cos, sin), None, None
        dyf = dy.float()
        g1 = dyf[..., 0::2]
        g2 = dyf[..., 1::2]
        c = cos.view(cos.shape[0], 1, 1, -1)
        s = sin.view(sin.shape[0], 1, 1, -1)
        d1 = g1 * c + g2 * s
        d2 = g2 * c - g1 * s
        dx = torch.stack([d1, d2], dim=-1).flatten(-2)
        return dx.to(dy.dtype), None, None


def apply_rope(x, cos, sin):
    return RoPEFunction.apply(x, cos, sin)


# ---------------------------------------------------------------------------
# Rotary embedding in any layout: interleaved or half pairs, part of the head,
# a position per token, query and key in one launch (csrc/rotary.hip).

def rotate_reference(x, cos, sin, interleaved):
    """x [s, b, n, h] turned by cos, sin [s, b or 1, r] in their own type,
    rounded once; values past 2r are left as they are."""
    r = cos.shape[-1]
    c, s = cos.unsqueeze(2), sin.unsqueeze(2)
    t, rest = x[..., : 2 * r].to(cos.dtype), x[..., 2 * r:]
    if interleaved:
        x1, x2 = t[..., 0::2], t[..., 1::2]
        y = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).flatten(-2)
    else:
        x1, x2 = t[..., :r], t[..., r:]
        y = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
    return torch.cat([y.to(x.dtype), rest], dim=-1)


def _rotate_pair(query, key, cos, sin, positions, interleaved, inverse):
    """query and key (either may be None) turned, or turned back."""
    ext = _C(cos)
    if ext is not None:
        # the kernel reads strided views with a dense head_dim
        if query is not None and query.stride(-1) != 1:
            query = query.contiguous()
        if key is not None and key.stride(-1) != 1:
            key = key.contiguous()
        first, second = (key, None) if query is None else (query, key)
        out = ext.rotary_apply(first, second, cos, sin, positions,
                               interleaved, inverse)
        if query is None:
            return None, out[0]
        return out[0], (out[1] if key is not None else None)
    if positions is None:
        s = (query if query is not None else key).shape[0]
        c, s = (t[:s].unsqueeze(1) for t in (cos, sin))
    else:
        c, s = (t[positions.t()] for t in (cos, sin))
    if inverse:
        s = -s
    return tuple(None if t is None else rotate_reference(t, c, s, interleaved)
                 for t in (query, key))


_ROTARY_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _has_tangent(*tensors):
    """Whether one of them is dual in forward-mode differentiation."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # none can be: cheap
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None
               for t in tensors)


def _turn(query, key, cos, sin, positions, interleaved, inverse, tracked):
    """As _rotate_pair, by an autograd node where something asks for one."""
    turn = (RotaryForwardFunction.apply if _has_tangent(query, key)
            else RotaryFunction.apply if tracked else _rotate_pair)
    return turn(query, key, cos, sin, positions, interleaved, inverse)


class RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, cos, sin, positions, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.mode = (interleaved, inverse)
        ctx.set_materialize_grads(False)
        return _rotate_pair(query, key, cos, sin, positions, interleaved,
                            inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        # the transpose of the rotation: the same with the angle negated
        if dq is not None or dk is not None:
            cos, sin, positions = ctx.saved_tensors
            interleaved, inverse = ctx.mode
            dq, dk = _turn(dq, dk, cos, sin, positions, interleaved,
                           not inverse, torch.is_grad_enabled())
        return dq, dk, None, None, None, None, None


class RotaryForwardFunction(RotaryFunction):
    """With forward-mode derivatives, also under torch.func. A node of its own:
    one whose context is set up apart costs the host 40 us more a call."""

    @staticmethod
    def forward(query, key, cos, sin, positions, interleaved, inverse):
        return _rotate_pair(query, key, cos, sin, positions, interleaved,
                            inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, _, cos, sin, positions, *ctx.mode = inputs
        ctx.save_for_backward(cos, sin, positions)
        ctx.save_for_forward(cos, sin, positions)
        ctx.set_materialize_grads(False)
        ctx.like = [None if y is None else (y.shape, y.dtype, y.device)
                    for y in output]

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # linear: tangents turn as their tensors do. Every output needs one.
        tangents = [
            t if t is not None or like is None
            else torch.zeros(like[0], dtype=like[1], device=like[2])
            for t, like in zip((tq, tk), ctx.like)]
        return RotaryForwardFunction.apply(*tangents, *ctx.saved_tensors,
                                           *ctx.mode)


def rotary_embedding(query, key, cos, sin, positions=None, interleaved=True):
    """Rotate query [s, b, n, h] and key [s, b, nkv, h] (or None) by their
    tokens' positions; returns both.

    cos, sin: fp32 [S, r] with r <= h / 2, from precompute_rotary_tables
    (models/rope.py): the first 2r values of a head are rotated, the others
    pass through. positions: int64 [b, s], rows of the tables; None means
    0..s-1 in every sequence. interleaved: pairs are (2j, 2j + 1), else
    (j, j + r). Positions outside the tables are refused on the CPU and give
    NaN on the GPU. Differentiable in query and key, backward and forward."""
    shape = query.shape
    if len(shape) != 4:
        raise ValueError("query must be [s, b, heads, head_dim]")
    s, b, _, h = shape
    dtype, device = query.dtype, query.device
    if dtype not in _ROTARY_TYPES:
        raise ValueError(f"rotary_embedding takes fp32, bf16 or fp16, not "
                         f"{dtype}")
    if key is not None:
        of_key = key.shape
        if (len(of_key) != 4 or of_key[0] != s or of_key[1] != b
                or of_key[3] != h or key.dtype != dtype
                or key.device != device):
            raise ValueError("key must match the query but for its heads")
    table = cos.shape
    rows, r = table if len(table) == 2 else (0, 0)
    if (not 1 <= r <= h // 2 or sin.shape != table
            or cos.dtype != torch.float32 or sin.dtype != torch.float32
            or cos.device != device or sin.device != device):
        raise ValueError("cos and sin must be float32 [positions, up to "
                         f"{h // 2}] on {device}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("cos and sin have no gradient")
    if positions is None:
        if rows < s:
            raise ValueError(f"tables of {rows} positions for {s} tokens")
    else:
        if (positions.shape != (b, s) or positions.dtype != torch.int64
                or positions.device != device):
            raise ValueError(f"positions must be int64 [{b}, {s}] on "
                             f"{device}")
        if not positions.is_cuda and positions.numel() and (
                int(positions.min()) < 0 or int(positions.max()) >= rows):
            raise ValueError("a position lies outside the tables")
    cos, sin = cos.contiguous(), sin.contiguous()
    tracked = torch.is_grad_enabled() and (
        query.requires_grad or (key is not None and key.requires_grad))
    return _turn(query, key, cos, sin, positions, interleaved, False, tracked)


# ---------------------------------------------------------------------------
# bias + dropout + residual add (reference transformer.py:596-609)

class BiasDropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, residual, p, training):
        ext = _C(x)
        ctx.p = p
        ctx.training = training
        ctx.has_bias = bias is not None
        if not training or p == 0.0:
            y = x + bias + residual if bias is not None else x + residual
            ctx.save_for_backward(torch.tensor([]))
            ctx.no_drop = True
            return y
        ctx.no_drop = False
        if ext is not None:
            seed, offset = _philox_seed(x)
            y, mask = ext.bias_dropout_add_fwd(
                x.contiguous(),
                bias.contiguous() if bias is not None else None,
                residual.contiguous(), float(p), int(seed), int(offset))
            ctx.save_for_backward(mask)
            return y
        z = x + bias if bias is not None else x
        mask = (torch.rand_like(z, dtype=torch.float32) >= p)
        y = z * mask.to(z.dtype) / (1.0 - p) + residual
        ctx.save_for_backward(mask)
        return y

    @staticmethod
    def backward(ctx, dy):
        if ctx.no_drop:
            dx = dy
        else:
            (mask,) = ctx.saved_tensors
            ext = _C(dy)
            if ext is not None:
                dx = ext.dropout_bwd(dy.contiguous(), mask, float(ctx.p))
            else:
                dx = dy * mask.to(dy.dtype) / (1.0 - ctx.p)
        dbias = None
        if ctx.has_bias:
            dbias = dx.reshape(-1, dx.shape[-1]).sum(0)
        return dx, dbias, dy, None, None


def _philox_seed(x):
    gen = torch.cuda.default_generators[x.device.index]
    state = gen.get_state()
    # consume; use torch's philox offset protocol
    seed = gen.initial_seed()
    offset = int(state[-8:].view(torch.int64).item()) if state.numel() >= 8 else 0
    # advance the generator offset by a chunk
    try:
        gen.set_offset(gen.get_offset() + ((x.numel() + 255) // 256) * 4)
        offset = gen.get_offset()
    except Exception:
        offset += x.numel()
    return seed, offset


def bias_dropout_add(x, bias, residual, p, training):
    return BiasDropoutAdd.apply(x, bias, residual, p, training)


# ---------------------------------------------------------------------------
# Flash attention (CDNA4 kernel; CPU reference = plain softmax attention)
# q,k,v: (b, s, n, h) bf16/fp16.  GQA: k/v have n_kv heads, n % n_kv == 0.

class FlashAttnFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, softmax_scale, window_size, dropout_p,
                training):
        ext = _C(q)
        use_drop = bool(training and dropout_p and dropout_p > 0.0)
        if softmax_scale is None:
            softmax_scale = 1.0 / math.sqrt(q.shape[-1])
        ctx.causal = causal
        ctx.softmax_scale = softmax_scale
        ctx.window_size = window_size
        # philox-in-kernel attention dropout on the P strip, regenerated
        # bit-exactly in backward (reference transformer.py:544 dropout via
        # flash-attn)
        ctx.dropout_p = float(dropout_p) if use_drop else 0.0
        ctx.drop_seed = 0
        ctx.drop_offset = 0
        if use_drop:
            if q.is_cuda:
                gen = torch.cuda.default_generators[q.device.index]
                ctx.drop_seed = gen.initial_seed()
                try:
                    ctx.drop_offset = gen.get_offset()
                    gen.set_offset(ctx.drop_offset + 4)
                except Exception:
                    ctx.drop_offset = int(
                        torch.randint(0, 2**31, (1,)).item()
                    )
            else:
                ctx.drop_seed = torch.initial_seed() & (2**63 - 1)
                ctx.drop_offset = int(torch.randint(0, 2**31, (1,)).item())
        if ext is not None:
            # kernels are stride-aware over batch/seq/head (head_dim must be
            # dense, strides 16B-aligned): sbhd transposes and QKV-projection
            # head slices pass with no copy
            def ok(t):
                return t.stride(-1) == 1 and all(
                    t.stride(i) % 8 == 0 for i in range(3)
                )

            q = q if ok(q) else q.contiguous()
            k = k if ok(k) else k.contiguous()
            v = v if ok(v) else v.contiguous()
            out, lse = ext.flash_attn_fwd(
                q, k, v,
                bool(causal), float(softmax_scale),
                int(window_size) if window_size is not None else -1,
                ctx.dropout_p, ctx.drop_seed, ctx.drop_offset,
            )
            ctx.save_for_backward(q, k, v, out, lse)
            return out
        out, lse = _sdpa_reference(
            q, k, v, causal, softmax_scale, window_size,
            dropout_p=ctx.dropout_p, drop_seed=ctx.drop_seed,
            drop_offset=ctx.drop_offset,
        )
        ctx.save_for_backward(q, k, v, out, lse)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        ext = _C(dout)
        if ext is not None:
            if not (dout.stride(-1) == 1
                    and all(dout.stride(i) % 8 == 0 for i in range(3))):
                dout = dout.contiguous()
            dq, dk, dv = ext.flash_attn_bwd(
                dout, q, k, v, out, lse,
                bool(ctx.causal), float(ctx.softmax_scale),
                int(ctx.window_size) if ctx.window_size is not None else -1,
                ctx.dropout_p, ctx.drop_seed, ctx.drop_offset,
            )
            return dq, dk, dv, None, None, None, None, None
        dq, dk, dv = _sdpa_reference_bwd(
            dout, q, k, v, out, lse, ctx.causal, ctx.softmax_scale,
            ctx.window_size, dropout_p=ctx.dropout_p,
            drop_seed=ctx.drop_seed, drop_offset=ctx.drop_offset,
        )
        return dq, dk, dv, None, None, None, None, None


def _attn_mask(sq, sk, causal, window_size, device):
    m = torch.zeros(sq, sk, dtype=torch.bool, device=device)
    if causal:
        m |= torch.ones(sq, sk, dtype=torch.bool, device=device).triu(sk - sq + 1)
    if window_size is not None and window_size > 0:
        # Sliding-window convention (canonical here = HF/Mistral): each query
        # attends to exactly `window_size` keys INCLUDING itself, i.e. keys
        # with q_idx - window_size + 1 <= k_idx <= q_idx. Note the reference
        # passes window_size=(w, w) to flash-attn, which keeps w+1 keys — a
        # deliberate one-key departure, documented in PARITY.md; Mistral
        # checkpoints are trained with the HF convention.
        q_idx = torch.arange(sq, device=device).unsqueeze(1) + (sk - sq)
        k_idx = torch.arange(sk, device=device).unsqueeze(0)
        m |= k_idx < (q_idx - window_size + 1)
    return m


def _drop_keep_mask(bsz, heads, sq, sk, dropout_p, drop_seed, drop_offset,
                    device):
    """[b, n, sq, sk] bool keep-mask, bit-exact vs the HIP kernels."""
    import numpy as np

    from .philox_ref import attn_dropout_mask

    m = np.stack([
        np.stack([
            attn_dropout_mask(drop_seed, drop_offset, b, h, heads, sq, sk,
                              dropout_p)
            for h in range(heads)
        ])
        for b in range(bsz)
    ])
    return torch.from_numpy(m).to(device)


def _sdpa_reference(q, k, v, causal, scale, window_size, dropout_p=0.0,
                    drop_seed=0, drop_offset=0):
    b, sq, n, h = q.shape
    n_kv = k.shape[2]
    rep = n // n_kv
    qf = q.float().permute(0, 2, 1, 3)  # b n s h
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    scores = torch.matmul(qf, kf.transpose(-2, -1)) * scale
    mask = _attn_mask(sq, k.shape[1], causal, window_size, q.device)
    scores = scores.masked_fill(mask, float("-inf"))
    lse = torch.logsumexp(scores, dim=-1)  # b n s
    p = torch.softmax(scores, dim=-1)
    if dropout_p and dropout_p > 0.0:
        keep = _drop_keep_mask(b, n, sq, k.shape[1], dropout_p, drop_seed,
                               drop_offset, q.device)
        p = p * keep.to(p.dtype) / (1.0 - dropout_p)
    of = torch.matmul(p, vf)
    return of.permute(0, 2, 1, 3).to(q.dtype), lse


def _sdpa_reference_bwd(dout, q, k, v, out, lse, causal, scale, window_size,
                        dropout_p=0.0, drop_seed=0, drop_offset=0):
    b, sq, n, h = q.shape
    n_kv = k.shape[2]
    rep = n // n_kv
    qf = q.float().permute(0, 2, 1, 3).requires_grad_(True)
    kf = k.float().permute(0, 2, 1, 3).requires_grad_(True)
    vf = v.float().permute(0, 2, 1, 3).requires_grad_(True)
    with torch.enable_grad():
        kr = kf.repeat_interleave(rep, dim=1)
        vr = vf.repeat_interleave(rep, dim=1)
        scores = torch.matmul(qf, kr.transpose(-2, -1)) * scale
        mask = _attn_mask(sq, k.shape[1], causal, window_size, q.device)
        scores = scores.masked_fill(mask, float("-inf"))
        p = torch.softmax(scores, dim=-1)
        if dropout_p and dropout_p > 0.0:
            keep = _drop_keep_mask(b, n, sq, k.shape[1], dropout_p,
                                   drop_seed, drop_offset, q.device)
            p = p * keep.to(p.dtype) / (1.0 - dropout_p)
        of = torch.matmul(p, vr)
    df = dout.float().permute(0, 2, 1, 3)
    dq, dk, dv = torch.autograd.grad(of, (qf, kf, vf), grad_outputs=df)
    return (
        dq.permute(0, 2, 1, 3).to(q.dtype),
        dk.permute(0, 2, 1, 3).to(k.dtype),
        dv.permute(0, 2, 1, 3).to(v.dtype),
    )


def flash_attention(q, k, v, causal=True, softmax_scale=None, window_size=None,
                    dropout_p=0.0, training=False):
    return FlashAttnFunction.apply(
        q, k, v, causal, softmax_scale, window_size, dropout_p, training
    )


class FusedQKVSplitRope(torch.autograd.Function):
    """Split the fused QKV projection output [s,b,g,(nq+2)h] into q/k/v and
    rotate q/k, assembling d_mixed in ONE buffer in the backward.

    Plain autograd slicing costs 3 zeros-fills + 3 copies + 2 full-size adds
    per layer in the backward (narrow-backward per slice, then fan-in sums);
    here the stride-aware RoPE kernel writes d(q)/d(k) straight into the
    corresponding regions of d_mixed and d(v) is one strided copy. q/k are
    read as strided views (no forward copies). v is deliberately returned as
    a strided VIEW of the input (saves a full copy, ~2 GB at seq 32k);
    autograd tracks it as a view output, so any in-place write to v
    downstream raises loudly rather than corrupting gradients — all
    consumers (FA kernel, CoreAttention, KV-cache fill) only read it.
    """

    @staticmethod
    def forward(ctx, mixed, cos, sin, np_, nkv, hn):
        ext = _C(mixed)
        sq, b, g, _ = mixed.shape
        nq = np_ // nkv
        q = mixed[..., : nq * hn]
        if nq > 1:
            q = q.reshape(sq, b, np_, hn)
        k = mixed[..., nq * hn : (nq + 1) * hn]
        v = mixed[..., (nq + 1) * hn :]
        if cos is not None:
            q_rot = ext.rope_fwd(q, cos, sin)
            k_rot = ext.rope_fwd(k, cos, sin)
        else:
            q_rot = q.contiguous()
            k_rot = k.contiguous()
        ctx.save_for_backward(cos, sin) if cos is not None else ctx.save_for_backward()
        ctx.dims = (sq, b, g, nq, hn, np_, nkv, cos is not None)
        # v is returned as a strided VIEW of the input (no copy, no extra
        # memory — ~2 GB at seq 32k); autograd tracks it as a view output
        return q_rot, k_rot, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        ext = _C(dq)
        sq, b, g, nq, hn, np_, nkv, have_rope = ctx.dims
        d_mixed = torch.empty(sq, b, g, (nq + 2) * hn, dtype=dq.dtype,
                              device=dq.device)
        dq_slice = d_mixed[..., : nq * hn]
        dk_slice = d_mixed[..., nq * hn : (nq + 1) * hn]
        dv_slice = d_mixed[..., (nq + 1) * hn :]
        if have_rope:
            cos, sin = ctx.saved_tensors
            if nq == 1:
                ext.rope_bwd_into(dq.contiguous(), cos, sin, dq_slice)
            else:
                # GQA q region is not uniformly strided over heads: rotate
                # densely, then one strided copy (5-D view splits the dense
                # nq*hn run of each group)
                dq_slice.view(sq, b, g, nq, hn).copy_(
                    ext.rope_bwd(dq.contiguous(), cos, sin).view(
                        sq, b, g, nq, hn
                    )
                )
            ext.rope_bwd_into(dk.contiguous(), cos, sin, dk_slice)
        else:
            dq_slice.view(sq, b, g, nq, hn).copy_(
                dq.reshape(sq, b, g, nq, hn)
            )
            dk_slice.copy_(dk)
        dv_slice.copy_(dv)
        return d_mixed, None, None, None, None, None


def fused_qkv_split_rope(mixed, cos, sin, np_, nkv, hn):
    return FusedQKVSplitRope.apply(mixed, cos, sin, np_, nkv, hn)


# ---------------------------------------------------------------------------
# Next tokens from filtered logits and given uniform numbers
# (csrc/sample.hip).

def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=0.0,
                  min_p=0.0):
    """Draw one token per row of logits [b, v]; int64 [b].

    uniform: float32 [b] in [0, 1). The settings are numbers, or tensors [b]
    for a setting per row (float32; top_k int64). Tokens are ordered by logit,
    equal ones by index. Of the weights exp((x - max) / temperature), top_k
    keeps the first k tokens (0: all), top_p of those each whose predecessors
    weigh at most top_p of them all (0 or 1: all), min_p those that weigh at
    least min_p times the largest. The token drawn is the first index whose
    kept weights up to it exceed uniform times all kept weights. temperature 0
    takes the largest logit, the lowest index of equal ones.

    A row with a NaN, or without a logit above -inf, gives -1."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [b, vocabulary]")
    b, v = logits.shape
    if v > 1 << 20:
        raise ValueError("at most 2^20 tokens")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"sample_tokens takes fp32, bf16 or fp16, not "
                         f"{logits.dtype}")
    settings = dict(uniform=uniform, temperature=temperature, top_k=top_k,
                    top_p=top_p, min_p=min_p)
    rows, numbers = {}, {}
    for name, x in settings.items():
        want = torch.int64 if name == "top_k" else torch.float32
        if isinstance(x, torch.Tensor):
            if (x.shape != (b,) or x.dtype != want
                    or x.device != logits.device):
                raise ValueError(f"{name} must be a number or a {want} "
                                 f"tensor [{b}] on {logits.device}")
            rows[name], numbers[name] = x.contiguous(), 0
        elif name == "uniform":
            raise ValueError("uniform must be a tensor")
        else:
            rows[name] = None
            numbers[name] = int(x) if name == "top_k" else float(x)
    if not 0.0 <= numbers["temperature"] < math.inf:
        raise ValueError("temperature must be finite and not negative")
    if numbers["top_k"] < 0:
        raise ValueError("top_k must not be negative")
    for name in ("top_p", "min_p"):
        if not 0.0 <= numbers[name] <= 1.0:
            raise ValueError(f"{name} must be in 0..1")
    if logits.requires_grad and torch.is_grad_enabled():
        logits = logits.detach()  # a drawn token has no gradient
    ext = _C(logits)
    if ext is not None:
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        return ext.sample_tokens(
            logits, rows["uniform"], rows["temperature"], rows["top_k"],
            rows["top_p"], rows["min_p"], numbers["temperature"],
            numbers["top_k"], numbers["top_p"], numbers["min_p"])

    def setting(name):
        if rows[name] is not None:
            return rows[name].double()[:, None]
        return torch.full((b, 1), numbers[name], dtype=torch.float64)

    return _sample_reference(logits.double(), *(
        setting(x) for x in ("temperature", "top_k", "top_p", "min_p")),
        uniform.double()[:, None])


def _sample_reference(x, temperature, top_k, top_p, min_p, uniform):
    top = x.amax(-1, keepdim=True)
    greedy = ~(temperature > 0)
    top_k = torch.where(greedy, torch.ones_like(top_k), top_k)
    temperature = torch.where(greedy, torch.ones_like(temperature),
                              temperature).clamp(max=1e30)
    weight = torch.where(x == top, torch.ones_like(x),
                         ((x - top) / temperature).exp())
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ranked = weight.gather(-1, order)
    rank = torch.arange(x.shape[-1], device=x.device)
    keep = (rank < top_k) | (top_k <= 0)
    ranked = ranked * keep
    before = ranked.cumsum(-1) - ranked
    keep &= ((before <= top_p * ranked.sum(-1, keepdim=True))
             | ~((top_p > 0) & (top_p < 1)))
    keep &= ~(ranked < min_p.clamp(max=1.0))
    kept = torch.zeros_like(keep).scatter(-1, order, keep)
    upto = (weight * kept).cumsum(-1)
    total = upto[:, -1:]
    target = torch.minimum(uniform * total, total * (1 - 2.0 ** -53))
    token = (upto <= target).sum(-1)
    # uniform numbers outside 0..1 still fall on a kept token
    index = torch.arange(x.shape[-1], device=x.device)
    some = kept & (weight > 0)
    last = torch.where(some, index, torch.full_like(index, -1)).amax(-1)
    first = torch.where(some, index,
                        torch.full_like(index, x.shape[-1])).amin(-1)
    token = torch.maximum(torch.minimum(token, last), first)
    void = x.isnan().any(-1) | (top[:, 0] == float("-inf"))
    return torch.where(void, torch.full_like(token, -1), token)
