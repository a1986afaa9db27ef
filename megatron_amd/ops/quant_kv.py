"""Key/value cache of one attention layer held in 4 bits (5 with the scales):
append, read-back and attention over it.

On the GPU everything runs in csrc/quant_kv.hip; on the CPU the same layout is
filled and read with plain torch operations.

What is held: groups of 32 values of a head share a zero point z = fp16(min)
and a scale s = fp16((max - z) / 15); a value is held as the nearest code 0..15
(ties to even) and stands for z + s * code. Magnitudes above 57344 are held as
that. A token whose key or value holds a NaN in some head makes every query of
that head that sees it NaN, and no other query.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import ext as _ext
from .functional import _has_tangent, rotate_reference

GROUP = 32
HELD_MAX = 57344.0
HEAD_DIMS = (32, 64, 128, 256)
_ROOM = 64  # buffers hold a multiple of this many tokens


def _round_up(n: int, to: int) -> int:
    return (n + to - 1) // to * to


class QuantKVCache:
    """Static cache of `max_sequence_len` tokens for `batch_size` sequences.

    Keys and values come as [s, b, heads, head_dim] in `dtype` (bf16 or fp16),
    `start` tells at which position a sequence's first token goes: an int, or
    an int64 tensor with 1 or `batch_size` elements on the cache's device,
    which a captured graph may change between replays. A negative start marks
    an idle sequence: nothing is written for it and its attention gives zeros.
    Tokens at or behind `max_sequence_len` are refused where the host can see
    them (an int start, or the CPU); on the GPU they are not written, and read
    back or attended from they give NaN.

    The object keeps nothing from call to call but the buffers, which are
    written in place. Calls that write and calls that read the same positions
    have to be ordered by the caller's streams."""

    def __init__(self, max_sequence_len: int, batch_size: int,
                 num_heads_kv: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, "
                             f"not {head_dim}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a 4-bit cache takes bf16 or fp16, not {dtype}")
        if min(max_sequence_len, batch_size, num_heads_kv) < 1:
            raise ValueError("max_sequence_len, batch_size and num_heads_kv "
                             "must be positive")
        self.max_sequence_len = max_sequence_len
        self.batch_size = batch_size
        self.num_heads_kv = num_heads_kv
        self.head_dim = head_dim
        self.dtype = dtype
        room = _round_up(max_sequence_len, _ROOM)
        heads = (batch_size, num_heads_kv)
        groups = head_dim // GROUP
        self._quarters = max(1, head_dim // 64)
        self.k_codes = torch.zeros(*heads, room, head_dim // 2,
                                   dtype=torch.uint8, device=device)
        self.k_meta = torch.zeros(*heads, room, groups, 2,
                                  dtype=torch.float16, device=device)
        self.v_codes = torch.zeros(*heads, room // 4, 128 * self._quarters,
                                   dtype=torch.uint8, device=device)
        self.v_meta = torch.zeros(*heads, groups, room // 4, 2, 4,
                                  dtype=torch.float16, device=device)

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def buffers(self):
        return [self.k_codes, self.k_meta, self.v_codes, self.v_meta]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.buffers)

    # -- argument checks ----------------------------------------------------

    # (on the way of each layer's decode step: attributes are read once)

    def _check_rows(self, x, name, device, heads=None):
        shape = x.shape
        if (len(shape) != 4 or shape[1] != self.batch_size
                or shape[3] != self.head_dim):
            raise ValueError(
                f"{name} must be [s, {self.batch_size}, heads, "
                f"{self.head_dim}], not {tuple(shape)}")
        if heads is not None and shape[2] != heads:
            raise ValueError(f"{name} must have {heads} heads, "
                             f"not {shape[2]}")
        if x.dtype != self.dtype or x.device != device:
            raise ValueError(
                f"{name} must be {self.dtype} on {device}, "
                f"not {x.dtype} on {x.device}")
        return x if x.stride(3) == 1 else x.contiguous()

    def _check_start(self, start, s,
                     device) -> Tuple[Optional[torch.Tensor], int]:
        if isinstance(start, torch.Tensor):
            shape = start.shape
            if (len(shape) != 1 or shape[0] not in (1, self.batch_size)
                    or start.dtype != torch.int64 or start.device != device):
                raise ValueError(
                    "start must be an int or an int64 tensor with 1 or "
                    f"{self.batch_size} elements on {device}")
            if not start.is_cuda and start.numel():
                if int(start.max()) + s > self.max_sequence_len:
                    raise ValueError(
                        f"start {int(start.max())} + {s} tokens exceed the "
                        f"cache's {self.max_sequence_len}")
            return start, 0
        start = int(start)
        if start + s > self.max_sequence_len:
            raise ValueError(f"start {start} + {s} tokens exceed the cache's "
                             f"{self.max_sequence_len}")
        return None, start

    @staticmethod
    def _check_no_grad(*tensors):
        if torch.is_grad_enabled() and any(
                t is not None and t.requires_grad for t in tensors):
            raise ValueError("the 4-bit cache has no gradient: call it under "
                             "torch.no_grad()")
        if _has_tangent(*tensors):
            raise ValueError("the 4-bit cache has no forward-mode derivative")

    # -- operations -----------------------------------------------------------

    def append(self, key: torch.Tensor, value: torch.Tensor,
               start: Union[int, torch.Tensor],
               query: Optional[torch.Tensor] = None,
               cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None,
               interleaved: bool = True) -> Optional[torch.Tensor]:
        """Hold `key` and `value` from position `start` on.

        With `query`, `cos` and `sin` (the decode step) query and key are
        rotated first, by the tables' rows at the tokens' positions as in
        rotary_embedding, and the rotated query is returned; an idle
        sequence's is zero. The key is rounded to its type between rotation
        and quantization."""
        if (query is None) != (cos is None) or (cos is None) != (sin is None):
            raise ValueError("query, cos and sin come together")
        self._check_no_grad(key, value, query)
        device = self.device
        key = self._check_rows(key, "key", device, self.num_heads_kv)
        value = self._check_rows(value, "value", device, self.num_heads_kv)
        s = key.shape[0]
        if value.shape[0] != s:
            raise ValueError("key and value must have the same shape")
        at, at_s = self._check_start(start, s, device)
        if query is not None:
            query = self._check_rows(query, "query", device)
            if query.shape[0] != s:
                raise ValueError("query and key must have as many tokens")
            _check_tables(cos, sin, self.head_dim, device)
        if device.type == "cuda":
            return _ext.load(required=True).quant_kv_append(
                self.buffers, self.max_sequence_len, key, value, at, at_s,
                query, cos, sin, interleaved)
        return self._append_reference(key, value, at, at_s, query, cos, sin,
                                      interleaved)

    def dequantize(self, start: Union[int, torch.Tensor] = 0,
                   length: Optional[int] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
        """What is held at `length` positions from `start` on (default: all):
        keys and values [length, b, heads, head_dim] in the cache's dtype."""
        if length is None:
            if isinstance(start, torch.Tensor):
                raise ValueError("a tensor start needs a length")
            length = self.max_sequence_len - int(start)
        if length < 0:
            raise ValueError("length must not be negative")
        device = self.device
        at, at_s = self._check_start(start, length, device)
        if device.type == "cuda":
            return tuple(_ext.load(required=True).quant_kv_dequantize(
                self.buffers, self.max_sequence_len, at, at_s, length,
                self.dtype == torch.bfloat16))
        pos = self._positions(at, at_s, length)
        out = []
        for held in self._held(pos.clamp(min=0)):
            held = held.masked_fill((pos < 0)[..., None, None], math.nan)
            out.append(held.transpose(0, 1).to(self.dtype).contiguous())
        return tuple(out)

    def attention(self, query: torch.Tensor, start: Union[int, torch.Tensor],
                  softmax_scale: Optional[float] = None,
                  window_size: Optional[int] = None,
                  sink_size: int = 0) -> torch.Tensor:
        """Causal attention of `query` [s, b, heads, head_dim] over what is
        held; heads must be a multiple of the cache's. Token i of a sequence
        stands at position start + i, has to be appended already, and sees the
        positions up to its own: with `window_size` w the last w of them, its
        own among them, and the first `sink_size`. Returns
        [s, b, heads * head_dim].

        On the GPU held keys and values and the softmax's weights are operands
        in fp16 and sums in 32 bits; in an fp16 cache what the operands'
        rounding left out is added."""
        self._check_no_grad(query)
        device = self.device
        query = self._check_rows(query, "query", device)
        s, b, n, h = query.shape
        if n < 1 or n % self.num_heads_kv:
            raise ValueError(f"{n} query heads are no multiple of "
                             f"{self.num_heads_kv} key heads")
        if window_size is not None and window_size < 1:
            raise ValueError("window_size must be positive, or None")
        if sink_size < 0:
            raise ValueError("sink_size must not be negative")
        if sink_size and window_size is None:
            raise ValueError("sink_size needs a window_size")
        at, at_s = self._check_start(start, s, device)
        if softmax_scale is None:
            softmax_scale = 1.0 / math.sqrt(h)
        if not math.isfinite(softmax_scale):
            raise ValueError("softmax_scale must be finite")
        # beyond the cache both mean all of it
        if window_size is not None:
            window_size = min(window_size, self.max_sequence_len)
        sink_size = min(sink_size, self.max_sequence_len)
        if device.type == "cuda":
            return _ext.load(required=True).quant_kv_attention(
                self.buffers, self.max_sequence_len, query, at, at_s,
                float(softmax_scale), window_size or 0, sink_size)
        pos = self._positions(at, at_s, s)  # [b, s]
        length = int(pos.max()) + 1 if pos.numel() else 0
        if length <= 0:
            return query.new_zeros(s, b, n * h)
        everything = torch.arange(length).expand(b, length)
        key, value = (x.permute(0, 2, 1, 3).repeat_interleave(
            n // self.num_heads_kv, dim=1) for x in self._held(everything))
        score = torch.matmul(query.float().permute(1, 2, 0, 3),
                             key.transpose(-2, -1)) * softmax_scale
        seen = everything[:, None] <= pos[..., None]
        if window_size is not None:
            seen &= (everything[:, None] > pos[..., None] - window_size) | (
                everything[:, None] < sink_size)
        seen &= (self._positions(at, at_s, 1) >= 0)[..., None]
        score = score.masked_fill(~seen[:, None], float("-inf"))
        prob = torch.softmax(score, dim=-1)
        prob = prob.masked_fill(~seen[:, None], 0.0)
        # a value that no query may see must not reach one as 0 * NaN; where
        # a query does see a NaN its key's NaN has reached it already
        out = torch.matmul(prob, value.nan_to_num(nan=0.0))
        return out.permute(2, 0, 1, 3).reshape(s, b, n * h).to(self.dtype)

    def reorder(self, batch_idx: torch.Tensor) -> None:
        """Sequence i becomes what sequence batch_idx[i] was (beam search).
        In place: a captured graph keeps its pointers."""
        if batch_idx.dim() != 1 or batch_idx.shape[0] != self.batch_size:
            raise ValueError(f"batch_idx must have {self.batch_size} elements")
        for t in self.buffers:
            t.copy_(t[batch_idx])

    # -- plain torch on the same layout (CPU) --------------------------------

    def _positions(self, at, at_s, s):
        first = at if at is not None else torch.tensor([at_s])
        return (first.expand(self.batch_size)[:, None]
                + torch.arange(s)[None, :])

    def _value_bytes(self, pos):
        """Index in a block of four tokens of each byte of a token's value
        codes: pairs of values, in the order of the values."""
        q = self._quarters
        piece = torch.arange(16 * q)
        chunk, quarter = piece // q, piece % q
        within = pos[..., None] % 4
        half = ((chunk * 2 + within // 2) * q + quarter) * 2 + within % 2
        both = torch.stack([2 * half, 2 * half + 1], -1).flatten(-2)
        return both if self.head_dim >= 64 else both[..., 0::2]

    def _append_reference(self, key, value, at, at_s, query, cos, sin,
                          interleaved):
        s = key.shape[0]
        pos = self._positions(at, at_s, s)
        idle = (pos[:, :1] < 0).expand_as(pos) if s else pos < 0
        rotated = None
        if query is not None:
            if bool((pos[~idle] >= cos.shape[0]).any()):
                raise ValueError("a position exceeds the rotary tables")
            # in 64 bits: the codes hang on the rounded keys
            rows = pos.clamp(min=0).t()
            c, sn = (t[rows].double() for t in (cos, sin))
            key = rotate_reference(key, c, sn, interleaved)
            rotated = rotate_reference(query, c, sn, interleaved)
            rotated = rotated.masked_fill(idle.t()[..., None, None], 0.0)
        rows = torch.arange(self.batch_size)[:, None].expand_as(pos)[~idle]
        pos = pos[~idle]
        k, v = (x.transpose(0, 1)[~idle] for x in (key, value))  # [t, n, h]
        (kc, ks, kz, kn), (vc, vs, vz, vn) = _quantize(k), _quantize(v)
        ks = ks.masked_fill((kn | vn).any(-1, keepdim=True), math.nan)
        vs = vs.masked_fill(vn, math.nan)
        word = kc.unflatten(-1, (-1, 4, 2)).transpose(-2, -1)  # [2, 4] a dword
        word = word.reshape(*word.shape[:-2], 4, 2)
        self.k_codes[rows, :, pos] = (
            word[..., 0] | (word[..., 1] << 4)).flatten(-2)
        self.k_meta[rows, :, pos] = torch.stack([ks, kz], -1)
        self.v_meta[rows, :, :, pos // 4, 0, pos % 4] = vs
        self.v_meta[rows, :, :, pos // 4, 1, pos % 4] = vz
        byte = vc[..., 0::2] | (vc[..., 1::2] << 4)
        where = self._value_bytes(pos)[:, None].expand_as(byte)
        heads = torch.arange(self.num_heads_kv)[None, :, None]
        self.v_codes[rows[:, None, None], heads, (pos // 4)[:, None, None],
                     where] = byte
        return rotated

    def _held(self, pos):
        """Keys and values at positions [b, t]: [b, t, heads, h] fp32."""
        rows = torch.arange(self.batch_size)[:, None].expand_as(pos)
        byte = self.k_codes[rows, :, pos].unflatten(-1, (-1, 4))
        word = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
        code = word.unflatten(-1, (2, 4)).transpose(-2, -1).flatten(-3)
        key = _values(code, *self.k_meta[rows, :, pos].unbind(-1))
        where = self._value_bytes(pos)[:, :, None]
        heads = torch.arange(self.num_heads_kv)[:, None]
        byte = self.v_codes[rows[..., None, None], heads,
                            (pos // 4)[..., None, None], where]
        code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
        scale = self.v_meta[rows, :, :, pos // 4, 0, pos % 4]
        zero = self.v_meta[rows, :, :, pos // 4, 1, pos % 4]
        return key, _values(code, scale, zero)


def _check_tables(cos, sin, head_dim, device):
    shape = cos.shape
    if (len(shape) != 2 or not 1 <= shape[1] <= head_dim // 2
            or sin.shape != shape
            or cos.dtype != torch.float32 or sin.dtype != torch.float32
            or cos.device != device or sin.device != device
            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(
            "cos and sin must be contiguous float32 tables [positions, "
            f"up to {head_dim // 2}] on {device}")


def _quantize(x):
    """[..., h] -> codes, fp16 scale and zero [..., groups], NaN per group."""
    x = x.double().unflatten(-1, (-1, GROUP))
    broken = x.isnan().any(-1)
    x = x.nan_to_num(nan=0.0, posinf=HELD_MAX, neginf=-HELD_MAX)
    x = x.clamp(-HELD_MAX, HELD_MAX)
    zero = x.amin(-1).to(torch.float16)
    above = zero.double()
    scale = ((x.amax(-1) - above) / 15.0).to(torch.float16)
    step = scale.double().unsqueeze(-1)
    code = ((x - above.unsqueeze(-1)) / step.clamp(min=2.0 ** -30)).round()
    code = code.clamp(0, 15).masked_fill(step == 0, 0)
    return code.to(torch.uint8).flatten(-2), scale, zero, broken


def _values(code, scale, zero):
    code = code.float().unflatten(-1, (-1, GROUP))
    return (zero.float().unsqueeze(-1)
            + scale.float().unsqueeze(-1) * code).flatten(-2)
