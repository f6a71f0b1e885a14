"""Generation with keys, values and weights held in 4 bits.

A group of numbers is held as codes 0 .. 15 with the group's lowest value and a step, both of the model's 16-bit type T:

    low = min x,   scale = T((max x - low) / 15),   code = min(15, round_half_even((x - low) / scale))  (0 where scale is 0),   x ~ scale * code + low

so a value is off by at most half a step (and 15 roundings of the step).  A group that holds an infinity or a NaN reads back as NaN, finite numbers as finite ones: where the
rounded step leaves a value above the type's largest number, that number is read back.

* `Int4KVCache`: a dense cache [slots, room, n_kv, hd] with groups of 32 channels of a key (after the rotation a few channels are far larger than the
  others, and a small group keeps them to themselves) and of 64 channels of a value: 4.75 bits a number, 3.4 times less than 16.  `store` quantises the
  keys and values of packed sequences, `load` reads them back, `decode_attention_int4` appends a token and attends to all rows as the cache holds them.
* `Int4Linear`: a weight [N, K] with groups of 32, 64 or 128 along K and its products with rows of any number; made for the few rows of a decode step,
  where the weights' bytes are the time.

None of these has a gradient.  A product or an attention step whose rows, or whose call's bias, would need one is refused; `store`, a weight and the bias that is kept with it are taken
as numbers.

The layout in memory is `csrc/int4.cuh`'s; `Int4KVCache.store`, `.load`, `decode_attention_int4` and `Int4Linear` on CPU tensors are plain PyTorch over the
same layout.  The reference generates in the training dtype only (`realhf/impl/model/nn/real_llm_generate.py`); both are opt-in
(`GenerationHyperparameters.kv_cache_bits`, `.int4_weights`), since what is sampled then is the quantised policy's.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from realhf_b200.ops import lib, use_native

KEY_GROUP, VALUE_GROUP, TILE_ROWS = 32, 64, 16
HEAD_DIMS = (64, 128)
GROUPS = (32, 64, 128)
# Rows up to which a product with a 4-bit weight takes less time than with a 16-bit one (4096 -> 11008: 16 rows 14.8 us against 17.6, 17 rows 23.8 against 17.9; 11008 -> 4096: 14.6
# against 17.7, 18.7 against 18.0; 4096 -> 12288: 17.7 against 19.0, 34.6 against 19.1)
FAST_ROWS = 16
# where channel i of a word's eight has its bits, in a key's, a value's and a weight's word
_KEY, _VALUE, _WEIGHT = [8 * (i & 3) + 4 * (i >> 2) for i in range(8)], [4 * i for i in range(8)], [4 * (i >> 1) + 16 * (i & 1) for i in range(8)]


# ------------------------------------------------------------------------------------------------ groups


def quantize_groups(x: torch.Tensor, group: int, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [..., n] of a 16-bit type (or of fp32, with the type of the steps in `dtype`) -> (codes uint8 [..., n], scale [..., n / group], low): the rule in plain
    PyTorch."""
    dtype = dtype or x.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"4-bit groups: steps are bfloat16 or float16, not {dtype}")
    if group <= 0 or x.shape[-1] % group:
        raise ValueError(f"4-bit groups: {x.shape[-1]} numbers in groups of {group}")
    xg = x.to(dtype).float().unflatten(-1, (-1, group))
    lo, hi = xg.amin(-1), xg.amax(-1)
    # (by 1/16, an exact factor: the widest group of bfloat16 stays inside fp32; a tensor by a tensor is a correctly rounded division)
    scale = ((hi * 0.0625 - lo * 0.0625) / torch.full_like(lo, 0.9375)).to(dtype)
    fine = torch.isfinite(lo) & torch.isfinite(hi)
    scale = torch.where(fine, scale, torch.full_like(scale, float("nan")))
    low = torch.where(fine, lo, torch.full_like(lo, float("nan"))).to(dtype)
    step = scale.float()[..., None]
    c = (xg * 0.0625 - lo[..., None] * 0.0625) / torch.where(step > 0, step * 0.0625, torch.ones_like(step))
    c = torch.where(step > 0, c.round().clamp(max=15), torch.zeros_like(c))
    return c.to(torch.uint8).flatten(-2), scale, low


def dequantize_groups(codes: torch.Tensor, scale: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """fp32 scale * code + low, rounded once."""
    xg = codes.unflatten(-1, (scale.shape[-1], -1)).double()
    return (xg * scale.double()[..., None] + low.double()[..., None]).float().flatten(-2)


def _to_type(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Rounded to the type; finite numbers stay finite (a step that was rounded up can leave 15 steps above the type's largest number)."""
    most = torch.finfo(dtype).max
    return torch.where(torch.isfinite(x), x.clamp(-most, most), x).to(dtype)


def _words(codes: torch.Tensor, shifts) -> torch.Tensor:
    """uint8 [..., 8 n] -> int32 [..., n], channels in order."""
    sh = torch.tensor(shifts, dtype=torch.int64, device=codes.device)
    w = (codes.unflatten(-1, (-1, 8)).long() << sh).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _codes(words: torch.Tensor, shifts) -> torch.Tensor:
    sh = torch.tensor(shifts, dtype=torch.int32, device=words.device)
    return ((words[..., None] >> sh) & 15).to(torch.uint8).flatten(-2)


def _group_words(scale: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    return (scale.view(torch.int16).int() << 16) | (low.view(torch.int16).int() & 0xFFFF)


def _group_numbers(words: torch.Tensor, dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    low = words & 0xFFFF
    return (words >> 16).to(torch.int16).view(dtype), torch.where(low >= 1 << 15, low - (1 << 16), low).to(torch.int16).view(dtype)


def _row_order(words: torch.Tensor) -> torch.Tensor:
    """[..., 4 J] words of a row in the order of the channels -> the order in memory, (t, j) with word 4 j + t."""
    return words.unflatten(-1, (-1, 4)).transpose(-1, -2).flatten(-2)


def _channel_order(words: torch.Tensor) -> torch.Tensor:
    return words.unflatten(-1, (4, -1)).transpose(-1, -2).flatten(-2)


# ------------------------------------------------------------------------------------------------ cache


def _inference_only(x: torch.Tensor, name: str) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or on detached tensors")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError(f"{name} has no forward-mode derivative: call it on tensors without a tangent")


class Int4KVCache:
    """Keys and values of `slots` sequences of up to `room` tokens, in 4 bits.  `dtype`: the model's type."""

    __slots__ = ("data", "slots", "room", "n_kv", "hd", "dtype")

    def __init__(self, slots: int, room: int, n_kv: int, hd: int, dtype=torch.bfloat16, device="cuda"):
        if hd not in HEAD_DIMS:
            raise ValueError(f"Int4KVCache: heads of 64 or 128 channels, not {hd}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"Int4KVCache: bfloat16 or float16, not {dtype}")
        if slots < 0 or room < 0 or n_kv <= 0:
            raise ValueError(f"Int4KVCache: {slots} slots of {room} tokens, {n_kv} heads")
        self.slots, self.room, self.n_kv, self.hd, self.dtype = int(slots), int(room), int(n_kv), int(hd), dtype
        words = TILE_ROWS * (hd // 4 + hd // KEY_GROUP + hd // VALUE_GROUP)
        self.data = torch.zeros(slots, n_kv, -(-room // TILE_ROWS), words, dtype=torch.int32, device=device)

    @property
    def shape(self) -> Tuple[int, int, int, int]:
        """The shape of a 16-bit cache of the same rows."""
        return (self.slots, self.room, self.n_kv, self.hd)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def nbytes(self) -> int:
        return self.data.numel() * 4

    def _fields(self):
        """Views: key words [slots, n_kv, tiles, 16, W], value halves int16 [.., W, 4, 2, 2, 2] (channels / 8, (row & 7) / 2, row / 8, quad of channels, row & 1), key groups
        [.., 16, hd / 32], value groups [.., 16, hd / 64]."""
        W, a = self.hd // 8, TILE_ROWS * self.hd // 8
        kg, vg = self.hd // KEY_GROUP, self.hd // VALUE_GROUP
        d = self.data
        return (d[..., :a].unflatten(-1, (TILE_ROWS, W)), d.view(torch.int16)[..., 2 * a:4 * a].unflatten(-1, (W, 4, 2, 2, 2)),
                d[..., 2 * a:2 * a + TILE_ROWS * kg].unflatten(-1, (TILE_ROWS, kg)), d[..., 2 * a + TILE_ROWS * kg:].unflatten(-1, (TILE_ROWS, vg)))

    def _check(self, cu_seqlens, slots, start):
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("Int4KVCache: cu_seqlens holds one number more than there are sequences")
        n = cu_seqlens.numel() - 1
        for name, t in (("slots", slots), ("start", start)):
            if t is not None and tuple(t.shape) != (n,):
                raise ValueError(f"Int4KVCache: `{name}` holds one number a sequence ({n}), not {tuple(t.shape)}")
        return self._whole(cu_seqlens), self._whole(slots), self._whole(start)

    def _whole(self, t):
        """int32 beside the cache."""
        if t is None or (t.dtype is torch.int32 and t.device == self.data.device and t.is_contiguous()):
            return t
        return t.to(device=self.data.device, dtype=torch.int32).contiguous()

    def _rows(self, cu, slots, start, tokens: int):
        """(token, slot, row) of every packed token whose row is inside the cache."""
        tok = torch.arange(tokens, device=cu.device)
        seq = torch.searchsorted(cu[1:].long().contiguous(), tok, right=True)
        inside = (seq < cu.numel() - 1) & (tok >= int(cu[0]))
        tok, seq = tok[inside], seq[inside]
        row = tok - cu.long()[seq] + (start.long()[seq] if start is not None else 0)
        slot = slots.long()[seq] if slots is not None else seq
        ok = (slot >= 0) & (slot < self.slots) & (row >= 0) & (row < self.room)
        return tok[ok], slot[ok], row[ok]

    def store(self, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: Optional[int] = None, slots: Optional[torch.Tensor] = None,
              start: Optional[torch.Tensor] = None) -> None:
        """Writes packed keys (rotated) and values [T, n_kv, hd]: the tokens cu_seqlens[i] .. of sequence i go to the rows start[i] .. (0 ..) of slot slots[i] (i).
        Rows and slots outside the cache are left out, all others of the cache keep what they hold.  No row may be named twice in a call.  `max_seqlen` sets the
        size of the launch alone.  What is stored is numbers: no gradient goes back to `k` and `v`."""
        if use_native(self.data) and k.dtype is self.dtype and k.is_cuda:      # (the op checks the rest)
            lib().int4_cache_store(k, v, self.data, self._whole(cu_seqlens), self._whole(slots), self._whole(start), self.room, self.hd, max_seqlen or 0)
            return
        if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (self.n_kv, self.hd):
            raise ValueError(f"Int4KVCache.store: keys and values [tokens, {self.n_kv}, {self.hd}], not {tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype != self.dtype or v.dtype != self.dtype or k.device != self.device or v.device != self.device:
            raise ValueError(f"Int4KVCache.store: keys and values are {self.dtype} on {self.device}, as the cache")
        cu, slots, start = self._check(cu_seqlens, slots, start)
        tok, slot, row = self._rows(cu, slots, start, k.shape[0])
        self._put(k.detach()[tok], v.detach()[tok], slot, row)

    def _at(self, slot, row):
        """Index of rows in the fields of keys and of the groups, and in the values with the row's three dims in front."""
        tile, r = row // TILE_ROWS, row % TILE_ROWS
        at = (slot[:, None], torch.arange(self.n_kv, device=slot.device)[None], tile[:, None])
        return at + (r[:, None],), at + ((r[:, None] & 7) >> 1, r[:, None] >> 3, r[:, None] & 1)

    def _put(self, k, v, slot, row):
        kw, vw, kg, vg = self._fields()
        at, place = self._at(slot, row)
        c, s, lo = quantize_groups(k, KEY_GROUP)
        kw[at] = _row_order(_words(c, _KEY))
        kg[at] = _group_words(s, lo)
        c, s, lo = quantize_groups(v, VALUE_GROUP)
        vw.permute(0, 1, 2, 4, 5, 7, 3, 6)[place] = _words(c, _VALUE).view(torch.int16).unflatten(-1, (-1, 2))
        vg[at] = _group_words(s, lo)

    def _get(self, slot, row):
        kw, vw, kg, vg = self._fields()
        at, place = self._at(slot, row)
        k = dequantize_groups(_codes(_channel_order(kw[at]), _KEY), *_group_numbers(kg[at], self.dtype))
        words = vw.permute(0, 1, 2, 4, 5, 7, 3, 6)[place].contiguous().flatten(-2).view(torch.int32)
        return k, dequantize_groups(_codes(words, _VALUE), *_group_numbers(vg[at], self.dtype))

    def load(self, cu_seqlens: torch.Tensor, tokens: int, max_seqlen: Optional[int] = None, slots: Optional[torch.Tensor] = None,
             start: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The reverse of `store`: keys and values [tokens, n_kv, hd] of the cache's type, each number rounded once.  Tokens whose row or slot is outside the cache,
        or that belong to no sequence, are 0."""
        if use_native(self.data):
            k, v = lib().int4_cache_load(self.data, self._whole(cu_seqlens), self._whole(slots), self._whole(start), self.room, self.hd, tokens, max_seqlen or 0, self.dtype)
            return k, v
        if tokens < 0:
            raise ValueError(f"Int4KVCache.load: {tokens} tokens")
        cu, slots, start = self._check(cu_seqlens, slots, start)
        out = torch.zeros(2, tokens, self.n_kv, self.hd, dtype=self.dtype, device=self.device)
        tok, slot, row = self._rows(cu, slots, start, tokens)
        k, v = self._get(slot, row)
        out[0, tok], out[1, tok] = _to_type(k, self.dtype), _to_type(v, self.dtype)
        return out[0], out[1]


# ------------------------------------------------------------------------------------------------ attention


def _rotated(x, cos, sin, rot_dim: int, interleaved: bool):
    """fp32 x [B, heads, hd], cos / sin [B, rot_dim / 2]."""
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:rot_dim:2], x[..., 1:rot_dim:2]) if interleaved else (x[..., : rot_dim // 2], x[..., rot_dim // 2: rot_dim])
    y = (a * c - b * s, b * c + a * s)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, x[..., rot_dim:]], -1)


def decode_attention_int4_ref(qkv, cache: Int4KVCache, cache_lens, n_q: int, n_kv: int, hd: int, scale: float, cos=None, sin=None, rot_dim: Optional[int] = None,
                              interleaved: bool = False):
    """`decode_attention_int4` in plain PyTorch, on any device and for fp32 projections too."""
    B, lens = qkv.shape[0], cache_lens.long()
    live = (lens >= 0) & (lens < cache.room)
    q, k, v = (t.reshape(B, -1, hd).float() for t in qkv.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
    if cos is not None:
        at = lens.clamp(0, max(cache.room - 1, 0))
        q, k = (_rotated(t, cos[at], sin[at], rot_dim or hd, interleaved) for t in (q, k))
    slot = torch.nonzero(live).flatten()
    cache._put(k[slot].to(cache.dtype), v[slot].to(cache.dtype), slot, lens[slot])
    out = torch.zeros(B, n_q, hd, dtype=torch.float32, device=qkv.device)
    for b in slot.tolist():
        n = int(lens[b]) + 1
        kk, vv = (t.repeat_interleave(n_q // n_kv, 1) for t in cache._get(torch.full((n,), b, device=qkv.device), torch.arange(n, device=qkv.device)))
        out[b] = torch.einsum("hn,nhd->hd", torch.softmax(torch.einsum("hd,nhd->hn", q[b], kk) * scale, -1), vv)
    return _to_type(out.reshape(B, n_q * hd), qkv.dtype)


def decode_attention_int4(qkv: torch.Tensor, cache: Int4KVCache, cache_lens: torch.Tensor, n_q: int, n_kv: int, hd: int, scale: Optional[float] = None, cos=None,
                          sin=None, rot_dim: Optional[int] = None, interleaved: bool = False) -> torch.Tensor:
    """One decode step over a 4-bit cache, as `attention.decode_attention` over a 16-bit one: row b of qkv [slots, (n_q + 2 n_kv) * hd] is the fused projection of
    the token at position cache_lens[b] of slot b.  Its queries and key are rotated (cos / sin [room or more, rot_dim / 2] given), the key is rounded to the cache's
    type, key and value are quantised and written, and the queries attend to the rows [0, cache_lens[b]] as the cache holds them, the new one among them.
    Returns [slots, n_q * hd], with no gradient (a call that would need one is refused).  A row whose length is not in [0, room) changes nothing and returns 0.  Does not advance cache_lens."""
    _inference_only(qkv, "decode_attention_int4")
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    if use_native(qkv) and qkv.dtype is cache.dtype:                           # (the op checks the rest)
        return lib().decode_attention_int4(qkv, cache.data, cache._whole(cache_lens), n_q, n_kv, hd, cache.room, scale, cos, sin, rot_dim or hd, interleaved)
    if (n_kv, hd) != (cache.n_kv, cache.hd) or n_q <= 0 or n_q % n_kv:
        raise ValueError(f"decode_attention_int4: {n_q} query heads over {n_kv} of {hd} channels, a cache of {cache.n_kv} heads of {cache.hd}")
    if tuple(qkv.shape) != (cache.slots, (n_q + 2 * n_kv) * hd) or tuple(cache_lens.shape) != (cache.slots,):
        raise ValueError(f"decode_attention_int4: projections [{cache.slots}, {(n_q + 2 * n_kv) * hd}] and as many lengths, not {tuple(qkv.shape)} and "
                         f"{tuple(cache_lens.shape)}")
    rot = rot_dim or hd
    if (cos is None) != (sin is None) or (cos is not None and (rot > hd or rot % (2 if interleaved else 16) or tuple(cos.shape[1:]) != (rot // 2,) or
                                                               cos.shape != sin.shape or cos.shape[0] < cache.room)):
        raise ValueError(f"decode_attention_int4: cosines and sines are tables [{cache.room} or more, {rot // 2}], both or neither")
    if use_native(qkv) or use_native(cache.data):
        raise ValueError(f"decode_attention_int4: projections are {cache.dtype} on {cache.device}, as the cache")
    return decode_attention_int4_ref(qkv, cache, cache_lens, n_q, n_kv, hd, scale, cos, sin, rot, interleaved)


# ------------------------------------------------------------------------------------------------ weights


class Int4Linear:
    """One weight matrix [N, K] in 4 bits, groups of `group` along K (+ optional bias).  `__call__(x)`: x @ w^T + bias for x [..., K] of the weight's type."""

    __slots__ = ("q", "bias", "N", "K", "group", "dtype")

    def __init__(self, w: torch.Tensor, bias: Optional[torch.Tensor] = None, group: int = 128):
        self._plan(w.shape, group, w.dtype, w.device, bias)
        self.requantize(w)

    def _plan(self, shape, group: int, dtype, device, bias):
        if len(shape) != 2 or group not in GROUPS or shape[0] <= 0 or shape[1] <= 0 or shape[1] % group:
            raise ValueError(f"Int4Linear: a weight [N, K] with groups of 32, 64 or 128 along K, not {tuple(shape)} in groups of {group}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"Int4Linear: bfloat16 or float16, not {dtype}")
        self.N, self.K, self.group, self.dtype = int(shape[0]), int(shape[1]), int(group), dtype
        if bias is not None and (tuple(bias.shape) != (self.N,) or bias.dtype != dtype):
            raise ValueError(f"Int4Linear: a bias [{self.N}] of {dtype}")
        self.bias = None if bias is None else bias.detach()                    # (its numbers alone, as the weight's)
        self.q = torch.zeros(-(-self.N // 128), -(-self.K // 128), 8, TILE_ROWS * 16 + TILE_ROWS * (128 // group), dtype=torch.int32, device=device)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, low: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "Int4Linear":
        """codes uint8 [N, K] (0 .. 15), scale and low [N, K / group] of the model's type: a weight that was quantised elsewhere."""
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scale.shape != low.shape or scale.dtype != low.dtype or scale.dim() != 2 or scale.shape[0] != codes.shape[0] \
                or scale.shape[1] == 0 or codes.shape[1] % scale.shape[1]:
            raise ValueError("Int4Linear.from_codes: codes uint8 [N, K], scale and low [N, K / group] of one type")
        if codes.numel() and int(codes.max()) > 15:
            raise ValueError("Int4Linear.from_codes: a code is 0 .. 15")
        self = cls.__new__(cls)
        self._plan(codes.shape, codes.shape[1] // scale.shape[1], scale.dtype, codes.device, bias)
        if use_native(codes):
            lib().int4_pack(codes, scale, low, self.q, self.group)
        else:
            self._fill(codes, scale, low)
        return self

    def _fill(self, codes, scale, low):
        nt, kb, _, _ = self.q.shape
        self.q.zero_()
        w = torch.zeros(nt * 128, kb * 16, dtype=torch.int32, device=codes.device)
        w[: self.N, : self.K // 8] = _words(codes, _WEIGHT)
        self.q[..., :256] = _row_order(w.view(nt, 8, TILE_ROWS, kb, 16)).permute(0, 3, 1, 2, 4).flatten(-2)
        g = torch.zeros(nt * 128, kb * (128 // self.group), dtype=torch.int32, device=codes.device)
        g[: self.N, : self.K // self.group] = _group_words(scale.contiguous(), low.contiguous())
        self.q[..., 256:] = g.view(nt, 8, TILE_ROWS, kb, -1).permute(0, 3, 1, 2, 4).flatten(-2)

    def requantize(self, w: torch.Tensor):
        """Refresh the 4-bit copy in place after the weight changed (same buffers: a kept CUDA graph stays valid)."""
        if tuple(w.shape) != (self.N, self.K) or w.dtype != self.dtype or w.device != self.q.device:
            raise ValueError(f"Int4Linear: a weight [{self.N}, {self.K}] of {self.dtype} on {self.q.device}")
        w = w.detach()
        if use_native(w):
            lib().int4_quantize(w, self.q, self.group)
        else:
            self._fill(*quantize_groups(w, self.group))

    def codes(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(codes uint8 [N, K], scale, low [N, K / group])."""
        nt, kb, _, _ = self.q.shape
        w = _channel_order(self.q[..., :256].unflatten(-1, (TILE_ROWS, 16))).permute(0, 2, 3, 1, 4).reshape(nt * 128, kb * 16)
        g = self.q[..., 256:].unflatten(-1, (TILE_ROWS, -1)).permute(0, 2, 3, 1, 4).reshape(nt * 128, -1)
        return (_codes(w[: self.N, : self.K // 8], _WEIGHT),) + _group_numbers(g[: self.N, : self.K // self.group], self.dtype)

    def dequantize(self) -> torch.Tensor:
        """fp32 [N, K]."""
        return dequantize_groups(*self.codes())

    def __call__(self, x: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.K:
            raise ValueError(f"Int4Linear: rows of {self.K}, not {tuple(x.shape)}")
        _inference_only(x, "Int4Linear")
        if bias is None:
            bias = self.bias
        else:
            _inference_only(bias, "Int4Linear")
        if use_native(x):
            if x.dtype is not self.dtype or x.device != self.q.device:
                raise ValueError(f"Int4Linear: rows of {self.dtype} on {self.q.device}")
            if x.dim() == 2:
                return lib().int4_linear(x, self.q, bias, self.N, self.group)
            y = lib().int4_linear(x.reshape(-1, self.K), self.q, bias, self.N, self.group)
        else:
            x2 = x.reshape(-1, self.K)
            y = x2.float() @ self.dequantize().t()
            y = (y if bias is None else y + bias.float()).to(x.dtype)
        return y.view(*x.shape[:-1], self.N)

    def nbytes(self) -> int:
        return 4 * self.q.numel()


def supported(w: torch.Tensor, group: int = 128) -> bool:
    """Weights that a 4-bit copy can be made of."""
    return bool(w.dim() == 2 and w.dtype in (torch.bfloat16, torch.float16) and w.shape[0] > 0 and w.shape[1] > 0 and w.shape[1] % group == 0)
