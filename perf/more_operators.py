"""Generation with 4-bit caches and weights, measured through the framework's public entry points.

A group of numbers is held as 4-bit codes c with the group's lowest value `low` and a step `scale`, both of the model's 16-bit type T:
    low = min x,   scale = T((max x - low) / 15),   c = min(15, round_half_even((x - low) / scale))  (0 where scale is 0),   x ~ scale c + low.

Kinds:
  cache   keys and values of packed sequences written to a 4-bit cache and read back: what a prompt's pass stores, and what a program that goes
          on in 16 bits reads.  Groups: 32 channels of a key, 64 of a value.  Sequences may go on behind rows that are there ("start").
  decode  one generation step's attention over such a cache: queries and key are rotated, key (rounded to T, as a 16-bit cache would hold it)
          and value are quantised and appended, the queries attend to all rows as the cache holds them; and the appended rows read back.
  linear  products of a few rows with a weight [N, K] in 4 bits, groups of `group` along K.

A case is a dict of plain values.  With `own` false `run` computes the plain forms, elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random
from typing import Dict, List

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
KEY_GROUP, VALUE_GROUP = 32, 64


# ------------------------------------------------------------------------------------------------ the cases


def listed() -> List[dict]:
    return [
        # three short prompts of a GPT-2 sized model: latency counts
        dict(name="cache_3x29_12x64", kind="cache", seqs=3, lo=9, hi=29, lens_seed=1, start=0, nkv=12, hd=64, dtype="bf16"),
        # the PPO benchmark's prompts, one layer: 128 sequences of 128 tokens, LLaMA-7B heads
        dict(name="cache_128x128_32x128", kind="cache", seqs=128, lo=128, hi=128, lens_seed=2, start=0, nkv=32, hd=128, dtype="bf16"),
        # long ragged prompts with grouped heads, stored in pieces: this piece begins inside the cache
        dict(name="cache_8x4096_8x128_piece", kind="cache", seqs=8, lo=1500, hi=4096, lens_seed=3, start=777, nkv=8, hd=128, dtype="fp16"),
        # one user's long conversation, grouped heads
        dict(name="decode_1x3900_32over8x128", kind="decode", batch=1, lo=3900, hi=3900, lens_seed=4, room=4096, nq=32, nkv=8, hd=128, dtype="bf16"),
        # a small batch with seven queries a key head
        dict(name="decode_5x700_14over2x64", kind="decode", batch=5, lo=37, hi=700, lens_seed=5, room=701, nq=14, nkv=2, hd=64, dtype="bf16"),
        # generation with 16 sequences per GPU (the benchmark's share on 8 GPUs)
        dict(name="decode_16x639_32x128", kind="decode", batch=16, lo=128, hi=639, lens_seed=6, room=640, nq=32, nkv=32, hd=128, dtype="bf16"),
        # serving long contexts with grouped heads
        dict(name="decode_32x4095_32over8x128", kind="decode", batch=32, lo=1300, hi=4095, lens_seed=7, room=4096, nq=32, nkv=8, hd=128, dtype="fp16"),
        # generation with the benchmark's whole batch on one GPU
        dict(name="decode_128x639_32x128", kind="decode", batch=128, lo=128, hi=639, lens_seed=8, room=640, nq=32, nkv=32, hd=128, dtype="bf16"),
        # one sequence through an attention output projection
        dict(name="linear_1x4096x4096", kind="linear", rows=1, width=4096, out=4096, group=128, bias=False, dtype="bf16"),
        # a GPT-2 sized head over an odd vocabulary, small groups
        dict(name="linear_7x1024x50257_g32", kind="linear", rows=7, width=1024, out=50257, group=32, bias=False, dtype="fp16"),
        # the LLaMA-7B gate and up projection at 16 sequences
        dict(name="linear_16x4096x22016", kind="linear", rows=16, width=4096, out=22016, group=128, bias=False, dtype="bf16"),
        # the down projection with the benchmark's whole batch
        dict(name="linear_128x11008x4096", kind="linear", rows=128, width=11008, out=4096, group=64, bias=True, dtype="bf16"),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12, 64), (16, 4, 128), (32, 32, 128), (32, 8, 128), (16, 16, 64), (14, 2, 64), (8, 1, 128), (20, 4, 128), (16, 1, 64)]


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["cache", "decode", "decode", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    nq, nkv, hd = rng.choice(HEADS)
    seed = rng.randrange(1 << 20)
    if kind == "cache":
        hi = _log(rng, 1, 4096)
        most = max(1, min(128, 128 * 128 * 32 * 128 // (hi * nkv * hd)))
        return dict(kind=kind, seqs=_log(rng, 1, most), lo=max(1, hi // rng.choice([1, 2, 5])), hi=hi, lens_seed=seed,
                    start=rng.choice([0, 0, rng.randint(1, 1000)]), nkv=nkv, hd=hd, dtype=dtype)
    if kind == "decode":
        room = _log(rng, 2, 8192)
        hi = rng.randint(room // 2, room - 1)
        most = max(1, min(128, 128 * 640 * 32 * 128 // (room * nkv * hd)))
        return dict(kind=kind, batch=_log(rng, 1, most), lo=hi // rng.choice([1, 3, 10]), hi=hi, lens_seed=seed, room=room, nq=nq, nkv=nkv, hd=hd, dtype=dtype)
    group, rows = rng.choice([32, 64, 128]), _log(rng, 1, 128)
    width = group * _log(rng, 256 // group, 11008 // group)
    most = min(4096 * 22016 // width, 128 * 11008 * 4096 // (rows * width))
    return dict(kind=kind, rows=rows, width=width, out=_log(rng, 300, min(50257, most)), group=group, bias=rng.random() < 0.3, dtype=dtype)


def _lens(case) -> List[int]:
    rng = random.Random(case["lens_seed"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"] if case["kind"] == "cache" else case["batch"])]


def work(case: dict) -> Dict[str, float]:
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["width"], case["out"]
        return {"bytes": N * K / 2 + 4 * N * K / case["group"] + 2 * (M * K + M * N + (N if case["bias"] else 0)), "flops": 2.0 * M * N * K}
    nkv, hd, lens = case["nkv"], case["hd"], _lens(case)
    held = nkv * (hd + 4 * hd // KEY_GROUP + 4 * hd // VALUE_GROUP)   # bytes of a token's key and value with their steps and lowest values
    plain = 4 * nkv * hd                                              # the same in 16 bits
    if case["kind"] == "cache":
        n = sum(lens)
        return {"bytes": n * (2 * plain + 2 * held), "flops": n * nkv * hd * 16.0}
    B, nq = case["batch"], case["nq"]
    return {"bytes": sum(lens) * held + B * (2 * nq * hd * 2 + plain + held + held + plain), "flops": 4.0 * sum(n + 1 for n in lens) * nq * hd}


# ------------------------------------------------------------------------------------------------ inputs


def _rows(g, n, heads, hd, dtype, dev, keys):
    """Keys (a few channels far larger than the others, as trained models have them) or values of n tokens, [n, heads, hd]."""
    x = torch.randn(n, heads, hd, generator=g, device=dev)
    if keys:
        x *= 1 + 6 * (torch.rand(heads, hd, generator=g, device=dev) < 0.04)
    return x.to(dtype)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["width"], case["out"]
        s["x"] = torch.randn(M, K, generator=g, device=dev).to(dt)
        w = torch.randn(N, K, generator=g, device=dev).mul_(1 / math.sqrt(K)).to(dt)
        s["bias"] = torch.randn(N, generator=g, device=dev).to(dt) if case["bias"] else None
        codes, scale, low = _quantise(w.float(), case["group"], dt)
        if own:
            from realhf_b200.ops import int4
            s["linear"] = int4.Int4Linear.from_codes(codes, scale, low, s["bias"])
        else:
            s.update(codes=codes, scale=scale, low=low)
        return s
    lens = _lens(case)
    nkv, hd, B = case["nkv"], case["hd"], len(lens)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    k, v = _rows(g, cu[-1], nkv, hd, dt, dev, True), _rows(g, cu[-1], nkv, hd, dt, dev, False)
    cu, total, longest = torch.tensor(cu, dtype=torch.int32, device=dev), cu[-1], max(lens)
    if case["kind"] == "cache":
        rows = case["start"] + longest
        kv = torch.cat([k, v], 1)   # as the projection gives them: keys | values
        s.update(k=kv[:, :nkv], v=kv[:, nkv:], cu=cu, total=total, longest=longest)
        s["start"] = torch.full((B,), case["start"], dtype=torch.int32, device=dev) if case["start"] else None
    else:
        rows = case["room"]
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["qkv"] = torch.cat([_rows(g, B, case["nq"], hd, dt, dev, False), _rows(g, B, nkv, hd, dt, dev, True), _rows(g, B, nkv, hd, dt, dev, False)], 1).view(B, -1)
        angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["one"] = torch.arange(B + 1, dtype=torch.int32, device=dev)   # one row a sequence
    if own:
        from realhf_b200.ops import int4
        s["cache"] = int4.Int4KVCache(B, rows, nkv, hd, dt, dev)
        if case["kind"] == "decode" and total:   # what the cache holds before the step
            s["cache"].store(k, v, cu, longest)
    else:
        s["held"] = {name: (torch.zeros(B, rows, nkv, hd, dtype=torch.uint8, device=dev), torch.zeros(B, rows, nkv, hd // group, dtype=dt, device=dev),
                            torch.zeros(B, rows, nkv, hd // group, dtype=dt, device=dev)) for name, group in (("k", KEY_GROUP), ("v", VALUE_GROUP))}
        if case["kind"] == "decode" and total:
            at = _where(cu, total, None)
            _put(s["held"]["k"], at, k, KEY_GROUP)
            _put(s["held"]["v"], at, v, VALUE_GROUP)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _quantise(x, group, dt):
    """fp32 x [..., n] -> (codes uint8 [..., n], scale, low [..., n / group] of the type dt)."""
    xg = x.unflatten(-1, (-1, group))
    low = xg.amin(-1)
    scale = ((xg.amax(-1) - low) / torch.full_like(low, 15.0)).to(dt)   # (a tensor by a tensor: a division, correctly rounded)
    step = scale.float()[..., None]
    c = torch.where(step > 0, (xg - low[..., None]) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(xg))
    return torch.round(c).clamp_(max=15).to(torch.uint8).flatten(-2), scale, low.to(dt)


def _value(codes, scale, low):
    """fp32 scale c + low."""
    group = codes.shape[-1] // scale.shape[-1]
    return (codes.unflatten(-1, (-1, group)).float() * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


def _put(held, at, x, group):
    codes, scale, low = _quantise(x.float(), group, x.dtype)
    held[0][at], held[1][at], held[2][at] = codes, scale, low


def _get(held, at):
    return _value(held[0][at], held[1][at], held[2][at])


def _where(cu, total, start):
    """(slot, row) of every packed token."""
    tok = torch.arange(total, device=cu.device)
    slot = torch.searchsorted(cu[1:].long(), tok, right=True)
    return slot, tok - cu.long()[slot] + (start.long()[slot] if start is not None else 0)


def _plain_cache(s):
    at, dt = _where(s["cu"], s["total"], s["start"]), s["k"].dtype
    _put(s["held"]["k"], at, s["k"], KEY_GROUP)
    _put(s["held"]["v"], at, s["v"], VALUE_GROUP)
    return dict(k=_get(s["held"]["k"], at).to(dt), v=_get(s["held"]["v"], at).to(dt))


def _turn(x, cos, sin):
    """x [B, heads, hd] fp32, cos / sin [B, hd / 2]: the first half of the channels against the second."""
    a, b = x.chunk(2, -1)
    c, z = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * z, b * c + a * z], -1)


def _attend(q, k, v, lens):
    """q [B, nq, hd], k / v [B, S, nkv, hd], rows [0, lens] of each sequence; in the type of q."""
    B, nq, hd = q.shape
    nkv = k.shape[2]
    q = q.view(B, nkv, nq // nkv, hd)
    z = torch.einsum("bgrd,bsgd->bgrs", q, k) * hd ** -0.5
    z = torch.where(torch.arange(k.shape[1], device=q.device) <= lens.long()[:, None, None, None], z, torch.full_like(z, float("-inf")))
    w = torch.exp(z - z.amax(-1, keepdim=True))
    return (torch.einsum("bgrs,bsgd->bgrd", w, v) / w.sum(-1, keepdim=True)).reshape(B, nq * hd)


def _plain_decode(s):
    c, dt, lens = s["case"], s["qkv"].dtype, s["lens"].long()
    B, nq, nkv, hd = c["batch"], c["nq"], c["nkv"], c["hd"]
    q, k, v = (t.view(B, -1, hd) for t in s["qkv"].split([nq * hd, nkv * hd, nkv * hd], 1))
    cos, sin = s["cos"][lens], s["sin"][lens]
    at = (torch.arange(B, device=lens.device), lens)
    _put(s["held"]["k"], at, _turn(k.float(), cos, sin).to(dt), KEY_GROUP)
    _put(s["held"]["v"], at, v, VALUE_GROUP)
    out = _attend(_turn(q.float(), cos, sin), _value(*s["held"]["k"]), _value(*s["held"]["v"]), lens)
    return dict(out=out.to(dt), k=_get(s["held"]["k"], at).to(dt), v=_get(s["held"]["v"], at).to(dt))


def _plain_linear(s):
    y = s["x"].float() @ _value(s["codes"], s["scale"], s["low"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return dict(y=y.to(s["x"].dtype))


# ------------------------------------------------------------------------------------------------ one pass


def _own(s):
    from realhf_b200.ops import int4
    c = s["case"]
    if c["kind"] == "linear":
        return dict(y=s["linear"](s["x"]))
    if c["kind"] == "cache":
        s["cache"].store(s["k"], s["v"], s["cu"], s["longest"], start=s["start"])
        k, v = s["cache"].load(s["cu"], s["total"], s["longest"], start=s["start"])
        return dict(k=k, v=v)
    out = int4.decode_attention_int4(s["qkv"], s["cache"], s["lens"], c["nq"], c["nkv"], c["hd"], cos=s["cos"], sin=s["sin"])
    k, v = s["cache"].load(s["one"], c["batch"], 1, start=s["lens"])
    return dict(out=out, k=k, v=v)


def run(state: dict):
    if own:
        return _own(state)
    return {"cache": _plain_cache, "decode": _plain_decode, "linear": _plain_linear}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ 64 bits


def _exact_values(x, group, dt):
    """The values that a 4-bit group stands for, from the definition: steps and lowest values as they are stored, all else in 64 bits."""
    parts = x.double().split(group, -1)
    done = []
    for p in parts:
        low = p.min(-1, keepdim=True).values
        step = ((p.max(-1, keepdim=True).values - low) / 15.0).float().to(dt).double()
        code = torch.nan_to_num((p - low) / step, nan=0.0, posinf=0.0).round().clamp(0, 15)
        done.append(low + step * code)
    return torch.cat(done, -1)


def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "linear":
        x, (N, K), group = s["x"].double(), s["codes"].shape, case["group"]
        y = torch.zeros(case["rows"], N, dtype=torch.float64, device=x.device)
        for n in range(0, N, 4096):
            w = s["codes"][n:n + 4096].double()
            for j in range(K // group):
                cols = slice(j * group, (j + 1) * group)
                y[:, n:n + 4096] += (x[:, cols] @ w[:, cols].T) * s["scale"][n:n + 4096, j].double() + x[:, cols].sum(1, keepdim=True) * s["low"][n:n + 4096, j].double()
        return dict(y=y if s["bias"] is None else y + s["bias"].double())
    if case["kind"] == "cache":
        return dict(k=_exact_values(s["k"], KEY_GROUP, dt), v=_exact_values(s["v"], VALUE_GROUP, dt))
    B, nq, nkv, hd, lens = case["batch"], case["nq"], case["nkv"], case["hd"], s["lens"].tolist()
    q, k, v = (t.reshape(B, -1, hd) for t in s["qkv"].split([nq * hd, nkv * hd, nkv * hd], 1))
    out, ks, vs = [], [], []
    for b, n in enumerate(lens):
        turn = torch.complex(s["cos"][n].double(), s["sin"][n].double())
        z = torch.complex(*q[b].double().chunk(2, -1)) * turn
        qb = torch.cat([z.real, z.imag], -1)
        # (the key is rotated in 32 bits and rounded to the type before it is quantised: that is what the cache is given)
        kn = _exact_values(_turn(k[b:b + 1].float(), s["cos"][n:n + 1], s["sin"][n:n + 1]).to(dt)[0], KEY_GROUP, dt)
        vn = _exact_values(v[b], VALUE_GROUP, dt)
        rows = []
        for held, new in ((s["held"]["k"], kn), (s["held"]["v"], vn)):
            codes, scale, low = (t[b, :n].double() for t in held)
            rep = hd // scale.shape[-1]
            rows.append(torch.cat([codes * scale.repeat_interleave(rep, -1) + low.repeat_interleave(rep, -1), new[None]]).repeat_interleave(nq // nkv, 1))
        w = torch.softmax((rows[0] * qb).sum(-1) / math.sqrt(hd), 0)
        out.append((w[..., None] * rows[1]).sum(0).flatten())
        ks.append(kn)
        vs.append(vn)
    return dict(out=torch.stack(out), k=torch.stack(ks), v=torch.stack(vs))
