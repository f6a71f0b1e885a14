"""Keys, values and weights in 4 bits against plain 64-bit implementations, on the CPU and on the GPU.

Bounds.  A group's step is (max - min) / 15 rounded to the type (relative error u = eps / 2), so a number is off by half a step, plus 15 roundings of the step where
the code is cut at 15: step * (0.5 + 15 u), plus a rounding of fp32.  What is read back as 16-bit numbers is rounded once, u relative.  Attention over a cache and
products with a weight are compared with 64 bits over the numbers that the cache and the weight hold, so that quantising is no part of those bounds.
"""
import math

import pytest
import torch

from realhf_b200.ops import int4

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16]
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of the type, relative
# ... and where the type has no relative step any more: fp16's numbers below 2^-14 lie 2^-24 apart, bf16's below 2^-126 2^-133
SMALL = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def rows(g, *shape, dtype, device, outliers=False):
    x = torch.randn(*shape, generator=g)
    if outliers:
        x *= 1 + 6 * (torch.rand(shape[-2:], generator=g) < 0.05)
    return x.to(dtype).to(device)


def groups64(x, group, dtype):
    """(values, steps) of the definition, in 64 bits but for the step's rounding to the type; [..., n] both."""
    xs, out, steps = x.double().unflatten(-1, (-1, group)), [], []
    lo, hi = xs.min(-1).values, xs.max(-1).values
    step = ((hi - lo) / 15).float().to(dtype).double()
    code = torch.where(step[..., None] > 0, (xs - lo[..., None]) / step[..., None].clamp(min=1e-300), torch.zeros_like(xs)).round().clamp(0, 15)
    return (lo[..., None] + code * step[..., None]).flatten(-2), step.repeat_interleave(group, -1).reshape(x.shape)


def check_groups(got, x, group, dtype, rounded=True):
    """`got`, read back of x, against the definition and against x."""
    want, step = groups64(x, group, dtype)
    u = EPS[dtype]
    tol = (u if rounded else 2.0 ** -23) * want.abs() + (SMALL[dtype] if rounded else 1e-30)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert bool(((got.double() - x.double()).abs() <= step * (0.5 + 15 * u) + tol + 2.0 ** -23 * x.double().abs()).all())


def packed(lens, device):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------------ the rule


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_of_special_values(dtype):
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(dtype).max
    x = torch.zeros(7, 32)
    x[1] = 3.5                                             # one value throughout: step 0, exact
    x[2, 5], x[3, 7] = inf, nan                            # read back as NaN, the whole group
    x[4], x[4, :16] = big, -big                            # the widest group
    x[5] = torch.linspace(-1, 1, 32)
    x[6, 3] = torch.finfo(dtype).tiny                      # a step that rounds to a subnormal number
    c, s, lo = int4.quantize_groups(x.to(dtype), 32)
    y = int4.dequantize_groups(c, s, lo)
    assert (c[:2] == 0).all() and (y[0] == 0).all() and (y[1] == 3.5).all()
    assert y[2:4].isnan().all() and (c[2:4] == 0).all() and torch.isfinite(y[[0, 1, 4, 5, 6]]).all()
    assert (y[4, :16] == -big).all() and bool(((y[4, 16:].double() - big).abs() <= 30 * EPS[dtype] * big).all())
    check_groups(y[5], x[5].to(dtype), 32, dtype, rounded=False)
    assert float((y[6] - x[6].to(dtype).float()).abs().max()) <= torch.finfo(dtype).tiny
    with pytest.raises(ValueError):
        int4.quantize_groups(x, 32)
    with pytest.raises(ValueError):
        int4.quantize_groups(x.to(dtype), 33)


def test_ties_go_to_the_even_code():
    x = torch.zeros(1, 32)
    x[0, 0], x[0, 1:5] = 15.0, torch.tensor([0.5, 1.5, 2.5, 13.5])
    c, s, lo = int4.quantize_groups(x.bfloat16(), 32)
    assert float(s) == 1.0 and float(lo) == 0.0 and c[0, :5].tolist() == [15, 0, 2, 2, 14]


# ------------------------------------------------------------------------------------------------ the cache


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nkv,hd,lens,start", [
    (2, 64, [1], None), (3, 128, [16, 1, 0, 17, 15, 33], None), (1, 64, [0, 0], None), (12, 64, [5, 40], [3, 16]), (2, 128, [1, 1, 1, 1], [0, 15, 16, 70]),
    (8, 128, [130, 7], [31, 1]),
])
def test_store_and_load(device, dtype, nkv, hd, lens, start):
    g = torch.Generator().manual_seed(len(lens) * 100 + hd)
    T, n = sum(lens), len(lens)
    wide = rows(g, T, 2 * nkv + 1, hd, dtype=dtype, device=device, outliers=True)
    k, v = wide[:, :nkv], wide[:, nkv:2 * nkv]             # views with strides
    room = max(a + b for a, b in zip(lens, start or [0] * n)) + 3
    cache = int4.Int4KVCache(n + 2, room, nkv, hd, dtype, device)
    cache.data.random_(-(1 << 31), (1 << 31) - 1)          # rows that nobody has written
    before = cache.data.clone()
    cu = packed(lens, device)
    slots = torch.randperm(n + 2, generator=g)[:n].int().to(device)
    st = None if start is None else torch.tensor(start, dtype=torch.int32, device=device)
    cache.store(k, v, cu, max(lens), slots=slots, start=st)
    k2, v2 = cache.load(cu, T, max(lens), slots=slots, start=st)
    assert k2.dtype == v2.dtype == dtype and k2.shape == k.shape
    check_groups(k2, k, 32, dtype)
    check_groups(v2, v, 64, dtype)
    # what was there before and behind is as it was: the words that changed are those of the stored rows
    mark = int4.Int4KVCache(n + 2, room, nkv, hd, dtype, device)
    for i, m in enumerate(lens):
        for r in range((start or [0] * n)[i], (start or [0] * n)[i] + m):
            t, q = r // 16, r % 16
            a, b, c, d = (f[int(slots[i]), :, t] for f in mark._fields())
            a[:, q], c[:, q], d[:, q] = 0x10001, 0x10001, 0x10001
            b[:, :, (q & 7) >> 1, q >> 3, :, q & 1] = 1
    halves = lambda x: x.view(torch.int16)   # noqa: E731
    mine = halves(mark.data) == 1
    assert torch.equal(halves(cache.data)[~mine], halves(before)[~mine])
    # a hint that is far off, and none, change nothing
    for hint in (1, 100000, None):
        again = int4.Int4KVCache(n + 2, room, nkv, hd, dtype, device)
        again.store(k, v, cu, hint, slots=slots, start=st)
        assert torch.equal(halves(again.data)[mine], halves(cache.data)[mine])
        k3, v3 = cache.load(cu, T, hint, slots=slots, start=st)
        assert torch.equal(k3, k2) and torch.equal(v3, v2)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_outside_the_cache_are_left_out(device):
    g = torch.Generator().manual_seed(0)
    k, v = (rows(g, 12, 2, 64, dtype=torch.bfloat16, device=device) for _ in range(2))
    cache = int4.Int4KVCache(2, 20, 2, 64, torch.bfloat16, device)
    cu = torch.tensor([1, 5, 9, 11], dtype=torch.int32, device=device)           # tokens 0 and 11 belong to nobody
    slots = torch.tensor([0, 5, 1], dtype=torch.int32, device=device)            # slot 5 is not there
    start = torch.tensor([18, 0, -1], dtype=torch.int32, device=device)          # rows 20, 21 and -1 are not
    cache.store(k, v, cu, 4, slots=slots, start=start)
    k2, v2 = cache.load(cu, 12, 4, slots=slots, start=start)
    held = torch.tensor([1, 2, 10], device=device)
    check_groups(k2[held], k[held], 32, torch.bfloat16)
    gone = torch.tensor([i for i in range(12) if i not in (1, 2, 10)], device=device)
    assert (k2[gone] == 0).all() and (v2[gone] == 0).all()
    one = int4.Int4KVCache(2, 20, 2, 64, torch.bfloat16, device)
    one.store(k[held[:2]], v[held[:2]], packed([2], device), 2, start=start[:1])
    one.store(k[10:11], v[10:11], packed([1], device), 1, slots=slots[2:])
    assert torch.equal(one.data, cache.data)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_cache_bits_are_the_same_on_both_devices(dtype, hd):
    """Values whose quotients lie on and next to ties, groups of one value, of infinities and of NaN: word for word."""
    g = torch.Generator().manual_seed(hd)
    k = torch.randint(-40, 41, (300, 3, hd), generator=g).to(dtype) / 4           # quotients by few-bit steps: many ties
    v = rows(g, 300, 3, hd, dtype=dtype, device="cpu") * (2.0 ** torch.randint(-8, 8, (300, 3, 1), generator=g)).to(dtype)
    k[5, 1, :40], k[6, 0, 3], v[7, 2, 9], v[8, 1, 5] = 2.0, float("inf"), float("nan"), -float("inf")
    cu = packed([300], "cpu")
    a, b = (int4.Int4KVCache(1, 300, 3, hd, dtype, d) for d in ("cpu", "cuda"))
    a.store(k, v, cu)
    b.store(k.cuda(), v.cuda(), cu.cuda(), 300)
    kw, vw, kg, vg = a._fields()
    for x, y in zip((kw, vw), b._fields()[:2]):
        assert torch.equal(x, y.cpu())
    for x, y in zip((kg, vg), b._fields()[2:]):
        for p, q in zip(int4._group_numbers(x, dtype), int4._group_numbers(y.cpu(), dtype)):
            torch.testing.assert_close(p, q, rtol=0, atol=0, equal_nan=True)
    ka, va = a.load(cu, 300)
    kb, vb = b.load(cu.cuda(), 300, 300)
    torch.testing.assert_close(ka, kb.cpu(), rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(va, vb.cpu(), rtol=0, atol=0, equal_nan=True)
    assert kb[6, 0, :32].isnan().all() and not kb[6, 0, 32:].isnan().any() and vb[7, 2, :64].isnan().all() and vb[8, 1, :64].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_group_bits_at_any_size(dtype):
    """Groups of every power of two of the type, the smallest numbers and the widest range among them, word for word as on the CPU: in a cache and in a weight."""
    g = torch.Generator().manual_seed(3)
    bits = torch.randint(0, 1 << 15, (256, 2, 64), generator=g).short().view(dtype)                # numbers of any size, side by side
    bits = torch.where(torch.isfinite(bits), bits, torch.ones_like(bits))
    info = torch.finfo(dtype)
    powers = range(int(math.log2(info.smallest_normal)) - 8, int(math.log2(info.max)) - 3)
    scaled = torch.stack([(rows(g, 2, 64, dtype=torch.float32, device="cpu").double() * 2.0 ** p).to(dtype) for p in powers])
    ties = torch.stack([(torch.randint(-30, 31, (2, 64), generator=g).double() / 2 * 2.0 ** p).to(dtype) for p in powers])
    ends = torch.zeros(4, 2, 64, dtype=dtype)
    ends[0, :, ::2], ends[1, :, ::2], ends[1, :, 1::2], ends[2], ends[3, :, :5] = info.max, info.max, -info.max, -0.0, info.smallest_normal
    x = torch.cat([bits, -bits, scaled, scaled + 1, ties, ends])
    n = x.shape[0]
    a, b = (int4.Int4KVCache(1, n, 2, 64, dtype, d) for d in ("cpu", "cuda"))
    a.store(x, x.flip(0), packed([n], "cpu"))
    b.store(x.cuda(), x.flip(0).cuda(), packed([n], "cuda"))
    for p, q in zip(a.load(packed([n], "cpu"), n), b.load(packed([n], "cuda"), n)):
        assert torch.equal(p, q.cpu())
    for p, q in zip(a._fields()[:2], b._fields()[:2]):
        assert torch.equal(p, q.cpu())
    for group in int4.GROUPS:
        w = x.reshape(-1, 128)
        p, q = int4.Int4Linear(w, group=group), int4.Int4Linear(w.cuda(), group=group)
        for s, t in zip(p.codes(), q.codes()):
            assert torch.equal(s, t.cpu())


# ------------------------------------------------------------------------------------------------ attention


def attend64(q, k, v, scale):
    """q [nq, hd], k / v [n, nkv, hd] -> [nq, hd]; 64 bits."""
    rep = q.shape[0] // k.shape[1]
    k, v = (t.double().repeat_interleave(rep, 1) for t in (k, v))
    return torch.einsum("hn,nhd->hd", torch.softmax(torch.einsum("hd,nhd->hn", q.double(), k) * scale, -1), v)


def turned64(x, cos, sin, rot, interleaved):
    x = x.double()
    c, s = cos.double(), sin.double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    y = (a * c - b * s, b * c + a * s)
    return torch.cat([torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1), x[..., rot:]], -1)


def held64(cache, slot, n):
    """The numbers that the cache holds, not rounded to its type."""
    kw, vw, kg, vg = (f[slot].cpu() for f in cache._fields())
    r = torch.arange(n)
    c = int4.Int4KVCache(1, cache.room, cache.n_kv, cache.hd, cache.dtype, "cpu")
    c.data.copy_(cache.data[slot: slot + 1].cpu())
    k, v = c._get(torch.zeros(n, dtype=torch.long), r)
    return k.double(), v.double()


def check_step(cache, qkv, lens, nq, nkv, hd, scale=None, cos=None, sin=None, rot=None, interleaved=False):
    """One step against 64 bits over what the cache holds afterwards, and the new rows.

    Bound of the outputs: their rounding, u relative, and what fp32 scores and sums leave: scores |s| < 64 hold sums of 128 products and of a few factors, each of
    relative error 2^-22 or less (queries in parts of 22 bits), so weights differ by less than 64 * 2 * 2^-22 * 2 < 1e-4 relative at the very most and by a
    tenth of that where errors do not all agree: 1e-5 of the largest value."""
    B, dtype = len(lens), cache.dtype
    scale = hd ** -0.5 if scale is None else scale
    before = cache.data.clone()
    kw = {} if cos is None else dict(cos=cos, sin=sin, rot_dim=rot, interleaved=interleaved)
    out = int4.decode_attention_int4(qkv, cache, torch.tensor(lens, dtype=torch.int32, device=qkv.device), nq, nkv, hd, scale, **kw).cpu().view(B, nq, hd)
    q, k, v = (t.reshape(B, -1, hd).cpu() for t in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    for b, n in enumerate(lens):
        if not 0 <= n < cache.room:
            assert (out[b] == 0).all() and torch.equal(cache.data[b], before[b])
            continue
        kk, vv = held64(cache, b, n + 1)
        kn, qn = k[b], q[b].double()
        if cos is not None:
            kn = int4._rotated(k[b: b + 1].float(), cos[n: n + 1].cpu(), sin[n: n + 1].cpu(), rot, interleaved).to(dtype)[0]
            qn = turned64(q[b], cos[n].cpu(), sin[n].cpu(), rot, interleaved)
        check_groups(kk[n], kn, 32, dtype, rounded=False)
        check_groups(vv[n], v[b], 64, dtype, rounded=False)
        ref = attend64(qn, kk, vv, scale)
        bound = EPS[dtype] * ref.abs() + SMALL[dtype] + 1e-5 * vv.abs().amax(0).amax(-1).repeat_interleave(nq // nkv)[:, None]
        assert bool(((out[b].double() - ref).abs() <= bound).all()), (b, n, float(((out[b].double() - ref).abs() - bound).max()))
        old = int4.Int4KVCache(1, cache.room, nkv, hd, dtype, "cpu")
        old.data.copy_(before[b: b + 1].cpu())
        if n:
            a, c = old._get(torch.zeros(n, dtype=torch.long), torch.arange(n))
            torch.testing.assert_close(kk[:n], a.double(), rtol=0, atol=0, equal_nan=True)
            torch.testing.assert_close(vv[:n], c.double(), rtol=0, atol=0, equal_nan=True)
    return out


def filled(g, B, room, nkv, hd, dtype, device, scale=1.0):
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, device)
    k, v = (rows(g, B * room, nkv, hd, dtype=dtype, device=device, outliers=i == 0) * scale for i in range(2))
    cache.store(k, v, packed([room] * B, device), room)
    return cache


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,nkv,hd,room", [(4, 4, 64, 70), (6, 3, 128, 131), (7, 1, 64, 300), (14, 2, 128, 33), (8, 1, 128, 40), (12, 1, 64, 50), (20, 1, 128, 66), (5, 5, 128, 1),
                                            (10, 2, 64, 90)])
def test_decode_lengths_and_groups(device, dtype, nq, nkv, hd, room):
    """Lengths of zero, around tiles of 16, the last row, and outside; groups of 1 to 20 queries."""
    g = torch.Generator().manual_seed(nq * 10 + hd)
    lens = [n for n in (0, 1, 14, 15, 16, 17, 31, 32, 63, 64, 65, 128) if n < room] + [room - 1, room, -1]
    cache = filled(g, len(lens), room, nkv, hd, dtype, device)
    qkv = rows(g, len(lens), (nq + 2 * nkv), hd, dtype=dtype, device=device).view(len(lens), -1)
    qkv[:, : nq * hd] *= 2
    check_step(cache, qkv, lens, nq, nkv, hd)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (128, 64), (128, 32), (64, 16)])
def test_decode_rotations(device, interleaved, hd, rot):
    from realhf_b200.ops import functional as OF
    g = torch.Generator().manual_seed(rot)
    nq, nkv, room = 6, 2, 100
    lens = [0, 3, 99, 50]
    cache = filled(g, 4, room, nkv, hd, torch.bfloat16, device)
    cos, sin = OF.rope_tables(128, rot, 10000.0, device)
    wide = rows(g, 4, nq + 2 * nkv + 1, hd, dtype=torch.bfloat16, device=device).view(4, -1)
    check_step(cache, wide[:, : (nq + 2 * nkv) * hd], lens, nq, nkv, hd, 0.2, cos, sin, rot, interleaved)


@pytest.mark.parametrize("device", DEVICES)
def test_decode_rows_that_hold_infinities_and_nan(device):
    """A key group that is NaN makes its head's scores NaN; a value group its own channels; other heads and sequences are not touched.  Rows behind the length may hold
    anything."""
    g = torch.Generator().manual_seed(3)
    nq, nkv, hd, room, B = 4, 2, 128, 80, 4
    cache = filled(g, B, room, nkv, hd, torch.bfloat16, device)
    lens = [70, 70, 70, 33]
    k, v = (rows(g, 2, nkv, hd, dtype=torch.bfloat16, device=device) for _ in range(2))
    k[0, 1, 5], v[1, 0, 70] = float("nan"), float("inf")
    cu, st = packed([1, 1], device), torch.tensor([20, 40], dtype=torch.int32, device=device)
    cache.store(k, v, cu, 1, start=st)                                        # slots 0 and 1
    for f in cache._fields():                                                 # behind the length of sequence 3: all bits set, NaN among them
        f[3, :, 3:] = -1
    qkv = rows(g, B, nq + 2 * nkv, hd, dtype=torch.bfloat16, device=device).view(B, -1)
    out = int4.decode_attention_int4(qkv, cache, torch.tensor(lens, dtype=torch.int32, device=device), nq, nkv, hd).view(B, nq, hd).cpu()
    for b, n in enumerate(lens):
        kk, vv = held64(cache, b, n + 1)
        ref = attend64(qkv[b, : nq * hd].view(nq, hd).cpu(), kk, vv, hd ** -0.5)
        assert torch.equal(out[b].isnan(), ref.isnan())
        ok = ~ref.isnan()
        assert bool(((out[b].double() - ref).abs()[ok] <= (2.0 ** -8 * ref.abs() + 1e-4)[ok]).all())
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and out[1, :2, 64:].isnan().all() and not out[1, :2, :64].isnan().any() and not out[2:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [-40, -12, 0, 10])
def test_decode_values_of_any_size(dtype, power):
    """Values far below and above one, and a sequence in which they grow by 2^12 from tile to tile and shrink again: the bound is relative to the largest value in reach."""
    if dtype == torch.float16 and power == -40:
        pytest.skip("below fp16's range")
    g = torch.Generator().manual_seed(power + 50)
    nq, nkv, hd, room = 8, 2, 128, 200
    cache = int4.Int4KVCache(3, room, nkv, hd, dtype, "cuda")
    k, v = (rows(g, 3 * room, nkv, hd, dtype=dtype, device="cuda") for _ in range(2))
    v *= 2.0 ** power
    if power == 0:
        v[room:2 * room] *= (2.0 ** (torch.arange(room, device="cuda") // 16 % 5 * 3 - 6.0)).to(dtype)[:, None, None]
        v[2 * room:] = 0
    cache.store(k, v, packed([room] * 3, "cuda"), room)
    qkv = rows(g, 3, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(3, -1)
    qkv[:, -nkv * hd:] *= 2.0 ** power
    check_step(cache, qkv, [room - 1, room - 2, 150], nq, nkv, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,nq,nkv,hd,room", [(1, 8, 1, 128, 9000), (2, 4, 4, 64, 5001), (1, 32, 8, 128, 4096), (300, 2, 2, 64, 40), (64, 32, 32, 128, 130), (200, 4, 4, 64, 300), (256, 8, 2, 128, 33),
                                               (33, 64, 64, 64, 50)])
def test_decode_long_and_wide(dtype, B, nq, nkv, hd, room):
    """Few long sequences (split over blocks) and many short ones."""
    g = torch.Generator().manual_seed(B + room)
    cache = filled(g, B, room, nkv, hd, dtype, "cuda")
    lens = torch.randint(0, room, (B,), generator=g).tolist()
    lens[0] = room - 1
    qkv = rows(g, B, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(B, -1)
    check_step(cache, qkv, lens[:B], nq, nkv, hd)


@pytest.mark.gpu
def test_decode_at_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes: the last slot's rows lie where they should."""
    g = torch.Generator().manual_seed(9)
    nq, nkv, hd, room, B = 2, 2, 128, 16 * 4000, 16                            # 2 x 4000 tiles of 2432 bytes a slot: 311 MB of 4.98 GB
    cache = int4.Int4KVCache(B, room, nkv, hd, torch.bfloat16, "cuda")
    n = 1000
    k, v = (rows(g, n, nkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cu, slot = packed([n], "cuda"), torch.tensor([B - 1], dtype=torch.int32, device="cuda")
    cache.store(k, v, cu, n, slots=slot)
    k2, v2 = cache.load(cu, n, n, slots=slot)
    check_groups(k2, k, 32, torch.bfloat16)
    st = torch.tensor([room - n], dtype=torch.int32, device="cuda")
    cache.store(k, v, cu, n, slots=slot, start=st)
    assert torch.equal(cache.load(cu, n, n, slots=slot, start=st)[0], k2)
    assert int(cache.data[: B - 1].count_nonzero()) == 0
    lens = [-1] * (B - 1) + [n]
    qkv = rows(g, B, nq + 2 * nkv, hd, dtype=torch.bfloat16, device="cuda").view(B, -1)
    out = int4.decode_attention_int4(qkv, cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), nq, nkv, hd).view(B, nq, hd)
    kk, vv = held64(cache, B - 1, n + 1)
    ref = attend64(qkv[B - 1, : nq * hd].view(nq, hd).cpu(), kk, vv, hd ** -0.5)
    assert bool(((out[B - 1].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-4).all())


@pytest.mark.gpu
def test_decode_captured_and_replayed():
    """A captured step reads its lengths and projections anew at each replay; two graphs on two streams."""
    g = torch.Generator().manual_seed(11)
    nq, nkv, hd, room, B = 8, 2, 128, 300, 3
    caches = [filled(g, B, room, nkv, hd, torch.bfloat16, "cuda") for _ in range(2)]
    twins = []
    for c in caches:
        t = int4.Int4KVCache(B, room, nkv, hd, torch.bfloat16, "cuda")
        t.data.copy_(c.data)
        twins.append(t)
    lens = [torch.full((B,), 250, dtype=torch.int32, device="cuda") for _ in range(2)]
    qkv = [torch.zeros(B, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    int4.decode_attention_int4(qkv[0], caches[0], torch.full((B,), -1, dtype=torch.int32, device="cuda"), nq, nkv, hd)   # (loaded outside the capture)
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(int4.decode_attention_int4(qkv[i], caches[i], lens[i], nq, nkv, hd))
            lens[i] += 1
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(3):
        for i in range(2):
            qkv[i].copy_(rows(g, B, nq + 2 * nkv, hd, dtype=torch.bfloat16, device="cuda").view(B, -1))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = int4.decode_attention_int4(qkv[i], twins[i], torch.full((B,), 250 + step, dtype=torch.int32, device="cuda"), nq, nkv, hd)
            assert torch.equal(want, outs[i]) and torch.equal(twins[i].data, caches[i].data)


# ------------------------------------------------------------------------------------------------ weights


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (33, 192, 64), (300, 1024, 64), (40, 896, 128)])
def test_weight_round_trip(device, dtype, N, K, group):
    g = torch.Generator().manual_seed(N + K)
    w = (rows(g, N, K + 8, dtype=dtype, device=device) * 0.1)[:, :K]           # strided rows
    lin = int4.Int4Linear(w, group=group)
    y = lin.dequantize()
    check_groups(y, w, group, dtype, rounded=False)
    c, s, lo = (t.cpu() for t in int4.quantize_groups(w.cpu(), group))
    for a, b in zip(lin.codes(), (c, s, lo)):
        assert torch.equal(a.cpu(), b)
    again = int4.Int4Linear.from_codes(*lin.codes())
    assert torch.equal(again.q, lin.q)
    lin.requantize(w * 2)
    check_groups(lin.dequantize(), w * 2, group, dtype, rounded=False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (33, 192, 64), (130, 384, 128), (300, 160, 32)])
def test_weights_of_codes(device, dtype, N, K, group):
    g = torch.Generator().manual_seed(N)
    c = torch.randint(0, 16, (N, K + 3), generator=g, dtype=torch.uint8).to(device)[:, 3:]          # strided, off by three bytes
    s, lo = (rows(g, K // group, N, dtype=dtype, device=device).t() for _ in range(2))
    lin = int4.Int4Linear.from_codes(c, s, lo)
    for a, b in zip(lin.codes(), (c, s, lo)):
        assert torch.equal(a, b)
    assert torch.equal(lin.q.cpu(), int4.Int4Linear.from_codes(c.cpu(), s.cpu(), lo.cpu()).q)       # ... and zeros beyond N and K


def check_linear(lin, x, bias=None):
    """Against 64 bits over the numbers that the weight holds.  Bound: the output's rounding, and sums in fp32 of K products whose factors hold 22 bits or more: each
    product and partial sum is off by 2^-22 of its size at most, errors of sqrt(K) partial sums add up: 2^-22 sqrt(K) sum |x w| is far above what is seen."""
    y = lin(x, bias) if bias is not None else lin(x)
    w, x2 = lin.dequantize().double().cpu(), x.reshape(-1, lin.K).double().cpu()
    b = lin.bias if bias is None else bias
    ref, size = x2 @ w.t(), x2.abs() @ w.abs().t()
    # (codes and lowest values are summed apart and cancel: the sizes of both count)
    size = size + 2 * x2.abs() @ torch.ones(lin.K, 1, dtype=torch.float64) * w.abs().amax(1)
    if b is not None:
        ref = ref + b.double().cpu()
    got = y.reshape(-1, lin.N).double().cpu()
    bound = EPS[lin.dtype] * ref.abs() + SMALL[lin.dtype] + 2.0 ** -22 * size
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], lin.N)
    assert bool(((got - ref).abs() <= bound).all()), float(((got - ref).abs() - bound).max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 32, 32), (1, 16, 128, 128), (2, 17, 160, 32), (3, 300, 896, 128), (8, 64, 256, 64), (9, 129, 192, 64), (16, 48, 1024, 32),
                                         (33, 100, 128, 128), (65, 40, 384, 64), (130, 20, 256, 128), (0, 16, 128, 128)])
def test_linear(device, dtype, M, N, K, group):
    g = torch.Generator().manual_seed(M + N + K)
    w = rows(g, N, K, dtype=dtype, device=device) * K ** -0.5
    bias = rows(g, N, 1, dtype=dtype, device=device)[:, 0] if M % 2 else None
    lin = int4.Int4Linear(w, bias, group)
    x = rows(g, M, K + 8, dtype=dtype, device=device)[:, :K]
    check_linear(lin, x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group", [(1, 4096, 4096, 128), (7, 5000, 1024, 32), (16, 22016, 4096, 128), (128, 4096, 11008, 64), (32, 300, 11008, 128), (5, 50257, 768, 64),
                                         (24, 12288, 4096, 128), (63, 2000, 14336, 128), (1, 40, 16384, 128)])
def test_linear_sizes_of_models(dtype, M, N, K, group):
    g = torch.Generator().manual_seed(M + N + K)
    lin = int4.Int4Linear(rows(g, N, K, dtype=dtype, device="cuda") * K ** -0.5, group=group)
    check_linear(lin, rows(g, M, K, dtype=dtype, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_rows_of_any_size(dtype):
    """Rows of very large and very small numbers side by side, rows of zeros, and infinities and NaN, which stay in their rows."""
    g = torch.Generator().manual_seed(4)
    N, K = 80, 1024
    lin = int4.Int4Linear(rows(g, N, K, dtype=dtype, device="cuda"), group=64)
    x = rows(g, 12, K, dtype=dtype, device="cuda").float()
    x *= (2.0 ** torch.tensor([0, 30, -30, 5, 0, -10, 0, 8, 0, -20, 3, 0] if dtype == torch.bfloat16 else [0, 3, -12, 5, 0, -10, 0, 2, 0, -9, 3, 0], device="cuda"))[:, None]
    x[4] = 0
    x[6, ::2] *= 2.0 ** -12
    check_linear(lin, x.to(dtype))
    x[8, 100], x[10, 3] = float("inf"), float("nan")
    y = lin(x.to(dtype))
    assert not torch.isfinite(y[8]).any() and y[10].isnan().all()
    keep = [i for i in range(12) if i not in (8, 10)]
    assert torch.isfinite(y[keep]).all() and torch.equal(y[keep], lin(x.to(dtype)[keep].contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,group", [(17, 32), (40, 128), (100, 64)])
def test_many_rows_of_any_size(dtype, M, group):
    g = torch.Generator().manual_seed(M)
    lin = int4.Int4Linear(rows(g, 200, 1152 + group, dtype=dtype, device="cuda"), group=group)
    x = rows(g, M, lin.K, dtype=dtype, device="cuda").float()
    x *= (2.0 ** torch.randint(-12, 4, (M, 1), generator=g)).cuda()
    x[4] = 0
    check_linear(lin, x.to(dtype))
    x[8, 100], x[10, 3], x[M - 1, lin.K - 1] = float("inf"), float("nan"), -float("inf")
    y = lin(x.to(dtype))
    bad = [8, 10, M - 1]
    assert not torch.isfinite(y[bad]).any()
    keep = [i for i in range(M) if i not in bad]
    x[bad] = 0
    assert torch.isfinite(y[keep]).all() and torch.equal(y[keep], lin(x.to(dtype))[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [5, 20, 128])
def test_linear_of_the_widest_groups(dtype, M):
    """Steps beyond an eighth of the type's largest number, and of the smallest ones.  Where there are more than 16 rows, 8 steps would overflow there and are two halves, the second of
    which is rounded to the type: off by EPS of half of |scale (c - 8)| <= 8 scale more than `check_linear` allows (and a factor 1 + EPS for the half that was rounded)."""
    g = torch.Generator().manual_seed(M)
    big = 0.97 * torch.finfo(dtype).max
    w = (torch.rand(40, 256, generator=g).double() * 2 - 1) * big
    w[:, ::32], w[:, 1::32] = big, -big
    lin = int4.Int4Linear(w.to(dtype).cuda(), group=32)
    limit = torch.finfo(dtype).max / 8
    assert float(lin.codes()[1].double().min()) > limit
    x = (torch.randn(M, 256, generator=g).double() * 2.0 ** (-14 if dtype == torch.float16 else -120)).to(dtype).cuda()
    y, wd, x2 = lin(x).double().cpu(), lin.dequantize().double().cpu(), x.double().cpu()
    ref, size = x2 @ wd.t(), 3 * x2.abs().sum(1, keepdim=True) * wd.abs().amax(1)
    extra = EPS[dtype] / 2 * (1 + EPS[dtype]) * x2.abs().sum(1, keepdim=True) * 8 * lin.codes()[1].double().cpu().amax(1) if M > 16 else 0
    assert bool(((y - ref).abs() <= EPS[dtype] * ref.abs() + SMALL[dtype] + 2.0 ** -22 * size + extra).all())
    if dtype == torch.float16:                              # steps that are subnormal numbers: products are taken whole
        lin = int4.Int4Linear((torch.randn(40, 256, generator=g) * 2.0 ** -17).to(dtype).cuda(), group=32)
        check_linear(lin, torch.randn(M, 256, generator=g).to(dtype).cuda() * 64)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 20, 64, 150])
def test_linear_captured_on_two_streams(M):
    """Two graphs of one weight, replayed at once, and a weight quantised anew between the replays."""
    g = torch.Generator().manual_seed(M)
    w = [rows(g, 700, 2048, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    lin, xs = int4.Int4Linear(w[0]), [rows(g, M, 2048, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    want = [[int4.Int4Linear(v)(x) for x in xs] for v in w]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    lin(xs[0])
    for gr, x in zip(graphs, xs):
        with torch.cuda.graph(gr):
            outs.append(lin(x))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for v, ref in zip(w, want):
        lin.requantize(v)
        torch.cuda.synchronize()
        for _ in range(3):
            for gr, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref[0]) and torch.equal(outs[1], ref[1])


@pytest.mark.gpu
def test_linear_of_leading_dimensions_streams_and_graphs():
    g = torch.Generator().manual_seed(5)
    lin = int4.Int4Linear(rows(g, 500, 512, dtype=torch.bfloat16, device="cuda"), rows(g, 500, 1, dtype=torch.bfloat16, device="cuda")[:, 0])
    x = rows(g, 6, 512, dtype=torch.bfloat16, device="cuda")
    y = lin(x)
    assert torch.equal(lin(x.view(2, 3, 512)), y.view(2, 3, 500))
    other = rows(g, 500, 1, dtype=torch.bfloat16, device="cuda")[:, 0]
    check_linear(lin, x, other)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = lin(x)
    s.synchronize()
    assert torch.equal(z, y)
    graphs, outs, xs = [], [], [x.clone(), x.clone()]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(lin(xs[i]))
        graphs.append(gr)
    xs[1] *= 2
    want = lin(xs[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], y) and torch.equal(outs[1], want)
    lin.requantize(rows(g, 500, 512, dtype=torch.bfloat16, device="cuda"))     # (a kept graph reads the weight anew)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], lin(x)) and not torch.equal(outs[0], y)


# ------------------------------------------------------------------------------------------------ refusals


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    bf, z = torch.bfloat16, lambda *s, **k: torch.zeros(*s, device=device, **{"dtype": torch.bfloat16, **k})   # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)   # noqa: E731
    for bad in (dict(hd=96), dict(dtype=torch.float32), dict(n_kv=0), dict(slots=-1), dict(room=-1)):
        with pytest.raises(ValueError):
            int4.Int4KVCache(**{**dict(slots=1, room=8, n_kv=1, hd=64, dtype=bf, device=device), **bad})
    c = int4.Int4KVCache(2, 8, 2, 64, bf, device)
    for k, v, cu, kw in ((z(3, 2, 128), z(3, 2, 128), i32(0, 3), {}), (z(3, 1, 64), z(3, 1, 64), i32(0, 3), {}), (z(3, 2, 64), z(2, 2, 64), i32(0, 3), {}),
                         (z(3, 2, 64, dtype=torch.float16), z(3, 2, 64, dtype=torch.float16), i32(0, 3), {}), (z(3, 2, 64), z(3, 2, 64), z(0, dtype=torch.int32), {}),
                         (z(3, 2, 64), z(3, 2, 64), i32(0, 3), dict(slots=i32(0, 1))), (z(3, 2, 64), z(3, 2, 64), i32(0, 3), dict(start=i32()))):
        with pytest.raises(ValueError):
            c.store(k, v, cu, **kw)
    with pytest.raises(ValueError):
        c.load(i32(0, 3), -1)
    tab = torch.zeros(8, 32, device=device)
    for qkv, lens, a, kw in ((z(2, 8 * 64), i32(0, 0), (4, 2, 64), dict(cos=tab)), (z(2, 8 * 64), i32(0, 0), (4, 2, 64), dict(cos=tab[:4], sin=tab[:4])),
                             (z(2, 8 * 64), i32(0, 0), (4, 2, 64), dict(cos=tab, sin=tab, rot_dim=32)), (z(2, 8 * 64), i32(0, 0), (4, 2, 128), {}),
                             (z(3, 8 * 64), i32(0, 0, 0), (4, 2, 64), {}), (z(2, 7 * 64), i32(0, 0), (3, 2, 64), {}), (z(2, 8 * 64), i32(0), (4, 2, 64), {}),
                             (z(2, 9 * 64), i32(0, 0), (4, 2, 64), {})):
        with pytest.raises(ValueError):
            int4.decode_attention_int4(qkv, c, lens, *a, **kw)
    for w, kw in ((z(4, 100), {}), (z(4, 128, dtype=torch.float32), {}), (z(128), {}), (z(0, 128), {}), (z(4, 128), dict(group=16)), (z(4, 128), dict(bias=z(3))),
                  (z(4, 128), dict(bias=z(4, dtype=torch.float32)))):
        with pytest.raises(ValueError):
            int4.Int4Linear(w, **kw)
    lin = int4.Int4Linear(z(4, 128))
    with pytest.raises(ValueError):
        lin(z(3, 64))
    with pytest.raises(ValueError):
        lin.requantize(z(4, 256))
    for codes, s in ((z(4, 128, dtype=torch.uint8) + 16, z(4, 1)), (z(4, 128, dtype=torch.int32), z(4, 1)), (z(4, 128, dtype=torch.uint8), z(4, 3)), (z(4, 128, dtype=torch.uint8), z(3, 1))):
        with pytest.raises(ValueError):
            int4.Int4Linear.from_codes(codes, s, s)


@pytest.mark.parametrize("device", DEVICES)
def test_no_gradient_is_refused_not_lost(device):
    z = lambda *s: torch.zeros(*s, device=device, dtype=torch.bfloat16)   # noqa: E731
    w = z(16, 128).requires_grad_()
    lin, c, lens = int4.Int4Linear(w), int4.Int4KVCache(1, 8, 1, 64, torch.bfloat16, device), torch.zeros(1, dtype=torch.int32, device=device)
    lin.requantize(w)
    c.store(z(3, 1, 64).requires_grad_(), z(3, 1, 64), packed([3], device))
    for f, x in ((lin, z(2, 128).requires_grad_()), (lambda t: int4.decode_attention_int4(t, c, lens, 2, 1, 64), z(1, 256).requires_grad_())):
        with pytest.raises(RuntimeError):
            f(x)
        with torch.no_grad():
            assert not f(x).requires_grad
        f(x.detach())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M", [3, 20, 70, 130])
def test_linear_of_repeated_and_overlapping_rows(device, M):
    g = torch.Generator().manual_seed(M)
    lin = int4.Int4Linear(rows(g, 48, 256, dtype=torch.bfloat16, device=device) * 0.1, group=64)
    flat = rows(g, 256 + 8 * M, dtype=torch.bfloat16, device=device)
    check_linear(lin, flat[:256].expand(M, 256))
    check_linear(lin, flat.as_strided((M, 256), (8, 1)))
    check_linear(lin, flat[:256].expand(2, M, 256))


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    """What Python's checks let through to the binding: devices and types that do not go together."""
    from realhf_b200.ops import lib
    c = int4.Int4KVCache(1, 8, 1, 64, torch.bfloat16, "cuda")
    with pytest.raises(ValueError):
        int4.decode_attention_int4(torch.zeros(1, 3 * 64, device="cuda"), c, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 1, 64)
    with pytest.raises(ValueError):
        int4.Int4Linear(torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16))(torch.zeros(4, 128, device="cuda"))
    with pytest.raises(ValueError):
        lib().decode_attention_int4(torch.zeros(1, 192, device="cuda", dtype=torch.bfloat16), c.data, torch.zeros(1, dtype=torch.int32), 1, 1, 64, 8, 1.0, None, None, 64, False)
    with pytest.raises(ValueError):
        lib().int4_linear(torch.zeros(1, 128, device="cuda", dtype=torch.bfloat16), c.data, None, 4, 128)
    with pytest.raises(ValueError):
        lib().int4_cache_store(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), c.data, torch.zeros(2, dtype=torch.int32), None, None, 8, 64, 1)
