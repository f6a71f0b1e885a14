"""4-bit caches whose numbers lie near the ends of their types, against 64 bits over what the cache holds."""
import pytest
import torch

from realhf_b200.ops import int4
from test_int4 import EPS, SMALL, TYPES, check_step, packed, rows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [100.0, -1000.0, 65504.0, 2.0 ** 100])
def test_decode_of_many_rows_of_one_value(dtype, hd, value):
    """Value groups with a step of 0 and a lowest value far from 0, thousands of them in one warp (more works than the GPU has places, so that none is split), some of them behind rows
    of ordinary steps.  All weights are about the same: outputs are means of n rows.  Sums of n numbers of one size in fp32 are off by n 2^-24 relative at the very most, 1.8e-4 for
    3000 rows, and the numbers of a lane, four warps' shares and so on are added up apart: a quarter of that."""
    value = torch.tensor(value if dtype == torch.bfloat16 else max(min(value, 65504.0), -65504.0)).to(dtype).item()
    g = torch.Generator().manual_seed(hd)
    B, nq, nkv, room = 320, 4, 4, 3000
    one = int4.Int4KVCache(1, room, nkv, hd, dtype, "cuda")
    k, v = rows(g, room, nkv, hd, dtype=dtype, device="cuda"), torch.full((room, nkv, hd), value, dtype=dtype, device="cuda")
    v[: room // 3, 2:] = rows(g, room // 3, nkv - 2, hd, dtype=dtype, device="cuda")
    one.store(k, v, packed([room], "cuda"), room)
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, "cuda")
    cache.data.copy_(one.data.expand_as(cache.data))
    qkv = rows(g, 1, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(1, -1) * 0.01
    qkv[:, -nkv * hd:] = value
    out = int4.decode_attention_int4(qkv.expand(B, -1), cache, torch.full((B,), room - 1, dtype=torch.int32, device="cuda"), nq, nkv, hd).view(B, nq, hd)
    kk, vv = (t[0].double() for t in _held(cache, room))
    w = torch.softmax(torch.einsum("hd,nhd->hn", qkv[0, : nq * hd].view(nq, hd).double(), kk) * hd ** -0.5, -1)
    ref = torch.einsum("hn,nhd->hd", w, vv)
    assert torch.isfinite(out).all()
    assert bool(((out.double() - ref).abs() <= EPS[dtype] * ref.abs() + SMALL[dtype] + 4.5e-5 * vv.abs().amax()).all())


def _held(cache, n):
    """The numbers of the first n rows of slot 0, in 64 bits, [1, n, heads, channels]."""
    c = int4.Int4KVCache(1, cache.room, cache.n_kv, cache.hd, cache.dtype, cache.device)
    c.data.copy_(cache.data[:1])
    return (t[None].double() for t in c._get(torch.zeros(n, dtype=torch.long, device=cache.device), torch.arange(n, device=cache.device)))


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv", [(4, 4), (6, 3), (4, 1), (8, 1)])
@pytest.mark.parametrize("power", [112, 116, 118, 120])
def test_decode_of_the_largest_values(nq, nkv, power):
    """Values up to 2^123 and steps beyond 2^114: sums of them stay inside fp32 (40 rows, weights of 2^4 at most: below 2^5.4 2^4 of a value, and most weights are far smaller)."""
    g = torch.Generator().manual_seed(power + nq)
    hd, room, B, dtype = 128, 40, 3, torch.bfloat16
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, "cuda")
    k, v = (rows(g, B * room, nkv, hd, dtype=dtype, device="cuda") for _ in range(2))
    v[: B * room // 2] *= 2.0 ** power
    v[B * room // 2:] *= 2.0 ** (power - 3)
    cache.store(k, v, packed([room] * B, "cuda"), room)
    qkv = rows(g, B, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(B, -1)
    qkv[:, -nkv * hd:] *= 2.0 ** power
    check_step(cache, qkv, [room - 1, 20, 0], nq, nkv, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 2), (8, 1)])
@pytest.mark.parametrize("power,one_value", [(122, False), (124, True), (119, False), (-78, False), (-100, False)])
def test_decode_of_the_largest_and_smallest_queries(nq, nkv, power, one_value):
    """Queries of 2^power against keys of 2^-power: scores of ordinary size.  With one value throughout, the sum of a query over 32 channels, which the keys' lowest values are taken by,
    is 2^5 times an element."""
    g = torch.Generator().manual_seed(power + 200 + nq)
    hd, room, B, dtype = 128, 70, 3, torch.bfloat16
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, "cuda")
    k, v = (rows(g, B * room, nkv, hd, dtype=dtype, device="cuda") for _ in range(2))
    cache.store(k * 2.0 ** -power, v, packed([room] * B, "cuda"), room)
    qkv = rows(g, B, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(B, -1)
    if one_value:
        qkv[:, : nq * hd] = 1
    qkv[:, : nq * hd] *= 2.0 ** power
    qkv[:, nq * hd: (nq + nkv) * hd] *= 2.0 ** -power
    check_step(cache, qkv, [room - 1, 31, 0], nq, nkv, hd, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv", [(4, 4), (6, 2), (8, 1)])
@pytest.mark.parametrize("room,low", [(1, -1.0), (40, -1.0), (1, 0.5), (500, 0.25), (1000, 1.0), (1000, -0.5)])
def test_decode_of_sums_beyond_fp32(nq, nkv, room, low):
    """Values up to 0.97 of bfloat16's largest number, groups that span the whole type among them: their means are finite, sums over rows are not in fp32.  The parts of a value (lowest value
    and 15 steps) are rounded apart, 2^-23 of twice the largest number, on top of what `check_step` allows relative to it: 1e-5 covers it."""
    g = torch.Generator().manual_seed(room + nq)
    hd, B, dtype = 128, 160, torch.bfloat16
    most = 0.97 * torch.finfo(dtype).max
    one = int4.Int4KVCache(1, room, nkv, hd, dtype, "cuda")
    k, v = rows(g, room, nkv, hd, dtype=dtype, device="cuda"), torch.full((room, nkv, hd), most, device="cuda")
    v[..., ::3] *= low
    one.store(k, v.to(dtype), packed([room], "cuda"), room)
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, "cuda")
    cache.data.copy_(one.data.expand_as(cache.data))
    qkv = (rows(g, 1, nq + 2 * nkv, hd, dtype=dtype, device="cuda").view(1, -1) * 0.25).expand(B, -1).contiguous()
    qkv[:, -nkv * hd:] = v[0].to(dtype).flatten()
    check_step(cache, qkv, [room - 1] + [-1] * (B - 1), nq, nkv, hd)
    check_step(cache, qkv, [room - 1] * 2 + [room // 2] * (B - 2), nq, nkv, hd)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", [0.0, -1.0, -0.5, -0.25, -0.77, 0.3])
def test_finite_numbers_read_back_finite(device, dtype, low):
    """Groups up to the type's largest number whose step is rounded up: 15 steps above the lowest value are more than that number, off by 15 roundings of the step at most.  Outputs of
    the attention, means of such values, are finite too; infinities stay NaN."""
    most, nkv, hd, room = torch.finfo(dtype).max, 2, 64, 20
    x = torch.full((room, nkv, hd), most)
    x[..., ::2] *= low
    x = x.to(dtype).to(device)
    cache = int4.Int4KVCache(1, room, nkv, hd, dtype, device)
    cu = packed([room], device)
    cache.store(x, -x, cu, room)
    k, v = cache.load(cu, room, room)
    for got, want in ((k, x), (v, -x)):
        assert torch.isfinite(got).all()
        assert bool(((got.double() - want.double()).abs() <= 15 * EPS[dtype] * 2 * most / 15 + EPS[dtype] * most).all())
    cache.store(torch.zeros_like(x), x, cu, room)
    qkv = torch.cat([torch.zeros(1, 2 * nkv * hd, dtype=dtype, device=device), x[:1].reshape(1, -1)], 1)
    out = int4.decode_attention_int4(qkv, cache, torch.tensor([room - 1], dtype=torch.int32, device=device), nkv, nkv, hd).view(nkv, hd)
    assert torch.isfinite(out).all()
    assert bool(((out.double() - x[0].double()).abs() <= 15 * EPS[dtype] * 2 * most / 15 + 2 * EPS[dtype] * most).all())
    bad = x.clone()
    bad[3, 1, 5] = float("inf")
    cache.store(bad, bad, cu, room)
    k, v = cache.load(cu, room, room)
    assert k[3, 1, :32].isnan().all() and v[3, 1].isnan().all() and int(k.isnan().sum()) == 32 and int(v.isnan().sum()) == 64


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 4), (8, 2), (8, 1)])
def test_decode_sums_are_rounded_not_cut(nq, nkv, hd):
    """Means of 4000 rows of one warp whose values cancel to a thousandth of their size, so that fp16 shows the sums' own errors.  A value is a code times its step and the lowest value, summed
    apart: 2.5 of either a row at most here.  250 partial sums rounded to nearest are off by 2^-24 of that each at most, at random: 2^-24 / sqrt(3) sqrt(250) is a standard deviation, of which six
    are allowed for each of the two sums; what is cut off within a tile's products, 2^-23 of them and two parts, is a bias of 2^-22 of a sum.  Weights of equal scores are equal.  The mean error
    over all channels has a standard deviation smaller by the root of their number: what is left of it is a bias."""
    g = torch.Generator().manual_seed(nq + hd)
    B, room, dtype = 1300 // nkv + 20, 4000, torch.float16
    x = rows(g, room // 2, nkv, hd, dtype=dtype, device="cuda")
    one = int4.Int4KVCache(1, room, nkv, hd, dtype, "cuda")
    one.store(rows(g, room, nkv, hd, dtype=dtype, device="cuda"), torch.stack([x, -x], 1).flatten(0, 1), packed([room], "cuda"), room)
    cache = int4.Int4KVCache(B, room, nkv, hd, dtype, "cuda")
    cache.data.copy_(one.data.expand_as(cache.data))
    qkv = torch.zeros(B, (nq + 2 * nkv) * hd, dtype=dtype, device="cuda")
    qkv[:, -nkv * hd:] = -x[-1].flatten()
    out = int4.decode_attention_int4(qkv, cache, torch.full((B,), room - 1, dtype=torch.int32, device="cuda"), nq, nkv, hd).view(B, nq, hd)
    ref = next(t for i, t in enumerate(_held(cache, room)) if i)[0].mean(0).repeat_interleave(nq // nkv, 0)
    bound = 2.5 * (2 * 6 * 2.0 ** -24 * (250 / 3) ** 0.5 + 2 * 2.0 ** -22)
    worst = float(((out.double() - ref).abs() - EPS[dtype] * ref.abs()).max())
    bias, most = abs(float((out.double() - ref)[0].mean())), 2.5 * (2 * 6 * 2.0 ** -24 * (250 / 3) ** 0.5 / (nkv * hd) ** 0.5 + 2 * 2.0 ** -22)
    assert bias <= most, (bias, most)
    assert worst <= bound + SMALL[dtype], (worst, bound)
