"""Token statistics, top alternatives, distillation and the head's forms of them against plain 64-bit implementations.

Bounds.  u = 2^-24.  A scaled logit z = c x is formed with one rounding of at most A u (A: the largest |z|), its power of two with 2^-22; a thread adds V / 512 terms
in turn and its sums are merged over at most 10 levels: the relative error of a row's sum, and so the absolute one of its log-sum-exp, stays below
  E = u (2 A + 8 + V / 512 + 64)          (64: exponents down to 2^-64, below which a term is nothing, rounded by 64 u).
A 16-bit result adds half a step of its type, `eps / 2`, of its value."""

import math

import pytest
import torch

from realhf_b200.ops import functional as OF

U = 2.0 ** -24
INF = float("inf")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def err(z, V):
    z = z.detach()
    a = float(z[z.isfinite()].abs().max()) if bool(z.isfinite().any()) else 0.0
    return U * (2 * a + 72 + V / 512)


def strided(x, layout):
    """The same values as a packed matrix, as rows of a wider one, at an odd offset, or transposed in memory."""
    T, V = x.shape
    if layout == "packed":
        return x.clone()
    if layout == "wide":
        wide = torch.full((T, V + 24), 77.0, dtype=x.dtype, device=x.device)
        wide[:, :V] = x
        return wide[:, :V]
    if layout == "odd":
        wide = torch.full((T, V + 3), 77.0, dtype=x.dtype, device=x.device)
        wide[:, 3:] = x
        return wide[:, 3:]
    return x.t().contiguous().t()


def make_logits(T, V, dtype, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, V, generator=g) * 2.2
    at = torch.randint(0, V, (T, min(V, 6)), generator=g)
    x.scatter_add_(1, at, torch.rand(T, min(V, 6), generator=g) * 10)
    labels = torch.randint(0, V, (T,), generator=g)
    return x.to(dtype).to(device), labels.to(device)


def scaled(logits, mask, c):
    z = logits.detach().cpu().double() * c
    return z if mask is None else z.masked_fill(mask.cpu(), -INF)


def stats64(z, labels):
    lse = torch.logsumexp(z, -1)
    y = z - lse[:, None]
    p = y.exp()
    H = torch.special.entr(p).sum(-1)
    return y, p, y.gather(1, labels[:, None]).squeeze(1), H


def grad64(y, p, H, labels, gl, ge, c):
    d = -p * (gl[:, None] + ge[:, None] * (torch.where(p > 0, y, 0.0) + H[:, None]))
    return d.scatter_add(1, labels[:, None], gl[:, None]) * c


def check_stats(dev, T, V, dtype, layout, masked, temp, seed):
    x, labels = make_logits(T, V, dtype, seed, dev)
    mask = bits = None
    if masked:
        g = torch.Generator().manual_seed(seed + 1)
        mask = torch.rand(T, V, generator=g) < 0.7
        mask.scatter_(1, labels.cpu()[:, None], False)
        mask = mask.to(dev)
        bits = OF.pack_mask_bits(mask)
    c = 1.0 / temp
    leaf = strided(x, layout).requires_grad_(True)
    logp, H = OF.logprob_entropy_from_logits(leaf, labels, bits, inv_temp=c)
    g = torch.Generator().manual_seed(seed + 2)
    gl, ge = torch.randn(T, generator=g), torch.randn(T, generator=g)
    (d,) = torch.autograd.grad([logp, H], [leaf], [gl.to(dev), ge.to(dev)])
    z = scaled(x, mask, c)
    y, p, want_logp, want_H = stats64(z, labels.cpu())
    e = err(z, V)
    assert logp.dtype == H.dtype == torch.float32 and d.dtype == dtype and d.shape == x.shape
    assert ((logp.cpu().double() - want_logp).abs() <= e + U * want_logp.abs()).all()
    assert ((H.cpu().double() - want_H).abs() <= 2 * e * (1 + want_H) + U).all()
    want = grad64(y, p, want_H, labels.cpu(), gl.double(), ge.double(), c)
    size = c * p * (gl.abs()[:, None] + ge.abs()[:, None] * (torch.where(p > 0, -y, 0.0) + want_H[:, None] + 1))
    tiny = torch.finfo(dtype).tiny  # results below the normal numbers have steps of their own
    allowed = half_step(dtype) * want.abs() + size * 4 * e + c * U * (gl.abs()[:, None] + 1) + tiny
    assert ((d.cpu().double() - want).abs() <= allowed).all()
    with torch.no_grad():
        again = OF.logprob_entropy_from_logits(leaf, labels, bits, inv_temp=c)
    assert torch.equal(again[0], logp) and torch.equal(again[1], H)


STATS = [(1, 1, "packed", False, 1.0), (3, 7, "packed", True, 0.7), (2, 8, "odd", False, 1.0), (5, 33, "wide", True, 1.5), (17, 1000, "packed", False, 1.0),
         (4, 4099, "odd", True, 0.7), (3, 4097, "packed", False, 2.0), (2, 777, "transposed", False, 1.0), (9, 32000, "packed", True, 1.0), (3, 50257, "packed", False, 0.8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,layout,masked,temp", STATS[:6])
def test_stats_cpu(T, V, layout, masked, temp, dtype):
    check_stats("cpu", T, V, dtype, layout, masked, temp, seed=T + V)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,layout,masked,temp", STATS + [(300, 32000, "packed", False, 1.0), (2, 131072, "packed", True, 1.0), (1, 300001, "packed", False, 1.0)])
def test_stats_gpu(T, V, layout, masked, temp, dtype):
    check_stats("cuda", T, V, dtype, layout, masked, temp, seed=T + V)


def check_special_rows(dev, dtype, V):
    """A row under a mask that leaves nothing, one of -inf alone, one with -inf among its tokens, a NaN, a +inf, one token, a negative label, a label beyond."""
    x, labels = make_logits(9, V, dtype, 5, dev)
    mask = torch.zeros(9, V, dtype=torch.bool, device=dev)
    mask[0] = True
    x[1] = -INF
    x[2, ::2] = -INF
    x[3, V // 2] = float("nan")
    x[4, V - 1] = INF
    mask[5] = True
    mask[5, 1] = False
    labels[2], labels[5], labels[6], labels[7] = 0, 1, -100, V
    labels[8] = 3
    mask[8, 3] = True
    leaf = x.clone().requires_grad_(True)
    logp, H = OF.logprob_entropy_from_logits(leaf, labels, OF.pack_mask_bits(mask))
    (d,) = torch.autograd.grad([logp, H], [leaf], [torch.ones_like(logp), torch.ones_like(H)])
    logp, H, d = logp.tolist(), H.tolist(), d.float()
    assert logp[0] == logp[1] == -INF and H[0] == H[1] == 0 and not d[0].any() and not d[1].any()
    assert logp[2] == -INF and math.isfinite(H[2]) and H[2] > 0 and not d[2, ::2][1:].any() and d[2].isfinite().all()
    assert all(math.isnan(v) for v in (logp[3], H[3], logp[4], H[4]))
    assert logp[5] == 0 and H[5] == 0 and not d[5].any()
    assert logp[6] == 0 and H[6] > 0
    assert math.isnan(logp[7]) and H[7] > 0
    assert logp[8] == -INF and H[8] > 0
    # a negative label: the entropy's gradient alone
    one = x[6:7].clone().requires_grad_(True)
    lp, h = OF.logprob_entropy_from_logits(one, labels[6:7])
    (only,) = torch.autograd.grad([h], [one], [torch.ones_like(h)])
    # (a row's sums run in an order that goes by its first address modulo 16, which differs for the copy: two results, each off by at most 4 E of the
    # gradient's parts and half a step)
    z = scaled(x[6:7], None, 1.0)
    y, p, _, h64 = stats64(z, labels[6:7].cpu().clamp(min=0))
    slack = 2 * (p * (h64[:, None] + 1 - y) * 4 * err(z, V) + half_step(dtype) * d[6].cpu().double().abs() + U + torch.finfo(dtype).tiny)
    assert ((only.float()[0] - d[6]).abs().cpu().double() <= slack[0]).all()
    # rows that nothing is asked of get zeros, whatever they hold
    leaf = x.clone().requires_grad_(True)
    lp, h = OF.logprob_entropy_from_logits(leaf, labels.clamp(0, V - 1))
    lp.backward(torch.zeros_like(lp))
    if dev == "cuda":
        assert not leaf.grad.any()


@pytest.mark.parametrize("V", [9, 130])
def test_special_rows_cpu(V):
    check_special_rows("cpu", torch.float32, V)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 130, 5000, 40001])
def test_special_rows_gpu(V, dtype):
    check_special_rows("cuda", dtype, V)


# ------------------------------------------------------------------------------------------------ alternatives


def check_top(dev, T, V, k, dtype, layout, masked, temp, seed, x=None):
    labels = None
    if x is None:
        x, labels = make_logits(T, V, dtype, seed, dev)
    mask = bits = None
    if masked:
        g = torch.Generator().manual_seed(seed + 1)
        mask = (torch.rand(T, V, generator=g) < 0.8).to(dev)
        bits = OF.pack_mask_bits(mask)
    c = 1.0 / temp
    o = OF.top_logprobs_from_logits(strided(x, layout), k, labels, bits, inv_temp=c)
    raw = x.cpu().double() + 0.0
    raw = raw if mask is None else raw.masked_fill(mask.cpu(), -INF)
    z = raw * c
    ids = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :k]
    lse = torch.logsumexp(z, -1)
    top = z.gather(1, ids) - lse[:, None]
    none = z.gather(1, ids) == -INF
    rest = torch.logsumexp(z.scatter(1, ids, -INF), -1) - lse
    e = err(z, V)
    empty = lse == -INF
    assert o.top_ids.dtype == torch.int64 and torch.equal(o.top_ids.cpu(), ids.masked_fill(none, -1))
    got = o.top_logp.cpu().double()
    assert (got[none] == -INF).all()
    assert ((got - top).abs()[~none] <= e + U * top.abs()[~none]).all()
    got = o.rest_logp.cpu().double()
    gone = (rest == -INF) | empty
    assert (got[gone] == -INF).all() and ((got - rest).abs()[~gone] <= 2 * e + U * rest.abs()[~gone]).all()
    H = torch.special.entr((z - lse.masked_fill(empty, 0.0)[:, None]).exp()).sum(-1)
    assert ((o.entropy.cpu().double() - H).abs() <= 2 * e * (1 + H) + U).all()
    if labels is None:
        assert o.logp is None
    else:
        want = z.gather(1, labels.cpu()[:, None]).squeeze(1) - lse.masked_fill(empty, 0.0)
        ok = want > -INF
        assert (o.logp.cpu()[~ok] == -INF).all() and ((o.logp.cpu().double() - want).abs()[ok] <= e + U * want.abs()[ok]).all()
    again = OF.top_logprobs_from_logits(strided(x, layout), k, labels, bits, inv_temp=c)
    for a, b in zip(o, again):
        assert a is None or torch.equal(a, b)


TOPS = [(1, 1, 1, "packed", False, 1.0), (3, 7, 7, "packed", False, 0.7), (2, 40, 40, "odd", True, 1.0), (5, 300, 256, "wide", False, 1.0),
        (4, 1000, 20, "packed", True, 1.5), (3, 4099, 1, "odd", False, 1.0), (3, 4099, 255, "odd", True, 1.0)]


@pytest.mark.parametrize("T,V,k,layout,masked,temp", TOPS)
def test_top_cpu(T, V, k, layout, masked, temp):
    check_top("cpu", T, V, k, torch.float32, layout, masked, temp, seed=V + k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,k,layout,masked,temp", TOPS + [(9, 32000, 20, "packed", False, 1.0), (5, 50257, 64, "packed", True, 0.8), (3, 32003, 256, "packed", False, 1.0),
                                                             (3, 32003, 1024, "packed", False, 1.0), (2, 131072, 100, "packed", False, 1.0),
                                                             (300, 2050, 5, "packed", False, 1.0), (1, 300001, 33, "packed", False, 1.0)])
def test_top_gpu(T, V, k, layout, masked, temp, dtype):
    check_top("cuda", T, V, k, dtype, layout, masked, temp, seed=V + k)


def tie_rows(V, dtype, dev):
    """Rows whose order is decided by ties, or that defeat a bound taken from parts of the row."""
    x = torch.zeros(9, V)
    x[1] = torch.arange(V).float() % 3                       # a third of the row shares the largest value
    x[2, V // 2:] = -0.0                                     # -0 equals 0
    x[3] = torch.arange(V).float() / V                       # ascending (many equal ones in 16 bits)
    x[4] = -torch.arange(V).float() / V
    x[5, :: max(1, V // 300)] = 5.0                          # some 300 equal ones all over the row
    x[6, -2:] = 1.0
    x[7] = -INF
    x[7, [V // 3, V - 1]] = 2.0                              # two tokens in all
    x[8, : V // 2] = 30.0                                    # the rest's mass is e^-30 of the row's
    return x.to(dtype).to(dev)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(8, 3), (1001, 10), (4096, 256), (20000, 64), (50257, 256), (50257, 1000)])
def test_top_ties_gpu(V, k, dtype):
    x = tie_rows(V, dtype, "cuda")
    check_top("cuda", 9, V, k, dtype, "packed", False, 1.0, 3, x=x)


def test_top_ties_cpu():
    check_top("cpu", 9, 40, 11, torch.float32, "packed", False, 1.0, 3, x=tie_rows(40, torch.float32, "cpu"))


# many alternatives: nearly every token of the row, more than its groups or pieces can bound, more than the room for candidates
MANY = [(4, 257, 257, "packed", False, 1.0), (3, 1025, 1024, "odd", False, 0.7), (5, 1300, 256, "packed", True, 1.0), (3, 2000, 256, "wide", False, 1.0),
        (3, 2048, 1000, "packed", True, 1.0), (3, 2049, 1024, "odd", False, 1.0), (2, 4500, 512, "odd", True, 1.5), (2, 9001, 1024, "packed", False, 1.0),
        (2, 20481, 512, "odd", False, 1.0), (2, 50257, 300, "odd", True, 0.8), (2, 151936, 1024, "packed", False, 1.0), (1, 400003, 300, "packed", False, 1.0)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,k,layout,masked,temp", MANY)
def test_top_many_gpu(T, V, k, layout, masked, temp, dtype):
    check_top("cuda", T, V, k, dtype, layout, masked, temp, seed=V + k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(1500, 257), (2048, 1024), (5000, 300), (20000, 700), (450001, 257)])
def test_top_many_ties_gpu(V, k, dtype):
    check_top("cuda", 9, V, k, dtype, "packed", False, 1.0, 3, x=tie_rows(V, dtype, "cuda"))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_many_of_few_kept_gpu(dtype):
    """Fewer tokens kept than alternatives asked for, of either sign."""
    x, _ = make_logits(4, 33000, dtype, 5, "cuda")
    keep = torch.randperm(33000, generator=torch.Generator().manual_seed(6))[:500].to("cuda")
    few = torch.full_like(x, -INF)
    few[:, keep] = x[:, keep]
    few[1] = few[1].abs().neg()
    few[2, keep] = -0.0
    check_top("cuda", 4, 33000, 600, dtype, "packed", False, 1.0, 3, x=few)


@gpu
@pytest.mark.parametrize("V", [50, 30000])
def test_top_rows_without_a_softmax_gpu(V):
    x, labels = make_logits(3, V, torch.bfloat16, 1, "cuda")
    x[0, 5], x[1, V - 1] = float("nan"), INF
    o = OF.top_logprobs_from_logits(x, 4, labels)
    assert o.top_logp[:2].isnan().all() and (o.top_ids[:2] == -1).all() and o.rest_logp[:2].isnan().all() and o.entropy[:2].isnan().all() and o.logp[:2].isnan().all()
    assert o.top_logp[2].isfinite().all() and o.rest_logp[2].isfinite()


# ------------------------------------------------------------------------------------------------ distillation


def make_teacher(x, k, seed, rest):
    g = torch.Generator().manual_seed(seed)
    lt = torch.log_softmax(x.detach().cpu().double() * 0.8 + torch.randn(x.shape, generator=g).double(), -1)
    t, ids = torch.topk(lt, k, -1)
    r = torch.logsumexp(lt.scatter(1, ids, -INF), -1) if rest else None
    return ids, t.float(), None if r is None else r.float()


def distill64(z, ids, t, tr, reverse):
    """Loss, d loss / d z and the sizes that bound their errors; ids as the operator takes them."""
    T, V = z.shape
    loss, grad, size, lsize = torch.zeros(T).double(), torch.zeros(T, V).double(), torch.zeros(T, V).double(), torch.zeros(T).double()
    for r in range(T):
        seen, idx, tk = set(), [], []
        for i, v in zip(ids[r].tolist(), t[r].double().tolist()):
            if i >= 0 and i not in seen:
                seen.add(i)
                idx.append(i)
                tk.append(v)
        other = [j for j in range(V) if j not in seen]
        lse = torch.logsumexp(z[r], -1)
        y = z[r] - lse
        tk = torch.tensor(tk, dtype=torch.float64)
        if tr is None:
            tk = torch.log_softmax(tk, 0)
            t_rest = torch.tensor(-INF).double()
        else:
            t_rest = tr[r].double()
        y_rest = torch.logsumexp(y[other], 0) if other else torch.tensor(-INF).double()
        yb, tb = torch.cat([y[idx], y_rest[None]]), torch.cat([tk, t_rest[None]])
        q, p = yb.exp(), tb.exp()
        if reverse:
            f = torch.where(q > 0, yb - tb, 0.0)
            loss[r] = (q * f).sum()
            gb = q * (f - loss[r])
            sb = q * (torch.where(q > 0, yb.abs() + tb.abs(), 0.0) + loss[r].abs() + 2)
            lsize[r] = (q * (torch.where(q > 0, yb.abs() + tb.abs(), 0.0) + 2)).sum()
        else:
            loss[r] = torch.where(p > 0, p * (tb - yb), 0.0).sum()
            gb = p.sum() * q - p
            sb = 2 * (p.sum() * q + p)
            lsize[r] = torch.where(p > 0, p * (tb.abs() + yb.abs() + 2), 0.0).sum()
        grad[r, idx], size[r, idx] = gb[:-1], sb[:-1]
        if other:
            share = (y[other] - y_rest).exp() if y_rest > -INF else torch.zeros(len(other)).double()
            grad[r, other], size[r, other] = share * gb[-1], share * sb[-1]
    return loss, grad, size, lsize


def check_distill(dev, T, V, k, dtype, layout, reverse, rest, temp, seed, spoil=False):
    x, _ = make_logits(T, V, dtype, seed, dev)
    ids, t, tr = make_teacher(x, k, seed + 1, rest)
    if spoil:  # unused places, a token listed twice, a listed token without mass
        ids[0, -1] = -1
        t[0, -1] = -INF
        if k > 2:
            ids[T - 1, 2] = ids[T - 1, 0]
            if not reverse:
                t[0, 1] = -INF
    c = 1.0 / temp
    leaf = strided(x, layout).requires_grad_(True)
    g = torch.rand(T, generator=torch.Generator().manual_seed(seed + 2)) + 0.3
    loss = OF.distill_loss_from_logits(leaf, ids.to(dev), t.to(dev), None if tr is None else tr.to(dev), reverse=reverse, inv_temp=c)
    (d,) = torch.autograd.grad([loss], [leaf], [g.to(dev)])
    z = scaled(x, None, c)
    want, grad, size, lsize = distill64(z, ids, t, tr, reverse)
    e = 2 * err(z, V) + U * k
    assert loss.dtype == torch.float32 and d.dtype == dtype
    assert ((loss.detach().cpu().double() - want).abs() <= 2 * e * lsize + U).all()
    scale = (g.double() * c)[:, None]
    allowed = half_step(dtype) * (grad * scale).abs() + scale * size * 3 * e + torch.finfo(dtype).tiny
    assert ((d.cpu().double() - grad * scale).abs() <= allowed).all()
    with torch.no_grad():
        assert torch.equal(OF.distill_loss_from_logits(leaf, ids.int().to(dev), t.to(dev), None if tr is None else tr.to(dev), reverse=reverse, inv_temp=c), loss)


DISTILL = [(1, 1, 1, "packed", False, False, 1.0), (2, 7, 7, "packed", False, True, 1.0), (3, 40, 5, "odd", True, True, 0.7), (3, 130, 17, "wide", False, False, 2.0),
           (2, 1000, 64, "packed", True, True, 1.0), (2, 1001, 1, "transposed", False, True, 1.0)]


@pytest.mark.parametrize("T,V,k,layout,reverse,rest,temp", DISTILL)
@pytest.mark.parametrize("spoil", [False, True])
def test_distill_cpu(T, V, k, layout, reverse, rest, temp, spoil):
    if spoil and k < 2:
        pytest.skip("nothing to spoil")
    check_distill("cpu", T, V, k, torch.float32, layout, reverse, rest, temp, V + k, spoil)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,k,layout,reverse,rest,temp", DISTILL + [(3, 4099, 33, "odd", False, True, 1.0), (2, 32000, 64, "packed", False, True, 1.0),
                                                                      (2, 50257, 256, "packed", True, True, 0.8), (2, 50257, 1024, "packed", False, False, 1.0),
                                                                      (1, 300001, 20, "packed", True, True, 1.0)])
@pytest.mark.parametrize("spoil", [False, True])
def test_distill_gpu(T, V, k, layout, reverse, rest, temp, spoil, dtype):
    if spoil and k < 2:
        pytest.skip("nothing to spoil")
    check_distill("cuda", T, V, k, dtype, layout, reverse, rest, temp, V + k, spoil)


def check_distill_special(dev, dtype):
    V, k = 50, 4
    x, _ = make_logits(6, V, dtype, 1, dev)
    ids, t, tr = (v.to(dev) for v in make_teacher(x, k, 2, True))
    x[0, 7] = float("nan")
    x[1, 7] = INF
    ids[2, 1] = V                                              # beyond the vocabulary
    x[3, ids[3, 0]] = -INF                                     # the student excludes what the teacher wants
    ids[4], t[4] = -1, -INF                                    # an empty list: the rest is everything
    leaf = x.clone().requires_grad_(True)
    loss = OF.distill_loss_from_logits(leaf, ids, t, tr)
    out = loss.tolist()
    assert all(math.isnan(v) for v in out[:3]) and out[3] == INF and math.isfinite(out[5])
    p = math.exp(float(tr[4]))
    assert abs(out[4] - p * float(tr[4])) <= 8 * U * (1 + abs(float(tr[4])))
    g = torch.ones_like(loss)
    g[:4] = 0
    (d,) = torch.autograd.grad([loss], [leaf], [g])
    if dev == "cuda":
        assert not d[:4].any()
    assert d[4:].isfinite().all()
    everything = OF.distill_loss_from_logits(x[4:5], ids[4:5], t[4:5])   # no token and no rest: nothing to learn from
    assert float(everything) == 0


def test_distill_special_cpu():
    check_distill_special("cpu", torch.float32)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_special_gpu(dtype):
    check_distill_special("cuda", dtype)


# ------------------------------------------------------------------------------------------------ gradients against differences


def test_references_against_differences():
    torch.manual_seed(0)
    x = torch.randn(3, 11, dtype=torch.float64, requires_grad=True)
    labels = torch.tensor([2, 10, -1])
    mask = torch.rand(3, 11) < 0.3
    mask[0, 2] = mask[1, 10] = False
    bits = OF.pack_mask_bits(mask)
    assert torch.autograd.gradcheck(lambda v: OF.logprob_entropy_from_logits(v, labels, bits, 0.7), (x,))
    o = OF.top_logprobs_from_logits(torch.randn(3, 11, dtype=torch.float64), 4)
    ids = o.top_ids.clone()
    ids[1, 3] = -1
    ids[2, 3] = ids[2, 0]
    for reverse, rest in ((False, o.rest_logp), (False, None), (True, o.rest_logp)):
        assert torch.autograd.gradcheck(lambda v: OF.distill_loss_from_logits(v, ids, o.top_logp, rest, reverse, 1.3), (x,))


@gpu
@pytest.mark.parametrize("what", ["logp", "entropy", "forward", "reverse"])
def test_gradients_against_differences_gpu(what):
    """The kernel's gradient along a direction against the 64-bit function's difference quotient with step s: its own error is s^2 / 6 of a third derivative
    (at most some 10 |v|^3 here), 1e-9; the gradient's is bounded as above (fp32)."""
    T, V, k, s = 2, 3001, 20, 1e-5
    x, labels = make_logits(T, V, torch.float32, 4, "cuda")
    ids, t, tr = make_teacher(x, k, 5, True)
    v = torch.randn(T, V, generator=torch.Generator().manual_seed(6)).double()

    def f64(z):
        if what in ("logp", "entropy"):
            return stats64(z, labels.cpu())[2 if what == "logp" else 3].sum()
        return distill64(z, ids, t, tr, what == "reverse")[0].sum()

    leaf = x.clone().requires_grad_(True)
    if what in ("logp", "entropy"):
        out = OF.logprob_entropy_from_logits(leaf, labels)[0 if what == "logp" else 1]
    else:
        out = OF.distill_loss_from_logits(leaf, ids.cuda(), t.cuda(), tr.cuda(), reverse=what == "reverse")
    out.sum().backward()
    z = x.cpu().double()
    want = (f64(z + s * v) - f64(z - s * v)) / (2 * s)
    got = (leaf.grad.cpu().double() * v).sum()
    assert abs(float(got - want)) <= 1e-6 + 200 * err(z, V) * T


# ------------------------------------------------------------------------------------------------ through the head


def make_head(T, H, V, dtype, seed, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=g) / math.sqrt(H)
    labels = torch.randint(0, V, (T,), generator=g)
    h = torch.randn(T, H, generator=g) * 1.5 + w[labels] * (torch.rand(T, 1, generator=g) * 8)
    return h.to(dtype).to(dev), w.to(dtype).to(dev), labels.to(dev)


def head_errors(h, w, c, V):
    """(scaled logits, bound on their error): products of 16-bit numbers are exact in fp32, the tensor core's accumulator cuts off once for 16 of them,
    at most 2^-22 of the largest partial sum, itself at most the sum of the products' sizes; fp32 operands round each of their products and sums."""
    z = h.double() @ w.double().t() * c
    size = h.double().abs() @ w.double().abs().t() * c
    return z, size * (h.shape[1] / 16 + 4) * 2.0 ** -22 + U * z.abs()


def check_head(dev, T, H, V, dtype, masked, temp, chunk, seed, buffer=None, keep=1 << 31):
    h, w, labels = make_head(T, H, V, dtype, seed)
    c = 1.0 / temp
    mask = bits = None
    if masked:
        mask = torch.rand(T, V, generator=torch.Generator().manual_seed(seed + 1)) < 0.6
        mask.scatter_(1, labels[:, None], False)
        if T > 2:
            mask[1] = True                                    # a row that keeps nothing
        bits = OF.pack_mask_bits(mask).to(dev)
    g = torch.Generator().manual_seed(seed + 2)
    gl, ge = torch.randn(T, generator=g), torch.randn(T, generator=g)
    hd = h.to(dev).requires_grad_(True)
    wd = torch.nn.Parameter(w.to(dev))
    old = torch.zeros(V, H).double()
    if buffer is not None:
        old = (torch.randn(V, H, generator=g) * 0.1).to(dtype if buffer == "weight_type" else torch.float32)
        if buffer == "weight_type":
            wd.grad, wd._grad_in_flat_buffer = old.to(dev).clone(), True
        else:
            wd.main_grad = old.to(dev).clone()
        old = old.double()
    logp, ent = OF.lm_head_logprobs_entropy(hd, wd, labels.to(dev), bits, temperature=temp, chunk=chunk, keep_bytes=keep)
    torch.autograd.backward([logp, ent], [gl.to(dev), ge.to(dev)])
    z, ez = head_errors(h, w, c, V)
    if mask is not None:
        z, ez = z.masked_fill(mask, -INF), ez.masked_fill(mask, 0.0)
    empty = (z == -INF).all(-1)
    zz = z.masked_fill(empty[:, None], 0.0)
    y, p, want_logp, want_H = stats64(zz, labels)
    e = (err(z, V) + ez.max(-1).values)[:, None]
    ok = ~empty
    assert (logp.cpu()[empty] == -INF).all() and (ent.cpu()[empty] == 0).all()
    assert ((logp.detach().cpu().double() - want_logp).abs() <= 2 * e[:, 0] + U * want_logp.abs())[ok].all()
    assert ((ent.detach().cpu().double() - want_H).abs() <= 2 * e[:, 0] * (1 + want_H) * 2 + U)[ok].all()
    d = grad64(y, p, want_H, labels, gl.double(), ge.double(), c).masked_fill(empty[:, None], 0.0)
    size = c * p * (gl.abs()[:, None] + ge.abs()[:, None] * (torch.where(p > 0, -y, 0.0) + want_H[:, None] + 1)) * 4 * e + c * U * (gl.abs()[:, None] + 1)
    r = half_step(dtype)
    # kept weights e, relative to the largest of 128 columns, are rounded by at most 2^-11 of e (fp16), their logarithm by as much, which moves the gradient by at most
    # 2^-11 of the size of its parts; below 2^-29 by 2^-40, which is no more than 2^-40 of what a probability of 1 would give
    kept = T > 256 and H >= 1024 and keep > 0 and dtype != torch.float32
    whole = c * (gl.abs()[:, None] + ge.abs()[:, None] * (want_H[:, None] + 30))
    more = (2.0 ** -11 * (size / (4 * e)) + 2.0 ** -40 * whole) if kept else 0.0
    ed = (r * d.abs() + size + more + torch.finfo(dtype).tiny).masked_fill(empty[:, None], 0.0)
    W, Hh = w.double(), h.double()
    for got, want, slack, n in ((hd.grad, d @ W, ed @ W.abs() + (d.abs() @ W.abs()) * (V / 16 + 4) * 2.0 ** -22, 1),
                                (wd.main_grad if buffer == "fp32" else wd.grad, d.t() @ Hh + old, ed.t() @ Hh.abs() + (d.abs().t() @ Hh.abs()) * (T / 16 + 4) * 2.0 ** -22,
                                 2 if buffer == "weight_type" else 1)):
        step = r if got.dtype == dtype else U
        assert ((got.cpu().double() - want).abs() <= slack + n * step * (want.abs() + slack) + n * torch.finfo(dtype).tiny + U * (want.abs() + old.abs().max())).all()
    if buffer == "fp32":
        assert wd.grad is None


HEADS = [(5, 64, 40, False, 1.0, 8192), (33, 64, 130, True, 0.7, 16), (3, 24, 33, True, 1.0, 1)]


@pytest.mark.parametrize("T,H,V,masked,temp,chunk", HEADS)
def test_head_cpu(T, H, V, masked, temp, chunk):
    check_head("cpu", T, H, V, torch.float32, masked, temp, chunk, seed=T)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,V,masked,temp,chunk", HEADS + [(1, 64, 1000, False, 1.0, 8192), (130, 256, 1001, True, 1.3, 8192), (300, 136, 5003, False, 1.0, 128),
                                                             (257, 512, 2048, True, 1.0, 8192), (513, 64, 32000, False, 1.0, 8192), (40, 60, 100, False, 1.0, 8192),
                                                             (270, 1032, 1001, True, 0.8, 8192), (300, 1024, 4096, False, 1.0, 128)])
def test_head_gpu(T, H, V, masked, temp, chunk, dtype):
    check_head("cuda", T, H, V, dtype, masked, temp, chunk, seed=T)
    if T > 256:
        check_head("cuda", T, H, V, dtype, masked, temp, chunk, seed=T, keep=0)


@gpu
@pytest.mark.parametrize("buffer", ["weight_type", "fp32"])
@pytest.mark.parametrize("T,chunk", [(64, 8192), (77, 8192), (77, 32)])
def test_head_gradient_into_a_buffer_gpu(T, chunk, buffer):
    if buffer == "weight_type" and T > chunk:
        pytest.skip("several chunks keep an fp32 sum and leave the buffer to autograd")
    check_head("cuda", T, 128, 1000, torch.bfloat16, False, 1.0, chunk, 7, buffer=buffer)


@gpu
@pytest.mark.parametrize("buffer", ["weight_type", "fp32"])
def test_head_gradient_is_given_to_who_asks_for_it_gpu(buffer):
    """With a gradient buffer on the weight, `torch.autograd.grad` returns the gradient and leaves the buffer as it was."""
    h, w, labels = make_head(70, 64, 500, torch.bfloat16, 3, "cuda")
    w = torch.nn.Parameter(w)
    logp, ent = OF.lm_head_logprobs_entropy(h, w, labels)
    (want,) = torch.autograd.grad(logp.sum() + ent.sum(), [w])
    old = torch.ones(500, 64, dtype=w.dtype if buffer == "weight_type" else torch.float32, device="cuda")
    if buffer == "weight_type":
        w.grad, w._grad_in_flat_buffer = old.clone(), True
    else:
        w.main_grad = old.clone()
    logp, ent = OF.lm_head_logprobs_entropy(h, w, labels)
    (got,) = torch.autograd.grad(logp.sum() + ent.sum(), [w])
    assert torch.equal(got, want) and torch.equal(w.grad if buffer == "weight_type" else w.main_grad, old)


@gpu
def test_inside_function_transforms_gpu():
    x, labels = make_logits(3, 50, torch.float32, 1, "cuda")
    o = OF.top_logprobs_from_logits(x, 4)
    e = err(x.cpu().double(), 50)
    for f in (lambda v: OF.logprob_entropy_from_logits(v, labels)[1].sum(), lambda v: OF.distill_loss_from_logits(v * 0.5, o.top_ids, o.top_logp, o.rest_logp).sum()):
        got = torch.func.grad(f)(x)
        leaf = x.clone().requires_grad_(True)
        f(leaf).backward()
        # two results of the bounds above for gradients whose parts are at most 1 + the entropy's 4
        assert ((got - leaf.grad).abs() <= 2 * 4 * e * 5 + 8 * U).all()


@gpu
def test_head_strided_operands_gpu():
    h, w, labels = make_head(70, 64, 200, torch.bfloat16, 3, "cuda")
    wide = torch.zeros(70, 67, dtype=h.dtype, device="cuda")
    wide[:, 1:65] = h
    a = OF.lm_head_logprobs_entropy(h, w, labels)
    b = OF.lm_head_logprobs_entropy(wide[:, 1:65], w, labels)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def check_chain(dev, dtype):
    """A teacher's alternatives, the student's distillation and the policy's statistics in one training step, as they are used together."""
    T, H, V, k = 37, 64, 501, 8
    h, w, labels = make_head(T, H, V, dtype, 1, dev)
    ht, wt, _ = make_head(T, H, V, dtype, 2, dev)
    teacher = OF.lm_head_top_logprobs(ht, wt, k, labels, temperature=1.2, chunk=16)
    zt = ht.cpu().double() @ wt.cpu().double().t() / 1.2
    order = torch.sort(zt, -1, descending=True).values
    lt = torch.log_softmax(zt, -1)
    got = torch.exp(teacher.top_logp).sum(-1) + torch.exp(teacher.rest_logp)
    assert ((got - 1).abs() <= 1e-5).all() and teacher.top_ids.shape == (T, k)
    assert ((teacher.top_logp.cpu().double() - (order[:, :k] - torch.logsumexp(zt, -1)[:, None])).abs() <= 1e-4).all()
    assert ((teacher.logp.cpu().double() - lt.gather(1, labels.cpu()[:, None]).squeeze(1)).abs() <= 1e-4).all()
    for reverse in (False, True):
        hs, ws = h.clone().requires_grad_(True), torch.nn.Parameter(w.clone())
        loss = OF.lm_head_distill_loss(hs, ws, teacher.top_ids, teacher.top_logp, teacher.rest_logp, reverse=reverse, temperature=1.2, chunk=16)
        logp, ent = OF.lm_head_logprobs_entropy(hs, ws, labels, temperature=1.2, chunk=16)
        total = loss.mean() - 0.1 * ent.mean() - 0.2 * logp.mean()
        total.backward()
        z, ez = head_errors(h.cpu(), w.cpu(), 1 / 1.2, V)
        want, grad, size, lsize = distill64(z, teacher.top_ids.cpu(), teacher.top_logp.cpu(), teacher.rest_logp.cpu(), reverse)
        e = 2 * (err(z, V) + ez.max()) + U * k
        assert ((loss.detach().cpu().double() - want).abs() <= 2 * e * lsize + U).all()
        y, p, lp, H64 = stats64(z, labels.cpu())
        d1 = grad / T / 1.2
        d2 = grad64(y, p, H64, labels.cpu(), torch.full((T,), -0.2 / T).double(), torch.full((T,), -0.1 / T).double(), 1 / 1.2)
        r = half_step(dtype)
        W = w.cpu().double()
        # both parts' gradients of logits, the two parts' gradients of hidden states and their sum are rounded to the type
        slack = (r * (d1.abs() + d2.abs())) @ W.abs() + 2 * r * ((d1 @ W).abs() + (d2 @ W).abs()) + 4 * float(e) * (size / T + 0.3 / T * p * (2 - y + H64[:, None])) @ W.abs() \
            + torch.finfo(dtype).tiny * V
        assert ((hs.grad.cpu().double() - (d1 + d2) @ W).abs() <= slack + 1e-7).all()
        assert ws.grad.isfinite().all() and ws.grad.shape == w.shape


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_head_kept_logits_gpu(dtype):
    """Logits kept for the backward pass or formed again: the same gradients, also when it runs twice."""
    T, H, V, k = 37, 64, 501, 8
    h, w, labels = make_head(T, H, V, dtype, 1, "cuda")
    ids, t, tr = (v.cuda() for v in make_teacher(make_logits(T, V, torch.float32, 4)[0], k, 3, True))
    g = torch.linspace(-1, 2, T, device="cuda")
    results = []
    for keep in (4 * T * V, 4 * T * V - 1, 0):
        a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = OF.lm_head_distill_loss(a, b, ids, t, tr, temperature=1.2, chunk=16, keep_bytes=keep)
        for _ in range(2):
            results.append((loss.detach(), *torch.autograd.grad(loss, [a, b], g, retain_graph=True)))
    for r in results[1:]:
        for x, y in zip(results[0], r):
            assert torch.equal(x, y)


def test_chain_cpu():
    check_chain("cpu", torch.float32)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_chain_gpu(dtype):
    check_chain("cuda", dtype)


# ------------------------------------------------------------------------------------------------ a model's output, the actor's entropy bonus


def check_model_output(dev, dtype, softcap, scale):
    """`ModelOutput`'s calls against 64 bits, with a soft cap on the logits, a fixed factor, both and neither.  Bound: as for the head; a cap forms
    cap tanh(z / cap) in fp32, 8 u of it, from logits that the capped path rounds to the model's type."""
    from realhf_b200.models.real_model import ModelOutput
    T, H, V, k = 11, 64, 300, 6
    h, w, labels = make_head(T, H, V, dtype, 5, dev)
    rows = torch.tensor([0, 3, 4, 10], device=dev)
    lab = labels[rows]

    def z64(hidden):
        z = hidden.cpu().double()[rows.cpu()] @ w.cpu().double().t()
        z = z * (1.0 if scale is None else scale)
        return (z if softcap is None else softcap * torch.tanh(z / softcap)) / 0.9

    rounding = half_step(dtype) if softcap is not None and dtype != torch.float32 else 0.0
    z = z64(h)
    slack = 4 * (err(z, V) + float(z.abs().max()) * (2.0 ** -19 + rounding))
    out = ModelOutput(hidden=h.clone().requires_grad_(True), head_weight=w, ctx=None, softcap=softcap, logit_scale=scale)
    logp, ent = out.logprobs_entropy(lab, None, 0.9, rows)
    y, p, want_logp, want_H = stats64(z, lab.cpu())
    assert ((logp.detach().cpu().double() - want_logp).abs() <= slack * 2).all() and ((ent.detach().cpu().double() - want_H).abs() <= slack * (1 + want_H) * 2).all()
    top = out.top_logprobs(k, lab, None, 0.9, rows)
    assert ((top.top_logp.cpu().double() - torch.sort(y, -1, descending=True).values[:, :k]).abs() <= 2 * slack).all()
    assert ((top.logp.cpu().double() - want_logp).abs() <= 2 * slack).all()
    assert ((top.top_logp.exp().sum(-1) + top.rest_logp.exp() - 1).abs() <= 1e-5).all()
    ids, t, tr = make_teacher(z, k, 3, True)
    loss = out.distill_loss(ids.to(dev), t.to(dev), tr.to(dev), False, 0.9, rows)
    want = distill64(z, ids, t, tr, False)[0]
    assert ((loss.detach().cpu().double() - want).abs() <= slack * 4).all()
    (d,) = torch.autograd.grad([logp.sum() + ent.sum() + loss.sum()], [out.hidden])
    # against a difference quotient of the 64-bit function along a direction; the parts' gradients are rounded twice to the type on the way
    v = torch.randn(T, H, generator=torch.Generator().manual_seed(6)).double()

    def f(hidden):
        z = z64(hidden)
        return stats64(z, lab.cpu())[2].sum() + stats64(z, lab.cpu())[3].sum() + distill64(z, ids, t, tr, False)[0].sum()

    s = 1e-5
    want = (f(h.cpu().double() + s * v) - f(h.cpu().double() - s * v)) / (2 * s)
    got = (d.cpu().double() * v).sum()
    size = float((d.cpu().double().abs() * v.abs()).sum())
    assert abs(float(got - want)) <= size * (6 * half_step(dtype) + 20 * slack) + 1e-6
    assert not d[1].any()


@pytest.mark.parametrize("softcap,scale", [(None, None), (20.0, None), (None, 0.5), (20.0, 0.5)])
def test_model_output_cpu(softcap, scale):
    check_model_output("cpu", torch.float32, softcap, scale)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("softcap,scale", [(None, None), (20.0, None), (None, 0.5), (20.0, 0.5)])
def test_model_output_gpu(softcap, scale, dtype):
    check_model_output("cuda", dtype, softcap, scale)


def _sharded_output(rank, world):
    """Every rank's share of a vocabulary-sharded head: the calls and the gradient of the whole hidden states."""
    from realhf_b200.base.topology import ParallelContext, ProcessTopology
    from realhf_b200.models.real_model import ModelOutput
    ctx = ParallelContext.build(ProcessTopology(1, 1, world), list(range(world)), rank, backend="gloo")
    h, w, labels = make_head(9, 32, 64, torch.float32, 2)
    per = 64 // world
    hidden, shard = h.clone().requires_grad_(True), w[rank * per: (rank + 1) * per].clone().requires_grad_(True)
    out = ModelOutput(hidden=hidden, head_weight=shard, ctx=ctx)
    logp, ent = out.logprobs_entropy(labels)
    top = out.top_logprobs(5, labels)
    loss = out.distill_loss(top.top_ids, top.top_logp - 0.1, top.rest_logp)
    (logp.sum() + ent.sum() + loss.sum()).backward()
    return [t.detach().tolist() for t in (logp, ent, loss, top.top_logp, top.top_ids, hidden.grad, shard.grad)]


@pytest.mark.distributed
def test_model_output_with_a_sharded_head_cpu():
    from realhf_b200.base.testing import run_distributed
    one = run_distributed(_sharded_output, 1)[0]
    two = run_distributed(_sharded_output, 2)
    for r, got in enumerate(two):
        for a, b in zip(one[:6], got[:6]):
            torch.testing.assert_close(torch.tensor(a), torch.tensor(b), atol=1e-5, rtol=1e-5)
        torch.testing.assert_close(torch.tensor(one[6][32 * r: 32 * r + 32]), torch.tensor(got[6]), atol=1e-5, rtol=1e-5)


def test_actor_loss_with_an_entropy_bonus_cpu():
    """The bonus is the masked mean entropy times its coefficient; without one the loss is what it was."""
    from types import SimpleNamespace
    from realhf_b200.interfaces import ppo
    from realhf_b200.models.real_model import ModelOutput
    T, H, V = 12, 32, 50
    h, w, _ = make_head(T, H, V, torch.float32, 1)
    ids = torch.arange(T) % V
    n = T - 2
    mask = torch.ones(n, dtype=torch.bool)
    mask[:3] = False
    data = dict(packed_input_ids=ids, old_logp=torch.full((n,), -3.0), advantages=torch.linspace(-1, 1, n), ppo_loss_mask=mask)
    mb = SimpleNamespace(data=data, flat_seqlens=lambda key: [5, 7])
    kw = dict(kl_adapter=None, eps_clip=0.2, temperature=1.0, early_stop_imp_ratio=None, early_stop_kl=None)
    grads = []
    for coef in (0.0, 0.3):
        hidden = h.clone().requires_grad_(True)
        loss, stat = ppo._actor_loss_from_output(ModelOutput(hidden=hidden, head_weight=w, ctx=None), mb, entropy_coef=coef, **kw)
        loss.backward()
        grads.append((loss.detach(), stat, hidden.grad))
    rows = torch.tensor([0, 1, 2, 3, 5, 6, 7, 8, 9, 10])
    hidden = h.clone().requires_grad_(True)
    p = torch.softmax(hidden[rows] @ w.t(), -1)
    mean = (torch.special.entr(p).sum(-1) * mask).sum() / mask.sum()
    mean.backward()
    assert "entropy" not in grads[0][1] and abs(float(grads[1][1]["entropy"] - mean.detach())) < 1e-5
    assert abs(float(grads[1][0] - (grads[0][0] - 0.3 * mean.detach()))) < 1e-5
    torch.testing.assert_close(grads[1][2], grads[0][2] - 0.3 * hidden.grad, atol=1e-6, rtol=1e-4)


def test_ppo_iterations_with_an_entropy_bonus_cpu():
    from test_engine_cpu import make_model
    from realhf_b200.api.data import SequenceSample
    from realhf_b200.interfaces import basic, ppo
    torch.manual_seed(0)
    actor, critic = make_model("actor"), make_model("critic", critic=True)
    ref, rew = make_model("ref", train=False), make_model("reward", critic=True, train=False, seed=7)
    a = ppo.PPOActorInterface(n_minibatches=2, generation_config=dict(max_new_tokens=6, min_new_tokens=2, top_k=50, top_p=0.9), entropy_coef=0.01)
    c = ppo.PPOCriticInterface(n_minibatches=2)
    plens = [5, 7, 4, 6]
    prompts = SequenceSample.from_default(seqlens=plens, ids=list(range(4)), data=dict(packed_prompts=torch.randint(2, 128, (sum(plens),))))
    d = a.generate(actor, prompts, n_mbs=1)
    d.update_(a.inference(ref, d))
    d.update_(c.inference(critic, d))
    d.update_(basic.PairedRewardInterface().inference(rew, d))
    st = a.train_step(actor, d, n_mbs=1)
    assert 0 < st["entropy"] < math.log(128) and st["actor_loss"] == st["actor_loss"]


# ------------------------------------------------------------------------------------------------ streams, graphs, sizes, refusals


@gpu
def test_captured_and_replayed_gpu():
    T, V, k, H = 12, 3000, 16, 64
    x, labels = make_logits(T, V, torch.bfloat16, 1, "cuda")
    h, w, _ = make_head(T, H, V, torch.bfloat16, 2, "cuda")
    ids, t, tr = (v.cuda() for v in make_teacher(x, k, 3, True))

    def work():
        a = x.detach().requires_grad_(True)
        b, c = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        logp, ent = OF.logprob_entropy_from_logits(a, labels)
        loss = OF.distill_loss_from_logits(a, ids, t, tr)
        lp, en = OF.lm_head_logprobs_entropy(b, c, labels)
        hd = OF.lm_head_distill_loss(b, c, ids, t, tr)
        top, htop = OF.top_logprobs_from_logits(x, k, labels), OF.lm_head_top_logprobs(h, w, k, labels)
        grads = torch.autograd.grad([logp, ent, loss, lp, en, hd], [a, b, c], [torch.ones_like(logp)] * 6)
        return [logp, ent, loss, lp, en, hd, *top, *htop, *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        graphs.append((graph, out))
    x2, _ = make_logits(T, V, torch.bfloat16, 9, "cuda")
    x.copy_(x2)
    streams = [torch.cuda.Stream() for _ in graphs]     # at once: no workspace is shared
    for stream, (graph, out) in zip(streams, graphs):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(5):
                graph.replay()
    torch.cuda.synchronize()
    second = work()
    for graph, out in graphs:
        for a, b in zip(out, second):
            assert torch.equal(a, b)
    assert not torch.equal(first[0], second[0])


@gpu
def test_capture_beside_a_living_eager_graph_is_refused_gpu():
    T, V, k = 5, 3000, 4
    x, labels = make_logits(T, V, torch.bfloat16, 1, "cuda")
    ids, t, tr = (v.cuda() for v in make_teacher(x, k, 3, True))
    h, w, _ = make_head(T, 64, V, torch.bfloat16, 2, "cuda")
    a, b, c, f, g = (v.detach().requires_grad_(True) for v in (x, h, w, h.float(), w.float()))
    calls = [lambda: OF.logprob_entropy_from_logits(a, labels)[1], lambda: OF.distill_loss_from_logits(a, ids, t, tr), lambda: OF.lm_head_logprobs_entropy(b, w, labels)[0],
             lambda: OF.lm_head_logprobs_entropy(h, c, labels)[0], lambda: OF.lm_head_logprobs_entropy(f, g, labels)[0], lambda: OF.lm_head_distill_loss(b, c, ids, t, tr)]
    living = [call() for call in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            with pytest.raises(RuntimeError, match="release that call's results first"):
                call()
            with torch.no_grad():
                call()
    torch.autograd.grad(living, [a, b, c, f, g], [torch.ones_like(y) for y in living])
    want = [y.detach().clone() for y in living]
    del living
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        out = [call().detach() for call in calls]
    again.replay()
    torch.cuda.synchronize()
    for y, z in zip(out, want):
        assert torch.equal(y, z)


@gpu
def test_nothing_beside_the_rows_is_written_gpu():
    """Gradients of a slice of rows: what lies around inputs and outputs stays as it was."""
    T, V = 6, 1003
    x, labels = make_logits(T, V, torch.bfloat16, 1, "cuda")
    wide = torch.full((T + 2, V + 9), 3.0, dtype=x.dtype, device="cuda")
    wide[1:-1, 5:-4] = x
    keep = wide.clone()
    leaf = wide.detach().requires_grad_(True)
    logp, ent = OF.logprob_entropy_from_logits(leaf[1:-1, 5:-4], labels)
    (logp.sum() + ent.sum()).backward()
    assert torch.equal(wide, keep) and not leaf.grad[0].any() and not leaf.grad[-1].any() and not leaf.grad[:, :5].any() and not leaf.grad[:, -4:].any()
    one = x.clone().requires_grad_(True)
    lp, en = OF.logprob_entropy_from_logits(one, labels)
    (lp.sum() + en.sum()).backward()
    z = scaled(x, None, 1.0)   # (another order of the rows' sums, as their addresses modulo 16 differ)
    y, p, _, h64 = stats64(z, labels.cpu())
    slack = 2 * (p * (h64[:, None] + 2 - y) * 4 * err(z, V) + half_step(x.dtype) * one.grad.cpu().double().abs() + U)
    assert ((leaf.grad[1:-1, 5:-4] - one.grad).abs().cpu().double() <= slack).all()


@gpu
def test_offsets_beyond_32_bits_gpu():
    """Rows whose first element lies beyond 2^31: the last rows of a matrix of 33000 x 70001 in 16 bits against the same rows alone.  A block has another number of
    threads for few rows and with it another order of sums: two results of the bounds above."""
    T, V = 33000, 70001
    x = torch.empty(T, V, dtype=torch.bfloat16, device="cuda").normal_(0, 2)
    labels = torch.arange(T, device="cuda") % V
    o = OF.top_logprobs_from_logits(x, 3, labels)
    last = x[-8:].clone()
    few = OF.top_logprobs_from_logits(last, 3, labels[-8:])
    z = scaled(last, None, 1.0)
    y, p, _, H = stats64(z, labels[-8:].cpu())
    e, r = err(z, V), half_step(x.dtype)
    assert torch.equal(o.top_ids[-8:], few.top_ids)
    for a, b in ((o.top_logp, few.top_logp), (o.rest_logp, few.rest_logp), (o.logp, few.logp), (o.entropy, few.entropy)):
        assert ((a[-8:] - b).abs() <= 4 * e * (1 + b.abs())).all()
    leaf = x.requires_grad_(True)
    logp, ent = OF.logprob_entropy_from_logits(leaf, labels)
    (d,) = torch.autograd.grad([logp, ent], [leaf], [torch.ones_like(logp), torch.ones_like(ent)])
    last = last.requires_grad_(True)
    lp, en = OF.logprob_entropy_from_logits(last, labels[-8:])
    (dl,) = torch.autograd.grad([lp, en], [last], [torch.ones_like(lp), torch.ones_like(en)])
    slack = 2 * (r * dl.cpu().double().abs() + p * (2 - y + H[:, None]) * 4 * e + U)
    assert ((logp[-8:] - lp).abs() <= 4 * e * (1 + lp.abs())).all() and ((d[-8:] - dl).abs().cpu().double() <= slack).all()
    del d
    loss = OF.distill_loss_from_logits(leaf, o.top_ids, o.top_logp, o.rest_logp)
    (d,) = torch.autograd.grad([loss], [leaf], [torch.ones_like(loss)])
    l8 = OF.distill_loss_from_logits(last, few.top_ids, few.top_logp, few.rest_logp)
    (d8,) = torch.autograd.grad([l8], [last], [torch.ones_like(l8)])
    # the teacher is the student: a loss of 0 but for the roundings of log-probabilities up to 12, and a gradient of as little
    assert (loss[-8:].abs() <= 8 * e * 12).all() and (l8.abs() <= 8 * e * 12).all() and (d[-8:].abs() <= 8 * e * 12).all() and (d8.abs() <= 8 * e * 12).all()


def check_no_rows(dev):
    V = 50
    x = torch.zeros(0, V, device=dev, requires_grad=True)
    none = torch.zeros(0, dtype=torch.long, device=dev)
    logp, ent = OF.logprob_entropy_from_logits(x, none)
    loss = OF.distill_loss_from_logits(x, none.view(0, 1).expand(0, 3), torch.zeros(0, 3, device=dev))
    (logp.sum() + ent.sum() + loss.sum()).backward()
    assert logp.shape == ent.shape == loss.shape == (0,) and x.grad.shape == (0, V)
    assert OF.top_logprobs_from_logits(x, 3, none).top_ids.shape == (0, 3)
    h, w = torch.zeros(0, 16, device=dev, requires_grad=True), torch.ones(V, 16, device=dev, requires_grad=True)
    logp, ent = OF.lm_head_logprobs_entropy(h, w, none)
    loss = OF.lm_head_distill_loss(h, w, none.view(0, 1).expand(0, 3), torch.zeros(0, 3, device=dev))
    (logp.sum() + ent.sum() + loss.sum()).backward()
    assert h.grad.shape == (0, 16) and w.grad.shape == (V, 16) and not w.grad.any()
    assert OF.lm_head_top_logprobs(h, w, 2).top_logp.shape == (0, 2)


def test_no_rows_cpu():
    check_no_rows("cpu")


def check_scales_beyond_fp32(dev, dtype):
    """Logits whose scaled values leave fp32's range: above it no softmax, below it no token, and a row with its maximum at 0 has that token alone."""
    x = torch.full((3, 700), -1e10)
    x[0, 300], x[2, 301], x[2, 5] = 1e10, 0.0, -2e10
    x, labels = x.to(dtype).to(dev), torch.tensor([300, 300, 301], device=dev)
    leaf = x.clone().requires_grad_(True)
    logp, ent = OF.logprob_entropy_from_logits(leaf, labels, inv_temp=1e30)
    o = OF.top_logprobs_from_logits(x, 2, labels, inv_temp=1e30)
    for lp, en in ((logp, ent), (o.logp, o.entropy)):
        assert lp[0].isnan() and en[0].isnan() and lp[1] == -INF and lp[2] == 0 and en[1] == 0 and en[2] == 0
    assert o.top_logp[0].isnan().all() and (o.top_logp[1] == -INF).all() and o.top_ids.tolist()[:2] == [[-1, -1]] * 2
    assert o.top_logp[2, 0] == 0 and o.top_ids[2, 0] == 301 and o.rest_logp[2] == -INF
    d, = torch.autograd.grad((logp + ent)[1:].sum(), leaf)
    assert not d[1:].any()


def test_scales_beyond_fp32_cpu():
    check_scales_beyond_fp32("cpu", torch.float32)


@gpu
@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_scales_beyond_fp32_gpu(dtype):
    check_scales_beyond_fp32("cuda", dtype)


@gpu
def test_no_rows_gpu():
    check_no_rows("cuda")


def check_refusals(dev):
    x, labels = make_logits(3, 20, torch.float32, 1, dev)
    ids, t, tr = (v.to(dev) for v in make_teacher(x, 4, 2, True))
    w = torch.randn(20, 8, device=dev)
    h = torch.randn(3, 8, device=dev)
    bits = torch.zeros(3, 3, dtype=torch.uint8, device=dev)
    L, P, D, E = OF.logprob_entropy_from_logits, OF.top_logprobs_from_logits, OF.distill_loss_from_logits, OF.lm_head_logprobs_entropy
    bad = [
        lambda: L(x[0], labels[:1]), lambda: L(x, labels[:2]), lambda: L(x, labels.float()), lambda: L(x, labels[:, None]), lambda: L(x, labels, inv_temp=0.0),
        lambda: L(x, labels, inv_temp=float("nan")), lambda: L(x, labels, inv_temp=INF), lambda: L(x, labels, inv_temp=1e38), lambda: L(x, labels, inv_temp=1e-40), lambda: L(x.int(), labels), lambda: L(x, labels, bits[:, :2]), lambda: L(x, labels, bits[:2]),
        lambda: L(x, labels, bits.bool()), lambda: L(x[:, :0], labels),
        lambda: P(x, 0), lambda: P(x, 21), lambda: P(torch.zeros(1, 2000, device=dev), 1025), lambda: P(x, 2, labels[:2]), lambda: P(x, 2, inv_temp=-1.0),
        lambda: D(x, ids, t[:, :2]), lambda: D(x, ids[:2], t[:2]), lambda: D(x, ids, t, tr[:2]), lambda: D(x, ids, t, reverse=True), lambda: D(x, t, t),
        lambda: D(x, ids[:, :0], t[:, :0]), lambda: D(x, ids, t, tr[:, None]), lambda: D(x, ids[0], t[0]), lambda: D(x, ids, t.clone().requires_grad_(True)),
        lambda: D(torch.zeros(3, (1 << 20) + 1, device=dev), ids, t),
        lambda: E(h, w[:, :4], labels), lambda: E(h, w.to(torch.bfloat16), labels), lambda: E(h, w, labels, temperature=0.0), lambda: E(h, w, labels, temperature=1e38), lambda: E(h, w, labels, chunk=0),
        lambda: E(h, w, labels[:2]), lambda: E(h, w, labels, bits[:, :1]), lambda: OF.lm_head_top_logprobs(h, w, 0), lambda: OF.lm_head_top_logprobs(h, w, 3, chunk=0),
        lambda: OF.lm_head_distill_loss(h, w, ids, t, reverse=True), lambda: OF.lm_head_distill_loss(h[:2], w, ids, t),
    ]
    if dev == "cuda":
        bad += [lambda: L(x, labels.cpu()), lambda: D(x, ids.cpu(), t), lambda: D(x, ids, t.cpu()), lambda: E(h, w.cpu(), labels), lambda: L(x, labels, bits.cpu()),
                lambda: L(x.double(), labels)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)


def test_refusals_cpu():
    check_refusals("cpu")


@gpu
def test_refusals_gpu():
    check_refusals("cuda")


@gpu
def test_second_derivatives_are_refused_gpu():
    x, labels = make_logits(2, 30, torch.float32, 1, "cuda")
    leaf = x.requires_grad_(True)
    logp, ent = OF.logprob_entropy_from_logits(leaf, labels)
    (d,) = torch.autograd.grad([logp.sum() + ent.sum()], [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
