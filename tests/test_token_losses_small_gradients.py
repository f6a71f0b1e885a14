"""Gradients of the size that a mean loss has (1 / T a row) through the head and from rows of logits, against 64 bits.

Bounds as in test_token_losses.py, but a number below the normal ones is off by half of the smallest step of its type and no more (fp16 2^-25).  Where d logits are
stored in fp16 on the way to the products of the head, they are scaled by a power of two that brings B, a bound of all of them, into [2^14, 2^15): half a step there is
at most 2^-39 B."""

import math

import pytest
import torch

from realhf_b200.ops import functional as OF
from test_token_losses import DTYPES, INF, U, err, grad64, half_step, make_head, make_logits, make_teacher, scaled

gpu = pytest.mark.gpu


def half_smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def head64(h, w, c):
    """Scaled logits in 64 bits and a bound on the kernel's: 16-bit products are exact in fp32, the accumulator cuts off once for 16 of them; fp32 operands round
    products and sums, over a tree or blocks of the sum at most as often as one after the other."""
    z = h.double() @ w.double().t() * c
    size = h.double().abs() @ w.double().abs().t() * c
    steps = h.shape[1] if h.dtype == torch.float32 else h.shape[1] / 16 + 4
    return z, size * steps * (U if h.dtype == torch.float32 else 2.0 ** -22) + U * z.abs()


def check_products(h, w, d, ed, got_h, got_w, old=None, sums=1):
    """d hidden and d weight from d logits [T, V] that are off by at most ed; `old`: what the gradient buffer held."""
    r, W, H = half_step(h.dtype), w.double(), h.double()
    for got, want, slack, n, before in ((got_h, d @ W, ed @ W.abs(), d.abs() @ W.abs(), None), (got_w, d.t() @ H, ed.t() @ H.abs(), d.abs().t() @ H.abs(), old)):
        terms = w.shape[0] if got is got_h else h.shape[0]
        cut = U * terms if h.dtype == torch.float32 else (terms / 16 + 4) * 2.0 ** -22
        slack = slack + n * cut + U * want.abs()
        step = r if got.dtype == h.dtype else U
        if before is not None:
            want = want + before
        allowed = slack + step * (want.abs() + slack) * sums + half_smallest(got.dtype) * sums
        if before is not None:
            allowed = allowed + sums * U * before.abs()
        # a value that its own type does not hold (fp16: above 65504) is rounded to an infinity of its sign
        beyond = got.isinf() & (want.abs() + allowed > torch.finfo(got.dtype).max) & (got.sign() == want.sign())
        assert ((got.double() - want).abs() <= allowed)[~beyond].all()
        assert got.any() or want.abs().max() <= half_smallest(got.dtype)


def check_head_gradients(T, H, V, dtype, temp, chunk=8192, keep=1 << 31, buffer=None, masked=False, size=None):
    dev, c = "cuda", 1.0 / temp
    size = 1.0 / T if size is None else size
    h, w, labels = make_head(T, H, V, dtype, T + V, dev)
    g = torch.Generator().manual_seed(T)
    gl = (torch.randn(T, generator=g) * size).to(dev)
    ge = ((torch.rand(T, generator=g) * -0.05 - 0.01) * size).to(dev)
    mask = bits = None
    if masked:
        mask = (torch.rand(T, V, generator=g) < 0.6).to(dev)
        mask.scatter_(1, labels[:, None], False)
        bits = OF.pack_mask_bits(mask)
    hd, wd = h.clone().requires_grad_(True), torch.nn.Parameter(w.clone())
    old = None
    if buffer is not None:
        old = (torch.randn(V, H, generator=g) * size * 0.1).to(dtype if buffer == "weight_type" else torch.float32).to(dev)
        if buffer == "weight_type":
            wd.grad, wd._grad_in_flat_buffer = old.clone(), True
        else:
            wd.main_grad = old.clone()
        old = old.double()
    logp, ent = OF.lm_head_logprobs_entropy(hd, wd, labels, bits, temperature=temp, chunk=chunk, keep_bytes=keep)
    torch.autograd.backward([logp, ent], [gl, ge])
    z, ez = head64(h, w, c)
    if masked:
        z, ez = z.masked_fill(mask, -INF), ez.masked_fill(mask, 0.0)
    y = z - torch.logsumexp(z, -1, keepdim=True)
    p = y.exp()
    H64 = torch.special.entr(p).sum(-1)
    e = (err(z, V) + ez.max(-1).values)[:, None]
    d = grad64(y, p, H64, labels, gl.double(), ge.double(), c)
    parts = c * p * (gl.abs()[:, None] + ge.abs()[:, None] * (torch.where(p > 0, -y, 0.0) + H64[:, None] + 1))
    ed = half_step(dtype) * d.abs() + parts * 4 * e + c * U * (gl.abs()[:, None] + ge.abs()[:, None]) * (p > 0)
    ed = ed + U * c * torch.zeros_like(d).scatter_(1, labels[:, None], gl.double().abs()[:, None])
    bound = float((c * (gl.abs() + ge.abs() * (H64 + 0.37))).max())
    if dtype == torch.float16:
        ed = ed + bound * 2.0 ** -39
    if dtype != torch.float32 and T > 256 and H >= 1024 and keep > 0:     # kept softmax weights: 11 bits, below 2^-29 of the largest of 128 columns 2^-40 of it
        ed = ed + 2.0 ** -11 * parts + 2.0 ** -40 * c * (gl.abs()[:, None] + ge.abs()[:, None] * (H64[:, None] + 30))
    if masked:
        ed = ed.masked_fill(mask, bound * 2.0 ** -39 if dtype == torch.float16 else 0.0)
    check_products(h, w, d, ed, hd.grad, wd.main_grad if buffer == "fp32" else wd.grad, old, 2 if buffer == "weight_type" else 1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,V,temp,kw", [(512, 256, 32000, 1.0, {}), (2048, 256, 32000, 1.5, {}), (2048, 256, 32000, 1.0, dict(chunk=500)), (600, 1024, 8003, 1.0, {}),
                                           (600, 1024, 8003, 0.7, dict(chunk=256, masked=True)), (600, 1024, 8003, 1.0, dict(keep=0, masked=True)), (16, 512, 32000, 1.0, {})])
def test_head_gradients_of_a_mean_gpu(T, H, V, temp, kw, dtype):
    check_head_gradients(T, H, V, dtype, temp, **kw)


@gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("buffer,chunk", [("weight_type", 8192), ("fp32", 8192), ("fp32", 300)])
def test_head_gradients_of_a_mean_into_a_buffer_gpu(buffer, chunk, dtype):
    check_head_gradients(1024, 256, 32000, dtype, 1.0, chunk=chunk, buffer=buffer)


@gpu
@pytest.mark.parametrize("size", [2e5, 1e-30])
@pytest.mark.parametrize("keep", [0, 1 << 31])
def test_head_gradients_beyond_the_range_of_fp16_gpu(size, keep):
    """Row gradients that fp16 does not reach, above and below (the weight's gradient goes into an fp32 buffer)."""
    check_head_gradients(300, 1024, 2003, torch.float16, 1.0, keep=keep, buffer="fp32", size=size)


def distill_gradients(z, ids, t, tr, reverse):
    """d loss / d z [T, V] of every row, and the size of its parts."""
    T, V = z.shape
    listed = torch.zeros_like(z, dtype=torch.bool).scatter_(1, ids, True)
    lse = torch.logsumexp(z, -1, keepdim=True)
    y = z - lse
    yr = torch.logsumexp(y.masked_fill(listed, -INF), -1, keepdim=True)
    yb, tb = torch.cat([y.gather(1, ids), yr], 1), torch.cat([t.double(), tr.double()[:, None]], 1)
    q, p = yb.exp(), tb.exp()
    if reverse:
        L = (q * (yb - tb)).sum(-1, keepdim=True)
        gb, sb = q * (yb - tb - L), q * (yb.abs() + tb.abs() + L.abs() + 2)
    else:
        L = (p * (tb - yb)).sum(-1, keepdim=True)
        gb, sb = p.sum(-1, keepdim=True) * q - p, 2 * (p.sum(-1, keepdim=True) * q + p)
    share = (y - yr).exp()
    return L[:, 0], (share * gb[:, -1:]).scatter(1, ids, gb[:, :-1]), (share * sb[:, -1:]).scatter(1, ids, sb[:, :-1]), gb


def check_head_distill(T, H, V, k, dtype, reverse, temp, size=None, **kw):
    dev, c = "cuda", 1.0 / temp
    h, w, _ = make_head(T, H, V, dtype, T + V, dev)
    z, ez = head64(h, w, c)
    ids, t, tr = (v.to(dev) for v in make_teacher(z, k, 3, True))
    g = ((torch.rand(T, generator=torch.Generator().manual_seed(4)) + 0.2) * (1.0 / T if size is None else size)).to(dev)
    hd, wd = h.clone().requires_grad_(True), torch.nn.Parameter(w.clone())
    loss = OF.lm_head_distill_loss(hd, wd, ids, t, tr, reverse=reverse, temperature=temp, **kw)
    loss.backward(g)
    want, per, parts, gb = distill_gradients(z, ids, t, tr, reverse)
    e = (2 * (err(z, V) + ez.max(-1).values) + U * k)[:, None]
    rows = (g.double() * c)[:, None]
    d, parts = per * rows, parts * rows
    ed = half_step(dtype) * d.abs() + 3 * e * parts
    if dtype == torch.float16:
        ed = ed + float((rows * gb.abs()).max()) * 2.0 ** -39
    check_products(h, w, d, ed, hd.grad, wd.grad)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("T,H,V,k,temp,kw", [(37, 64, 501, 8, 1.2, dict(chunk=16)), (512, 256, 32000, 64, 1.0, {}), (512, 256, 32000, 64, 1.0, dict(keep_bytes=0, chunk=200)),
                                             (2048, 256, 16001, 20, 1.5, {})])
def test_head_distillation_gradients_of_a_mean_gpu(T, H, V, k, temp, kw, reverse, dtype):
    check_head_distill(T, H, V, k, dtype, reverse, temp, **kw)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_a_mean_from_logits_gpu(dtype):
    """Statistics and distillation from logits: the result alone is rounded, below the normal numbers by half the smallest step."""
    T, V, k = 256, 32000, 64
    x, labels = make_logits(T, V, dtype, 3, "cuda")
    z = x.double()
    y = z - torch.logsumexp(z, -1, keepdim=True)
    p = y.exp()
    H64 = torch.special.entr(p).sum(-1)
    e = err(z, V)
    g = torch.Generator().manual_seed(5)
    gl, ge = (torch.randn(T, generator=g) / T).cuda(), ((torch.rand(T, generator=g) * -0.05 - 0.01) / T).cuda()
    leaf = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(OF.logprob_entropy_from_logits(leaf, labels), leaf, [gl, ge])
    want = grad64(y, p, H64, labels, gl.double(), ge.double(), 1.0)
    parts = p * (gl.abs()[:, None] + ge.abs()[:, None] * (torch.where(p > 0, -y, 0.0) + H64[:, None] + 1))
    one = torch.zeros_like(z).scatter_(1, labels[:, None], gl.double().abs()[:, None])
    assert ((d.double() - want).abs() <= half_step(dtype) * want.abs() + half_smallest(dtype) + 4 * e * parts + 2 * U * one).all() and d.any()
    ids, t, tr = (v.cuda() for v in make_teacher(z, k, 3, True))
    for reverse in (False, True):
        d, = torch.autograd.grad(OF.distill_loss_from_logits(leaf, ids, t, tr, reverse), leaf, gl.abs())
        _, per, parts, _ = distill_gradients(z, ids, t, tr, reverse)
        rows = gl.double().abs()[:, None]
        want = per * rows
        assert ((d.double() - want).abs() <= half_step(dtype) * want.abs() + half_smallest(dtype) + 3 * (2 * e + U * k) * parts * rows).all() and d.any()


@gpu
def test_head_gradients_where_nothing_is_asked_or_a_row_is_bad_gpu():
    """No gradient at all: zeros.  A row whose gradient is NaN (a label beyond the vocabulary) leaves the other rows of d hidden as they are without it."""
    T, H, V = 300, 1024, 2003
    h, w, labels = make_head(T, H, V, torch.float16, 1, "cuda")
    for keep in (0, 1 << 31):
        results = []
        for bad in (False, True):
            hd, wd = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            lab = labels.clone()
            gl = torch.randn(T, generator=torch.Generator().manual_seed(2)).cuda() / T
            gl[7] = 0
            if bad:
                lab[7], gl[7] = V, 1.0
            logp, ent = OF.lm_head_logprobs_entropy(hd, wd, lab, keep_bytes=keep)
            a, b = torch.autograd.grad(logp, [hd, wd], gl, retain_graph=True)
            results.append(a)
            assert bool(b.isfinite().all()) != bad
            zero = torch.autograd.grad([logp, ent], [hd, wd], [torch.zeros_like(logp)] * 2)
            assert not zero[0].any() and not zero[1].any()
        assert results[1][7].isnan().all()
        results[1][7] = results[0][7]
        # (the bad row's own size takes part in the scale: below the normal numbers of fp16 a step of 2^-39 of 1, at most V of them of |W| <= 1)
        assert ((results[0].double() - results[1].double()).abs() <= 2 * (V * 2.0 ** -39 + half_step(torch.float16) * results[0].double().abs() + 2.0 ** -25)).all()


@gpu
def test_head_gradients_captured_gpu():
    """The scale goes by what a replay finds: row gradients 2^14 apart, each replay as an eager call."""
    T, H, V, k = 300, 1024, 2003, 5
    h, w, labels = make_head(T, H, V, torch.float16, 1, "cuda")
    ids, t, tr = (v.cuda() for v in make_teacher(make_logits(T, V, torch.float32, 4)[0], k, 3, True))
    g = torch.randn(T, generator=torch.Generator().manual_seed(2)).cuda()

    def work():
        a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        logp, ent = OF.lm_head_logprobs_entropy(a, b, labels)
        loss = OF.lm_head_distill_loss(a, b, ids, t, tr)
        return [*torch.autograd.grad([logp, ent], [a, b], [g, g]), *torch.autograd.grad(loss, [a, b], g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for scale in (1.0, 2.0 ** -14, 1.0):
        g.copy_(torch.randn(T, generator=torch.Generator().manual_seed(3)).cuda() * scale)
        graph.replay()
        for a, b in zip(out, work()):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("keep_bytes", [0, 1 << 31])
def test_head_distillation_gradients_that_are_next_to_nothing_gpu(keep_bytes):
    """A student that has learnt its teacher: every gradient below 1e-33 of an incoming one of 100, for which the scale of d logits is the largest there is."""
    T, H, V = 3, 64, 40
    w = torch.zeros(V, H, dtype=torch.float16)
    w[0, :] = 1.0
    h = torch.full((T, H), 85.0 / 64, dtype=torch.float16)           # logits 85 and 0: the others hold e^-85 = 1e-37 of the mass each
    hd, wd = h.cuda().requires_grad_(True), torch.nn.Parameter(w.cuda())
    wd.main_grad = torch.zeros(V, H, device="cuda")
    ids, t, tr = torch.zeros(T, 1, dtype=torch.long, device="cuda"), torch.zeros(T, 1, device="cuda"), torch.full((T,), -INF, device="cuda")
    loss = OF.lm_head_distill_loss(hd, wd, ids, t, tr, keep_bytes=keep_bytes)
    loss.backward(torch.full((T,), 100.0, device="cuda"))
    assert loss.abs().max() < 1e-30 and not hd.grad.any()
    assert wd.main_grad.isfinite().all() and wd.main_grad.abs().max() < 1e-30
