"""Token statistics and distillation through the head inside function transforms and forward-mode differentiation: plain torch operations answer."""

import pytest
import torch

from realhf_b200.ops import functional as OF
from test_token_losses import DTYPES, err, half_step, make_head, make_logits, make_teacher

gpu = pytest.mark.gpu


def functions(dev, dtype, T=7, H=64, V=50):
    h, w, labels = make_head(T, H, V, dtype, 1, dev)
    ids, t, tr = (v.to(dev) for v in make_teacher(make_logits(T, V, torch.float32, 4)[0], 4, 3, True))
    return h, w, [lambda a, b: (OF.lm_head_logprobs_entropy(a, b, labels)[0] - 0.5 * OF.lm_head_logprobs_entropy(a, b, labels, rounded=True)[1]).sum(),
                  lambda a, b: OF.lm_head_distill_loss(a, b, ids, t, tr).sum(), lambda a, b: OF.lm_head_distill_loss(a, b, ids, t, tr, reverse=True).sum()]


def check_transforms(dev, dtype):
    """Against autograd's own gradients of the same call.  Both are off by the roundings of test_token_losses.py: d logits, whose parts are at most 1 + the entropy's 4
    (reverse divergence: log-probabilities of up to 20 twice), by 8 E of them and two half steps, sums of 50 and 7 products by as much as their terms, the result by
    half a step."""
    h, w, fs = functions(dev, dtype)
    e, r = err(h.double() @ w.double().t(), 50) + 64 * 2.0 ** -22 * 40, half_step(dtype)
    for f, size in zip(fs, (5, 4, 45)):
        got = torch.func.grad(f, argnums=(0, 1))(h, w)
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        f(a, b).backward()
        for x, y, other in zip(got, (a.grad, b.grad), (w, h)):
            slack = size * (16 * e + 4 * r) * other.double().abs().sum(0)
            assert x.dtype == y.dtype and ((x.double() - y.double()).abs() <= slack + 2 * r * y.double().abs()).all()
        va, vb = torch.randn_like(h), torch.randn_like(w)
        _, along = torch.func.jvp(f, (h, w), (va, vb))
        want = sum((x.double() * v.double()).sum() for x, v in zip((a.grad, b.grad), (va, vb)))
        rounded = sum((size * (16 * e + 4 * r) * o.double().abs().sum(0) * v.double().abs()).sum() for o, v in ((w, va), (h, vb)))
        assert abs(float(along.double() - want)) <= float(rounded)


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_head_inside_function_transforms_cpu(dtype):
    check_transforms("cpu", dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_inside_function_transforms_gpu(dtype):
    check_transforms("cuda", dtype)


def check_alternatives(dev, dtype):
    """A list of alternatives taken inside a transform is that of the plain call, to the bounds of test_token_losses.py; what it is multiplied with has its gradient."""
    h, w, labels = make_head(6, 64, 50, dtype, 1, dev)
    x = make_logits(12, 50, dtype, 2, dev)[0].view(4, 3, 50)
    e = 4 * (err(h.double() @ w.double().t(), 50) + 64 * 2.0 ** -22 * 40)
    flat = OF.top_logprobs_from_logits(x.view(12, 50), 3, labels.repeat(2))
    got = torch.func.vmap(lambda a, b: OF.top_logprobs_from_logits(a, 3, b))(x, labels.repeat(2).view(4, 3))
    assert torch.equal(got.top_ids.view(12, 3), flat.top_ids)
    for a, b in ((got.top_logp, flat.top_logp), (got.rest_logp, flat.rest_logp), (got.logp, flat.logp), (got.entropy, flat.entropy)):
        assert ((a.reshape(b.shape) - b).abs() <= e * (1 + b.abs())).all()
    plain = OF.lm_head_top_logprobs(h, w, 3, labels, chunk=4)
    got = torch.func.vmap(lambda a: OF.lm_head_top_logprobs(a, w, 3, labels, chunk=4).top_logp)(torch.stack([h, h]))
    assert ((got - plain.top_logp).abs() <= e * (1 + plain.top_logp.abs())).all()
    top = torch.func.grad(lambda a: (a.float() * OF.lm_head_top_logprobs(a, w, 3).top_logp.sum()).sum())(h)
    want = plain.top_logp.double().sum()
    assert ((top.double() - want).abs() <= (18 * e * 21 + half_step(dtype) * want.abs())).all()
    per = torch.func.grad(lambda a: (a.float() * OF.top_logprobs_from_logits(a, 3).top_logp.sum()).sum())(x[0])
    want = flat.top_logp[:3].double().sum()
    assert ((per.double() - want).abs() <= (9 * e * 21 + half_step(dtype) * want.abs())).all()


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_alternatives_inside_function_transforms_cpu(dtype):
    check_alternatives("cpu", dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_inside_function_transforms_gpu(dtype):
    check_alternatives("cuda", dtype)
