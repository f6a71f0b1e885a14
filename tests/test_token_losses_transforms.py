"""Token statistics and distillation through the head inside function transforms and forward-mode differentiation: plain torch operations answer."""

import pytest
import torch

from realhf_b200.ops import functional as OF
from test_token_losses import DTYPES, U, err, half_step, make_head, make_logits, make_teacher

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
