"""Alternatives through the head at sizes that a teacher has: several chunks of rows, an odd vocabulary, lists of every variant of the kernel."""

import pytest
import torch

from realhf_b200.ops import functional as OF
from test_token_losses import DTYPES, INF, U, err, make_head
from test_token_losses_small_gradients import head64

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,V,k,chunk,masked,temp", [(600, 512, 50257, 20, 256, False, 1.0), (300, 1024, 32000, 64, 4096, True, 0.7), (130, 256, 32003, 256, 64, False, 1.0),
                                                       (70, 256, 20011, 700, 4096, False, 1.3), (5, 512, 200003, 10, 4096, False, 1.0), (1, 4096, 32000, 20, 4096, False, 1.0)])
def test_head_alternatives_gpu(T, H, V, k, chunk, masked, temp, dtype):
    """Values against 64 bits in the order that 64 bits give; a token that stands elsewhere is within the two logits' errors of the one it displaced."""
    c = 1.0 / temp
    h, w, labels = make_head(T, H, V, dtype, T + V, "cuda")
    z, ez = head64(h, w, c)
    bits = None
    if masked:
        mask = (torch.rand(T, V, generator=torch.Generator().manual_seed(1)) < 0.7).cuda()
        mask.scatter_(1, labels[:, None], False)
        bits, z, ez = OF.pack_mask_bits(mask), z.masked_fill(mask, -INF), ez.masked_fill(mask, 0.0)
    o = OF.lm_head_top_logprobs(h, w, k, labels, bits, temperature=temp, chunk=chunk)
    e = (err(z, V) + ez.max(-1).values)[:, None]
    lse = torch.logsumexp(z, -1, keepdim=True)
    y = z - lse
    want = torch.sort(y, -1, descending=True).values[:, :k]
    assert ((o.top_logp.double() - want).abs() <= 2 * e + U * want.abs()).all()
    assert o.top_ids.shape == (T, k) and (torch.sort(o.top_ids, -1).values.diff(dim=-1) > 0).all()
    assert ((y.gather(1, o.top_ids) - want).abs() <= 4 * e).all()
    got = o.top_logp.diff(dim=-1)
    assert (got <= 0).all()
    rest = torch.logsumexp(y.scatter(1, o.top_ids, -INF), -1)
    assert ((o.rest_logp.double() - rest).abs() <= 2 * e[:, 0] + U * rest.abs()).all()
    p = y.exp()
    H64 = torch.special.entr(p).sum(-1)
    assert ((o.entropy.double() - H64).abs() <= 4 * e[:, 0] * (1 + H64) + U).all()
    want = y.gather(1, labels[:, None])[:, 0]
    assert ((o.logp.double() - want).abs() <= 2 * e[:, 0] + U * want.abs()).all()


@gpu
def test_kernels_of_d_hidden_are_counted_gpu():
    from realhf_b200.ops import launches, lib
    d, w = torch.randn(64, 2048, dtype=torch.float16, device="cuda"), torch.randn(2048, 256, dtype=torch.float16, device="cuda")
    out = torch.empty(64, 256, dtype=torch.float16, device="cuda")
    results = []
    for splits, kernels in ((1, 1), (4, 2)):      # (parts are added up by a second kernel)
        before = launches.total
        lib().head_dhidden(d, w, out, splits, 148)
        assert launches.total - before == kernels
        results.append(out.double())
    want = d.double() @ w.double()
    size = d.double().abs() @ w.double().abs()
    for got in results:       # the accumulator cuts off once for 16 terms, at most 2^-22 of their sizes' sum; the result is rounded once
        assert ((got - want).abs() <= size * (2048 / 16 + 4) * 2.0 ** -22 + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
