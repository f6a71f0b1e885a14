"""The actor's ratio is formed from one definition of the log-probability, with an entropy bonus and without: that of logits rounded to the head's type."""

from types import SimpleNamespace

import pytest
import torch

from realhf_b200.interfaces import ppo
from realhf_b200.models.real_model import ModelOutput
from realhf_b200.ops import functional as OF
from test_token_losses import U, err, grad64, half_step, make_head, stats64
from test_token_losses_small_gradients import check_products, head64

gpu = pytest.mark.gpu


def check_unchanged_policy(dev, dtype, seqlens, H, V):
    """old_logp from the same weights: every ratio is 1, but for what the two kernels' sums of the same rounded logits differ by and, on a GPU, for logits that lie so near
    to the middle between two 16-bit numbers that the order of their products' sum decides: those may move by a step."""
    T = sum(seqlens)
    h, w, _ = make_head(T, H, V, dtype, 1, dev)
    ids = torch.arange(T, device=dev) * 7 % V
    n = T - len(seqlens)
    mask = torch.ones(n, dtype=torch.bool, device=dev)
    mask[:3] = False
    out = ModelOutput(hidden=h.clone().requires_grad_(True), head_weight=w, ctx=None)
    rows, labels = ppo.IF.shifted_rows_and_labels(seqlens, ids)
    with torch.no_grad():
        old = out.logprobs(labels, None, 1.0, rows)
    data = dict(packed_input_ids=ids, old_logp=old, advantages=torch.linspace(-1, 1, n, device=dev), ppo_loss_mask=mask)
    mb = SimpleNamespace(data=data, flat_seqlens=lambda key: seqlens)
    logp, _ = out.logprobs_entropy(labels, None, 1.0, rows, rounded=True)
    z, ez = head64(h[rows], w, 1.0)
    low, high = (z - ez).to(dtype).double(), (z + ez).to(dtype).double()
    step = (high - low) if dev == "cuda" and dtype != torch.float32 else torch.zeros_like(z)     # (on a CPU, and in fp32, both forms take the same product)
    y, p, _, _ = stats64(high, labels)
    allowed = 4 * err(z, V) + step.gather(1, labels[:, None])[:, 0] + (p * step).sum(-1) * 1.1
    assert ((logp.double() - old.double()).abs() <= allowed).all()
    assert (allowed < 1e-3).any()
    for coef in (0.0, 0.3):
        loss, stat = ppo._actor_loss_from_output(out, mb, kl_adapter=None, eps_clip=0.2, temperature=1.0, early_stop_imp_ratio=None, early_stop_kl=None, entropy_coef=coef)
        most = float(allowed.mean()) * n / int(mask.sum()) * 1.1
        assert abs(float(stat["importance_weight"]) - 1.0) <= most and abs(float(stat["ppo_approx_kl"])) <= most
        assert float(stat["actor_clip_ratio"]) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_unchanged_policy_cpu(dtype):
    check_unchanged_policy("cpu", dtype, [9, 14], 64, 304)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seqlens,H,V", [([9, 14], 64, 304), ([200, 1, 333], 1024, 8000), ([140, 60], 512, 32000), ([33], 60, 1003)])
def test_unchanged_policy_gpu(seqlens, H, V, dtype):
    check_unchanged_policy("cuda", dtype, seqlens, H, V)


def check_rounded_statistics(dev, dtype, T, H, V, masked, **kw):
    """Statistics and gradients of rounded logits.  Hidden states are whole numbers up to 8 and weights 64ths up to 1 / 8: every sum of products is exact in fp32, and the
    rounded logit known."""
    g = torch.Generator().manual_seed(T)
    h = torch.randint(-8, 9, (T, H), generator=g).to(dtype).to(dev)
    w = (torch.randint(-8, 9, (V, H), generator=g) / 64).to(dtype).to(dev)
    labels = torch.randint(0, V, (T,), generator=g).to(dev)
    gl, ge = (torch.randn(T, generator=g) / T).to(dev), (torch.randn(T, generator=g) * 0.1 / T).to(dev)
    z = (h.double() @ w.double().t()).to(dtype).double() / 1.3
    bits = None
    if masked:
        mask = (torch.rand(T, V, generator=g) < 0.6).to(dev).scatter_(1, labels[:, None], False)
        bits, z = OF.pack_mask_bits(mask), z.masked_fill(mask, float("-inf"))
    hd, wd = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    logp, ent = OF.lm_head_logprobs_entropy(hd, wd, labels, bits, 1.3, rounded=True, **kw)
    torch.autograd.backward([logp, ent], [gl, ge])
    y, p, want_logp, want_H = stats64(z, labels)
    e = err(z, V)
    assert ((logp.detach().double() - want_logp).abs() <= 2 * e + U * want_logp.abs()).all()
    assert ((ent.detach().double() - want_H).abs() <= 4 * e * (1 + want_H) + U).all()
    d = grad64(y, p, want_H, labels, gl.double(), ge.double(), 1 / 1.3)
    parts = p * (gl.abs()[:, None] + ge.abs()[:, None] * (torch.where(p > 0, -y, 0.0) + want_H[:, None] + 1))
    whole = gl.abs()[:, None] + ge.abs()[:, None] * (want_H[:, None] + 30)
    ed = half_step(dtype) * d.abs() + parts * 4 * e + 2 * U * torch.zeros_like(d).scatter_(1, labels[:, None], whole.double())
    if dtype != torch.float32:
        ed = ed + 2.0 ** -11 * parts + 2.0 ** -39 * float(whole.max())
    check_products(h, w, d, ed, hd.grad, wd.grad)


ROUNDED = [(5, 64, 40, False, {}), (33, 64, 130, True, dict(chunk=16))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,V,masked,kw", ROUNDED)
def test_rounded_statistics_cpu(T, H, V, masked, kw, dtype):
    check_rounded_statistics("cpu", dtype, T, H, V, masked, **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,V,masked,kw", ROUNDED + [(300, 1024, 5003, False, {}), (300, 1024, 5003, True, dict(chunk=128)), (300, 1024, 5003, True, dict(keep_bytes=0)),
                                                       (70, 512, 32000, False, {}), (40, 60, 100, True, {})])
def test_rounded_statistics_gpu(T, H, V, masked, kw, dtype):
    check_rounded_statistics("cuda", dtype, T, H, V, masked, **kw)


@gpu
def test_rounded_statistics_beside_a_gradient_buffer_gpu():
    """The route of weights with a gradient buffer beside .grad gives what the native one does."""
    h, w, labels = make_head(300, 1024, 2000, torch.bfloat16, 3, "cuda")
    results = []
    for own in (False, True):
        a, b = h.clone().requires_grad_(True), torch.nn.Parameter(w.clone())
        if own:
            b.main_grad = torch.zeros(b.shape, device="cuda")
        logp, ent = OF.lm_head_logprobs_entropy(a, b, labels, rounded=True)
        (logp.sum() + ent.sum()).backward()
        results.append((logp.detach(), ent.detach(), a.grad, (b.main_grad if own else b.grad).bfloat16()))
    for x, y in zip(*results):
        assert torch.equal(x, y)


def check_capped(dev, dtype, softcap, scale):
    """A capped or scaled head: both calls have the same log-probability, the cap's tanh apart (8 u of it)."""
    h, w, labels = make_head(21, 64, 304, dtype, 2, dev)
    out = ModelOutput(hidden=h, head_weight=w, ctx=None, softcap=softcap, logit_scale=scale)
    with torch.no_grad():
        old = out.logprobs(labels, None, 0.9)
    logp, _ = out.logprobs_entropy(labels, None, 0.9, rounded=True)
    z = out.logits.double() / 0.9
    assert ((logp.double() - old.double()).abs() <= 4 * err(z, 304) + 32 * U * float(z.abs().max())).all()


@pytest.mark.parametrize("softcap,scale", [(20.0, None), (20.0, 0.5), (None, 0.5)])
def test_capped_and_scaled_heads_cpu(softcap, scale):
    check_capped("cpu", torch.bfloat16, softcap, scale)


def _sharded_logprobs(rank, world):
    from realhf_b200.base.topology import ParallelContext, ProcessTopology
    ctx = ParallelContext.build(ProcessTopology(1, 1, world), list(range(world)), rank, backend="gloo")
    h, w, labels = make_head(9, 32, 64, torch.bfloat16, 2)
    per = 64 // world
    out = ModelOutput(hidden=h, head_weight=w[rank * per: (rank + 1) * per].clone(), ctx=ctx)
    return out.logprobs(labels, None, 0.9).tolist(), out.logprobs_entropy(labels, None, 0.9, rounded=True)[0].tolist()


@pytest.mark.distributed
def test_sharded_head_cpu():
    from realhf_b200.base.testing import run_distributed
    h, w, _ = make_head(9, 32, 64, torch.bfloat16, 2)
    z = h.double() @ w.double().t() / 0.9
    for old, new in run_distributed(_sharded_logprobs, 2):
        assert ((torch.tensor(old, dtype=torch.float64) - torch.tensor(new, dtype=torch.float64)).abs() <= 4 * err(z, 64)).all()
