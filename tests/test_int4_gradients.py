"""The 4-bit operators have no gradient: what would need one is refused on both devices, never dropped on one and kept on the other."""
import pytest
import torch
from torch.autograd import forward_ad

from realhf_b200.ops import int4

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]


def pieces(device):
    g = torch.Generator().manual_seed(0)
    z = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16)   # noqa: E731
    cache = int4.Int4KVCache(2, 8, 1, 64, torch.bfloat16, device)
    return z, z(16, 128), z(16), z(2, 128), z(2, 256), cache, torch.tensor([0, 3], dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_bias(device):
    z, w, b, x, _, _, _ = pieces(device)
    lin, plain = int4.Int4Linear(w, b.clone().requires_grad_()), int4.Int4Linear(w, b)
    assert torch.equal(lin(x), plain(x)) and not lin(x).requires_grad             # kept with the weight: numbers alone
    again = int4.Int4Linear.from_codes(*plain.codes(), b.clone().requires_grad_())
    assert torch.equal(again(x), plain(x)) and not again(x).requires_grad
    with pytest.raises(RuntimeError):
        plain(x, b.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(plain(x, b.clone().requires_grad_()), plain(x))


@pytest.mark.parametrize("device", DEVICES)
def test_a_kept_bias_follows_its_tensor(device):
    """It shares the tensor's numbers: an optimiser's step in place is seen by the next call."""
    z, w, b, x, _, _, _ = pieces(device)
    p = torch.nn.Parameter(b.clone())
    lin = int4.Int4Linear(w, p)
    before = lin(x)
    with torch.no_grad():
        p.add_(64)
    assert not torch.equal(lin(x), before) and torch.equal(lin(x), int4.Int4Linear(w, b + 64)(x))


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode(device):
    z, w, b, x, qkv, cache, lens = pieces(device)
    lin = int4.Int4Linear(w)
    step = lambda t: int4.decode_attention_int4(t, cache, lens, 2, 1, 64)   # noqa: E731
    want = lin(x), step(qkv)
    held = cache.data.clone()
    with forward_ad.dual_level():
        for f, t in ((lin, x), (step, qkv), (lambda c: lin(x, c), b)):
            with pytest.raises(RuntimeError):
                f(forward_ad.make_dual(t, torch.ones_like(t)))
        assert torch.equal(cache.data, held)
        assert torch.equal(lin(x), want[0]) and torch.equal(step(qkv), want[1])   # nothing to differentiate: as outside
    for f, t in ((lin, x), (step, qkv)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda y: f(y).float().sum())(t)
