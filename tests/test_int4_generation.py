"""Generation with a 4-bit cache and 4-bit weights: which rows and weights are quantised, where, and that captured and eager loops agree."""
import pytest
import torch

from realhf_b200.api.model import GenerationHyperparameters, ReaLModelConfig
from realhf_b200.models import generation as gen
from realhf_b200.models.real_model import ReaLModel
from realhf_b200.ops import attention as A
from realhf_b200.ops import int4

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]


def tiny(device, dtype, hd=64, nq=4, nkv=2, vocab=320, bias=True, **kw):
    cfg = ReaLModelConfig(n_layers=2, n_kv_heads=nkv, n_q_heads=nq, hidden_dim=nq * hd, intermediate_dim=3 * hd * nq, vocab_size=vocab, n_positions=512, embd_pdrop=0.0,
                          resid_pdrop=0.0, attn_pdrop=0.0, activation_function="silu", scale_attn_by_inverse_layer_idx=False, use_attention_bias=bias,
                          use_attn_proj_bias=False, use_mlp_bias=False, layer_norm_type="rms", mlp_type="llama", apply_rotary=True, **kw)
    m = ReaLModel(cfg, dtype=dtype, device=torch.device(device)).instantiate(seed=3, std=0.06)
    for p in m.parameters():
        p.requires_grad_(False)
    return m.eval()


def prompts(device, vocab=320, lens=(5, 17, 1, 40)):
    g = torch.Generator().manual_seed(2)
    return (torch.randint(3, vocab, (sum(lens),), generator=g).to(device),
            torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=device))


def rounded(x, group, dtype):
    return int4.dequantize_groups(*int4.quantize_groups(x.to(dtype), group)).to(x.dtype)


def held_decode(qkv, kc, vc, lens, nq, nkv, hd, scale=None, cos=None, sin=None, rot=None, inter=False):
    """A 16-bit cache's step with every row rounded as a 4-bit cache holds it."""
    B, dt = qkv.shape[0], torch.bfloat16
    q, k, v = (t.reshape(B, -1, hd).float() for t in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    if cos is not None:
        q, k = (int4._rotated(t, cos[lens.long()], sin[lens.long()], rot or hd, inter) for t in (q, k))
    idx = torch.arange(B)
    kc[idx, lens.long()], vc[idx, lens.long()] = rounded(k, 32, dt).to(kc.dtype), rounded(v, 64, dt).to(vc.dtype)
    return A.decode_attention_ref(q, kc, vc, lens + 1, scale).reshape(B, nq * hd).to(qkv.dtype)


def test_cache_wiring(monkeypatch):
    """The loop over a 4-bit cache is the loop over a cache whose rows, of the prompt and generated, are rounded as the 4-bit one holds them; its state is a quarter
    of the size."""
    m = tiny("cpu", torch.float32)
    ids, cu = prompts("cpu")
    kw = dict(max_new_tokens=12, min_new_tokens=12, greedy=True)
    out, state = gen.generate(m, ids, cu, GenerationHyperparameters(kv_cache_bits=4, **kw), eos_id=None, pad_id=0)
    assert state.kv_bits == 4 and all(isinstance(c, int4.Int4KVCache) for c in state.k) and state.k[0].shape == (4, 52, 2, 64)
    assert state.k[0].nbytes() * 3 < 2 * 2 * 4 * 64 * 2 * 64                     # (rooms are rounded up to 16 rows: 64)
    monkeypatch.setattr(A, "decode_attention", held_decode)
    fill = gen.prefill_into_state

    def held_fill(model, st, *a, **k):
        h = fill(model, st, *a, **k)
        for kc, vc in zip(st.k, st.v):
            kc.copy_(rounded(kc.contiguous(), 32, torch.bfloat16))
            vc.copy_(rounded(vc.contiguous(), 64, torch.bfloat16))
        return h
    monkeypatch.setattr(gen, "prefill_into_state", held_fill)
    ref, st16 = gen.generate(m, ids, cu, GenerationHyperparameters(**kw), eos_id=None, pad_id=0, state=state)   # (a state of another kind is not taken)
    assert st16.kv_bits == 16
    assert torch.equal(out.tokens, ref.tokens)
    torch.testing.assert_close(out.logprobs, ref.logprobs, atol=1e-4, rtol=1e-4)


def test_states_filled_both_ways_are_the_same():
    m = tiny("cpu", torch.float32)
    ids, cu = prompts("cpu")
    a, b = (gen.DecodeState(m, 4, 60, 4) for _ in range(2))
    gen.prefill_into_state(m, a, [0, 1, 2, 3], ids, cu)
    kv = []
    with torch.no_grad():
        m(input_ids=ids, cu_seqlens=cu, max_seqlen=40, kv_sink=kv)
    b.fill_from_prefill(kv, cu, cu[1:] - cu[:-1])
    assert all(torch.equal(x.data, y.data) for x, y in zip(a.k, b.k)) and torch.equal(a.cache_lens, b.cache_lens)


@pytest.mark.parametrize("tied", [False, True])
def test_weight_wiring(tied, monkeypatch):
    """Every block linear and the head of every decode step go through the 4-bit product, with the bias of the projection, and nothing is left behind.  The log-probabilities
    are those of a model whose weights are the numbers that the copies hold (rounded to bfloat16 once more there: a step of 2^-8 on weights of std 0.06)."""
    m = tiny("cpu", torch.bfloat16, tied_embedding=tied)
    ids, cu = prompts("cpu")
    calls = []
    real = int4.Int4Linear.__call__
    monkeypatch.setattr(int4.Int4Linear, "__call__", lambda self, x, bias=None: (calls.append((self.N, self.K, bias is not None)), real(self, x, bias))[1])
    n = 6
    g = GenerationHyperparameters(max_new_tokens=n, min_new_tokens=n, greedy=True, int4_weights=True)
    out, _ = gen.generate(m, ids, cu, g, eos_id=None, pad_id=0)
    qkv = ((4 + 2 * 2) * 64, 256, True)
    assert calls == ([qkv, (256, 256, False), (2 * 768, 256, False), (256, 768, False)] * 2 + [(320, 256, False)]) * (n - 1)
    assert m._int4 is None and not m._int4_active
    calls.clear()
    base, _ = gen.generate(m, ids, cu, GenerationHyperparameters(max_new_tokens=n, min_new_tokens=n, greedy=True), eos_id=None, pad_id=0)
    assert not calls
    assert torch.equal(out.tokens[:, 0], base.tokens[:, 0])                        # the prompt's pass reads the model's own weights
    if tied:
        return
    twin = tiny("cpu", torch.bfloat16)
    for name, p in m.p.items():
        if name in twin.p:
            twin.p[name].copy_(p)
    twin.enable_int4_decode()
    for name, f in twin._int4.items():
        (twin.head_weight() if name == "head" else twin.p[name]).copy_((int4.Int4Linear(m.head_weight(), group=f.group) if name == "head" else f).dequantize())
    twin.disable_int4_decode()
    st = gen.DecodeState(m, 4, 60)
    gen.prefill_into_state(m, st, [0, 1, 2, 3], ids, cu)
    with torch.no_grad():
        for step in range(n - 1):
            h = twin.decode_step(out.tokens[:, step], st.k, st.v, st.cache_lens)
            st.cache_lens += 1
            lp = torch.log_softmax(gen._final_logits(twin, h).float(), -1).gather(1, out.tokens[:, step + 1: step + 2])[:, 0]
            assert float((lp - out.logprobs[:, step + 1]).abs().max()) < 0.1


def test_options():
    for bad in (dict(kv_cache_bits=8), dict(kv_cache_bits=2), dict(int4_weights=True, fp8_weights=True)):
        with pytest.raises(ValueError):
            GenerationHyperparameters(**bad)
    with pytest.raises(ValueError):
        gen.DecodeState(tiny("cpu", torch.float32, hd=32), 1, 8, 4)
    with pytest.raises(ValueError):
        gen.DecodeState(tiny("cpu", torch.float32), 1, 8, 8)
    from realhf_b200.models import hf_io
    hetero = ReaLModel(hf_io.family("rapodra").make_test_config(), dtype=torch.float32, device=torch.device("cpu")).instantiate(seed=1)
    with pytest.raises(ValueError):
        gen.DecodeState(hetero, 1, 8, 4)
    assert not hetero.int4_decode_supported()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv", [(64, 8, 8), (128, 8, 2), (64, 14, 2)])
@pytest.mark.parametrize("bits,weights", [(4, False), (16, True), (4, True)])
def test_captured_and_eager_loops_agree(hd, nq, nkv, bits, weights):
    if bits == 16 and nq // nkv == 7:
        pytest.skip("the decode kernel over 16-bit caches takes groups of 1, 2, 4 and 8")
    m = tiny("cuda", torch.bfloat16, hd, nq, nkv)
    ids, cu = prompts("cuda")
    outs = []
    for graph in (False, True):
        g = GenerationHyperparameters(max_new_tokens=40, min_new_tokens=40, greedy=True, use_cuda_graph=graph, kv_cache_bits=bits, int4_weights=weights)
        outs.append(gen.generate(m, ids, cu, g, eos_id=None, pad_id=0)[0])
    assert torch.equal(outs[0].tokens, outs[1].tokens)
    torch.testing.assert_close(outs[0].logprobs, outs[1].logprobs, atol=1e-3, rtol=1e-3)
    assert m._int4 is None and not m._int4_active


@pytest.mark.gpu
def test_cache_on_the_gpu_is_the_cpus():
    """The same prompt and steps over a 4-bit cache on both devices: the log-probabilities of the same tokens."""
    a, b = tiny("cpu", torch.bfloat16), tiny("cuda", torch.bfloat16)
    for n, p in a.p.items():
        b.p[n].copy_(p)
    ids, cu = prompts("cpu")
    sa, sb = gen.DecodeState(a, 4, 64, 4), gen.DecodeState(b, 4, 64, 4)
    gen.prefill_into_state(a, sa, [0, 1, 2, 3], ids, cu)
    gen.prefill_into_state(b, sb, [0, 1, 2, 3], ids.cuda(), cu.cuda())
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for _ in range(5):
            tok = torch.randint(3, 320, (4,), generator=g)
            la, lb = (torch.log_softmax(gen._final_logits(m, m.decode_step(tok.to(m.device), s.k, s.v, s.cache_lens)).float(), -1).cpu() for m, s in ((a, sa), (b, sb)))
            sa.cache_lens += 1
            sb.cache_lens += 1
            assert float((la - lb).abs().max()) < 0.1          # (activations in bfloat16 on both, in another order of sums)


@pytest.mark.gpu
def test_kept_graph_reads_weights_anew():
    """`force_cudagraph_recapture=False`: the graph of the first call serves the second, whose weights are others."""
    m = tiny("cuda", torch.bfloat16)
    ids, cu = prompts("cuda")
    g = GenerationHyperparameters(max_new_tokens=10, min_new_tokens=10, greedy=True, use_cuda_graph=True, force_cudagraph_recapture=False, kv_cache_bits=4, int4_weights=True)
    _, state = gen.generate(m, ids, cu, g, eos_id=None, pad_id=0)
    graph = state.graph
    assert graph is not None and m._int4 is not None and not m._int4_active
    for n, p in m.p.items():
        if n.endswith("mlp.down.weight") or n.endswith("attn.qkv.weight"):
            p.mul_(-1)
    out, state = gen.generate(m, ids, cu, g, eos_id=None, pad_id=0, state=state)
    assert state.graph is graph
    fresh, _ = gen.generate(m, ids, cu, GenerationHyperparameters(max_new_tokens=10, min_new_tokens=10, greedy=True, kv_cache_bits=4, int4_weights=True), eos_id=None, pad_id=0)
    assert torch.equal(out.tokens, fresh.tokens)
    torch.testing.assert_close(out.logprobs, fresh.logprobs, atol=1e-3, rtol=1e-3)


@pytest.mark.parametrize("device", DEVICES)
def test_inflight_batching_over_a_4_bit_cache(device):
    """More prompts than slots: each request's tokens are those that it gets alone."""
    m = tiny(device, torch.float32 if device == "cpu" else torch.bfloat16)
    g = GenerationHyperparameters(max_new_tokens=9, min_new_tokens=9, greedy=True, kv_cache_bits=4)
    ids, cu = prompts(device, lens=(5, 17, 1, 30, 8))
    ps = [ids[int(cu[i]): int(cu[i + 1])] for i in range(5)]
    got = gen.InflightBatchingGenerator(m, g, None, 0, 2, 30).generate(ps)
    for p, (toks, lps, _) in zip(ps, got):
        one, _ = gen.generate(m, p, torch.tensor([0, p.numel()], dtype=torch.int32, device=device), g, eos_id=None, pad_id=0)
        same = [a == b for a, b in zip(toks, one.tokens[0].tolist())]
        assert len(toks) == 9 and (all(same) if device == "cpu" else same[0])
        if all(same):
            torch.testing.assert_close(torch.tensor(lps), one.logprobs[0].cpu(), atol=2e-2 if device == "cuda" else 1e-4, rtol=2e-2 if device == "cuda" else 1e-4)
