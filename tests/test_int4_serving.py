"""4-bit caches and weights in the loops around `generate`: in-flight batching, pipeline stages, and what is said where an option is not used."""
import pytest
import torch

from realhf_b200.api.model import GenerationHyperparameters, ReaLModelConfig
from realhf_b200.models import generation as gen
from realhf_b200.models.real_model import ReaLModel
from realhf_b200.ops import int4
from test_int4_generation import DEVICES, prompts, tiny


def said(monkeypatch):
    lines = []
    monkeypatch.setattr(gen, "_SAID", set())
    monkeypatch.setattr(gen.logging, "getLogger", lambda *a: type("L", (), {"warning": staticmethod(lines.append)}))
    return lines


@pytest.mark.parametrize("why", ["supported", "fp8", "sequences", "type", "batching"])
def test_a_loop_that_cannot_use_4_bit_weights_says_so(why, monkeypatch):
    lines, calls = said(monkeypatch), []
    real = int4.Int4Linear.__call__
    monkeypatch.setattr(int4.Int4Linear, "__call__", lambda self, x, bias=None: (calls.append(x.shape[0]), real(self, x, bias))[1])
    m = tiny("cpu", torch.float32 if why == "type" else torch.bfloat16)
    g = GenerationHyperparameters(max_new_tokens=2, min_new_tokens=2, greedy=True, int4_weights=True)
    ids, cu = prompts("cpu", lens=(2,) * 17) if why == "sequences" else prompts("cpu", lens=(2,) * 16) if why == "supported" else prompts("cpu")
    if why == "fp8":
        monkeypatch.setenv("REAL_FP8_EMULATE", "1")
        monkeypatch.setenv("REAL_GEN_FP8", "1")
    for _ in range(2):                                     # ... once
        if why == "batching":
            gen.InflightBatchingGenerator(m, g, None, 0, 2, 40).generate([ids[:5], ids[5:9], ids[9:12]])
        else:
            gen.generate(m, ids, cu, g, eos_id=None, pad_id=0)
    assert len(lines) == (why != "supported") and all("int4_weights is not used" in line for line in lines)
    assert set(calls) == ({16} if why == "supported" else set())


class Checked(gen.InflightBatchingGenerator):
    """In-flight batching that looks after each refill at what the slot's cache holds: bit by bit what a cache of its own would, whoever had the slot before."""
    refills = 0

    def _refill(self, slot, req_id, prompt):
        super()._refill(slot, req_id, prompt)
        alone = gen.DecodeState(self.model, 1, self.state.S, 4)
        n = prompt.numel()
        cu = torch.tensor([0, n], dtype=torch.int32, device=prompt.device)
        gen.prefill_into_state(self.model, alone, [0], prompt, cu, n)
        at = torch.tensor([slot], dtype=torch.int32, device=prompt.device)
        for a, b in zip(self.state.k, alone.k):
            for x, y in zip(a.load(cu, n, slots=at), b.load(cu, n)):
                assert torch.equal(x, y) and bool(x.abs().sum() > 0)
        assert int(self.state.cache_lens[slot]) == n
        self.refills += 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd,nq,nkv", [(64, 4, 2), (128, 2, 2)])
def test_inflight_slots_hold_their_own_requests(device, hd, nq, nkv):
    """More prompts than slots.  Each request's tokens, fed one by one to a state of its own, have the log-probabilities that the batch gave them: those of all tokens but the first are read from
    the cache.  Both sides quantise the same rows up to the rounding of bfloat16 activations, which products of one and of two rows sum in another order: as between two devices 0.1 (in fp32 1e-4)."""
    m = tiny(device, torch.float32 if device == "cpu" else torch.bfloat16, hd, nq, nkv)
    g = GenerationHyperparameters(max_new_tokens=9, min_new_tokens=9, greedy=True, kv_cache_bits=4)
    ids, cu = prompts(device, lens=(5, 17, 1, 30, 8, 16))
    ps = [ids[int(cu[i]): int(cu[i + 1])] for i in range(6)]
    batch = Checked(m, g, None, 0, 2, 30)
    got = batch.generate(ps)
    assert batch.refills == 6
    for p, (toks, lps, _) in zip(ps, got):
        st = gen.DecodeState(m, 1, 48, 4)
        h = gen.prefill_into_state(m, st, [0], p, torch.tensor([0, p.numel()], dtype=torch.int32, device=device), p.numel())[-1:]
        assert len(toks) == 9
        for tok, lp in zip(toks, lps):
            with torch.no_grad():
                want = float(torch.log_softmax(gen._final_logits(m, h).float(), -1)[0, tok])
                h = m.decode_step(torch.tensor([tok], device=device), st.k, st.v, st.cache_lens)
            st.cache_lens += 1
            assert abs(lp - want) < (1e-4 if device == "cpu" else 0.1)


def _stages(rank, world, layout, bits):
    import types

    from realhf_b200.api.config import ModelName
    from realhf_b200.api.data import SequenceSample
    from realhf_b200.api.model import FinetuneSpec, Model
    from realhf_b200.base.topology import ParallelContext, ProcessTopology
    from realhf_b200.engine.engine import InferenceBackend
    cfg = ReaLModelConfig(n_layers=4, n_kv_heads=2, n_q_heads=4, hidden_dim=256, intermediate_dim=512, vocab_size=320, n_positions=512, embd_pdrop=0.0, resid_pdrop=0.0, attn_pdrop=0.0,
                          activation_function="silu", scale_attn_by_inverse_layer_idx=False, use_attention_bias=True, use_attn_proj_bias=False, use_mlp_bias=False, layer_norm_type="rms",
                          mlp_type="llama", apply_rotary=True)
    ctx = ParallelContext.build(ProcessTopology(*layout), list(range(world)), rank, backend="gloo", sequence_parallel=False)
    m = ReaLModel(cfg, ctx, dtype=torch.float32, device=torch.device("cpu")).instantiate(seed=7, std=0.06)
    model = InferenceBackend().initialize(Model(ModelName("m", 0), m, None, "cpu"), FinetuneSpec(1, 10, 10))
    states, real = [], gen.DecodeState.fill_from_prefill

    def noted(self, kv, cu, lens):
        real(self, kv, cu, lens)
        states.append((self.kv_bits, len(self.k), all(c.nbytes() < 2 * 2 * 4 * c.slots * c.room * c.n_kv * c.hd // 3 for c in self.k) if self.kv_bits == 4 else False))
    gen.DecodeState.fill_from_prefill = noted
    lens = [4, 16, 5, 17]
    batch = SequenceSample.from_default(seqlens=lens, ids=list(range(4)), data=dict(packed_input_ids=torch.arange(2, 2 + sum(lens))))
    g = GenerationHyperparameters(max_new_tokens=14, min_new_tokens=14, greedy=True, kv_cache_bits=bits)
    outs = model.module.generate(batch, types.SimpleNamespace(eos_token_id=1, pad_token_id=0), g, num_micro_batches=1)
    return dict(states=states, tokens=None if outs is None else torch.cat([o.tokens for o in outs]).tolist(), logprobs=None if outs is None else torch.cat([o.logprobs for o in outs]).tolist())


@pytest.mark.distributed
@pytest.mark.parametrize("layout", [(2, 1, 1), (2, 1, 2)])
def test_pipeline_stages_over_a_4_bit_cache(layout):
    """Two stages, each with caches of its own blocks, give the tokens of one process over a 4-bit cache."""
    from realhf_b200.base.testing import run_distributed
    one = run_distributed(_stages, 1, layout=(1, 1, 1), bits=4)[0]
    plain = run_distributed(_stages, 1, layout=(1, 1, 1), bits=16)[0]
    res = run_distributed(_stages, layout[0] * layout[2], layout=layout, bits=4)
    for r in res:
        assert r["states"] and all(s == (4, 2, True) for s in r["states"])
    outs = [r for r in res if r["tokens"] is not None]
    assert outs
    for r in outs:
        assert r["tokens"] == one["tokens"]
        torch.testing.assert_close(torch.tensor(r["logprobs"]), torch.tensor(one["logprobs"]), atol=1e-4, rtol=1e-4)
    assert not torch.allclose(torch.tensor(plain["logprobs"]), torch.tensor(one["logprobs"]), atol=1e-4, rtol=1e-4)
