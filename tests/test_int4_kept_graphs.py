"""A captured decode step that is kept reads quantised copies of the weights: they live as long as the graph does, whatever other calls on the model do."""
import pytest
import torch

from realhf_b200.api.model import GenerationHyperparameters
from realhf_b200.models import generation as gen
from realhf_b200.ops import int4
from test_int4_generation import prompts, tiny


def options(n, **kw):
    return GenerationHyperparameters(max_new_tokens=n, min_new_tokens=n, greedy=True, **{"use_cuda_graph": True, **kw})


def test_a_state_renews_the_copies_that_its_graph_reads(monkeypatch):
    """(On the CPU nothing is captured: what stands in for a graph is a mark that there is one.)  A call with other options frees the model's copies, not the state's, and the next call with that
    state reads the state's."""
    m = tiny("cpu", torch.bfloat16)
    ids, cu = prompts("cpu")
    _, state = gen.generate(m, ids, cu, options(3), eos_id=None, pad_id=0)
    m.enable_int4_decode()
    copies = dict(m._int4)
    read = m.copies_read()
    assert len(read) == len(copies) == 9 and len(set(read)) == 9
    state.graph, state.copies = object(), (None, m._int4)
    m.disable_int4_decode(free=False)
    assert m.copies_read() == ()
    gen.generate(m, ids, cu, options(3, int4_weights=True), eos_id=None, pad_id=0)                 # another state
    assert m._int4 is None
    seen, real = [], int4.Int4Linear.__call__
    monkeypatch.setattr(int4.Int4Linear, "__call__", lambda self, x, bias=None: (seen.append(self), real(self, x, bias))[1])
    m.p["1.mlp.down.weight"].mul_(-1)
    out, _ = gen.generate(m, ids, cu, options(3, int4_weights=True), eos_id=None, pad_id=0, state=state)
    assert {id(f) for f in seen} == {id(f) for f in copies.values()}
    fresh, _ = gen.generate(m, ids, cu, options(3, int4_weights=True), eos_id=None, pad_id=0)
    assert torch.equal(out.tokens, fresh.tokens) and torch.equal(out.logprobs, fresh.logprobs)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int4_weights", "fp8_weights"])
def test_kept_graph_after_a_call_that_keeps_none(kind):
    """Kept graph, a call with the default options on another state, then the kept state again, with memory that the allocator could have taken from freed copies."""
    m = tiny("cuda", torch.bfloat16)
    ids, cu = prompts("cuda")
    keep = options(10, force_cudagraph_recapture=False, **{kind: True})
    _, state = gen.generate(m, ids, cu, keep, eos_id=None, pad_id=0)
    graph = state.graph
    assert graph is not None
    fresh, _ = gen.generate(m, ids, cu, options(10, **{kind: True}), eos_id=None, pad_id=0)
    junk = [torch.full((1 << 18,), -1, dtype=torch.int8, device="cuda") for _ in range(64)]
    out, state = gen.generate(m, ids, cu, keep, eos_id=None, pad_id=0, state=state)
    assert state.graph is graph and len(junk) == 64
    assert torch.equal(out.tokens, fresh.tokens)
    torch.testing.assert_close(out.logprobs, fresh.logprobs, atol=1e-3, rtol=1e-3)
    for n, p in m.p.items():
        if n.endswith("mlp.down.weight"):
            p.mul_(-1)
    out, state = gen.generate(m, ids, cu, keep, eos_id=None, pad_id=0, state=state)
    fresh, _ = gen.generate(m, ids, cu, options(10, **{kind: True}), eos_id=None, pad_id=0)
    assert state.graph is graph and torch.equal(out.tokens, fresh.tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int4_weights", "fp8_weights"])
def test_kept_graph_before_and_after_an_eager_call(kind, monkeypatch):
    """One state in three calls whose sampling lies outside the graph: captured, eager, captured."""
    monkeypatch.setenv("REAL_GEN_SAMPLE_IN_GRAPH", "0")
    m = tiny("cuda", torch.bfloat16)
    ids, cu = prompts("cuda")
    state, outs = None, []
    for graph in (True, False, True):
        g = options(10, force_cudagraph_recapture=False, use_cuda_graph=graph, **{kind: True})
        out, state = gen.generate(m, ids, cu, g, eos_id=None, pad_id=0, state=state)
        outs.append(out)
        assert state.graph is not None
        junk = [torch.full((1 << 18,), -1, dtype=torch.int8, device="cuda") for _ in range(64)]
        assert len(junk) == 64
    for out in outs[1:]:
        assert torch.equal(out.tokens, outs[0].tokens)
        torch.testing.assert_close(out.logprobs, outs[0].logprobs, atol=1e-3, rtol=1e-3)


@pytest.mark.parametrize("kind", ["int4_weights", "fp8_weights"])
def test_an_error_in_the_loop_leaves_no_copies_in_use(kind, monkeypatch):
    monkeypatch.setenv("REAL_FP8_EMULATE", "1")
    m = tiny("cpu", torch.bfloat16)
    ids, cu = prompts("cpu")
    real = gen.genstep

    def failing(logits, g, step, *a, **k):
        if step == 2:
            assert m._int4_active or m._fp8_active
            raise KeyError("sampling")
        return real(logits, g, step, *a, **k)
    monkeypatch.setattr(gen, "genstep", failing)
    with pytest.raises(KeyError):
        gen.generate(m, ids, cu, GenerationHyperparameters(max_new_tokens=5, min_new_tokens=5, greedy=True, **{kind: True}), eos_id=None, pad_id=0)
    assert not m._int4_active and not m._fp8_active and m._int4 is None and m._fp8 is None


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_kept_graph_after_a_longer_sequence(bits):
    """A sequence beyond the tables of cosines and sines makes the model take longer ones: the kept graph's live on, with the same numbers."""
    import weakref
    m = tiny("cuda", torch.bfloat16)
    ids, cu = prompts("cuda")
    keep = options(10, force_cudagraph_recapture=False, kv_cache_bits=bits)
    want, state = gen.generate(m, ids, cu, keep, eos_id=None, pad_id=0)
    graph, table, n = state.graph, weakref.ref(m._rope[0]), m._rope[0].shape[0]
    assert graph is not None
    m.rope_tables(2 * n)
    junk = [torch.full((n, 32), 7.0, device="cuda") for _ in range(16)]
    assert m._rope[0].shape[0] >= 2 * n and table() is not None and table() is not m._rope[0] and len(junk) == 16
    out, state = gen.generate(m, ids, cu, keep, eos_id=None, pad_id=0, state=state)
    assert state.graph is graph and torch.equal(out.tokens, want.tokens)
    torch.testing.assert_close(out.logprobs, want.logprobs, atol=1e-3, rtol=1e-3)
    _, state = gen.generate(m, ids, cu, options(10, kv_cache_bits=bits), eos_id=None, pad_id=0, state=state)      # (keeps none)
    assert state.graph is None and table() is None


def test_copies_that_were_in_use_before_a_call_stay_in_use():
    """Copies that a program has put to use by hand are its own: a call without the option leaves them so, with an error too."""
    m = tiny("cpu", torch.bfloat16)
    ids, cu = prompts("cpu")
    m.enable_int4_decode()
    copies = m._int4
    gen.generate(m, ids, cu, options(3), eos_id=None, pad_id=0)
    assert m._int4_active and m._int4 is copies
    with pytest.raises(AttributeError):
        gen.generate(m, ids, cu, None, eos_id=None, pad_id=0)
    assert m._int4_active and m._int4 is copies
