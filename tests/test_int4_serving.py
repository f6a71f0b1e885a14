"""4-bit caches and weights in the loops around `generate`: in-flight batching, pipeline stages, and what is said where an option is not used."""
import pytest
import torch

from realhf_b200.api.model import GenerationHyperparameters, ReaLModelConfig
from realhf_b200.models import generation as gen
from realhf_b200.models.real_model import ReaLModel
from test_int4_generation import DEVICES, prompts, tiny


def said(monkeypatch):
    lines = []
    monkeypatch.setattr(gen, "_SAID", set())
    monkeypatch.setattr(gen.logging, "getLogger", lambda *a: type("L", (), {"warning": staticmethod(lines.append)}))
    return lines


@pytest.mark.parametrize("why", ["supported", "fp8", "sequences", "type", "batching"])
def test_a_loop_that_cannot_use_4_bit_weights_says_so(why, monkeypatch):
    lines = said(monkeypatch)
    m = tiny("cpu", torch.float32 if why == "type" else torch.bfloat16)
    g = GenerationHyperparameters(max_new_tokens=2, min_new_tokens=2, greedy=True, int4_weights=True)
    ids, cu = prompts("cpu", lens=(2,) * 129) if why == "sequences" else prompts("cpu")
    if why == "fp8":
        monkeypatch.setenv("REAL_FP8_EMULATE", "1")
        monkeypatch.setenv("REAL_GEN_FP8", "1")
    for _ in range(2):                                     # ... once
        if why == "batching":
            gen.InflightBatchingGenerator(m, g, None, 0, 2, 40).generate([ids[:5], ids[5:9], ids[9:12]])
        else:
            gen.generate(m, ids, cu, g, eos_id=None, pad_id=0)
    assert len(lines) == (why != "supported") and all("int4_weights is not used" in line for line in lines)
