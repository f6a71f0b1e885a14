"""The distillation recipe of docs/customization.md, run as it is written: a teacher's inference, a student's training step on what it returns."""
import os
import re

import torch

from realhf_b200.api import model as model_api
from realhf_b200.api.data import SequenceSample
from realhf_b200.interfaces import functional as IF
from test_engine_cpu import make_model, sft_batch
from test_token_losses import distill64, make_teacher

DOC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "docs", "customization.md")


def recipe():
    blocks = re.findall(r"```python\n(.*?)```", open(DOC).read(), re.S)
    (code,) = [b for b in blocks if "def teacher_hook" in b]
    space = dict(torch=torch, IF=IF, SequenceSample=SequenceSample, model_api=model_api)
    exec(code, space)
    return space


def logits_of(model, batch):
    rows, _ = IF.shifted_rows_and_labels(batch.flat_seqlens("packed_input_ids"), batch.data["packed_input_ids"])
    return model.module.forward(batch, num_micro_batches=1, post_hook=lambda out, mb: out.logits[rows]).double()


def test_teacher_and_student_as_documented():
    space = recipe()
    teacher, student = make_model("teacher", train=False, seed=3), make_model("student", seed=5, lr=1e-3)
    itf = space["Distillation"]()
    batch = sft_batch(bs=5, seed=2)
    zt, zs = logits_of(teacher, batch), logits_of(student, batch)
    batch.update_(itf.inference(teacher, batch, n_mbs=2))
    lt, k = torch.log_softmax(zt, -1), batch.data["top_ids"].shape[1]
    assert batch.data["top_ids"].dtype == torch.int64 and 1 <= k < zt.shape[1]
    torch.testing.assert_close(batch.data["top_logp"].double(), torch.sort(lt, -1, descending=True).values[:, :k], atol=1e-5, rtol=1e-5)
    torch.testing.assert_close(lt.gather(1, batch.data["top_ids"]).float(), batch.data["top_logp"], atol=1e-5, rtol=1e-5)
    want = distill64(zs, batch.data["top_ids"], batch.data["top_logp"], batch.data["rest_logp"], False)[0].mean()
    before = student.module.module.flat_param.data.clone()
    st = itf.train_step(student, batch, n_mbs=1)
    assert abs(float(st["loss"]) - float(want)) <= 1e-5 * (1 + float(want)) and float(st["grad_norm"]) > 0
    assert not torch.equal(before, student.module.module.flat_param.data)
    # micro-batches cut what the teacher returned along its sequences
    st = itf.train_step(student, batch, n_mbs=3)
    assert float(st["loss"]) > 0


def test_what_a_teacher_returns_has_a_default_length():
    x = torch.randn(7, 20)
    ids, t, tr = make_teacher(x, 4, 1, True)
    s = SequenceSample.from_default(ids=[0, 1], seqlens=[5, 4], data=dict(top_ids=ids, top_logp=t, rest_logp=tr))
    first, second = s.split(2)
    assert first.data["top_ids"].shape[0] in (3, 4) and first.data["top_ids"].shape[0] + second.data["rest_logp"].shape[0] == 7
