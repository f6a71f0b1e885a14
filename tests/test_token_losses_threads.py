"""Calls from several host threads at once: rows of different lengths through one kernel, each with shared memory of its own size."""

import threading

import pytest
import torch

from realhf_b200.ops import functional as OF
from test_token_losses import make_logits, make_teacher

gpu = pytest.mark.gpu


def run_at_once(calls, times):
    """Every call in a thread and a stream of its own, again and again; the errors they met and their last results."""
    errors, results, ready = [], [None] * len(calls), threading.Barrier(len(calls))

    def loop(i):
        stream = torch.cuda.Stream()
        ready.wait()
        with torch.cuda.stream(stream), torch.no_grad():
            for _ in range(times):
                try:
                    results[i] = calls[i]()
                except Exception as e:      # noqa: BLE001
                    errors.append(e)
                    return
        stream.synchronize()

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors, results


@gpu
@pytest.mark.parametrize("what", ["top", "top_many", "distill"])
def test_lengths_at_once_gpu(what):
    k = 300 if what == "top_many" else 8
    calls = []
    for V in (262000, 300000, 350000) if what == "distill" else (130000, 160000, 190000):
        x, labels = make_logits(2, V, torch.bfloat16, V, "cuda")
        if what == "distill":
            ids, t, tr = (v.cuda() for v in make_teacher(x, k, 1, True))
            calls.append(lambda x=x, ids=ids, t=t, tr=tr: (OF.distill_loss_from_logits(x, ids, t, tr),))
        else:
            calls.append(lambda x=x, labels=labels: OF.top_logprobs_from_logits(x, k, labels))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    errors, results = run_at_once(calls * 2, 5000 if what == "distill" else 1500)
    torch.cuda.synchronize()
    assert not errors, errors[0]
    for i, r in enumerate(results):
        for a, b in zip(r, want[i % len(want)]):
            assert torch.equal(a, b)
