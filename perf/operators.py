"""Token statistics over a vocabulary and the losses built on them, measured through the framework's public entry points.

Kinds:
  logprobs  log-probability of a given token and entropy of its distribution from logits [T, V]: "infer", or "train" with the gradient of
            both with respect to the logits; optionally under the packed mask of the sampler's filters and a temperature.
  top       the k most likely tokens of every row, their log-probabilities, the log of the mass of all others, and what "logprobs" gives,
            in one call: what a teacher or a reporting server stores.
  distill   Kullback-Leibler divergence between a teacher known by its k most likely tokens and a student's logits, with the gradient:
            the k tokens are one outcome each, all others together are one more ("rest") or left out.
  head      log-probability and entropy from hidden states through the language-model head, without logits in memory: "infer", or
            "train" with the gradients of hidden states and head weight.

A case is a dict of plain values.  With `own` false `run` computes the plain forms, elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random
from typing import Dict, List

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_CELLS = 8192 * 131072
NEG = float("-inf")


# ------------------------------------------------------------------------------------------------ the cases


def listed() -> List[dict]:
    return [
        # one generation step of 16 sequences whose chosen tokens are scored: latency counts
        dict(name="logprobs_infer_16x32000", kind="logprobs", mode="infer", rows=16, vocab=32000, dtype="bf16", masked=False, temp=1.0),
        # the actor's minibatch of the PPO benchmark with an entropy bonus, logits at hand
        dict(name="logprobs_train_8192x32000", kind="logprobs", mode="train", rows=8192, vocab=32000, dtype="bf16", masked=False, temp=1.0),
        # GPT-2's vocabulary (odd rows), fp32 logits, under the sampler's filters and its temperature
        dict(name="logprobs_train_2047x50257_masked", kind="logprobs", mode="train", rows=2047, vocab=50257, dtype="fp32", masked=True, temp=0.7),
        # scoring a long batch over a large vocabulary
        dict(name="logprobs_infer_8192x131072", kind="logprobs", mode="infer", rows=8192, vocab=131072, dtype="bf16", masked=False, temp=1.0),
        # a serving step that reports twenty alternatives a sequence
        dict(name="top20_16x32000", kind="top", rows=16, vocab=32000, top=20, dtype="bf16", temp=1.0),
        # a teacher's pass over a training batch
        dict(name="top64_4096x131072", kind="top", rows=4096, vocab=131072, top=64, dtype="bf16", temp=1.0),
        # a ragged evaluation batch, fp32 logits of an odd vocabulary, a few alternatives
        dict(name="top5_1001x50257", kind="top", rows=1001, vocab=50257, top=5, dtype="fp32", temp=0.8),
        # distillation step: 64 teacher tokens and the rest, forward divergence
        dict(name="distill_fwd_8192x32000_k64", kind="distill", rows=8192, vocab=32000, top=64, dtype="bf16", reverse=False, rest=True, temp=1.0),
        # on-policy distillation: the student's own samples, reverse divergence, large vocabulary
        dict(name="distill_rev_2000x131072_k128", kind="distill", rows=2000, vocab=131072, top=128, dtype="bf16", reverse=True, rest=True, temp=1.0),
        # a short batch with the teacher renormalised over 256 tokens, fp32, temperature 2
        dict(name="distill_fwd_257x50257_k256", kind="distill", rows=257, vocab=50257, top=256, dtype="fp32", reverse=False, rest=False, temp=2.0),
        # the actor's minibatch of the PPO benchmark through the LLaMA-7B head
        dict(name="head_train_8192x4096x32000", kind="head", mode="train", rows=8192, width=4096, vocab=32000, dtype="bf16", temp=1.0),
        # reference scoring of a ragged batch through a GPT-2 head
        dict(name="head_infer_2047x1024x50257", kind="head", mode="infer", rows=2047, width=1024, vocab=50257, dtype="fp16", temp=1.0),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["logprobs", "logprobs", "top", "top", "distill", "distill", "head"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    temp = rng.choice([1.0, 1.0, 0.7, 1.5])
    if kind == "head":
        width, vocab = 8 * _log(rng, 32, 512), _log(rng, 1000, 50257)
        most = max(1, min(8192, 8192 * 4096 * 32000 // (width * vocab)))
        return dict(kind=kind, mode=rng.choice(["infer", "train"]), rows=_log(rng, 1, most), width=width, vocab=vocab, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    temp=temp)
    vocab = rng.choice([_log(rng, 300, 131072), _log(rng, 300, 131072), 32000, 50257])
    bytes_each = 4 if dtype == "fp32" else 2
    rows = _log(rng, 1, max(1, min(8192, MAX_CELLS // (vocab * bytes_each))))
    if kind == "logprobs":
        return dict(kind=kind, mode=rng.choice(["infer", "train"]), rows=rows, vocab=vocab, dtype=dtype, masked=rng.random() < 0.3, temp=temp)
    top = _log(rng, 1, 256)
    rows = min(rows, 4096)
    if kind == "top":
        return dict(kind=kind, rows=rows, vocab=vocab, top=top, dtype=dtype, temp=temp)
    reverse = rng.random() < 0.4
    return dict(kind=kind, rows=rows, vocab=vocab, top=top, dtype=dtype, reverse=reverse, rest=reverse or rng.random() < 0.6, temp=temp)


def work(case: dict) -> Dict[str, float]:
    T, V, b = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "head":
        H, train = case["width"], case["mode"] == "train"
        once = (T * H + V * H) * b
        return {"bytes": once * (2 if train else 1) + T * (16 + (8 if train else 0)), "flops": (6.0 if train else 2.0) * T * V * H}
    cells = T * V
    if case["kind"] == "logprobs":
        train = case["mode"] == "train"
        return {"bytes": cells * b * (2 if train else 1) + T * (16 + (8 if train else 0)) + (cells // 8 if case["masked"] else 0), "flops": cells * (8.0 if train else 4.0)}
    if case["kind"] == "top":
        return {"bytes": cells * b + T * (20 + case["top"] * 12), "flops": cells * 5.0}
    return {"bytes": 2 * cells * b + T * (12 + case["top"] * 12), "flops": cells * 8.0}


# ------------------------------------------------------------------------------------------------ inputs


def _logits(g, T, V, dtype, dev):
    """Rows as a trained model gives them: a broad bulk, a few tokens far above it, some rows nearly decided, others not."""
    x = torch.randn(T, V, generator=g, device=dev, dtype=torch.float32).mul_(2.2)
    n = min(V, 12)
    at = torch.randint(0, V, (T, n), generator=g, device=dev)
    lift = torch.rand(T, n, generator=g, device=dev) * 9 + torch.rand(T, 1, generator=g, device=dev) * 4
    x.scatter_add_(1, at, lift)
    return x.to(dtype), at[:, 0].contiguous()


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    T, V, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    s = dict(case=dict(case), inv_temp=1.0 / case["temp"])
    if case["kind"] == "head":
        H, train = case["width"], case["mode"] == "train"
        w = torch.randn(V, H, generator=g, device=dev).mul_(1 / math.sqrt(H))
        labels = torch.randint(0, V, (T,), generator=g, device=dev)
        h = torch.randn(T, H, generator=g, device=dev).mul_(1.8) + w[labels] * (torch.rand(T, 1, generator=g, device=dev) * 12)
        s.update(hidden=h.to(dt).requires_grad_(train), weight=w.to(dt).requires_grad_(train), labels=labels)
    else:
        logits, labels = _logits(g, T, V, dt, dev)
        s.update(logits=logits, labels=labels)
    if case["kind"] == "logprobs":
        s["mask_bits"] = None
        if case["masked"]:  # the sampler keeps about a tenth of the tokens, the sampled one among them; bit j % 8 of byte j // 8, set = filtered out
            keep = s["logits"] >= s["logits"].float().mean(1, keepdim=True) + 2.8
            keep.scatter_(1, labels[:, None], True)
            m = torch.nn.functional.pad((~keep).to(torch.uint8), (0, -V % 8)).view(T, -1, 8)
            s["mask_bits"] = (m << torch.arange(8, device=dev, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)
    if case.get("mode") == "train":
        s["g_logp"] = torch.randn(T, generator=g, device=dev) / T
        s["g_entropy"] = torch.rand(T, generator=g, device=dev).mul_(-0.05).sub_(0.01) / T
    if case["kind"] == "logprobs":
        s["logits"].requires_grad_(case["mode"] == "train")
    if case["kind"] == "distill":
        k = min(case["top"], V)
        teacher = s["logits"].float() * 0.8 + torch.randn(T, V, generator=g, device=dev)
        lt = torch.log_softmax(teacher * s["inv_temp"], -1)
        s["top_logp"], s["top_ids"] = torch.topk(lt, k, dim=-1)
        rest = torch.logsumexp(lt.scatter(1, s["top_ids"], NEG), -1)
        s["rest_logp"] = rest if case["rest"] else None
        del teacher, lt
        s["g_loss"] = (torch.rand(T, generator=g, device=dev) + 0.2) / T
        s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_stats(x, labels):
    """Scaled (and masked) fp32 logits x [T, V] -> (log-probabilities [T, V], probabilities, logp of the labels, entropy)."""
    m = x.max(-1, keepdim=True).values
    lse = m + torch.exp(x - m).sum(-1, keepdim=True).log()
    y = x - lse
    p = torch.exp(y)
    entropy = -torch.where(p > 0, p * y, torch.zeros_like(p)).sum(-1)
    return y, p, y.gather(1, labels[:, None]).squeeze(1), entropy


def _plain_grad(y, p, labels, entropy, g_logp, g_entropy):
    """d / dx of g_logp * y[label] + g_entropy * H: g_logp (onehot - p) - g_entropy p (y + H)."""
    d = -p * (g_logp[:, None] + g_entropy[:, None] * (torch.where(p > 0, y, torch.zeros_like(y)) + entropy[:, None]))
    return d.scatter_add_(1, labels[:, None], g_logp[:, None])


def _plain_logprobs(s):
    x = s["logits"].detach().float() * s["inv_temp"]
    if s["mask_bits"] is not None:
        bit = torch.arange(x.shape[1], device=x.device)
        x = torch.where(((s["mask_bits"][:, bit // 8] >> (bit % 8)) & 1).bool(), torch.full_like(x, NEG), x)
    y, p, logp, entropy = _plain_stats(x, s["labels"])
    if s["case"]["mode"] == "infer":
        return dict(logp=logp, entropy=entropy)
    d = _plain_grad(y, p, s["labels"], entropy, s["g_logp"], s["g_entropy"]) * s["inv_temp"]
    return dict(logp=logp, entropy=entropy, dlogits=d.to(s["logits"].dtype))


def _plain_top(s):
    raw = s["logits"].float()
    T, V = raw.shape
    x = raw * s["inv_temp"]
    y, p, logp, entropy = _plain_stats(x, s["labels"])
    bits = (raw + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) - torch.arange(V, device=raw.device)  # equal values: the lowest index first
    ids = torch.topk(key, min(s["case"]["top"], V), dim=-1).indices
    others = x.scatter(1, ids, NEG)
    m = others.max(-1, keepdim=True).values.clamp(min=-3e38)
    rest = m.squeeze(1) + torch.exp(others - m).sum(-1).log() - (x - y)[:, 0]
    return dict(top_logp=y.gather(1, ids), top_ids=ids, rest_logp=rest, logp=logp, entropy=entropy)


def _plain_distill(s):
    x = s["logits"].detach().float() * s["inv_temp"]
    ids, t = s["top_ids"], s["top_logp"]
    m = x.max(-1, keepdim=True).values
    lse = m + torch.exp(x - m).sum(-1, keepdim=True).log()
    xk = x.gather(1, ids)
    others = x.scatter(1, ids, NEG)
    mo = others.max(-1, keepdim=True).values.clamp(min=-3e38)
    lse_rest = mo + torch.exp(others - mo).sum(-1, keepdim=True).log()
    if s["rest_logp"] is None:  # the teacher's k tokens are its whole distribution
        mt = t.max(-1, keepdim=True).values
        t = t - mt - torch.exp(t - mt).sum(-1, keepdim=True).log()
        tr = torch.full_like(lse, NEG)
    else:
        tr = s["rest_logp"][:, None]
    t, y = torch.cat([t, tr], 1), torch.cat([xk, lse_rest], 1) - lse  # outcomes: the k tokens, then the rest
    e = torch.exp(others - lse_rest.clamp(min=-3e38))                 # a token's share of the rest
    if s["case"]["reverse"]:
        q = torch.exp(y)
        f = torch.where(q > 0, y - t, torch.zeros_like(y))
        loss = (q * f).sum(-1)
        per = q * (f - loss[:, None])
    else:
        p = torch.exp(t)
        loss = torch.where(p > 0, p * (t - y), torch.zeros_like(p)).sum(-1)
        per = p.sum(-1, keepdim=True) * torch.exp(y) - p
    per = per * (s["g_loss"] * s["inv_temp"])[:, None]
    d = (e * per[:, -1:]).scatter(1, ids, per[:, :-1])
    return dict(loss=loss, dlogits=d.to(s["logits"].dtype))


def _plain_head(s):
    h, w = s["hidden"].detach().float(), s["weight"].detach().float()
    y, p, logp, entropy = _plain_stats((h @ w.t()) * s["inv_temp"], s["labels"])
    if s["case"]["mode"] == "infer":
        return dict(logp=logp, entropy=entropy)
    d = _plain_grad(y, p, s["labels"], entropy, s["g_logp"], s["g_entropy"]) * s["inv_temp"]
    return dict(logp=logp, entropy=entropy, dhidden=(d @ w).to(s["hidden"].dtype), dweight=(d.t() @ h).to(s["weight"].dtype))


# ------------------------------------------------------------------------------------------------ one pass


def _own(s):
    from realhf_b200.ops import functional as OF
    c = s["case"]
    if c["kind"] == "top":
        o = OF.top_logprobs_from_logits(s["logits"], min(c["top"], c["vocab"]), s["labels"], inv_temp=s["inv_temp"])
        return dict(top_logp=o.top_logp, top_ids=o.top_ids, rest_logp=o.rest_logp, logp=o.logp, entropy=o.entropy)
    if c["kind"] == "distill":
        loss = OF.distill_loss_from_logits(s["logits"], s["top_ids"], s["top_logp"], s["rest_logp"], reverse=c["reverse"], inv_temp=s["inv_temp"])
        (d,) = torch.autograd.grad([loss], [s["logits"]], [s["g_loss"]])
        return dict(loss=loss.detach(), dlogits=d)
    if c["kind"] == "logprobs":
        logp, entropy = OF.logprob_entropy_from_logits(s["logits"], s["labels"], s["mask_bits"], inv_temp=s["inv_temp"])
        inputs, names = [s["logits"]], ["dlogits"]
    else:
        logp, entropy = OF.lm_head_logprobs_entropy(s["hidden"], s["weight"], s["labels"], temperature=c["temp"])
        inputs, names = [s["hidden"], s["weight"]], ["dhidden", "dweight"]
    if c["mode"] == "infer":
        return dict(logp=logp, entropy=entropy)
    grads = torch.autograd.grad([logp, entropy], inputs, [s["g_logp"], s["g_entropy"]])
    return dict(logp=logp.detach(), entropy=entropy.detach(), **dict(zip(names, grads)))


def run(state: dict):
    if own:
        return _own(state)
    return {"logprobs": _plain_logprobs, "top": _plain_top, "distill": _plain_distill, "head": _plain_head}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    T = case["rows"]
    names = {"logprobs": ["logp", "entropy"] + (["dlogits"] if case.get("mode") == "train" else []),
             "top": ["top_logp", "top_ids", "rest_logp", "logp", "entropy"], "distill": ["loss", "dlogits"],
             "head": ["logp", "entropy"] + (["dhidden", "dweight"] if case.get("mode") == "train" else [])}[case["kind"]]
    parts: Dict[str, list] = {n: [] for n in names}
    w = s["weight"].detach().double().requires_grad_(True) if case["kind"] == "head" else None
    step = max(1, (1 << 27) // case["vocab"])
    for a in range(0, T, step):
        r = slice(a, min(T, a + step))
        if w is None:
            leaf = s["logits"][r].detach().double().requires_grad_(True)
            z = leaf / case["temp"]
        else:
            leaf = s["hidden"][r].detach().double().requires_grad_(True)
            z = (leaf @ w.t()) / case["temp"]
        if case["kind"] == "logprobs" and s["mask_bits"] is not None:
            gone = torch.stack([(s["mask_bits"][r] >> j) & 1 for j in range(8)], -1).flatten(1)[:, : case["vocab"]].bool()
            z = z.masked_fill(gone, -1e6)  # (finite, so that 0 times it is 0; exp(-1e6) is 0)
        ls = torch.log_softmax(z, -1)
        if case["kind"] == "distill":
            t, ids = s["top_logp"][r].double(), s["top_ids"][r]
            inside = torch.zeros_like(z, dtype=torch.bool).scatter_(1, ids, True)
            q = ls.gather(1, ids)
            if s["rest_logp"] is None:
                t = torch.log_softmax(t, -1)
            else:
                q = torch.cat([q, torch.logsumexp(ls.masked_fill(inside, -1e6), -1, keepdim=True)], 1)
                t = torch.cat([t, s["rest_logp"][r].double()[:, None]], 1)
            loss = torch.nn.functional.kl_div(t, q, reduction="none", log_target=True).sum(-1) if case["reverse"] \
                else torch.nn.functional.kl_div(q, t, reduction="none", log_target=True).sum(-1)
            (d,) = torch.autograd.grad(loss, leaf, s["g_loss"][r].double())
            got = dict(loss=loss.detach(), dlogits=d)
        else:
            logp = ls.gather(1, s["labels"][r, None]).squeeze(1)
            entropy = torch.special.entr(ls.exp()).sum(-1) if case.get("mode") != "train" else -(ls.exp() * ls).sum(-1)
            got = dict(logp=logp.detach(), entropy=entropy.detach())
            if case["kind"] == "top":
                k = min(case["top"], case["vocab"])
                top = torch.sort(s["logits"][r].double(), dim=-1, descending=True, stable=True).indices[:, :k]
                rest = torch.logsumexp(ls.scatter(1, top, NEG), -1)
                got.update(top_logp=ls.gather(1, top), top_ids=top, rest_logp=rest)
                got = {n: v.detach() for n, v in got.items()}
            elif case["mode"] == "train":
                total = (logp * s["g_logp"][r].double()).sum() + (entropy * s["g_entropy"][r].double()).sum()
                if w is None:
                    got["dlogits"] = torch.autograd.grad(total, leaf)[0]
                else:
                    got["dhidden"], dw = torch.autograd.grad(total, [leaf, w])
                    parts["dweight"] = [parts["dweight"][0] + dw] if parts["dweight"] else [dw]
        for n, v in got.items():
            parts[n].append(v)
    return {n: parts[n][0] if n == "dweight" else torch.cat(parts[n]) for n in names}
