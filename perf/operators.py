"""Measured cases of the token log-probability and distillation operators.

    logprobs   log-probabilities of given tokens from logit rows, with the entropy of each row and its
               `top_k` most likely alternatives; with `train`, also the gradient of the logits
    distill    distillation from a teacher's top-K log-probabilities; with `train`, loss and gradient
    head       the same log-probabilities and entropies straight from hidden states and the output
               projection, without the logits; with `train`, also the gradients of both

`run` computes a case in plain torch operations (32 bits, one rounding at the end) or, with `own`
set, through the framework's entry points.  `exact` gives the definition's values in 64 bits.
"""
import math
import os
import sys

import torch

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    def logprobs(name, rows, vocab, dtype, top_k=0, entropy=True, temperature=1.0, softcap=0.0, train=False):
        return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
                "entropy": entropy, "temperature": temperature, "softcap": softcap, "train": train}

    def distill(name, rows, vocab, dtype, top_k, tail, temperature=1.0, softcap=0.0, train=True):
        return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
                "tail": tail, "temperature": temperature, "softcap": softcap, "train": train}

    def head(name, rows, dim, vocab, dtype, entropy=True, temperature=1.0, softcap=0.0, train=False):
        return {"name": name, "op": "head", "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype,
                "entropy": entropy, "temperature": temperature, "softcap": softcap, "train": train}

    return [
        # one decode step of one sequence that reports the sampled token and 20 alternatives
        logprobs("decode 1 row top 20", 1, 50304, "bf16", top_k=20, temperature=0.8),
        # one decode step of a batch with capped fp32 logits of a large vocabulary
        logprobs("decode 64 rows fp32 top 5", 64, 131072, "fp32", top_k=5, softcap=30.0),
        # scoring given text: no alternatives
        logprobs("score 4096 rows fp16", 4096, 32768, "fp16"),
        # a teacher's pass over a training batch: its 64 most likely tokens per position
        logprobs("teacher 8192 rows top 64", 8192, 50304, "bf16", top_k=64, entropy=False, temperature=2.0),
        # a short policy-gradient batch with an odd vocabulary
        logprobs("policy 37 rows fp32 odd", 37, 50257, "fp32", train=True),
        # a policy-gradient step with an entropy bonus
        logprobs("policy 8192 rows", 8192, 50304, "bf16", train=True),
        # a small batch distilled with the rest of the vocabulary as one bucket
        distill("distill 24 rows fp32", 24, 32000, "fp32", 8, tail=True),
        # fp16 with a loss scale, odd sizes, renormalised teacher
        distill("distill 1023 rows fp16 odd", 1023, 50257, "fp16", 33, tail=False, temperature=2.0),
        # a full distillation step
        distill("distill 8192 rows", 8192, 50304, "bf16", 64, tail=True, temperature=2.0),
        # the last positions of a few sequences scored from their hidden states
        head("head 8 rows", 8, 768, 50304, "bf16"),
        # scoring under a wider model, rows that fill no tile
        head("head 2001 rows fp16", 2001, 1536, 32000, "fp16"),
        # a policy-gradient step from the hidden states
        head("head 4096 rows train", 4096, 768, 50304, "bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "distill", "distill", "head"])
    train = rng.random() < 0.5
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
    if op == "head":
        dim = 8 * _log_int(rng, 16, 256)
        vocab = _log_int(rng, 1000, 65536)
        most = 4096 * 768 * 50304 // (dim * vocab)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(8192, most))), "dim": dim, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "entropy": rng.random() < 0.7,
                "temperature": temperature, "softcap": softcap, "train": train}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = _log_int(rng, 1000, 131072)
    rows = _log_int(rng, 1, max(1, 8192 * 50304 // vocab // (2 if dtype == "fp32" else 1)))
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "softcap": softcap,
            "train": train}
    if op == "logprobs":
        case.update(top_k=0 if train else rng.choice([0, 1, _log_int(rng, 2, 128)]), entropy=rng.random() < 0.7)
    else:
        case.update(top_k=_log_int(rng, 1, 128), tail=rng.random() < 0.5)
    return case


def work(case):
    n, v, es = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "head":
        d, gemms = case["dim"], 3 if case["train"] else 1
        moved = (n * d + v * d) * es * (2 if case["train"] else 1) + n * 8 + n * 12 + (n * 8 if case["train"] else 0)
        return {"bytes": moved, "flops": 2.0 * n * d * v * gemms}
    passes = 2 if case["train"] else 1  # the logits once, and their gradient once
    k = case["top_k"]
    if case["op"] == "logprobs":
        small = n * (8 + 8) + (n * 4 if case["entropy"] else 0) + n * k * 12 + (n * 8 if case["train"] else 0)
        return {"bytes": n * v * es * passes + small, "flops": 6.0 * n * v * passes}
    return {"bytes": n * v * es * passes + n * k * 12 + n + 4, "flops": 4.0 * n * v * passes}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    n, v = case["rows"], case["vocab"]

    def randn(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)

    s = {"case": case}
    s["targets"] = torch.randint(0, v, (n,), generator=g, device="cuda")
    if case["op"] != "distill" and n >= 16:  # padding positions
        s["targets"][torch.rand(n, generator=g, device="cuda") < 0.04] = IGNORE
    if case["op"] == "head":
        s["hidden"] = randn(n, case["dim"], dtype=dt)
        s["weight"] = randn(v, case["dim"], std=2.0 / math.sqrt(case["dim"]), dtype=dt)
    else:
        # broad noise with a raised target: the shape of a language model's logits
        x = randn(n, v, std=2.0, dtype=dt)
        at = s["targets"].clamp(min=0)[:, None]
        lift = torch.rand(n, 1, generator=g, device="cuda") * 12
        s["logits"] = x.scatter_(1, at, (x.gather(1, at).float() + lift).to(dt))
    if case["op"] == "distill":
        # the teacher agrees with the student in part; its log-probabilities leave some mass outside
        near = s["logits"].to(torch.float16 if dt == torch.float16 else torch.bfloat16)
        score = near * 0.5 + randn(n, v, dtype=near.dtype)
        top, at = torch.topk(score, case["top_k"], dim=1)
        rest = 0.05 + 0.4 * torch.rand(n, 1, generator=g, device="cuda")
        s["teacher_idx"] = at
        s["teacher_lp"] = torch.log_softmax(top.float() * 1.5, 1) + torch.log1p(-rest)
        s["mask"] = torch.rand(n, generator=g, device="cuda") >= (0.04 if n >= 16 else 0.0)
        # fp16 training scales its loss
        s["upstream"] = torch.full((), 1024.0 if dt == torch.float16 else 1.0, device="cuda")
    elif case["train"]:
        s["g_lp"] = randn(n)
        s["g_ent"] = randn(n, std=0.02)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["op"] == "logprobs":
        return _plain_logprobs(case, state)
    if case["op"] == "distill":
        return _plain_distill(case, state)
    return _plain_head(case, state)


def _own(case, s):
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autokernel-halo-strix_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    if case["op"] == "distill":
        from kernels.distill import distill_topk
        if not case["train"]:
            return {"loss": distill_topk(s["logits"], s["teacher_idx"], s["teacher_lp"], mask=s["mask"],
                                         temperature=case["temperature"], softcap=case["softcap"],
                                         tail=case["tail"])}
        x = s["logits"].detach().requires_grad_(True)
        loss = distill_topk(x, s["teacher_idx"], s["teacher_lp"], mask=s["mask"], temperature=case["temperature"],
                            softcap=case["softcap"], tail=case["tail"])
        grad, = torch.autograd.grad(loss, x, s["upstream"])
        return {"loss": loss.detach(), "grad": grad}
    kw = dict(temperature=case["temperature"], softcap=case["softcap"], ignore_index=IGNORE, entropy=case["entropy"])
    if case["op"] == "logprobs":
        from kernels.token_logprobs import token_logprobs
        leaves = [s["logits"].detach().requires_grad_(True)] if case["train"] else [s["logits"]]
        r = token_logprobs(leaves[0], s["targets"], top_k=case["top_k"], **kw)
    else:
        from kernels.token_logprobs import linear_token_logprobs
        leaves = [s["hidden"], s["weight"]]
        if case["train"]:
            leaves = [t.detach().requires_grad_(True) for t in leaves]
        r = linear_token_logprobs(leaves[0], leaves[1], s["targets"], **kw)
    out = {"logprobs": r.logprobs.detach(), "lse": r.lse}
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
    if case.get("top_k"):
        out.update(top_logprobs=r.top_logprobs, top_indices=r.top_indices)
    if case["train"]:
        outs, gs = ([r.logprobs, r.entropy], [s["g_lp"], s["g_ent"]]) if case["entropy"] else ([r.logprobs], [s["g_lp"]])
        out["grads"] = list(torch.autograd.grad(outs, leaves, gs))
    return out


def _squash(x, case):
    """Softcap and temperature in 32 bits."""
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    return x / case["temperature"] if case["temperature"] != 1.0 else x


def _unsquash(g, x, case):
    """Gradient through _squash at its output x."""
    if case["softcap"]:
        t = x * (case["temperature"] / case["softcap"])
        g = g * (1 - t * t)
    return g / case["temperature"] if case["temperature"] != 1.0 else g


def _stats(x, targets, entropy):
    """(logprobs, lse, entropy or None, row maximum, e = exp(x - max), its sum) of fp32 rows."""
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    valid = targets != IGNORE
    at = targets.clamp(min=0)[:, None]
    lp = torch.where(valid, (d.gather(1, at) - logz)[:, 0], 0.0)
    ent = torch.where(valid, (logz - (e * d).sum(1, keepdim=True) / z)[:, 0], 0.0) if entropy else None
    return lp, (m + logz)[:, 0], ent, m, e, z


def _grad_rows(x, m, e, z, ent, targets, g_lp, g_ent):
    """d(sum g_lp lp + g_ent H)/dx of fp32 rows."""
    valid = targets != IGNORE
    p = e / z
    gl = torch.where(valid, g_lp, 0.0)[:, None]
    grad = p * -gl
    if ent is not None:
        ge = torch.where(valid, g_ent, 0.0)[:, None]
        grad -= ge * p * (x - m - torch.log(z) + ent[:, None])
    return grad.scatter_add_(1, targets.clamp(min=0)[:, None], gl)


def _top(raw, k):
    """Indices of the k largest per row, equal values by lowest index."""
    v = raw.shape[1]
    bits = raw.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = (order << 32) | torch.arange(v - 1, -1, -1, device=raw.device)
    return v - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)


def _plain_logprobs(case, s):
    raw = s["logits"].float()
    x = _squash(raw, case)
    lp, lse, ent, m, e, z = _stats(x, s["targets"], case["entropy"])
    out = {"logprobs": lp, "lse": lse}
    if case["entropy"]:
        out["entropy"] = ent
    if case["top_k"]:
        at = _top(raw, case["top_k"])
        out.update(top_logprobs=x.gather(1, at) - m - torch.log(z), top_indices=at)
    if case["train"]:
        g = _unsquash(_grad_rows(x, m, e, z, ent, s["targets"], s["g_lp"], s["g_ent"]), x, case)
        out["grads"] = [g.to(s["logits"].dtype)]
    return out


def _plain_head(case, s):
    h, w = s["hidden"].float(), s["weight"].float()
    x = _squash(h @ w.t(), case)
    lp, lse, ent, m, e, z = _stats(x, s["targets"], case["entropy"])
    out = {"logprobs": lp, "lse": lse}
    if case["entropy"]:
        out["entropy"] = ent
    if case["train"]:
        g = _unsquash(_grad_rows(x, m, e, z, ent, s["targets"], s["g_lp"], s["g_ent"]), x, case)
        out["grads"] = [(g @ w).to(s["hidden"].dtype), (g.t() @ h).to(s["weight"].dtype)]
    return out


def _plain_distill(case, s):
    x = _squash(s["logits"].float(), case)
    tl, at, mask, t = s["teacher_lp"], s["teacher_idx"], s["mask"], case["temperature"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    lp = x.gather(1, at) - lse
    if case["tail"]:
        # the rest of both distributions, the student's as a sum of its own: 1 - sum would lose it
        q, logq = torch.exp(tl), tl
        r = (1 - torch.exp(tl.double()).sum(1, keepdim=True)).clamp(min=0).float()
        pr = e.scatter(1, at, 0.0).sum(1, keepdim=True) / z
        loss = (q * (logq - lp)).sum(1) + (r * (torch.log(r) - torch.log(pr)))[:, 0]
        rest = 1 - r / pr
    else:
        tm = tl.amax(1, keepdim=True)
        logq = tl - tm - torch.log(torch.exp(tl - tm).sum(1, keepdim=True))
        q = torch.exp(logq)
        loss = (q * (logq - lp)).sum(1)
        rest = None
    n = mask.sum().clamp(min=1)
    out = {"loss": torch.where(mask, loss, 0.0).sum() * (t * t) / n}
    if case["train"]:
        p = e / z
        g = p if rest is None else p * rest
        g = g.scatter(1, at, torch.exp(lp) - q) * (t * t / n * s["upstream"])
        g = torch.where(mask[:, None], g, 0.0)
        out["grad"] = _unsquash(g, x, case).to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    n, v = case["rows"], case["vocab"]
    step = max(1, (1 << 26) // v)
    parts = []
    valid_rows = float(max(1, int(s["mask"].sum()))) if case["op"] == "distill" else None
    dw = torch.zeros(v, case["dim"], dtype=torch.float64, device="cuda") if case["op"] == "head" else None
    for a in range(0, n, step):
        r = slice(a, min(n, a + step))
        if case["op"] == "head":
            raw = s["hidden"][r].double() @ s["weight"].double().T
        else:
            raw = s["logits"][r].double()
        y, dy = raw, torch.ones((), dtype=torch.float64, device="cuda")
        if case["softcap"]:
            th = torch.tanh(raw / case["softcap"])
            y, dy = case["softcap"] * th, 1 - th.square()
        y, dy = y / case["temperature"], dy / case["temperature"]
        logp = torch.log_softmax(y, 1)
        prob = logp.exp()
        if case["op"] == "distill":
            parts.append(_exact_distill(case, s, r, logp, prob, dy, valid_rows))
            continue
        tgt = s["targets"][r]
        live = (tgt != IGNORE).double()
        hot = torch.zeros_like(prob).scatter_(1, tgt.clamp(min=0)[:, None], live[:, None])
        part = {"logprobs": (hot * logp).sum(1), "lse": torch.logsumexp(y, 1)}
        ent = -(prob * logp).sum(1)
        if case["entropy"]:
            part["entropy"] = ent * live
        if case.get("top_k"):
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
            part.update(top_logprobs=logp.gather(1, order), top_indices=order)
        if case["train"]:
            gl = (s["g_lp"][r].double() * live)[:, None]
            ge = (s["g_ent"][r].double() * live)[:, None] * (1.0 if case["entropy"] else 0.0)
            g = (gl * (hot - prob) - ge * prob * (logp + ent[:, None])) * dy
            if case["op"] == "head":
                part["g0"] = g @ s["weight"].double()
                dw += g.T @ s["hidden"][r].double()
            else:
                part["g0"] = g
        parts.append(part)
    if case["op"] == "distill":
        out = {"loss": torch.stack([p["loss"] for p in parts]).sum()}
        if case["train"]:
            out["grad"] = torch.cat([p["grad"] for p in parts])
        return out
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0] if k != "g0"}
    if case["train"]:
        out["grads"] = [torch.cat([p["g0"] for p in parts])] + ([dw] if case["op"] == "head" else [])
    return out


def _exact_distill(case, s, r, logp, prob, dy, valid_rows):
    t2 = case["temperature"] ** 2
    tl, at, live = s["teacher_lp"][r].double(), s["teacher_idx"][r], s["mask"][r].double()
    q = tl.exp() if case["tail"] else torch.softmax(tl, 1)
    per = (q * (q.log() - logp.gather(1, at))).sum(1)
    ref = torch.zeros_like(prob).scatter_(1, at, q)
    if case["tail"]:
        outside = torch.ones_like(prob).scatter_(1, at, 0.0)
        r_t = 1 - q.sum(1)
        r_s = (prob * outside).sum(1)
        per = per + r_t * (r_t.log() - r_s.log())
        ref = ref + outside * prob * (r_t / r_s)[:, None]
    part = {"loss": (per * live).sum() * t2 / valid_rows}
    if case["train"]:
        part["grad"] = (prob - ref) * dy * (live * (t2 / valid_rows) * s["upstream"].double())[:, None]
    return part
