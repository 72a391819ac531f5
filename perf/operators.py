"""The losses of a language-model head: what they compute, in elementary torch operations, and the calls of the framework.

  linear_cross_entropy   softmax cross entropy of x w against token ids, from the hidden states x [tokens, hidden] and the head's
                         weights w [hidden, vocab]: loss, logsumexp and the gradients of x and w
  distillation           KL divergence of softmax(logits / temperature) from a teacher's top entries, times temperature squared:
                         loss, logsumexp and the gradient of the logits
  linear_distillation    the same loss of the logits x w, with the gradients of x and w

The widths are the LM's own (hidden 2048, vocabulary 32768) and generic ones around them.  Hidden states are N(0, 1) as behind the
final norm and lean towards their target's weights, head weights are N(0, 0.02); a teacher's entries fall off from its best one,
some rows hold fewer of them and some none, as where a batch is padded.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32


def listed():
    return [
        # One short sequence at the LM's width: reading the head's weights and writing their gradient is the whole cost.
        _case("lce_64", "lce", 64, 2048, 32768),
        # The LM's training batch: 8 sequences of 2048 tokens.
        _case("lce_16384", "lce", 16384, 2048, 32768),
        # A head that shares its weights with the embedding table, with an odd vocabulary and a ragged batch's padding.
        _case("lce_tied_odd", "lce", 1999, 1096, 50001, tied=True, ignored=0.2),
        # Evaluation: the loss alone.
        _case("lce_eval", "lce", 8192, 2048, 32768, grad=False),
        # A small model's head kept in f32, its sizes off every grid.
        _case("lce_f32", "lce", 700, 515, 8190, dtype="f32"),
        # A few rows of logits against a teacher's 16 best.
        _case("kd_64", "kd", 64, 0, 32768, k=16, tau=2.0),
        # A training batch of logits against a teacher's 64 best.
        _case("kd_8192", "kd", 8192, 0, 32768, k=64, tau=2.0),
        # f32 logits of a vocabulary off every grid, a hundred teacher entries a row.
        _case("kd_f32_odd", "kd", 1500, 0, 50001, k=100, tau=1.0, dtype="f32"),
        # A long vocabulary, rows of which exceed what one SM holds.
        _case("kd_wide", "kd", 1024, 0, 150000, k=20, tau=1.5),
        # Distillation from the hidden states, a short batch.
        _case("lkd_128", "lkd", 128, 2048, 32768, k=32, tau=1.0),
        # Distillation from the hidden states, a training batch.
        _case("lkd_8192", "lkd", 8192, 2048, 32768, k=64, tau=2.0),
        # Tied weights, odd sizes, few entries.
        _case("lkd_tied_odd", "lkd", 3001, 776, 20011, k=7, tau=1.3, tied=True, ignored=0.1),
    ]


def _case(name, op, tokens, hidden, vocab, k=0, tau=1.0, dtype="bf16", tied=False, ignored=0.01, grad=True):
    c = {"op": op, "tokens": tokens, "hidden": hidden, "vocab": vocab, "k": k, "tau": tau, "dtype": dtype, "tied": tied,
         "ignored": ignored, "grad": grad}
    return {"name": name, **c} if name else c


def draw(rng: random.Random):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("lce", "lce", "kd", "lkd", "lkd"))
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    vocab = log_uniform(500, 150000)
    if rng.random() < 0.5:
        vocab = vocab // 64 * 64 + 64
    hidden = 0
    if op != "kd":
        hidden = log_uniform(64, 4096)
        if rng.random() < 0.6:
            hidden = hidden // 64 * 64 + 64
    most = 16384
    if op == "kd":
        most = min(8192, (1 << 28) // vocab // (2 if dtype == "f32" else 1))
    else:  # no more work than the largest listed case, and no more than a few hundred milliseconds in f32
        most = min(most, (1 << (40 if dtype == "bf16" else 35)) // (vocab * hidden), (1 << 29) // vocab)
    tokens = log_uniform(1, max(2, most))
    k = 0 if op == "lce" else log_uniform(1, 256)
    tau = 1.0 if op == "lce" else round(rng.uniform(0.7, 4.0), 2)
    return _case(None, op, tokens, hidden, vocab, k=k, tau=tau, dtype=dtype, tied=rng.random() < 0.4,
                 ignored=rng.choice((0.0, 0.05, 0.3)), grad=rng.random() < 0.85)


# ------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, d, v, k = case["tokens"], case["hidden"], case["vocab"], case["k"]
    dt = BF16 if case["dtype"] == "bf16" else F32
    on = dict(generator=gen, device="cuda")
    out = {"case": case, "d_loss": 0.5 + torch.rand(t, **on), "grad_scale": 1.0 / t}
    best = torch.randint(0, v, (t,), **on)  # the token that a row leans towards
    skip = torch.rand(t, **on) < case["ignored"]
    if case["op"] == "kd":
        logits = torch.randn(t, v, **on)
        logits.scatter_add_(1, best[:, None], 6.0 * torch.rand(t, 1, **on))
        out["logits"] = logits.mul_(1.5).to(dt)
    else:
        w = (torch.randn(v, d, **on) * 0.02).to(dt)
        x = torch.randn(t, d, **on)
        lean = w[best].float()
        x += 8.0 * torch.rand(t, 1, **on) * lean / lean.norm(dim=1, keepdim=True)
        out["x"] = x.to(dt)
        out["w"] = w.t() if case["tied"] else w.t().contiguous()
    if case["op"] == "lce":
        targets = torch.where(torch.rand(t, **on) < 0.7, best, torch.randint(0, v, (t,), **on))
        out["targets"] = torch.where(skip, -1, targets).to(torch.int32)
    else:
        step = 1 + torch.randint(0, max(1, (v - 1) // max(1, k)), (t, 1), **on)
        ids = (best[:, None] + step * torch.arange(k, device="cuda")) % v
        falls = torch.rand(t, k, **on).mul_(0.8).cumsum(1)
        short = torch.randint(1, k + 1, (t, 1), **on)  # rows with fewer entries
        cut = (torch.rand(t, 1, **on) < 0.1) & (torch.arange(k, device="cuda") >= short)
        out["ids"] = torch.where(cut | skip[:, None], -1, ids).to(torch.int32)
        out["teacher"] = (12.0 - falls * 2.0).to(dt)
    return out


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import cleanlm_b200 as cdl

        s["ops"] = cdl.ops
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    ops, case = s["ops"], s["case"]
    if case["op"] == "kd":
        o = ops.distillation(s["logits"], s["ids"], s["teacher"], ops.DistillationOpts(
            temperature=case["tau"], grad_scale=s["grad_scale"], d_loss=s["d_loss"], grad=case["grad"]))
        return {"loss": o.loss, "lse": o.lse, "d_logits": o.d_logits}
    opts = ops.LinearLossOpts(temperature=case["tau"], grad_scale=s["grad_scale"], d_loss=s["d_loss"], grad=case["grad"])
    if case["op"] == "lce":
        o = ops.linear_cross_entropy(s["x"], s["w"], s["targets"], opts)
    else:
        o = ops.linear_distillation(s["x"], s["w"], s["ids"], s["teacher"], opts)
    return {"loss": o.loss, "lse": o.lse, "dx": o.dx, "dw": o.dw}


def _softmax(z):
    """The exponentials of z over their sum, in place, and the logarithm of the sum of the exponentials."""
    m = z.amax(1, keepdim=True)
    e = z.sub_(m).exp_()
    s = e.sum(1, keepdim=True)
    return e.div_(s), (m + s.log())[:, 0]


def _teacher(s, v):
    """The teacher's probabilities (0 at entries that do not count) and ids that may be used as indices."""
    ids, tau = s["ids"].long(), s["case"]["tau"]
    counts = (ids >= 0) & (ids < v)
    y = torch.where(counts, s["teacher"].float() / tau, -torch.inf)
    any_ = counts.any(1)
    y = y - torch.where(any_, y.amax(1), 0.0)[:, None]
    e = y.exp()
    total = e.sum(1, keepdim=True)
    p = torch.where(any_[:, None], e / total, 0.0)
    log_p = torch.where(counts & any_[:, None], y - total.log(), 0.0)
    return p, log_p, torch.where(counts, ids, 0), any_


def _plain(s):
    case = s["case"]
    tau, dt = case["tau"], (BF16 if case["dtype"] == "bf16" else F32)
    linear = case["op"] != "kd"
    if linear:
        x, w = s["x"].float(), s["w"].float()
        z = x @ w
    else:
        z = s["logits"].float()
    v = z.shape[1]
    if case["op"] == "lce":
        targets = s["targets"].long()
        counts = (targets >= 0) & (targets < v)
        ids = torch.where(counts, targets, 0)[:, None]
        at = z.gather(1, ids)
        q, lse = _softmax(z)
        loss = torch.where(counts, lse - at[:, 0], 0.0)
        p = counts.float()[:, None]
    else:
        p, log_p, ids, counts = _teacher(s, v)
        z = z / tau if tau != 1.0 else (z if linear else z.clone())
        at = z.gather(1, ids)
        q, lse = _softmax(z)
        loss = tau * tau * torch.where(p > 0, p * (log_p - at + lse[:, None]), 0.0).sum(1)
    out = {"loss": loss, "lse": lse, "dx": None, "dw": None} if linear else {"loss": loss, "lse": lse, "d_logits": None}
    if case["grad"]:
        scale = torch.where(counts, s["d_loss"] * (s["grad_scale"] * tau), 0.0)
        g = q.scatter_add_(1, ids, -p).mul_(scale[:, None])
        if linear:
            out["dx"], out["dw"] = (g @ w.t()).to(dt), (x.t() @ g).to(dt)
        else:
            out["d_logits"] = g.to(dt)
    return out


# ------------------------------------------------------------------------------------------ what it takes
def work(case):
    t, d, v, k = case["tokens"], case["hidden"], case["vocab"], case["k"]
    size = 2 if case["dtype"] == "bf16" else 4
    both = 2 if case["grad"] else 1
    rows = 12 * t + (4 * t if case["op"] == "lce" else (4 + size) * t * k)  # d_loss, loss, lse; targets or the teacher's entries
    if case["op"] == "kd":
        return {"bytes": float(both * size * t * v + rows), "flops": float((3 + 3 * both) * t * v)}
    return {"bytes": float(both * size * (t * d + d * v) + rows), "flops": (6.0 if case["grad"] else 2.0) * t * d * v}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    t, v, k, tau = case["tokens"], case["vocab"], case["k"], case["tau"]
    f64 = dict(dtype=torch.float64, device="cuda")
    linear = case["op"] != "kd"
    loss, lse = torch.zeros(t, **f64), torch.zeros(t, **f64)
    if linear:
        x, w = s["x"].double(), s["w"].double()
        dx, dw = torch.zeros(t, case["hidden"], **f64), torch.zeros(case["hidden"], v, **f64)
    else:
        d_logits = torch.zeros(t, v, **f64)
    block = max(1, min(t, (1 << 27) // v))
    for r0 in range(0, t, block):
        r = slice(r0, min(t, r0 + block))
        z = (x[r] @ w if linear else s["logits"][r].double()) / tau
        lse[r] = torch.logsumexp(z, 1)
        log_q = z - lse[r][:, None]
        want = torch.zeros_like(z)  # the distribution that the softmax is held against
        if case["op"] == "lce":
            tgt = s["targets"][r].long()
            rows = torch.nonzero(tgt >= 0)[:, 0]
            want[rows, tgt[rows]] = 1.0
            loss[r] = -(want * log_q).sum(1)
        else:
            ids, y = s["ids"][r].long(), s["teacher"][r].double() / tau
            rows, at = torch.nonzero(ids >= 0, as_tuple=True)
            log_p = torch.full_like(y, -torch.inf)
            log_p[rows, at] = y[rows, at]
            log_p = log_p - torch.logsumexp(log_p, 1, keepdim=True)
            lp = log_p[rows, at]
            p = lp.exp()
            want.index_put_((rows, ids[rows, at]), p, accumulate=True)
            loss[r] = loss[r].index_add(0, rows, tau ** 2 * p * (lp - log_q[rows, ids[rows, at]]))
        if case["grad"]:
            # rows without a target have no gradient
            g = log_q.exp_().mul_((want.sum(1, keepdim=True) > 0)).sub_(want)
            g.mul_((s["d_loss"][r].double() * s["grad_scale"] * tau)[:, None])
            if linear:
                dx[r] = g @ w.t()
                dw.addmm_(x[r].t(), g)
            else:
                d_logits[r] = g
    if linear:
        return {"loss": loss, "lse": lse, "dx": dx if case["grad"] else None, "dw": dw if case["grad"] else None}
    return {"loss": loss, "lse": lse, "d_logits": d_logits if case["grad"] else None}
