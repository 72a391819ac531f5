"""The losses of a language-model head in 64 bits, from their definitions, on the CPU or the GPU (torch float64).

  cross entropy  loss = lse - z[target]
  distillation   p = softmax(teacher / tau) over the entries that count,
                 loss = tau^2 sum_k p_k (log p_k - log softmax(z / tau)[id_k])
Rows in which nothing counts (target or every id outside [0, vocab), or logits of -inf) have loss 0 and no gradient."""
from __future__ import annotations

import torch


def _top(y):
    """[rows, 1]: what is subtracted before exponentials are taken.  (Logits may be masked with a type's lowest value, beside which
    even 64 bits have no room for the sum's logarithm.)"""
    if not y.shape[1]:
        return torch.zeros(y.shape[0], 1, dtype=y.dtype, device=y.device)
    top = y.amax(1, keepdim=True)
    return torch.where(top == -torch.inf, 0.0, top)


def entries(ids, teacher, vocab, tau):
    """(p, log p) [rows, K]: 0 where an entry does not count."""
    ids = ids.long()
    y = teacher.double() / tau
    counts = (ids >= 0) & (ids < vocab)
    y = torch.where(counts, y, -torch.inf)
    counts &= y != -torch.inf
    log_p = torch.where(counts, y - _top(y), 0.0)
    total = torch.where(counts, log_p.exp(), 0.0).sum(1)
    log_p = torch.where(counts, log_p - torch.where(counts.any(1), total, 1.0).log()[:, None], 0.0)
    return torch.where(counts, log_p.exp(), 0.0), log_p, counts


def distillation(z, ids, teacher, tau=1.0, scale=None):
    """z [rows, vocab] float64: loss, lse, gradient of sum(scale * loss)."""
    rows, vocab = z.shape
    p, log_p, counts = entries(ids, teacher, vocab, tau)
    some = counts.any(1)
    u = z / tau
    top = _top(u)
    u = u - top
    rest = u.exp().sum(1).log()
    lse = top[:, 0] + rest
    at = u.gather(1, torch.where(counts, ids.long(), 0)) if ids.shape[1] else u[:, :0]
    loss = tau * tau * torch.where(p > 0, p * (log_p - (at - rest[:, None])), 0.0).sum(1)
    loss = torch.where(some, loss, 0.0)
    want = torch.zeros_like(z)
    want.scatter_add_(1, torch.where(counts, ids.long(), 0), p)
    scale = torch.ones(rows, dtype=z.dtype, device=z.device) if scale is None else scale.double()
    grad = torch.where(some[:, None], (tau * scale)[:, None] * ((u - rest[:, None]).exp() - want), 0.0)
    return loss, lse, grad


def cross_entropy(z, targets, scale=None):
    zero = torch.zeros(z.shape[0], 1, dtype=torch.float64, device=z.device)
    return distillation(z, targets[:, None], zero, 1.0, scale)


def linear(x, w, loss_of):
    """The loss of z = x w by loss_of(z) -> (loss, lse, d z), and its gradients; rows without a gradient add nothing."""
    x, w = x.double(), w.double()
    loss, lse, g = loss_of(x @ w)
    keep = (g != 0).any(1, keepdim=True)
    return loss, lse, g, torch.where(keep, g @ w.t(), 0.0), torch.where(keep, x, 0.0).t() @ g
