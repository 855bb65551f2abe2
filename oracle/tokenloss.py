"""Label log-probabilities, preference loss, clipped policy loss, gradient clipping and Adam in 64 bits on the CPU, from
their formulas; gradients by autograd in 64 bits."""
import math

import torch


def token_logprobs(x, labels, class_dim=1, temperature=1.0, ignore_index=255):
    """x fp64; positions with ignore_index give 0, other labels outside the classes NaN."""
    x = x.movedim(class_dim, -1)
    keep = labels != ignore_index
    bad = keep & ((labels < 0) | (labels >= x.shape[-1]))
    at = torch.where(keep & ~bad, labels, 0)
    # ignored positions are not read: whatever stands there must not reach the others through autograd
    x = torch.where(keep.unsqueeze(-1), x, torch.zeros((), dtype=x.dtype))
    logp = torch.log_softmax(x / temperature, -1).gather(-1, at.unsqueeze(-1)).squeeze(-1)
    logp = torch.where(bad, torch.full((), math.nan, dtype=x.dtype), logp)
    return torch.where(keep, logp, torch.zeros((), dtype=x.dtype)), keep


def preference(x, labels, ref, beta=0.1, label_smoothing=0.0, loss_type="sigmoid", average=False, **how):
    logp, keep = token_logprobs(x, labels, **how)
    n = x.shape[0]
    diff = torch.where(keep, logp - torch.where(keep, ref.double(), 0.0), torch.zeros((), dtype=logp.dtype)).reshape(n, -1)
    r = diff.sum(1)
    if average:
        r = r / keep.reshape(n, -1).sum(1).clamp(min=1)
    h = r[: n // 2] - r[n // 2:]
    if loss_type == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - label_smoothing) * ls(beta * h) - label_smoothing * ls(-beta * h)
    else:
        loss = (h - 1 / (2 * beta)) ** 2
    return loss.mean(), beta * r


def policy(x, labels, old, adv, ref=None, clip_low=0.2, clip_high=0.2, kl_weight=0.0, reduction="token", **how):
    logp, keep = token_logprobs(x, labels, **how)
    n = x.shape[0]
    zero = torch.zeros((), dtype=logp.dtype)
    lp, k = logp.reshape(n, -1), keep.reshape(n, -1)
    a = adv.double().reshape(n, -1)
    ratio = torch.exp(torch.where(k, lp - old.double().reshape(n, -1), zero))
    free, held = ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a
    surrogate = torch.where(k, -torch.minimum(free, held), zero)
    far = zero.expand(lp.shape)
    if ref is not None:
        q = torch.where(k, ref.double().reshape(n, -1) - lp, zero)
        far = torch.where(k, torch.exp(q) - q - 1, zero)

    def mean(v):
        if reduction == "token":
            return v.sum() / k.sum().clamp(min=1)
        return (v.sum(1) / k.sum(1).clamp(min=1)).mean()

    clipped = ((free > held) & k).sum().double() / k.sum().clamp(min=1)
    s, f = mean(surrogate), mean(far)
    return (s + kl_weight * f if kl_weight else s), s, f, clipped, logp


def grad_norm(grads, norm_type=2.0):
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    return torch.linalg.vector_norm(flat, norm_type)


def clip_factor(norm, max_norm):
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def adam(p, g, m, v, t, factor=1.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False):
    """One step in 64 bits: (p, m, v)."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * factor
    if decoupled:
        p = p * (1 - lr * weight_decay)
    else:
        g = g + weight_decay * p
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    mh, vh = m / (1 - betas[0] ** t), v / (1 - betas[1] ** t)
    return p - lr * mh / (vh.sqrt() + eps), m, v
