"""Plain forms of the training operators of include/pmg_lm.h on CPU tensors, in fp64 unless said otherwise."""
from __future__ import annotations

import torch

BLOCK = 256


def embedding(weight, ids, scale):
    return weight.double()[ids] * scale


def embedding_grad(grad, ids, V, scale, padding_idx=-1):
    """(gradient of the table, sum of magnitudes, number of positions per token)."""
    E = grad.shape[-1]
    g, flat = grad.double().reshape(-1, E), ids.reshape(-1).long()
    if padding_idx >= 0:
        keep = flat != padding_idx
        g, flat = g[keep], flat[keep]
    out = torch.zeros(V, E, dtype=torch.float64)
    size = torch.zeros(V, E, dtype=torch.float64)
    out.index_add_(0, flat, g)
    size.index_add_(0, flat, g.abs())
    return out * scale, size * abs(scale), torch.bincount(flat, minlength=V)


def clip_factor(norm, max_norm):
    return min(1.0, max_norm / (float(norm) + 1e-6))


def sqrt(x):
    """Correctly rounded: fp64's root carries the 2 x 24 + 2 bits that make its rounding to fp32 the root's own
    (torch.sqrt of fp32 CPU tensors is off by one step for a fifth of the values)."""
    return torch.sqrt(x.double()).to(x.dtype)


def state_values(code, top):
    """fp32, every product rounded by itself: what codes of an 8-bit state stand for."""
    n = code.numel()
    c = torch.nn.functional.pad(code.reshape(-1).float(), (0, -n % BLOCK)).view(-1, BLOCK)
    if code.dtype == torch.int8:
        c = c * torch.tensor(1.0 / 127.0)
        x = (c * c.abs()) * top.unsqueeze(1)
    else:
        c = c * torch.tensor(1.0 / 255.0)
        c = c * c
        x = (c * c) * top.unsqueeze(1)
    return x.reshape(-1)[:n].view(code.shape)


def state_codes(x, signed):
    """fp32: (codes, scales) of the values of a state."""
    n = x.numel()
    f = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    top = f.abs().amax(1)
    share = torch.where(top >= torch.finfo(torch.float32).tiny, torch.ones_like(top) / top, torch.zeros_like(top))
    part = f.abs() * share.unsqueeze(1)
    if signed:
        q = torch.round(sqrt(part) * 127.0)
        q = torch.where(q.isnan(), torch.zeros_like(q), q) * torch.where(f < 0, -1.0, 1.0)
        code = q.to(torch.int8)
    else:
        q = torch.round(sqrt(sqrt(part)) * 255.0)
        q = torch.where(q.isnan(), torch.zeros_like(q), q)
        q = torch.where(f > 0, q.clamp(min=1.0), q)
        code = q.to(torch.uint8)
    return code.reshape(-1)[:n].view(x.shape), top


def adamw(p, g, m, v, t, lr, beta1, beta2, eps, wd, decoupled, factor=1.0):
    """One update in the type of ``p`` (fp64: the exact one; fp32: rounded operation by operation, the factors in t
    and lr formed in fp64).  Returns (p, m, v)."""
    as_ = lambda x: torch.tensor(x, dtype=torch.float64).to(p.dtype)      # noqa: E731
    rate, root = as_(lr / (1 - beta1 ** t)), as_(1 / (1 - beta2 ** t) ** 0.5)
    g = g * as_(factor)
    if not decoupled:
        g = g + as_(wd) * p
    m = m * as_(beta1) + g * as_(1 - beta1)
    v = v * as_(beta2) + (g * g) * as_(1 - beta2)
    move = (m * rate) / (sqrt(v) * root + as_(eps))
    return p * as_(1 - lr * wd if decoupled else 1.0) - move, m, v
