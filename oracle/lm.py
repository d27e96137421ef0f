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


def linear_ce(x, w, t, b=None, r=None, scale=1.0, reduction='mean', ignore=-100):
    """Loss and log-sum-exp of scale (x w^T + b), with ``size`` (the largest sum of magnitudes behind a row's logits),
    ``w`` (the rows' weights, 0 without a target) and ``count``."""
    H = x.shape[-1]
    X, W, T = x.double().reshape(-1, H), w.double(), t.reshape(-1).long()
    logits = X @ W.t()
    size = (X.abs() @ W.abs().t()).amax(1)
    if b is not None:
        logits = logits + b.double()
        size = size + b.double().abs().amax()
    logits = logits * scale
    lse = torch.logsumexp(logits, 1)
    keep = T != ignore
    weight = keep.double() * (r.double().reshape(-1) if r is not None else 1.0)
    nll = torch.where(keep, (lse - logits.gather(1, T.clamp(min=0).unsqueeze(1)).squeeze(1)) * weight, torch.zeros_like(lse))
    count = int(keep.sum())
    loss = nll if reduction == 'none' else nll.sum() if reduction == 'sum' else nll.sum() / max(1, count)
    return dict(loss=loss, lse=lse, size=size * abs(scale), w=weight, count=count, logits=logits, keep=keep)


def linear_ce_grads(x, w, t, b, r, scale, reduction, ignore, slope, lse_slope):
    """Gradients of sum(slope loss) + sum(lse_slope lse), and under |name| the sums of magnitudes that form them."""
    e = linear_ce(x, w, t, b, r, scale, reduction, ignore)
    H = x.shape[-1]
    X, W, T = x.double().reshape(-1, H), w.double(), t.reshape(-1).long()
    c = e['w'] * slope.double().reshape(-1)
    if reduction == 'mean':
        c = c / max(1, e['count'])
    a = c + (lse_slope.double().reshape(-1) if lse_slope is not None else 0.0)
    d = (e['logits'] - e['lse'].unsqueeze(1)).exp() * a.unsqueeze(1)
    mag = d.abs()
    row = torch.arange(len(T), device=T.device)[e['keep']]
    d[row, T[row]] -= c[row]
    mag[row, T[row]] += c[row].abs()
    d, mag = d * scale, mag * abs(scale)
    return {'x': (d @ W).view(x.shape), '|x|': (mag @ W.abs()).view(x.shape), 'w': d.t().contiguous() @ X, '|w|': mag.t().contiguous() @ X.abs(),
            'b': d.sum(0), '|b|': mag.sum(0)}
