"""The norm, the projection with its cross entropy and the balance loss in 64 bits (torch, on whatever device the
operands are on), written from their formulas, with bounds derived from the kernels' roundings.

u = 2^-24 is half a step of float32; half(t) half a step of type t, relative to the value. A float32 sum of n terms
whose partial sums stay below S errs by at most n u S; a tensor-core step adds 16 products to the sum and may truncate,
which is counted as 4 u S a step.
"""
import math

import torch

U = 2.0 ** -24
BLOCK = 128


def half(dtype):
    return torch.finfo(dtype).eps / 2


def d(t):
    return None if t is None else t.double()


# ------------------------------------------------------------------------------------- norm


def norm(x, residual, weight, eps):
    """(y, rstd, bound of y before its rounding) of the rows of x + residual, in 64 bits, the sum rounded to its type."""
    s = d(x) if residual is None else (d(x) + d(residual)).to(x.dtype).double()
    n = s.shape[-1]
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    y = s * rstd * d(weight)
    # squares and their sum (n / 32 terms a lane at least, and the lanes' joins), half of it in the root, the division,
    # the root, the reciprocal and two products
    return y, rstd, y.abs() * ((n / 32 + 8) / 2 + 8) * U


def scales(y, quant):
    n = y.shape[-1]
    width = n if quant == "row" else BLOCK
    amax = torch.stack([p.abs().amax(-1) for p in y.split(width, -1)], -1)
    s = torch.where(amax == 0, 1.0, amax / 448)
    return s, s.repeat_interleave(width, -1)[..., :n]


def norm_grad(up, s, weight, eps, passed):
    """grad_x, grad_weight and their bounds before rounding."""
    up, s, w = d(up), d(s), d(weight)
    n, rows = s.shape[-1], math.prod(s.shape[:-1])
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    h, g = s * rstd, up * w
    gx = rstd * (g - h * (g * h).mean(-1, keepdim=True))
    c = ((n / 32 + 8) * 1.5 + 16) * U
    bx = c * rstd * (g.abs() + h.abs() * (g * h).abs().mean(-1, keepdim=True))
    if passed is not None:
        gx = gx + d(passed)
        bx = bx + U * gx.abs()
    lead = tuple(range(s.dim() - 1))
    gw, aw = (up * h).sum(lead), (up * h).abs().sum(lead)
    return gx, bx, gw, aw * (rows + (n / 32 + 8) / 2 + 16) * U


# ------------------------------------------------------------------------------------- head


def head(hidden, weight, targets, weights, z_coef=0.0, temperature=1.0, grad=True, alike=1):
    """A dict of name: (value, bound). Rows whose weight is 0 may hold anything. alike: how many rows are the same hidden
    state; their logits' gradients round alike, so in grad_weight their errors add up as such, not as independent ones."""
    dim, vocab = hidden.shape[-1], weight.shape[0]
    rows = targets.numel()
    h, w, t = d(hidden).reshape(rows, dim), d(weight), targets.reshape(rows)
    share = torch.full((rows,), 1.0 / rows, dtype=torch.float64, device=h.device) if weights is None else \
        weights.double().expand(targets.shape).reshape(rows)
    on = share != 0
    h = torch.where(on[:, None], h, 0.0)
    t = torch.where(on, t, 0)
    z = h @ w.T / temperature
    lse = torch.logsumexp(z, 1)
    logp = z.gather(1, t[:, None])[:, 0] - lse
    loss = torch.where(on, -logp + z_coef * lse ** 2, 0.0)
    steps = (dim / 16 + 1) * 4 if hidden.dtype == torch.bfloat16 else dim + 1
    reach = h.norm(dim=1) * w.norm(dim=1).max() / temperature  # of every partial sum, by Cauchy and Schwarz
    dz = steps * U * reach
    # exponentials (2^-22), their sums (a tile's 256 terms, then the tiles), each result's rounding
    dlse = dz + 300 * U
    up = (1 + 2 * z_coef * lse.abs())
    out = {"loss": ((share * loss).sum(), (share.abs() * (2 * dlse * up)).sum() + U * (share * loss).sum().abs()),
           "row_loss": (loss, torch.where(on, 2 * dlse * up + 2 * U * loss.abs(), 0.0)),
           "lse": (torch.where(on, lse, 0.0), torch.where(on, dlse + 2 * U * lse.abs(), 0.0))}
    if grad:
        hot = torch.zeros_like(z).scatter_(1, t[:, None], 1.0)
        p = torch.exp(z - lse[:, None])
        g = (p * (1 + 2 * z_coef * lse)[:, None] - hot) * torch.where(on, share, 0.0)[:, None] / temperature
        half_g = half(hidden.dtype) if hidden.dtype == torch.bfloat16 else 0.0
        # of p (twice the logits' error, the held exponentials' 2^-12) and of the products' sums
        rel = 2 * dz + (2.0 ** -11 if half_g else 40 * U)
        sums = (vocab / 16 + 1) * 4 * U if half_g else (vocab + 1) * U
        # the logits' gradients' rounding: independent from term to term, so six standard deviations (half / sqrt 3)
        spread = 6 * half_g / math.sqrt(3)
        mag = torch.where(hot != 0, (p + 1) * share[:, None].abs() * up[:, None] / temperature, g.abs())
        # what is too small to be held: float32's smallest normal number; in 16 bits 2^-39 of a tile's largest exponential
        least = (2.0 ** -39 if half_g else 2.0 ** -125) * torch.where(on, share, 0.0).abs()[:, None] / temperature
        gh = g @ w
        bh = half(hidden.dtype) * gh.abs() + spread * torch.sqrt((g * g) @ (w * w)) + (rel[:, None] + sums) * (mag @ w.abs()) + \
            least * w.abs().sum(0)
        gw = g.T @ h
        sums = (rows / 16 + 1) * 4 * U if half_g else (rows + 1) * U
        bw = half(hidden.dtype) * gw.abs() + math.sqrt(alike) * spread * torch.sqrt((g * g).T @ (h * h)) + \
            ((rel[:, None] * mag).T @ h.abs() + sums * (mag.T @ h.abs()) + (least * h.abs()).sum(0))
        # what is too small for the results' own type: half of bfloat16's least number (float32's is smaller)
        out["grad_hidden"] = (gh.view(hidden.shape), bh.view(hidden.shape) + 2.0 ** -134)
        out["grad_weight"] = (gw, bw + 2.0 ** -134)
        # the norm of both if every logit's gradient were its row's weight at the target
        out["unit_grad_hidden"] = float(((hot @ w) * torch.where(on, share, 0.0)[:, None]).norm()) / temperature
        out["unit_grad_weight"] = float((h * torch.where(on, share, 0.0)[:, None]).norm()) / temperature
    out["alike"] = alike
    for k in ("row_loss", "lse"):
        out[k] = tuple(v.view(targets.shape) for v in out[k])
    return out


# ------------------------------------------------------------------------------------- balance


def balance(logits, experts, mask, groups, coef, z_coef):
    e, k = logits.shape[-1], experts.shape[-1]
    x, c = d(logits).reshape(-1, e), experts.reshape(-1, k).long()
    rows = x.shape[0]
    on = torch.ones(rows, dtype=torch.bool, device=x.device) if mask is None else (mask != 0).expand(logits.shape[:-1]).reshape(rows)
    x = torch.where(on[:, None], x, 0.0)
    p, lse = torch.softmax(x, 1), torch.logsumexp(x, 1)
    length = rows // groups
    where = torch.arange(rows, device=x.device) // max(length, 1)
    n = torch.zeros(groups, dtype=torch.float64, device=x.device).index_add_(0, where, on.double()).clamp_min(1)
    counts = torch.zeros(groups * e, dtype=torch.int64, device=x.device)
    ids = (where[:, None] * e + c)[on].reshape(-1)
    counts.index_add_(0, ids, torch.ones_like(ids))
    counts = counts.view(groups, e)
    probs = torch.zeros(groups, e, dtype=torch.float64, device=x.device).index_add_(0, where, p * on[:, None]) / n[:, None]
    slope = coef * e * counts / (n * k)[:, None]
    z2 = torch.zeros(groups, dtype=torch.float64, device=x.device).index_add_(0, where, lse ** 2 * on) / n
    loss = ((slope * probs).sum(1) + z_coef * z2).mean()
    a = slope[where]
    factor = (on / (n * groups)[where])[:, None]
    grad = p * (a - (a * p).sum(1, keepdim=True) + 2 * z_coef * lse[:, None]) * factor
    size = p * (a.abs() + (a.abs() * p).sum(1, keepdim=True) + 2 * abs(z_coef) * (1 + lse[:, None].abs())) * factor
    # a row's exponentials (2^-22 at most, and their argument's rounding where x is far below the maximum), its sum of
    # e / 32 + 5 additions, the division; then a lane's sum over its rows
    far = (x.amax(1, keepdim=True) - x).clamp(max=100)
    rel = (e / 32 + 24 + 2 * far) * U
    bp = torch.zeros(groups, e, dtype=torch.float64, device=x.device).index_add_(0, where, p * rel * on[:, None]) / n[:, None]
    bp = bp + probs * (length / 8 + 10) * U
    bound = half(logits.dtype) * grad.abs() + size * (rel + rel.mean(1, keepdim=True)) * 2 + 1e-40
    bl = ((slope.abs() * bp).sum(1) + abs(z_coef) * z2 * (e / 32 + 24) * U * 4).mean() + 4 * U * loss.abs()
    return {"loss": (loss, bl), "counts": (counts, 0), "probs": (probs, bp), "grad": (grad.view(logits.shape), bound.view(logits.shape))}
