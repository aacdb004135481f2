"""The losses over logits rows by their definitions, in float64 numpy, each with a bound on how far a
float32 evaluation may be off.

The bounds count the roundings of the kernels' own arithmetic (ctorch_b200/csrc/losses.cuh), u = 2^-24:
  * t = (x - m) * c2: the difference, c2 and the product are rounded once each, so exp(t) is off by
    3 u d relative, d = |x - m| / T;
  * the hardware's 2^t: 2^-22 relative (4 u), flushed to 0 below 2^-126;
  * s = sum of exp: each term's own error, and one u an addition along the longest chain of additions,
    at most V / 32 + 64 of them (a lane of a warp that has the row alone, then the joining tree), with
    one more exponential and product (6 u) at each of at most 32 rescalings of a running sum;
  * a result of p bits is rounded once more: half of torch.finfo(dtype).eps.
For float64 logits the same counts hold with u = 2^-53 and an exp good to 2 ulp. There the oracle's own
roundings, of the same counts, are as large as the kernel's, so every count is taken twice; and the
row's float64 arithmetic, which float32 results never see, counts: log p is a difference of numbers of
the size of d and log s (u each), a teacher's probability q = exp(z - lse) carries u (|z| + |lse|).
"""
import numpy as np

EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f64": 2.0 ** -53}  # half steps


class Row:
    """Statistics of rows [n, V] at temperature T, and the relative error bounds of p and of s."""

    def __init__(self, x, temperature, kind):
        u = EPS["f64"] if kind == "f64" else EPS["f32"]
        self.u = u
        x = x.astype(np.float64)
        v = x.shape[-1]
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            m = x.max(-1, keepdims=True)
            d = (x - m) / temperature
            d = np.where(x == m, np.where(np.isinf(m), np.nan, 0.0), d)  # +-inf alone has no softmax
            e = np.exp(d)
            s = e.sum(-1, keepdims=True)
            self.p = e / s
            self.lse = (m / temperature + np.log(s))[..., 0]
            self.lse = np.where(np.isneginf(m[..., 0]), -np.inf, self.lse)
            self.logp = d - np.log(s)
            far = np.where(np.isfinite(d), -d, 0.0)
            self.e_rel = 3 * u * far + 4 * u
            self.s_rel = ((self.p * self.e_rel).sum(-1) + (v / 32 + 64 + 6 * 32) * u)
        self.s_rel = np.where(np.isfinite(self.s_rel), self.s_rel, 0.0)
        self.p_rel = self.e_rel + self.s_rel[..., None] + 2 * u


def pick(a, t):
    return np.take_along_axis(a, t[..., None], -1)[..., 0]


def token(x, t, mask, temperature, kind):
    """(logp, its bound, lse, its bound); rows [n]."""
    r = Row(x, temperature, kind)
    bad = mask & ((t < 0) | (t >= x.shape[-1]))
    tt = np.where(mask & ~bad, t, 0)
    logp = np.where(bad, np.nan, pick(r.logp, tt))
    logp = np.where(mask, logp, 0.0)
    lse = np.where(mask, r.lse, 0.0)
    out = EPS["f64"] if kind == "f64" else EPS["f32"]
    with np.errstate(invalid="ignore"):
        # one u for the float64 row arithmetic's own inputs, which the element type holds exactly
        wide = 4 * EPS["f64"]
        logp_tol = r.s_rel + (out + wide) * np.abs(logp) + r.u
        lse_tol = r.s_rel + (out + wide) * (np.abs(lse) + 8) + r.u
    return logp, logp_tol, lse, lse_tol


def pull(x, t, g, g_tol, temperature, kind, extra=0.0):
    """The gradient of sum(g * logp) and its bound, for rows with g, which itself may be off by g_tol.
    extra: a relative error of every p on top (what the backward pass is given)."""
    r = Row(x, temperature, kind)
    n, v = x.shape
    ok = (t >= 0) & (t < v)
    tt = np.where(ok, t, 0)
    one = np.zeros((n, v))
    one[np.arange(n), tt] = 1.0
    on = g != 0
    with np.errstate(invalid="ignore"):
        c = (g / temperature)[:, None]
        grad = c * (one - r.p)
        # 1 - p at the target is computed as one number, from the log-probability
        slack = np.abs(c) * r.p * (r.p_rel + 4 * r.u + np.broadcast_to(extra, (n,))[:, None])
        slack += 4 * EPS["f64"] * np.abs(c)  # c and 1 - p in float64, on either side
        slack += (np.broadcast_to(g_tol, (n,)) / temperature)[:, None] * np.abs(one - r.p)
        grad = np.where(on[:, None], grad, 0.0)
        grad[on & ~ok] = np.nan
        tol = slack + EPS[kind] * (np.abs(grad) + slack) + 1e-37 * np.abs(c)
    return grad, np.where(on[:, None], tol, 0.0)


def policy(x, t, old, adv, ref, w, lo, hi, kl_coef, temperature, kind):
    on = w != 0
    logp, lt, _, _ = token(x, t, on, temperature, kind)
    out = EPS["f64"] if kind == "f64" else EPS["f32"]
    lt = lt - out * np.abs(logp)  # not rounded on the way into the loss
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.exp(logp - old)
        u, c = r * adv, np.clip(r, 1 - lo, 1 + hi) * adv
        free = ~(u > c)
        loss, slope = np.where(free, -u, -c), np.where(free, -u, 0.0)
        d = ref - logp if ref is not None else np.zeros_like(logp)
        kl = np.expm1(d) - d
        loss, slope = loss + kl_coef * kl, slope - kl_coef * np.expm1(d)
        slope_tol = (np.abs(u) + kl_coef * np.exp(d)) * 1.01 * lt
        loss_tol = (np.abs(u) + kl_coef * (1 + np.exp(d))) * 1.01 * lt + 4 * out * np.abs(loss)
        kl_tol = (1 + np.exp(d)) * 1.01 * lt + 4 * out * np.abs(kl)
    z = lambda a: np.where(on, a, 0.0)
    g = z(w * slope)
    grad, gtol = pull(x, t, g, np.abs(w) * slope_tol, temperature, kind)
    edge = z(np.minimum(np.abs(r - (1 - lo)), np.abs(r - (1 + hi))))
    return {"logprobs": (z(logp), z(lt) + out * np.abs(z(logp))), "row_loss": (z(loss), z(loss_tol)),
            "kl": (z(kl), z(kl_tol)) if ref is not None else (0 * z(kl), 0 * z(kl)),
            "loss": total(w, z(loss), z(loss_tol), out), "grad": (grad, gtol), "edge": np.where(on, edge, 1.0)}


def total(w, loss, tol, out):
    s = np.where(w != 0, w * loss, 0.0).sum()
    return s, (np.abs(w) * tol).sum() + out * abs(s) * 1.5


def distill(x, teacher, index, tlse, w, temperature, kind):
    """Rows [n, V], entries [n, K] (float64, -inf = padding)."""
    n, v = x.shape
    r = Row(x, temperature, kind)
    out = EPS["f64"] if kind == "f64" else EPS["f32"]
    row_loss, row_tol = np.zeros(n), np.zeros(n)
    grad, gtol = np.zeros((n, v)), np.zeros((n, v))
    for i in range(n):
        valid = teacher[i] != -np.inf
        if w[i] == 0 or not valid.any():
            continue
        k = index[i][valid]
        if ((k < 0) | (k >= v)).any() or len(set(k.tolist())) < len(k):
            row_loss[i], grad[i] = np.nan, np.nan
            continue
        zq = teacher[i][valid] / temperature
        if tlse is None:
            mx = zq.max()
            logq = zq - (mx + np.log(np.exp(zq - mx).sum()))
        else:
            logq = zq - tlse[i]
        q, logp, p = np.exp(logq), r.logp[i, k], r.p[i]
        # q is float64 on both sides
        q_rel = 2 * EPS["f64"] * (np.abs(zq) + np.abs(zq - logq) + 4)
        some = q > 0
        loss = (q[some] * (logq[some] - logp[some])).sum()
        tol = q.sum() * (r.s_rel[i] + 4 * r.u) + (q * q_rel * (1 + np.abs(logq - np.where(some, logp, 0.0))))[some].sum()
        a, big = 1.0, 1.0
        if tlse is not None:
            mass = q.sum()
            q_rest = max(0.0, 1.0 - mass) if len(k) < v else 0.0
            big = mass + q_rest
            others = np.delete(p, k)
            p_rest = others.sum()
            if q_rest > 0:
                with np.errstate(divide="ignore"):
                    loss += q_rest * (np.log(q_rest) - np.log(p_rest))
                tol += q_rest * 2 * r.p_rel[i].max()
            a = big - (q_rest / p_rest if p_rest > 0 else 0.0)
        c = w[i] / temperature
        g = c * a * p
        # where A is the difference Q - q'/p', its terms' own errors count
        gt = np.abs(c) * p * (r.p_rel[i] + 4 * r.u) * (np.abs(a) if tlse is None else big + abs(big - a)) * 2
        if tlse is not None and p_rest == 0:
            g[:] = 0.0
        g[k] = c * (big * p[k] - q)
        gt[k] = np.abs(c) * (big * p[k] * (r.p_rel[i][k] + 4 * r.u) + (4 * r.u + q_rel) * q)
        row_loss[i], row_tol[i] = loss, tol + 4 * out * abs(loss)
        grad[i], gtol[i] = g, gt
    gtol = gtol + EPS[kind] * (np.abs(grad) + gtol) + 1e-37 + 4 * EPS["f64"] * np.abs(grad)
    return {"row_loss": (row_loss, row_tol), "loss": total(w, row_loss, row_tol, out), "grad": (grad, gtol)}


def preference(x, t, ends, ref, mask, w, beta, eps, average, kind):
    """Rows [n, V]; ends [2 * pairs + 1]."""
    pairs = (len(ends) - 1) // 2
    n = x.shape[0]
    mask = mask & (np.arange(n) >= ends[0]) & (np.arange(n) < ends[-1])
    logp, lt, _, _ = token(x, t, mask, 1.0, kind)
    out = EPS["f64"] if kind == "f64" else EPS["f32"]
    inner = np.where(mask, lt - out * np.abs(logp), 0.0)
    diff = np.where(mask, logp - (ref if ref is not None else 0.0), 0.0)
    reward, rtol, share = np.zeros(2 * pairs), np.zeros(2 * pairs), np.ones(2 * pairs)
    for s in range(2 * pairs):
        b = slice(ends[s], ends[s + 1])
        if average:
            share[s] = 1.0 / max(1, mask[b].sum())
        reward[s] = beta * diff[b].sum() * share[s]
        rtol[s] = beta * share[s] * (inner[b].sum() + 2.0 ** -50 * np.abs(logp[b]).sum())
    h = reward[:pairs] - reward[pairs:]
    softplus = lambda z: np.maximum(z, 0) + np.log1p(np.exp(-np.abs(z)))
    sigma = lambda z: np.exp(-softplus(-z))
    loss = (1 - eps) * softplus(-h) + eps * softplus(h)
    ht = rtol[:pairs] + rtol[pairs:]
    loss_tol = ht + 4 * out * loss
    dh = eps * sigma(h) - (1 - eps) * sigma(-h)
    g, gt = np.zeros(n), np.zeros(n)
    for s in range(2 * pairs):
        b, i, sign = slice(ends[s], ends[s + 1]), s % pairs, 1 if s < pairs else -1
        if w[i] != 0:
            g[b] = sign * beta * w[i] * dh[i] * share[s] * mask[b]
            gt[b] = beta * abs(w[i]) * share[s] * 0.26 * ht[i]  # sigma' <= 1/4
    grad, gtol = pull(x, t, g, gt, 1.0, kind)
    return {"logprobs": (logp, np.where(mask, lt, 0.0)), "rewards": (reward, rtol + 2 * out * np.abs(reward)),
            "pair_loss": (loss, loss_tol), "loss": total(w, loss, loss_tol, out), "grad": (grad, gtol)}
