"""The end of a language model's step around the losses over logits rows, as it is measured: the norm with the
residual's addition (also to 8 bits) and its backward pass, the projection to the vocabulary with its cross entropy and
both gradients, and the balance loss of routed experts with its counts and gradient.

`run` computes them in their plain form (elementary torch operations and matrix products in 32 bits, long sums in 64),
or, where `own` is true, through ctorch_b200.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
E4M3_MAX = 448.0
BLOCK = 128  # columns that share a scale where the scales are not a row's


def listed():
    return [
        # one token scored against the whole vocabulary: forward only
        {"name": "head_token", "op": "head", "rows": 1, "dim": 2048, "vocab": 32768, "pad": 0, "dtype": "bf16",
         "grad": False, "kept": 1.0, "z": 0.0},
        # a small model in float32, every size odd
        {"name": "head_f32_odd", "op": "head", "rows": 509, "dim": 517, "vocab": 10007, "pad": 0, "dtype": "f32",
         "grad": True, "kept": 1.0, "z": 0.0},
        # an ordinary training step
        {"name": "head_step", "op": "head", "rows": 4096, "dim": 2048, "vocab": 32768, "pad": 0, "dtype": "bf16",
         "grad": True, "kept": 0.9, "z": 1e-4},
        # answers after masked prompts, a vocabulary of odd size, rows with a gap between them
        {"name": "head_masked", "op": "head", "rows": 2047, "dim": 1600, "vocab": 50021, "pad": 24, "dtype": "bf16",
         "grad": True, "kept": 0.6, "z": 0.0},
        # the largest: a long batch on a large vocabulary
        {"name": "head_large", "op": "head", "rows": 8192, "dim": 4096, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "grad": True, "kept": 1.0, "z": 0.0},
        # tokens that a server decodes for eight users, to 8 bits with a scale a row
        {"name": "norm_decode", "op": "norm", "rows": 8, "dim": 4096, "dtype": "bf16", "quant": "row", "train": False},
        # a prompt, to 8 bits with a scale for every 128 columns
        {"name": "norm_prompt", "op": "norm", "rows": 8192, "dim": 8192, "dtype": "bf16", "quant": "block",
         "train": False},
        # a training step, forward and backward
        {"name": "norm_train", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "quant": "", "train": True},
        # the same in float32 on rows of odd length
        {"name": "norm_train_odd", "op": "norm", "rows": 2047, "dim": 5003, "dtype": "f32", "quant": "", "train": True},
        # a few tokens on a few experts
        {"name": "balance_small", "op": "balance", "groups": 1, "length": 64, "experts": 8, "chosen": 2, "dtype": "f32",
         "kept": 1.0, "z": 0.0},
        # an ordinary step: the loss of each of sixteen sequences, padding left out
        {"name": "balance_step", "op": "balance", "groups": 16, "length": 1023, "experts": 60, "chosen": 4,
         "dtype": "bf16", "kept": 0.9, "z": 1e-3},
        # many experts, a long batch taken as one
        {"name": "balance_large", "op": "balance", "groups": 1, "length": 131072, "experts": 256, "chosen": 8,
         "dtype": "f32", "kept": 1.0, "z": 1e-3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["head", "head", "norm", "balance"])
    if op == "head":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        big = (8192, 4096, 131072) if dtype == "bf16" else (2048, 1024, 32768)
        dim = _log(rng, 64, big[1])
        if rng.random() < 0.7:
            dim -= dim % 8  # most models' sizes
        return {"op": op, "rows": _log(rng, 1, big[0]), "dim": dim, "vocab": _log(rng, 500, big[2]),
                "pad": rng.choice([0, 0, rng.randint(1, 40)]), "dtype": dtype, "grad": rng.random() < 0.8,
                "kept": rng.choice([1.0, round(rng.uniform(0.3, 1.0), 2)]), "z": rng.choice([0.0, 1e-4])}
    if op == "norm":
        dim = _log(rng, 64, 16384)
        train = rng.random() < 0.5
        return {"op": op, "rows": _log(rng, 1, 16384 * 4096 // max(dim, 4096)), "dim": dim,
                "dtype": rng.choice(["bf16", "f32"]), "quant": "" if train else rng.choice(["row", "block", ""]),
                "train": train}
    experts = _log(rng, 4, 512)
    rows = _log(rng, 8, 131072 * 256 // max(experts, 256))
    groups = rng.choice([1, min(rows, rng.randint(2, 64))])
    return {"op": op, "groups": groups, "length": rows // groups, "experts": experts,
            "chosen": rng.randint(1, min(8, experts)), "dtype": rng.choice(["bf16", "f32"]),
            "kept": rng.choice([1.0, round(rng.uniform(0.3, 1.0), 2)]), "z": rng.choice([0.0, 1e-3])}


# ------------------------------------------------------------------------------------- inputs


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _uniform(g, n):
    return torch.rand(n, generator=g, device="cuda")


def _keep(g, rows, share):
    """Which rows count; one of them at least."""
    keep = _uniform(g, rows) < share
    keep[0] = True
    return keep


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "head":
        rows, dim, vocab = case["rows"], case["dim"], case["vocab"]
        # logits of a spread of 2, and hidden states that lean towards their target as a trained model's do
        weight = _normal(g, vocab, dim, dtype=dtype, std=2.0 / math.sqrt(dim))
        targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
        hidden = _normal(g, rows, dim + case["pad"], dtype=dtype)
        hidden[:, :dim] += (3.0 * _uniform(g, rows)[:, None] * weight[targets]).to(dtype)
        weights = None
        if case["kept"] < 1:
            keep = _keep(g, rows, case["kept"])
            weights = keep.float() / keep.sum()
        return {"op": "head", "hidden": hidden[:, :dim], "weight": weight, "targets": targets, "weights": weights,
                "z": case["z"], "grad": case["grad"]}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s = {"op": "norm", "x": _normal(g, rows, dim, dtype=dtype, std=0.5), "quant": case["quant"] or None,
             "residual": _normal(g, rows, dim, dtype=dtype, std=2.0) * torch.exp(0.5 * _normal(g, rows, 1)).to(dtype),
             "weight": (1.0 + 0.3 * _normal(g, dim)).to(dtype), "eps": 1e-6, "train": case["train"]}
        if case["train"]:
            s["upstream"] = _normal(g, rows, dim, dtype=dtype, std=0.01)
            s["passed"] = _normal(g, rows, dim, dtype=dtype, std=0.01)
        return s
    rows, experts = case["groups"] * case["length"], case["experts"]
    # experts that the router prefers more and less
    logits = (_normal(g, rows, experts) + 0.7 * _normal(g, 1, experts)).to(dtype)
    chosen = torch.topk(logits.float(), case["chosen"], dim=-1).indices
    mask = _keep(g, rows, case["kept"]) if case["kept"] < 1 else None
    return {"op": "balance", "logits": logits, "experts": chosen, "mask": mask, "groups": case["groups"], "coef": 0.01,
            "z": case["z"]}


# ------------------------------------------------------------------------------------- one pass


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import ctorch_b200 as cb

    if s["op"] == "head":
        r = cb.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], weights=s["weights"], z_coef=s["z"],
                                    grad=s["grad"])
        out = {"loss": r.loss, "row_loss": r.row_loss, "lse": r.lse}
        if s["grad"]:
            out.update(grad_hidden=r.grad_hidden, grad_weight=r.grad_weight)
        return out
    if s["op"] == "norm":
        r = cb.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=s["eps"], quant=s["quant"])
        out = {"out": r.out, "summed": r.summed}
        if s["quant"]:
            out["scales"] = r.scales
        if s["train"]:
            b = cb.rms_norm_backward(s["upstream"], r.summed, s["weight"], r.rstd, grad_summed=s["passed"])
            out.update(grad_x=b.grad_x, grad_weight=b.grad_weight)
        return out
    r = cb.balance_loss(s["logits"], s["experts"], mask=s["mask"], groups=s["groups"], coef=s["coef"], z_coef=s["z"])
    return {"loss": r.loss, "counts": r.counts, "probs": r.probs, "grad": r.grad}


def _run_plain(s):
    return {"head": _plain_head, "norm": _plain_norm, "balance": _plain_balance}[s["op"]](s)


def _plain_head(s):
    h, w, t, dtype = s["hidden"].float(), s["weight"].float(), s["targets"], s["hidden"].dtype
    rows = h.shape[0]
    z = h @ w.t()
    top = z.amax(1, keepdim=True)
    zt = z.gather(1, t[:, None])
    e = torch.exp(z.sub_(top))
    total = e.sum(1, keepdim=True)
    rest = torch.log(total.double())
    lse = (top.double() + rest)[:, 0]
    loss = ((top - zt).double() + rest)[:, 0] + s["z"] * lse * lse
    r = torch.full((rows,), 1.0 / rows, device=h.device) if s["weights"] is None else s["weights"]
    on = r != 0
    loss, lse = loss.where(on, 0.0), lse.where(on, 0.0)
    out = {"loss": (r * loss).sum().float(), "row_loss": loss.float(), "lse": lse.float()}
    if s["grad"]:
        e *= (r.double() * (1 + 2 * s["z"] * lse) / total[:, 0]).float()[:, None]
        e.scatter_add_(1, t[:, None], -r[:, None])
        out["grad_hidden"] = (e @ w).to(dtype)
        out["grad_weight"] = (e.t() @ h).to(dtype)
    return out


def _plain_norm(s):
    dtype = s["x"].dtype
    summed = (s["x"].float() + s["residual"].float()).to(dtype)
    x, w = summed.float(), s["weight"].float()
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + s["eps"])
    hat = x * rstd
    y = hat * w
    out = {"summed": summed}
    if s["quant"]:
        rows, dim = y.shape
        block = dim if s["quant"] == "row" else BLOCK
        parts = -(-dim // block)
        padded = torch.nn.functional.pad(y, (0, parts * block - dim)).view(rows, parts, block)
        scales = padded.abs().amax(2, keepdim=True) / E4M3_MAX
        scales = scales.where(scales != 0, 1.0)
        q = (padded / scales).clamp(-E4M3_MAX, E4M3_MAX).view(rows, -1)[:, :dim]
        out["out"] = q.to(torch.float8_e4m3fn)
        out["scales"] = scales[:, 0] if s["quant"] == "row" else scales[:, :, 0]
        if s["quant"] == "row":
            out["scales"] = out["scales"][:, 0]
    else:
        out["out"] = y.to(dtype)
    if s["train"]:
        up = s["upstream"].float()
        gw = up * w
        grad = rstd * (gw - hat * (gw * hat).mean(1, keepdim=True))
        out["grad_x"] = (grad + s["passed"].float()).to(dtype)
        out["grad_weight"] = (up * hat).sum(0, dtype=torch.float64).to(dtype)
    return out


def _plain_balance(s):
    x, groups, experts = s["logits"].float(), s["groups"], s["logits"].shape[1]
    rows = x.shape[0]
    on = torch.ones(rows, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total))[:, 0].double().where(on, 0.0)
    live = on.view(groups, -1).sum(1).double()
    n = live.clamp_min(1.0)
    where = torch.arange(groups, device=x.device).repeat_interleave(rows // groups)
    flat = (where[:, None] * experts + s["experts"])[on].reshape(-1)
    counts = torch.bincount(flat, minlength=groups * experts).view(groups, experts)
    probs = p.where(on[:, None], 0.0).view(groups, -1, experts).sum(1, dtype=torch.float64) / n[:, None]
    share = counts / (n * s["experts"].shape[1])[:, None]
    inner = (share * probs).sum(1)
    loss = (s["coef"] * experts * inner + s["z"] * (lse * lse).view(groups, -1).sum(1) / n).mean()
    slope = s["coef"] * experts * share.float()[where]
    slope = slope - (slope * p).sum(1, keepdim=True)
    grad = p * (slope + (2 * s["z"] * lse).float()[:, None]) * (on / (n * groups)[where]).float()[:, None]
    return {"loss": loss.float(), "counts": counts, "probs": probs.float(), "grad": grad.to(s["logits"].dtype)}


# ------------------------------------------------------------------------------------- work


def work(case):
    """Each input read once and each output written once; rows that do not count are not read."""
    b = BYTES[case["dtype"]]
    if case["op"] == "head":
        rows, dim, vocab = case["rows"] * case["kept"], case["dim"], case["vocab"]
        twice = 2 if case["grad"] else 1  # both gradients have their operand's size
        return {"bytes": twice * (rows + vocab) * dim * b + 20 * case["rows"],
                "flops": (6 if case["grad"] else 2) * rows * dim * vocab}
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        if case["quant"]:
            scales = 1 if case["quant"] == "row" else -(-case["dim"] // BLOCK)
            return {"bytes": n * (3 * b + 1) + case["rows"] * scales * 4, "flops": 8 * n}
        return {"bytes": n * b * (8 if case["train"] else 4), "flops": (16 if case["train"] else 6) * n}
    rows = case["groups"] * case["length"]
    n = rows * case["experts"]
    return {"bytes": n * b * (1 + case["kept"]) + rows * case["chosen"] * 8, "flops": 8 * n}


# ------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The same outputs in 64 bits: the losses by their definitions, their gradients by differentiation."""
    s = prepare(case, seed)
    return {"head": _exact_head, "norm": _exact_norm, "balance": _exact_balance}[case["op"]](s)


def _exact_head(s):
    weight = s["weight"].double().requires_grad_(s["grad"])
    rows = s["targets"].shape[0]
    share = torch.ones(rows, dtype=torch.float64, device=weight.device) / rows if s["weights"] is None else s["weights"].double()
    row_loss, lse, grads = [], [], []
    for i in range(0, rows, 1024):
        h = s["hidden"][i:i + 1024].double().requires_grad_(s["grad"])
        z = torch.nn.functional.linear(h, weight)
        a = torch.logsumexp(z, 1)
        loss = torch.nn.functional.cross_entropy(z, s["targets"][i:i + 1024], reduction="none") + s["z"] * a.square()
        if s["grad"]:
            (loss * share[i:i + 1024]).sum().backward()
            grads.append(h.grad)
        row_loss.append(loss.detach())
        lse.append(a.detach())
        del z, loss, a
    row_loss, lse, on = torch.cat(row_loss), torch.cat(lse), share != 0
    zero = torch.zeros_like(lse)
    out = {"loss": (share * row_loss).sum(), "row_loss": torch.where(on, row_loss, zero), "lse": torch.where(on, lse, zero)}
    if s["grad"]:
        out.update(grad_hidden=torch.cat(grads), grad_weight=weight.grad)
    return out


def _exact_norm(s):
    total = s["x"].double() + s["residual"].double()
    rounded = total.to(s["x"].dtype).double().requires_grad_(s["train"])  # the norm is that of the sum as it is kept
    w = s["weight"].double().requires_grad_(s["train"])
    y = w * rounded / torch.sqrt(rounded.square().mean(1, keepdim=True) + s["eps"])
    out = {"summed": total, "out": y.detach()}
    if s["quant"]:
        rows, dim = y.shape
        width = dim if s["quant"] == "row" else BLOCK
        scales = torch.stack([part.abs().amax(1) / E4M3_MAX for part in y.split(width, 1)], 1)
        out["out"] = y / scales.repeat_interleave(width, 1)[:, :dim]
        out["scales"] = scales[:, 0] if s["quant"] == "row" else scales
    if s["train"]:
        (y * s["upstream"].double()).sum().backward()
        out["grad_x"] = rounded.grad + s["passed"].double()
        out["grad_weight"] = w.grad
    return out


def _exact_balance(s):
    x = s["logits"].double().requires_grad_(True)
    groups, (rows, experts) = s["groups"], x.shape
    on = torch.ones(rows, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"]
    counts, probs, loss = [], [], 0.0
    for rows_of, picked, live in zip(x.chunk(groups), s["experts"].chunk(groups), on.chunk(groups)):
        seen, n = rows_of[live], max(1, int(live.sum()))
        counts.append(torch.zeros(experts, dtype=torch.int64, device=x.device).scatter_add_(
            0, picked[live].reshape(-1), torch.ones_like(picked[live].reshape(-1))))
        probs.append(torch.softmax(seen, 1).sum(0) / n)
        share = counts[-1].double() / (n * picked.shape[1])
        loss = loss + s["coef"] * experts * (share * probs[-1]).sum() + s["z"] * torch.logsumexp(seen, 1).square().sum() / n
    loss = loss / groups
    loss.backward()
    return {"loss": loss.detach(), "counts": torch.stack(counts), "probs": torch.stack(probs).detach(), "grad": x.grad}
