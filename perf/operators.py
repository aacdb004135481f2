"""The losses over rows of a logits matrix, as they are measured: log-probabilities of chosen tokens
(and their backward pass), distillation from a teacher's top logits, the clipped policy loss with a
KL term, and the preference loss on pairs of sequences, each with the gradient of the logits.

`run` computes them in their plain form (elementary torch operations in 32 bits, row statistics that
cancel in 64), or, where `own` is true, through ctorch_b200.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # log-probabilities of the tokens that a server has just sampled for four users
        {"name": "logprobs_serve", "op": "logprobs", "rows": 4, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "backward": False, "kept": 1.0, "temperature": 0.7},
        # scoring of prompts: forward only, one row a position
        {"name": "logprobs_score", "op": "logprobs", "rows": 8192, "vocab": 32768, "pad": 0, "dtype": "bf16",
         "backward": False, "kept": 1.0, "temperature": 1.0},
        # a training step in float32 on a vocabulary of odd size (no row starts on 16 bytes but every fourth)
        {"name": "logprobs_train_odd", "op": "logprobs", "rows": 2047, "vocab": 50021, "pad": 0, "dtype": "f32",
         "backward": True, "kept": 0.9, "temperature": 1.0},
        # a small student: 64 rows of a small vocabulary, 8 teacher entries a row
        {"name": "distill_small", "op": "distill", "rows": 64, "vocab": 8192, "pad": 0, "dtype": "f32",
         "top": 8, "tail": False, "kept": 1.0, "temperature": 1.0},
        # an ordinary step: the teacher's 64 best, renormalised, softened
        {"name": "distill_step", "op": "distill", "rows": 4096, "vocab": 32768, "pad": 0, "dtype": "bf16",
         "top": 64, "tail": False, "kept": 0.9, "temperature": 2.0},
        # the large one: a wide vocabulary, the teacher's 128 best, and the mass of the rest as one event
        {"name": "distill_tail_large", "op": "distill", "rows": 4096, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "top": 128, "tail": True, "kept": 1.0, "temperature": 1.0},
        # a policy step on a handful of tokens
        {"name": "policy_small", "op": "policy", "rows": 32, "vocab": 4096, "pad": 0, "dtype": "f32",
         "kept": 1.0, "temperature": 1.0, "kl": 0.0},
        # an odd vocabulary inside rows padded to 64 columns, a sixth of the tokens not counted
        {"name": "policy_padded", "op": "policy", "rows": 3001, "vocab": 50021, "pad": 27, "dtype": "bf16",
         "kept": 0.85, "temperature": 1.0, "kl": 0.04},
        # the large one
        {"name": "policy_large", "op": "policy", "rows": 8192, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "kept": 0.9, "temperature": 1.0, "kl": 0.02},
        # one pair of short answers
        {"name": "preference_small", "op": "preference", "pairs": 1, "length": 31, "packed": True, "vocab": 8192,
         "pad": 0, "dtype": "f32", "kept": 0.7, "smoothing": 0.0, "average": False},
        # a padded batch, next-token positions of [sequences, length + 1, vocab], prompts not counted
        {"name": "preference_batch", "op": "preference", "pairs": 8, "length": 255, "packed": False, "vocab": 32768,
         "pad": 0, "dtype": "bf16", "kept": 0.6, "smoothing": 0.1, "average": False},
        # packed sequences of unequal lengths over a wide vocabulary of odd size
        {"name": "preference_packed", "op": "preference", "pairs": 4, "length": 500, "packed": True, "vocab": 100003,
         "pad": 0, "dtype": "bf16", "kept": 0.8, "smoothing": 0.0, "average": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: a vocabulary of 1000 to 131072, one row to as many as make 2 GB of logits in
    the work of the largest listed case, padded or odd rows, either type, every operator."""
    op = rng.choice(["logprobs", "distill", "policy", "preference"])
    vocab = _log_int(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = max(64, vocab // 64 * 64)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    pad = rng.choice([0, 0, -vocab % 64])
    most = (1 << 30) // (vocab * BYTES[dtype])
    case = {"op": op, "vocab": vocab, "pad": pad, "dtype": dtype, "kept": round(rng.uniform(0.5, 1.0), 2)}
    if op == "preference":
        rows = _log_int(rng, 8, max(8, min(16384, most)))
        pairs = max(1, min(rows // 4, _log_int(rng, 1, 64)))
        case.update(pairs=pairs, length=max(2, rows // (2 * pairs)), packed=rng.random() < 0.5,
                    smoothing=rng.choice([0.0, 0.1]), average=rng.random() < 0.5)
        return case
    case.update(rows=_log_int(rng, 1, min(16384, most)), temperature=rng.choice([1.0, 1.0, 0.8, 2.0]))
    if op == "logprobs":
        case.update(backward=rng.random() < 0.6)
    elif op == "distill":
        case.update(top=_log_int(rng, 1, min(256, vocab // 4)), tail=rng.random() < 0.5)
    else:
        case.update(kl=rng.choice([0.0, 0.05]))
    return case


def _rows_of(case):
    return 2 * case["pairs"] * case["length"] if case["op"] == "preference" else case["rows"]


# ------------------------------------------------------------------------------------- inputs


def _logits(g, shape, vocab, pad, dtype):
    """Logits of a trained model: a broad body, a few likely tokens, one of which is the target."""
    rows = math.prod(shape)
    x = torch.empty((rows, vocab + pad), dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=g)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    likely = torch.randint(vocab, (rows, 3), generator=g, device="cuda")
    at = torch.arange(rows, device="cuda")
    for k in range(3):
        x[at, likely[:, k]] = (9.0 + 3.0 * torch.rand(rows, generator=g, device="cuda")).to(dtype)
    x[at, targets] = (8.0 + 6.0 * torch.rand(rows, generator=g, device="cuda")).to(dtype)
    return x.view(*shape, vocab + pad)[..., :vocab], targets.view(shape)


def _keep(g, rows, share):
    """Which rows count; one of them at least."""
    keep = torch.rand(rows, generator=g, device="cuda") < share
    keep[0] = True
    return keep


def _near_logprobs(g, x, targets, temperature, spread):
    """Log-probabilities as another model's would be: these logits' own, moved a little."""
    out = torch.empty(targets.shape, dtype=torch.float32, device="cuda")
    for i in range(0, x.shape[0], 512):
        z = x[i:i + 512].float() / temperature
        out[i:i + 512] = z.gather(-1, targets[i:i + 512, None])[:, 0] - z.logsumexp(-1)
    return (out + spread * torch.randn(out.shape, generator=g, device="cuda")).clamp_max(0.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, vocab, dtype = case["op"], case["vocab"], DTYPES[case["dtype"]]
    if op == "preference":
        return _prepare_preference(case, g, vocab, dtype)
    rows = case["rows"]
    x, targets = _logits(g, (rows,), vocab, case["pad"], dtype)
    keep = _keep(g, rows, case["kept"])
    s = {"op": op, "logits": x, "temperature": case["temperature"]}
    if op == "logprobs":
        s.update(targets=targets, mask=keep if case["kept"] < 1 else None, backward=case["backward"])
        s["upstream"] = torch.randn(rows, generator=g, device="cuda") / rows
        return s
    s["weights"] = keep.float() / keep.sum()
    if op == "policy":
        s.update(targets=targets, kl=case["kl"])
        s["old"] = _near_logprobs(g, x, targets, case["temperature"], 0.15)
        s["ref"] = _near_logprobs(g, x, targets, case["temperature"], 0.3) if case["kl"] else None
        s["advantages"] = torch.randn(rows, generator=g, device="cuda")
        return s
    # the teacher's best entries: the target among the student's likely ones, and others at random, all
    # different (one from each of `top` equal parts of the vocabulary)
    top = case["top"]
    part = vocab // top
    index = torch.arange(top, device="cuda") * part + torch.randint(part, (rows, top), generator=g, device="cuda")
    index.scatter_(1, (targets // part).clamp_max(top - 1)[:, None], targets[:, None])
    teacher = x.gather(1, index).float() + torch.randn((rows, top), generator=g, device="cuda")
    teacher, order = teacher.sort(dim=1, descending=True)
    s.update(index=index.gather(1, order), teacher=teacher, lse=None)
    if case["tail"]:
        rest = 0.05 + 0.4 * torch.rand(rows, generator=g, device="cuda")  # the teacher's mass outside
        s["lse"] = (teacher / case["temperature"]).logsumexp(1) - torch.log1p(-rest)
    return s


def _prepare_preference(case, g, vocab, dtype):
    pairs, length = case["pairs"], case["length"]
    n = 2 * pairs
    if case["packed"]:
        # every sequence gives some of its share to the next one
        move = torch.randint(max(1, length // 2), (n + 1,), generator=g, device="cuda")
        move[0] = move[n] = 0
        offsets = torch.arange(n + 1, device="cuda") * length + move
        x, targets = _logits(g, (n * length,), vocab, case["pad"], dtype)
    else:
        offsets = None
        x, targets = _logits(g, (n, length + 1), vocab, case["pad"], dtype)
        x, targets = x[:, :-1], targets[:, :-1]
    keep = _keep(g, targets.numel(), case["kept"]).view(targets.shape)
    flat = [_near_logprobs(g, x.flatten(0, -2)[i:i + 512] if case["packed"] else x[i // length], t, 1.0, 0.1)
            for i, t in zip(range(0, n * length, 512 if case["packed"] else length),
                            targets.split(512) if case["packed"] else targets)]
    ref = torch.cat(flat).view(targets.shape)
    return {"op": "preference", "logits": x, "targets": targets, "mask": keep, "offsets": offsets, "ref": ref,
            "pairs": pairs, "beta": 0.1, "smoothing": case["smoothing"], "average": case["average"]}


# ------------------------------------------------------------------------------------- one pass


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import ctorch_b200 as cb

    if s["op"] == "logprobs":
        r = cb.token_logprobs(s["logits"], s["targets"], mask=s["mask"], temperature=s["temperature"])
        if not s["backward"]:
            return {"logprobs": r.logprobs, "lse": r.lse}
        grad = cb.token_logprobs_backward(s["upstream"], s["logits"], s["targets"], r.logprobs, r.lse,
                                          mask=s["mask"], temperature=s["temperature"])
        return {"logprobs": r.logprobs, "lse": r.lse, "grad": grad}
    if s["op"] == "distill":
        r = cb.distill_loss(s["logits"], s["teacher"], s["index"], teacher_lse=s["lse"], weights=s["weights"],
                            temperature=s["temperature"])
        return {"loss": r.loss, "row_loss": r.row_loss, "grad": r.grad}
    if s["op"] == "policy":
        r = cb.policy_loss(s["logits"], s["targets"], s["old"], s["advantages"], ref_logprobs=s["ref"],
                           weights=s["weights"], clip_low=0.2, clip_high=0.2, kl_coef=s["kl"],
                           temperature=s["temperature"])
        return {"loss": r.loss, "row_loss": r.row_loss, "logprobs": r.logprobs, "grad": r.grad}
    r = cb.preference_loss(s["logits"], s["targets"], s["pairs"], ref_logprobs=s["ref"], mask=s["mask"],
                           offsets=s["offsets"], beta=s["beta"], label_smoothing=s["smoothing"],
                           average=s["average"])
    return {"loss": r.loss, "pair_loss": r.pair_loss, "rewards": r.rewards, "logprobs": r.logprobs, "grad": r.grad}


def _softmax_parts(x, temperature):
    """exp(z - max), its sum, and the pieces of log-sum-exp (the maximum and the logarithm, in 64 bits)."""
    z = x.float() / temperature
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    return e, total, top.double(), torch.log(total.double())


def _picked(x, index, temperature, top, log_total):
    """Log-probabilities of x's entries at `index`, in 64 bits."""
    return x.gather(-1, index).double() / temperature - top - log_total


def _pull(e, total, targets, upstream, temperature, dtype):
    """The gradient of sum(upstream * log p[target]): upstream / T * (1[target] - p)."""
    c = (upstream / temperature).unsqueeze(-1)
    grad = e * (-c / total)
    grad.scatter_add_(-1, targets.unsqueeze(-1), c)
    return grad.to(dtype)


def _run_plain(s):
    x, dtype = s["logits"], s["logits"].dtype
    if s["op"] == "distill":
        return _plain_distill(s)
    temperature = s.get("temperature", 1.0)
    e, total, top, log_total = _softmax_parts(x, temperature)
    logp = _picked(x, s["targets"].unsqueeze(-1), temperature, top, log_total).squeeze(-1)
    if s["op"] == "logprobs":
        lse = (top + log_total).squeeze(-1)
        if s["mask"] is not None:
            logp, lse = logp.where(s["mask"], 0.0), lse.where(s["mask"], 0.0)
        out = {"logprobs": logp.float(), "lse": lse.float()}
        if s["backward"]:
            up = s["upstream"] if s["mask"] is None else s["upstream"].where(s["mask"], 0.0)
            out["grad"] = _pull(e, total, s["targets"], up, temperature, dtype)
        return out
    if s["op"] == "policy":
        counts = s["weights"] != 0
        ratio = torch.exp(logp - s["old"])
        a = s["advantages"].double()
        u, c = ratio * a, ratio.clamp(0.8, 1.2) * a
        loss, slope = -torch.minimum(u, c), -u * (u <= c)
        if s["kl"]:
            d = s["ref"].double() - logp
            loss = loss + s["kl"] * (torch.exp(d) - d - 1)
            slope = slope + s["kl"] * (1 - torch.exp(d))
        loss, logp = loss.where(counts, 0.0), logp.where(counts, 0.0)
        up = (s["weights"] * slope).where(counts, 0.0).float()
        return {"loss": (s["weights"] * loss).sum().float(), "row_loss": loss.float(), "logprobs": logp.float(),
                "grad": _pull(e, total, s["targets"], up, temperature, dtype)}
    # preference
    n = 2 * s["pairs"]
    mask, shape = s["mask"], logp.shape
    logp = logp.where(mask, 0.0)
    if s["offsets"] is None:
        seq = torch.arange(n, device=x.device).repeat_interleave(shape[-1])
    else:
        seq = torch.searchsorted(s["offsets"], torch.arange(logp.numel(), device=x.device), right=True) - 1
    diff = (logp - s["ref"].where(mask, 0.0)).reshape(-1)
    ratio = torch.zeros(n, dtype=torch.float64, device=x.device).index_add_(0, seq, diff)
    scale = torch.ones_like(ratio)
    if s["average"]:
        scale = 1 / torch.zeros_like(ratio).index_add_(0, seq, mask.reshape(-1).double()).clamp_min(1)
    rewards = s["beta"] * ratio * scale
    h = rewards[: s["pairs"]] - rewards[s["pairs"]:]
    eps = s["smoothing"]
    pair = (1 - eps) * torch.log1p(torch.exp(-h)) + eps * torch.log1p(torch.exp(h))
    dh = s["beta"] / s["pairs"] * (eps / (1 + torch.exp(-h)) - (1 - eps) / (1 + torch.exp(h)))
    up = (torch.cat([dh, -dh]) * scale)[seq].view(shape).where(mask, 0.0).float()
    return {"loss": pair.mean().float(), "pair_loss": pair.float(), "rewards": rewards.float(),
            "logprobs": logp.float(), "grad": _pull(e, total, s["targets"], up, 1.0, dtype)}


def _plain_distill(s):
    x, t = s["logits"], s["temperature"]
    e, total, top, log_total = _softmax_parts(x, t)
    logp = _picked(x, s["index"], t, top, log_total)
    zq = s["teacher"].double() / t
    lse = torch.log(torch.exp(zq - zq.amax(1, keepdim=True)).sum(1, keepdim=True)) + zq.amax(1, keepdim=True)
    logq = zq - (lse if s["lse"] is None else s["lse"].double()[:, None])
    q = torch.exp(logq)
    loss = (q * (logq - logp)).sum(1)
    w = s["weights"].double()
    inner = (w / t)[:, None]
    if s["lse"] is None:
        grad = e * (inner / total).float()
    else:
        others = e.scatter(1, s["index"], 0.0).sum(1, keepdim=True).double()
        q_rest, p_rest = 1 - q.sum(1, keepdim=True), others / total
        loss = loss + (q_rest * (torch.log(q_rest) - torch.log(p_rest)))[:, 0]
        grad = e * (inner * (1 - q_rest / p_rest) / total).float()
    grad.scatter_(1, s["index"], (inner * (torch.exp(logp) - q)).float())
    loss = loss.where(w != 0, 0.0)
    return {"loss": (w * loss).sum().float(), "row_loss": loss.float(), "grad": grad.to(x.dtype)}


# ------------------------------------------------------------------------------------- work


def work(case):
    """Each counted row's logits read once (a row that does not count is not read), the whole gradient
    written once, the rows' own numbers; an exponential, a multiply-add and an addition an element forward,
    an exponential and a multiply backward."""
    rows, v, b = _rows_of(case), case["vocab"], BYTES[case["dtype"]]
    read = rows * case["kept"] * v * b
    op = case["op"]
    if op == "logprobs":
        return {"bytes": read + rows * 20 + (rows * v * b + 4 * rows if case["backward"] else 0),
                "flops": rows * v * (6 if case["backward"] else 4)}
    extra = {"policy": 28 if case.get("kl") else 24, "preference": 17,
             "distill": 12 * case.get("top", 0) + 12}[op]
    return {"bytes": read + rows * v * b + rows * extra, "flops": rows * v * 6}


# ------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The same outputs by the definitions in 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    x, v = s["logits"], case["vocab"]
    shape = x.shape[:-1]
    rows = math.prod(shape)
    t = s.get("temperature", 1.0)
    blocks = [slice(i, min(i + 256, rows)) for i in range(0, rows, 256)]

    def row_block(b):
        if x.dim() == 2:
            return x[b].double() / t
        i = torch.arange(b.start, b.stop, device=x.device)
        return x[i // shape[1], i % shape[1]].double() / t

    lse = torch.cat([torch.logsumexp(row_block(b), -1) for b in blocks])

    def gradient(of_block):
        return torch.cat([of_block(b, torch.exp(row_block(b) - lse[b, None])).to(torch.float64) for b in blocks]).view(*shape, v)

    if case["op"] == "distill":
        out = _exact_distill(s, row_block, lse, blocks, t, gradient)
        return out
    target = s["targets"].reshape(-1)
    logp = torch.cat([row_block(b).gather(1, target[b, None])[:, 0] for b in blocks]) - lse

    def pulled(up):
        def of_block(b, p):
            y = -p * up[b, None]
            y[torch.arange(b.stop - b.start, device=x.device), target[b]] += up[b]
            return y / t
        return gradient(of_block)

    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    if case["op"] == "logprobs":
        on = torch.ones_like(target, dtype=torch.bool) if s["mask"] is None else s["mask"]
        out = {"logprobs": torch.where(on, logp, zero), "lse": torch.where(on, lse, zero)}
        if case["backward"]:
            out["grad"] = pulled(torch.where(on, s["upstream"].double(), zero))
        return out
    if case["op"] == "policy":
        w, a = s["weights"].double(), s["advantages"].double()
        ratio = torch.exp(logp - s["old"].double())
        low, high = 1 - 0.2, 1 + 0.2
        held = torch.clamp(ratio, low, high)
        free = ratio * a <= held * a
        loss = -torch.where(free, ratio * a, held * a)
        slope = torch.where(free, -ratio * a, zero)
        if s["ref"] is not None:
            d = s["ref"].double() - logp
            loss = loss + case["kl"] * (torch.expm1(d) - d)
            slope = slope - case["kl"] * torch.expm1(d)
        on = w != 0
        loss = torch.where(on, loss, zero)
        return {"loss": (w * loss).sum(), "row_loss": loss, "logprobs": torch.where(on, logp, zero),
                "grad": pulled(torch.where(on, w * slope, zero))}
    pairs, n = s["pairs"], 2 * s["pairs"]
    ends = s["offsets"].tolist() if s["offsets"] is not None else [i * shape[1] for i in range(n + 1)]
    on, ref = s["mask"].reshape(-1), s["ref"].reshape(-1).double()
    part = [slice(ends[i], ends[i + 1]) for i in range(n)]
    sums = torch.stack([((logp[b] - ref[b]) * on[b]).sum() for b in part])
    share = torch.stack([1.0 / on[b].sum().clamp_min(1).double() if s["average"] else zero + 1.0 for b in part])
    rewards = s["beta"] * sums * share
    h, eps = rewards[:pairs] - rewards[pairs:], s["smoothing"]
    logsigmoid = torch.nn.functional.logsigmoid
    loss = -(1 - eps) * logsigmoid(h) - eps * logsigmoid(-h)
    dh = (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)) * s["beta"] / pairs
    up = torch.zeros_like(logp)
    for i, b in enumerate(part):
        up[b] = (dh[i] if i < pairs else -dh[i - pairs]) * share[i] * on[b]
    return {"loss": loss.mean(), "pair_loss": loss, "rewards": rewards,
            "logprobs": torch.where(on, logp, zero).view(shape), "grad": pulled(up)}


def _exact_distill(s, row_block, lse, blocks, t, gradient):
    zq = s["teacher"].double() / t
    logq = torch.log_softmax(zq, 1) if s["lse"] is None else zq - s["lse"].double()[:, None]
    q, w = logq.exp(), s["weights"].double()
    logp = torch.cat([row_block(b).gather(1, s["index"][b]) for b in blocks]) - lse[:, None]
    loss = (q * (logq - logp)).sum(1)
    rest_q = rest_p = None
    if s["lse"] is not None:
        rest_q = 1 - q.sum(1)
        rest_p = torch.cat([torch.exp(row_block(b) - lse[b, None]).scatter(1, s["index"][b], 0).sum(1) for b in blocks])
        loss = loss + rest_q * (rest_q.log() - rest_p.log())

    def of_block(b, p):
        y = p.clone() if rest_q is None else p * (1 - rest_q[b] / rest_p[b])[:, None]
        y.scatter_(1, s["index"][b], p.gather(1, s["index"][b]) - q[b])
        return y * (w[b] / t)[:, None]

    loss = torch.where(w != 0, loss, torch.zeros_like(loss))
    return {"loss": (w * loss).sum(), "row_loss": loss, "grad": gradient(of_block)}
