"""GPU checks of the losses over logits rows against the float64 oracle (tests/losses_oracle.py), within
the bounds that it derives from the kernels' roundings."""
import numpy as np
import pytest
import torch

import losses_oracle as O

pytestmark = pytest.mark.gpu

KIND = {"f32": torch.float32, "bf16": torch.bfloat16, "f64": torch.float64}


def cb():
    import ctorch_b200

    return ctorch_b200


def dev(a, dtype=None):
    return torch.as_tensor(a, dtype=dtype).cuda()


def host(t):
    return t.detach().double().cpu().numpy()


def check(got, want, what=""):
    value, tol = want
    value, tol = np.asarray(value), np.asarray(tol)
    g = host(got)
    assert g.shape == value.shape, (what, g.shape, value.shape)
    assert (np.isnan(g) == np.isnan(value)).all(), f"{what}: NaN positions differ"
    inf = np.isinf(value)
    assert (g[inf] == value[inf]).all(), f"{what}: infinities differ"
    fine = ~(np.isnan(value) | inf)
    off = np.abs(g[fine] - value[fine]) - np.broadcast_to(tol, value.shape)[fine]
    if off.size and off.max() > 0:
        k = int(off.argmax())
        raise AssertionError(f"{what}: {g[fine][k]!r} for {value[fine][k]!r}, allowed "
                             f"{np.broadcast_to(tol, value.shape)[fine][k]:.3g}")


def make(rng, rows, v, kind, spread=3.0):
    x = dev(rng.normal(0, spread, (rows, v)), torch.float64).to(KIND[kind])
    return x, host(x)


def layouts(x, how):
    """The same [rows, V] values in other memory."""
    n, v = x.shape
    if how == "contiguous":
        return x.contiguous()
    if how == "pitched":  # rows padded to 128 bytes
        w = torch.full((n, -(-v * x.element_size() // 128) * 128 // x.element_size()), 7.0, dtype=x.dtype, device=x.device)
        w[:, :v] = x
        return w[:, :v]
    if how == "offset":  # rows that start anywhere
        w = torch.full((n * (v + 3) + 5,), 7.0, dtype=x.dtype, device=x.device)
        y = w[5:].view(n, v + 3)[:, 1:v + 1]
        y.copy_(x)
        return y
    if how == "columns":  # the vocabulary strided
        return x.t().contiguous().t()
    raise ValueError(how)


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 33), (6, 257), (7, 1000), (2, 5003), (3, 4096), (300, 64), (2, 40000), (1, 131072)]
LAYOUTS = ["contiguous", "pitched", "offset", "columns"]


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,v", SHAPES)
def test_token_logprobs(rows, v, kind, how):
    rng = np.random.default_rng(rows * v)
    x, hx = make(rng, rows, v, kind)
    t, mask = rng.integers(0, v, rows), rng.random(rows) < 0.7
    temperature = 1.0 if rows % 2 else 1.7
    y = layouts(x, how)
    for m in (None, mask):
        on = np.ones(rows, bool) if m is None else m
        r = cb().token_logprobs(y, dev(t), None if m is None else dev(m), temperature)
        logp, lt, lse, st = O.token(hx, t, on, temperature, kind)
        check(r.logprobs, (logp, np.where(on, lt, 0)), "logprobs")
        check(r.lse, (lse, np.where(on, st, 0)), "lse")
        up = rng.normal(size=rows).astype(np.float32)
        up[0] = 0.0 if rows > 2 else up[0]
        grad = cb().token_logprobs_backward(dev(up), y, dev(t), r.logprobs, r.lse, None if m is None else dev(m), temperature)
        # what it is given is off by the smaller of the two roundings, and the forward's own error
        extra = np.minimum(lt, st) + 2 * O.EPS["f64" if kind == "f64" else "f32"] * np.abs(logp)
        want, tol = O.pull(hx, t, np.where(on, up, 0.0).astype(np.float64), 0.0, temperature, kind, extra)
        check(grad, (want, tol), "grad")


# 16-byte packs of a row around every number of them that a warp holds, and what is too long for a warp
PACKS = [0, 1, 31, 32, 33, 64, 65, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 1700]


@pytest.mark.parametrize("how", ["contiguous", "pitched", "offset"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("packs", PACKS)
def test_rows_by_length(packs, kind, how):
    size = 4 if kind == "f32" else 2
    for more in (0, 16 // size - 1):
        rows, v = 21, packs * 16 // size + more
        if v == 0:
            continue
        rng = np.random.default_rng(v)
        x, hx = make(rng, rows, v, kind)
        t = rng.integers(0, v, rows)
        t[:4] = [0, v - 1, v // 2, min(v - 1, 8)]
        w = np.where(rng.random(rows) < 0.7, rng.random(rows), 0.0).astype(np.float32)
        w[:4] = 0.5
        on = w != 0
        y = layouts(x, how)
        r = cb().token_logprobs(y, dev(t), dev(w))
        logp, lt, lse, st = O.token(hx, t, on, 1.0, kind)
        check(r.logprobs, (logp, np.where(on, lt, 0)), "logprobs")
        check(r.lse, (lse, np.where(on, st, 0)), "lse")
        up = rng.normal(size=rows).astype(np.float32)
        extra = np.minimum(lt, st) + 2 * O.EPS["f32"] * np.abs(logp)
        want, tol = O.pull(hx, t, np.where(on, up, 0.0).astype(np.float64), 0.0, 1.0, kind, extra)
        check(cb().token_logprobs_backward(dev(up), y, dev(t), r.logprobs, r.lse, dev(w)), (want, tol), "grad")
        other = torch.full((rows, v + 1), 5.0, dtype=y.dtype, device="cuda")  # rows aligned unlike the logits'
        cb().token_logprobs_backward(dev(up), y, dev(t), r.logprobs, r.lse, dev(w), out=other[:, 1:])
        check(other[:, 1:], (want, tol), "grad into a view")
        assert (other[:, 0] == 5.0).all()
        old = (O.token(hx, t, np.ones(rows, bool), 1.0, "f64")[0] + 0.3 * rng.normal(size=rows)).astype(np.float32)
        f = lambda a: a.astype(np.float64)
        want = O.policy(hx, t, f(old), f(up), f(old), f(w), 0.1, 0.3, 0.1, 1.0, kind)
        assert want["edge"].min() > 1e-6
        got = cb().policy_loss(y, dev(t), dev(old), dev(up), dev(old), dev(w), 0.1, 0.3, 0.1)
        for name in ("logprobs", "row_loss", "kl", "loss", "grad"):
            check(getattr(got, name), want[name], name)
        same = cb().policy_loss(y, dev(t), dev(old), dev(up), dev(old), dev(w), 0.1, 0.3, 0.1, out_grad=y)
        assert same.grad is y and torch.equal(y, got.grad)


@pytest.mark.parametrize("kind,rows,v", [("bf16", 50, 65536), ("bf16", 2, 262144), ("bf16", 2, 262147), ("bf16", 1, 600001),
                                         ("f32", 3, 131075), ("f32", 40, 100000), ("f32", 20, 50000)])
def test_long_rows(kind, rows, v):
    """Rows split over clusters of every size, up to the longest that a cluster holds, and beyond that."""
    rng = np.random.default_rng(v)
    x, hx = make(rng, rows, v, kind)
    t = rng.integers(0, v, rows)
    on = np.ones(rows, bool)
    r = cb().token_logprobs(x, dev(t))
    logp, lt, lse, st = O.token(hx, t, on, 1.0, kind)
    check(r.logprobs, (logp, lt), "logprobs")
    old, adv, w = (logp + 0.05).astype(np.float32), rng.normal(size=rows).astype(np.float32), np.full(rows, 0.5, np.float32)
    f = lambda a: a.astype(np.float64)
    want = O.policy(hx, t, f(old), f(adv), None, f(w), 0.2, 0.2, 0.0, 1.0, kind)
    assert want["edge"].min() > 1e-5
    got = cb().policy_loss(x, dev(t), dev(old), dev(adv), weights=dev(w))
    for name in ("logprobs", "row_loss", "loss", "grad"):
        check(getattr(got, name), want[name], name)
    for top in (100, 2048):
        index = np.stack([rng.permutation(v)[:top] for _ in range(rows)])
        teacher = rng.normal(size=(rows, top)).astype(np.float32)
        tl = (np.log(np.exp(f(teacher)).sum(1)) + 0.3).astype(np.float32)
        want = O.distill(hx, f(teacher), index, f(tl), f(w), 1.0, kind)
        got = cb().distill_loss(x, dev(teacher), dev(index), dev(tl), dev(w))
        for name in ("row_loss", "loss", "grad"):
            check(getattr(got, name), want[name], name)
    import ctorch_b200._capi as C
    assert C.wait_timeouts() == 0


def test_leading_dims_and_broadcast_operands():
    rng = np.random.default_rng(5)
    b, l, v = 3, 5, 130
    full = dev(rng.normal(0, 2, (b, l + 1, v)), torch.float32)
    x = full[:, :-1]
    t = rng.integers(0, v, (b, l))
    adv = rng.normal(size=(b, 1)).astype(np.float32)
    old = -rng.random(l).astype(np.float32) * 4
    w = rng.random((b, 1)).astype(np.float32)
    r = cb().policy_loss(x, dev(t.astype(np.int32)), dev(old), dev(adv), weights=dev(w))
    flat = lambda a: np.broadcast_to(a, (b, l)).reshape(-1).astype(np.float64)
    want = O.policy(host(x).reshape(-1, v), t.reshape(-1), flat(old), flat(adv), None, flat(w), 0.2, 0.2, 0.0, 1.0, "f32")
    assert want["edge"].min() > 1e-5
    assert r.grad.shape == x.shape and r.logprobs.shape == (b, l)
    for k in ("loss", "row_loss", "logprobs", "kl", "grad"):
        value, tol = want[k]
        got = getattr(r, k)
        check(got.reshape(-1, v) if k == "grad" else got.reshape(-1) if k != "loss" else got, (value, tol), k)
    # one vector of logits is one row; an expanded one is the same row many times
    one = cb().token_logprobs(x[0, 0], dev(np.int64(3)))
    assert one.logprobs.shape == ()
    many = cb().token_logprobs(x[0, 0].expand(4, v), dev(np.full(4, 3)))
    assert torch.equal(many.logprobs, one.logprobs.expand(4))
    # permuted leading dims of rank 3, and target strides of their own
    p = dev(rng.normal(0, 2, (2, 3, 4, 65)), torch.float32).permute(2, 0, 1, 3)
    tp = dev(rng.integers(0, 65, (3, 4, 2))).permute(1, 2, 0)
    # (rows that start elsewhere on a 16-byte boundary are added in another order: equal within the bound)
    logp, lt, lse, st = O.token(host(p).reshape(-1, 65), tp.cpu().numpy().reshape(-1), np.ones(24, bool), 1.0, "f32")
    for q, tq in ((p, tp), (p.contiguous(), tp.contiguous())):
        got = cb().token_logprobs(q, tq)
        check(got.logprobs.reshape(-1), (logp, lt), "logprobs")
        check(got.lse.reshape(-1), (lse, st), "lse")


@pytest.mark.parametrize("kind", list(KIND))
def test_unusual_values(kind):
    lowest = torch.finfo(KIND[kind]).min
    v = 300
    rng = np.random.default_rng(11)
    x = rng.normal(size=(10, v))
    x[0, 10:] = -np.inf            # most of the row masked
    x[1] = -np.inf                 # all of it
    x[2] = lowest                  # the type's lowest throughout: uniform
    x[3, ::2] = lowest             # and in part
    x[4, 7] = np.inf
    x[5, 9] = np.nan
    x[6] += 1000.0                 # a common offset
    x[7, 1:] = -200.0              # one logit holds everything
    x[8, 20] = -np.inf             # the target itself is masked
    x[9] = 0.0
    t = np.array([3, 3, 3, 3, 3, 3, 3, 0, 20, 299])
    y = dev(x, torch.float64).to(KIND[kind])
    hx = host(y)
    r = cb().token_logprobs(y, dev(t))
    on = np.ones(10, bool)
    logp, lt, lse, st = O.token(hx, t, on, 1.0, kind)
    logp[4] = np.nan
    lse[4] = np.nan
    check(r.logprobs, (logp, lt), "logprobs")
    check(r.lse, (lse, st), "lse")
    grad = cb().token_logprobs_backward(torch.ones(10, device="cuda"), y, dev(t), r.logprobs, r.lse)
    ok = np.array([0, 2, 3, 6, 7, 8, 9])
    extra = np.minimum(lt, st) + 2 * O.EPS["f64" if kind == "f64" else "f32"] * np.where(np.isfinite(logp), np.abs(logp), 30.0)
    want, tol = O.pull(hx, t, np.ones(10), 0.0, 1.0, kind, extra)
    check(grad[ok], (want[ok], tol[ok]), "grad")
    assert torch.isnan(grad[[1, 4, 5]]).any(-1).all()
    # the same rows, not counted
    off = torch.zeros(10, dtype=torch.bool, device="cuda")
    r = cb().token_logprobs(y, dev(np.full(10, -100)), off)
    assert not r.logprobs.any() and not r.lse.any()
    g = cb().token_logprobs_backward(torch.full((10,), float("nan"), device="cuda"), y, dev(t), r.logprobs, r.lse, off)
    assert not g.any()
    nan = torch.full((10,), float("nan"), device="cuda")
    r = cb().policy_loss(y, dev(np.full(10, -100)), nan, nan, nan, off, kl_coef=0.1)
    assert all(not a.any() for a in (r.loss, r.row_loss, r.logprobs, r.kl, r.grad))
    e = torch.full((10, 2), float("nan"), device="cuda")
    r = cb().distill_loss(y, e, dev(np.full((10, 2), -1)), nan, off)
    assert all(not a.any() for a in (r.loss, r.row_loss, r.grad))


@pytest.mark.parametrize("kind", list(KIND))
def test_bad_targets(kind):
    v = 50
    x = torch.randn(4, v, device="cuda").to(KIND[kind])
    t = torch.tensor([3, v, -1, 4], device="cuda")
    status = cb().index_status()
    cb().check_index_status(status)
    r = cb().token_logprobs(x, t, status=status)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, False]
    assert not torch.isnan(r.lse).any()
    with pytest.raises(cb().ShapeError, match="index (50|-1) out of range"):
        cb().check_index_status(status)
    status.zero_()
    z = torch.zeros(4, device="cuda")
    p = cb().policy_loss(x, t, z, z + 1, status=status)
    bad = torch.isnan(p.grad).any(-1)
    assert bad.tolist() == [False, True, True, False] and torch.isnan(p.loss)
    with pytest.raises(cb().ShapeError):
        cb().check_index_status(status)
    g = cb().token_logprobs_backward(z + 1, x, t, r.logprobs, r.lse)
    assert torch.isnan(g).any(-1).tolist() == [False, True, True, False]
    good = torch.tensor([True, False, False, True], device="cuda")
    status.zero_()
    p = cb().policy_loss(x, t, z, z + 1, weights=good, status=status)
    assert torch.isfinite(p.grad).all() and torch.isfinite(p.loss)
    cb().check_index_status(status)


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,v", SHAPES)
def test_policy_loss(rows, v, kind, how):
    rng = np.random.default_rng(rows + v)
    x, hx = make(rng, rows, v, kind)
    t = rng.integers(0, v, rows)
    w = np.where(rng.random(rows) < 0.8, rng.random(rows), 0.0).astype(np.float32)
    temperature = 0.8 if rows % 2 else 1.0
    logp = O.token(hx, t, np.ones(rows, bool), temperature, "f64")[0]
    old = (logp + 0.3 * rng.normal(size=rows)).astype(np.float32)
    ref = (logp + 0.3 * rng.normal(size=rows)).astype(np.float32)
    adv = rng.normal(size=rows).astype(np.float32)
    if rows > 2:
        adv[1] = 0.0
    for r_, k in ((None, 0.0), (ref, 0.1), (ref, 0.0)):
        f = lambda a: None if a is None else a.astype(np.float64)
        want = O.policy(hx, t, f(old), f(adv), f(r_), f(w), 0.1, 0.3, k, temperature, kind)
        assert want["edge"].min() > 1e-5
        got = cb().policy_loss(layouts(x, how), dev(t), dev(old), dev(adv), None if r_ is None else dev(r_), dev(w),
                               0.1, 0.3, k, temperature)
        for name in ("logprobs", "row_loss", "kl", "loss", "grad"):
            check(getattr(got, name), want[name], name)
    only = cb().policy_loss(layouts(x, how), dev(t), dev(old), dev(adv), dev(ref), dev(w), 0.1, 0.3, 0.0, temperature, grad=False)
    assert only.grad is None and torch.equal(only.loss, got.loss) and torch.equal(only.row_loss, got.row_loss)


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,v,top,tail", [
    (3, 2, 1, True), (2, 1, 1, False), (2, 1, 1, True), (5, 7, 7, True), (5, 7, 3, False), (6, 257, 1, True),
    (4, 1000, 64, False), (4, 1000, 64, True), (2, 5003, 300, True), (3, 4096, 8, False), (2, 40000, 2048, True),
    (1, 131072, 100, True), (200, 64, 5, False)])
def test_distill_loss(rows, v, top, tail, kind, how):
    rng = np.random.default_rng(rows + v + top)
    x, hx = make(rng, rows, v, kind)
    index = np.stack([rng.permutation(v)[:top] for _ in range(rows)])
    teacher = (np.take_along_axis(hx, index, 1) + rng.normal(size=(rows, top))).astype(np.float32)
    if top > 2:
        teacher[0, 1] = -np.inf
        index[0, 1] = -5  # padding: not looked at
    if rows > 3:
        teacher[2] = -np.inf
    temperature = 2.0 if rows % 2 else 1.0
    with np.errstate(divide="ignore"):
        lse = (np.log(np.exp(teacher.astype(np.float64) / temperature).sum(1)) + 0.3).astype(np.float32) if tail else None
    w = np.where(rng.random(rows) < 0.8, rng.random(rows), 0.0).astype(np.float32)
    w[0] = 1.0
    f = lambda a: None if a is None else a.astype(np.float64)
    want = O.distill(hx, f(teacher), index, f(lse), f(w), temperature, kind)
    ti = dev(index.astype(np.int32 if rows % 2 else np.int64))
    got = cb().distill_loss(layouts(x, how), dev(teacher), ti, None if lse is None else dev(lse), dev(w), temperature)
    for name in ("row_loss", "loss", "grad"):
        check(getattr(got, name), want[name], name)
    only = cb().distill_loss(layouts(x, how), dev(teacher), ti, None if lse is None else dev(lse), dev(w), temperature, grad=False)
    assert only.grad is None and torch.equal(only.loss, got.loss)


@pytest.mark.parametrize("kind", list(KIND))
def test_distill_edges(kind):
    v, top = 700, 6
    rng = np.random.default_rng(2)
    x, hx = make(rng, 6, v, kind)
    index = np.stack([rng.permutation(v)[:top] for _ in range(6)])
    teacher = rng.normal(size=(6, top))
    index[1, 4] = index[1, 2]      # the same index twice
    index[2, 0] = v                # outside
    index[3, 5] = -1
    for lse in (None, np.log(np.exp(teacher).sum(1)) + 0.5):
        status = cb().index_status()
        f = lambda a: None if a is None else dev(a, torch.float32)
        got = cb().distill_loss(x, f(teacher), dev(index), f(lse), status=status)
        assert torch.isnan(got.row_loss).tolist() == [False, True, True, True, False, False]
        assert torch.isnan(got.grad).all(-1).tolist() == [False, True, True, True, False, False]
        with pytest.raises(cb().ShapeError):
            cb().check_index_status(status)
        # the next call finds nothing left of the bad rows
        good = np.stack([rng.permutation(v)[:top] for _ in range(6)])
        t32 = teacher.astype(np.float32).astype(np.float64)
        l32 = None if lse is None else lse.astype(np.float32).astype(np.float64)
        want = O.distill(hx, t32, good, l32, np.full(6, 1 / 6), 1.0, kind)
        got = cb().distill_loss(x, f(teacher), dev(good), f(lse))
        for name in ("row_loss", "loss", "grad"):
            check(getattr(got, name), want[name], name)
    # bfloat16 entries, strided lists, broadcast over the rows
    tb = dev(teacher[0]).to(torch.bfloat16)
    pair = torch.stack([dev(good[0]), dev(good[1])], -1)[:, 0]
    got = cb().distill_loss(x, tb, pair)
    want = O.distill(hx, np.tile(host(tb), (6, 1)), np.tile(good[0], (6, 1)), None, np.full(6, 1 / 6), 1.0, kind)
    for name in ("row_loss", "loss", "grad"):
        check(getattr(got, name), want[name], name)
    # a student certain of the teacher's entries: the rest's share of its own sum is about 1e-9
    y = x.clone()
    y[torch.arange(6, device="cuda")[:, None], dev(good)] = 24.0
    hy = host(y)
    lse = dev(np.log(np.exp(t32).sum(1)) + 0.3, torch.float32)
    got = cb().distill_loss(y, f(teacher), dev(good), lse)
    want = O.distill(hy, t32, good, host(lse), np.full(6, 1 / 6), 1.0, kind)
    for name in ("row_loss", "loss", "grad"):
        check(getattr(got, name), want[name], name)
    # -inf outside the entries: no mass there, an infinite loss, and no gradient on those logits
    y[:] = -np.inf
    y[torch.arange(6, device="cuda")[:, None], dev(good)] = 1.0
    got = cb().distill_loss(y, f(teacher), dev(good), lse)
    assert torch.isinf(got.row_loss).all() and torch.isfinite(got.grad).all()


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("v,ends", [(33, [0, 4, 9, 9, 12]), (1000, [2, 3, 7]), (5003, [0, 5, 8]), (64, [0, 0, 0])])
def test_preference_loss_packed(v, ends, kind, how):
    rng = np.random.default_rng(v)
    rows = max(ends) + 2  # rows behind the last sequence
    pairs = (len(ends) - 1) // 2
    x, hx = make(rng, rows, v, kind)
    t = rng.integers(0, v, rows)
    t[ends[-1]:] = -100
    t[:ends[0]] = -100
    mask = rng.random(rows) < 0.8
    ref = -rng.random(rows).astype(np.float32) * 5
    for r_, avg, eps, w in ((ref, False, 0.1, None), (None, True, 0.0, rng.random(pairs).astype(np.float32))):
        status = cb().index_status()
        got = cb().preference_loss(layouts(x, how), dev(t), pairs, None if r_ is None else dev(r_), dev(mask),
                                   dev(np.array(ends, np.int32 if avg else np.int64)), None if w is None else dev(w),
                                   0.3, eps, avg, status=status)
        hw = np.full(pairs, 1 / pairs) if w is None else w.astype(np.float64)
        want = O.preference(hx, t, ends, None if r_ is None else r_.astype(np.float64), mask, hw, 0.3, eps, avg, kind)
        for name in ("logprobs", "rewards", "pair_loss", "loss", "grad"):
            check(getattr(got, name), want[name], name)
        cb().check_index_status(status)
    only = cb().preference_loss(layouts(x, how), dev(t), pairs, None, dev(mask), dev(np.array(ends)), dev(w), 0.3, 0.0, True, grad=False)
    assert only.grad is None and torch.equal(only.loss, got.loss)


def test_preference_loss_padded_batch_and_bad_offsets():
    rng = np.random.default_rng(9)
    pairs, l, v = 3, 17, 260
    full = dev(rng.normal(0, 2, (2 * pairs, l + 1, v)), torch.float32).to(torch.bfloat16)
    x = full[:, :-1]
    t = rng.integers(0, v, (2 * pairs, l))
    mask = rng.random((2 * pairs, l)) < 0.6
    mask[1] = False  # a sequence with nothing to say
    w = np.array([0.5, 0.0, 2.0], np.float32)
    got = cb().preference_loss(x, dev(t), pairs, mask=dev(mask), weights=dev(w), beta=0.05)
    ends = [i * l for i in range(2 * pairs + 1)]
    want = O.preference(host(x).reshape(-1, v), t.reshape(-1), ends, None, mask.reshape(-1), w.astype(np.float64), 0.05,
                        0.0, False, "bf16")
    check(got.grad.reshape(-1, v), want["grad"], "grad")
    check(got.logprobs.reshape(-1), want["logprobs"], "logprobs")
    for name in ("rewards", "pair_loss", "loss"):
        check(getattr(got, name), want[name], name)
    flat = x.reshape(-1, v)
    for bad in ([0, 5, 3], [0, 5, 10 ** 6], [-1, 5, 9]):
        status = cb().index_status()
        got = cb().preference_loss(flat, dev(t.reshape(-1)), 1, offsets=dev(np.array(bad)), status=status)
        assert torch.isnan(got.loss) and torch.isnan(got.rewards).all() and torch.isnan(got.pair_loss).all()
        with pytest.raises(cb().ShapeError):
            cb().check_index_status(status)
    # very unequal pairs: both ends of the sigmoid
    y = torch.zeros(2, 4, device="cuda")
    y[0, 0], y[1, 0] = 500.0, -500.0
    for t0, want_loss in (([0, 0], 0.0), ([1, 1], None)):
        got = cb().preference_loss(y, dev(np.array(t0)), 1, beta=10.0)
        assert torch.isfinite(got.grad).all() and torch.isfinite(got.loss)
        if want_loss is not None:
            assert got.loss.item() == want_loss


@pytest.mark.parametrize("kind", list(KIND))
def test_gradient_in_place_and_into_views(kind):
    rng = np.random.default_rng(4)
    for rows, v in ((5, 1003), (3, 40000)):
        x, hx = make(rng, rows, v, kind)
        t, up = dev(rng.integers(0, v, rows)), dev(rng.normal(size=rows), torch.float32)
        r = cb().token_logprobs(x, t)
        want = cb().token_logprobs_backward(up, x, t, r.logprobs, r.lse)
        y = x.clone()
        assert cb().token_logprobs_backward(up, y, t, r.logprobs, r.lse, out=y) is y
        assert torch.equal(y, want)
        old, adv = r.logprobs.float() - 0.05, up
        want = cb().policy_loss(x, t, old, adv).grad
        for how in LAYOUTS:
            y = layouts(x.clone(), how)
            assert cb().policy_loss(y, t, old, adv, out_grad=y).grad is y
            # another layout may take another kernel, with sums in another order
            assert (y.double() - want.double()).abs().max() <= 4 * torch.finfo(x.dtype).eps * want.abs().max()
        index = torch.stack([torch.randperm(v, device="cuda")[:9] for _ in range(rows)])
        teacher = x.gather(1, index).float() + 0.5
        lse = teacher.logsumexp(1) + 0.2
        want = cb().distill_loss(x, teacher, index, lse).grad
        y = x.clone()
        cb().distill_loss(y, teacher, index, lse, out_grad=y)
        assert torch.equal(y, want)
        if rows % 2:
            continue
    x, _ = make(rng, 4, 1003, kind)
    t = dev(rng.integers(0, 1003, 4))
    want = cb().preference_loss(x, t, 1).grad
    y = x.clone()
    cb().preference_loss(y, t, 1, out_grad=y)
    assert torch.equal(y, want)
    # what lies between the rows of a view stays as it was
    for how, rest in (("pitched", lambda w, v: w[:, v:]), ):
        w = torch.full((4, 1024), 7.0, dtype=x.dtype, device="cuda")
        cb().preference_loss(x, t, 1, out_grad=w[:, :1003])
        assert (rest(w, 1003) == 7).all()
        assert (w[:, :1003].double() - want.double()).abs().max() <= 4 * torch.finfo(x.dtype).eps * want.abs().max()
    w = torch.full((5 * 1003 + 8,), 7.0, dtype=x.dtype, device="cuda")
    for off in (0, 1, 3):
        w.fill_(7.0)
        view = w[off:off + 4 * 1003].view(4, 1003)
        cb().preference_loss(x, t, 1, out_grad=view)
        assert (w[:off] == 7).all() and (w[off + 4 * 1003:] == 7).all()
        assert (view.double() - want.double()).abs().max() <= 4 * torch.finfo(x.dtype).eps * want.abs().max()
    with pytest.raises(cb().AliasError):
        cb().preference_loss(w[:4 * 1003].view(4, 1003), t, 1, out_grad=w[1:1 + 4 * 1003].view(4, 1003))
    with pytest.raises(cb().DTypeError):
        cb().preference_loss(x, t, 1, out_grad=torch.empty(4, 1003, dtype=torch.int32, device="cuda"))
    with pytest.raises(cb().ShapeError):
        cb().preference_loss(x, t, 1, out_grad=torch.empty(4, 1002, dtype=x.dtype, device="cuda"))


def test_float64_gradient_against_differences_of_the_kernel():
    rng = np.random.default_rng(8)
    n, v, h = 4, 11, 1e-5
    x = dev(rng.normal(size=(n, v)), torch.float64)
    t = dev(rng.integers(0, v, n))
    logp = cb().token_logprobs(x, t).logprobs
    old, adv = (logp + 0.07).float(), dev(rng.normal(size=n), torch.float32)
    index = dev(np.stack([rng.permutation(v)[:4] for _ in range(n)]))
    teacher = dev(rng.normal(size=(n, 4)), torch.float64)
    calls = {
        "policy": lambda y: cb().policy_loss(y, t, old, adv, old, kl_coef=0.3, temperature=1.3),
        "distill": lambda y: cb().distill_loss(y, teacher, index, temperature=1.3),
        "tail": lambda y: cb().distill_loss(y, teacher, index, teacher.logsumexp(1) + 0.4),
        "preference": lambda y: cb().preference_loss(y, t, 2, beta=0.5, label_smoothing=0.1, average=True),
    }
    for name, f in calls.items():
        got = f(x).grad
        for i in range(n):
            for j in range(v):
                a, b = x.clone(), x.clone()
                a[i, j] += h
                b[i, j] -= h
                d = (f(a).loss.item() - f(b).loss.item()) / (2 * h)
                assert abs(d - got[i, j].item()) < 1e-9, (name, i, j)


def test_empty_calls():
    x = torch.empty(0, 16, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    z = torch.empty(0, device="cuda")
    assert cb().token_logprobs(x, t).logprobs.shape == (0,)
    assert cb().token_logprobs_backward(z, x, t, z, z).shape == (0, 16)
    r = cb().policy_loss(x, t, z, z)
    assert r.loss.item() == 0.0 and r.grad.shape == (0, 16)
    r = cb().distill_loss(x, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int64, device="cuda"))
    assert r.loss.item() == 0.0
    r = cb().preference_loss(x, t, 2)  # empty sequences: h = 0
    assert abs(r.loss.item() - np.log(2)) < 1e-7
    x = torch.empty(2, 0, 16, device="cuda")
    assert cb().token_logprobs(x, torch.empty(2, 0, dtype=torch.int64, device="cuda")).lse.shape == (2, 0)
    with pytest.raises(cb().ShapeError):
        cb().token_logprobs(torch.empty(3, 0, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"))


def _step(x, t, ref, teacher, index, mask, pairs, grads):
    """The losses as a training program would run them after one another: a reference's log-probabilities
    into the preference and policy losses, and the teacher's entries."""
    c = cb()
    r = c.token_logprobs(ref, t, mask)
    a = c.preference_loss(x, t, pairs, r.logprobs, mask, out_grad=grads[0])
    b = c.policy_loss(x, t, a.logprobs - 0.05, r.logprobs, r.logprobs, mask, kl_coef=0.1, out_grad=grads[1])
    d = c.distill_loss(x, teacher, index, weights=mask, out_grad=grads[2])
    e = c.token_logprobs_backward(r.logprobs, ref, t, r.logprobs, r.lse, mask, out=grads[3])
    return [a.loss, a.rewards, a.grad, b.loss, b.kl, b.grad, d.loss, d.row_loss, d.grad, e]


def _inputs(seed, rows, v, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x, ref = (torch.randn(rows, v, generator=g, device="cuda").to(dtype) for _ in range(2))
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    index = torch.arange(8, device="cuda") * (v // 8) + torch.randint(v // 8, (rows, 8), generator=g, device="cuda")
    teacher = torch.randn(rows, 8, generator=g, device="cuda")
    mask = torch.rand(rows, generator=g, device="cuda") < 0.8
    return [x, t, ref, teacher, index, mask]


@pytest.mark.parametrize("rows,v,dtype", [(8, 1003, torch.float32), (512, 32768, torch.bfloat16), (8, 131072, torch.bfloat16)])
def test_run_together_repeated_on_streams_and_captured(rows, v, dtype):
    ins = [_inputs(s, rows, v, dtype) for s in (1, 2)]
    new = lambda: [torch.empty(rows, v, dtype=dtype, device="cuda") for _ in range(4)]
    want = [[o.clone() for o in _step(*i, pairs=2, grads=new())] for i in ins]
    for w, i in zip(want, ins):  # equal calls, equal bits
        for a, b in zip(w, _step(*i, pairs=2, grads=new())):
            assert torch.equal(a, b)
    # two streams at once, each on its own inputs
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = _step(*ins[k], pairs=2, grads=new())
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))
    # captured once, replayed on other inputs in the same buffers
    static = [t.clone() for t in ins[0]]
    grads = new()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*static, pairs=2, grads=grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*static, pairs=2, grads=grads)
    for k in (1, 0, 1):
        for s, t in zip(static, ins[k]):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[k], out))


@pytest.mark.parametrize("v,dtype", [(50021, torch.float32), (32768, torch.float32), (100003, torch.bfloat16)])
def test_every_element_of_many_rows(v, dtype):
    """Enough rows for every stage of the kernels' rings to be refilled many times: every gradient element
    against float64, so that one pack read from the wrong copy shows. A pack of another row is off by a
    factor; the bound is 2^-15 of each element (64 roundings of float32 and more, see losses_oracle), and half a
    step of bfloat16."""
    every_element(2000, v, dtype)


@pytest.mark.parametrize("rows,v,dtype", [(2100, 20001, torch.bfloat16), (2200, 9003, torch.float32), (20000, 1003, torch.float32),
                                          (20000, 2048, torch.bfloat16), (50000, 130, torch.bfloat16), (6000, 8192, torch.bfloat16)])
def test_every_element_of_rows_that_a_warp_takes_whole(rows, v, dtype):
    every_element(rows, v, dtype)


def every_element(rows, v, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    x = (2 * torch.randn(rows, v, generator=g, device="cuda")).to(dtype)
    t = torch.randint(v, (rows,), generator=g, device="cuda")
    up = torch.ones(rows, device="cuda")
    r = cb().token_logprobs(x, t)
    pull = cb().token_logprobs_backward(up, x, t, r.logprobs, r.lse)
    old = r.logprobs.clone()
    held = cb().policy_loss(x, t, old, -up, weights=up).grad  # ratio r = 1, A = -1: loss r, gradient r (1[t] - p)
    index = (torch.arange(4, device="cuda") * (v // 4)).expand(rows, 4)
    top = cb().distill_loss(x, torch.zeros(rows, 4, device="cuda"), index, weights=up).grad
    half = 2.0 ** -9 if dtype == torch.bfloat16 else 0.0
    for i in range(0, rows, 200):
        b = slice(i, i + 200)
        p = torch.softmax(x[b].double(), -1)
        want = -p
        want.scatter_add_(1, t[b, None], torch.ones(len(want), 1, dtype=torch.float64, device="cuda"))
        bound = (2.0 ** -15 + 2 * half) * want.abs() + 1e-30
        assert ((pull[b].double() - want).abs() <= bound).all()
        assert ((held[b].double() - want).abs() <= bound).all()
        p[:, index[0]] -= 0.25
        bound = (2.0 ** -15 + 2 * half) * p.abs() + 1e-30
        bound[:, index[0]] += 2.0 ** -20
        assert ((top[b].double() - p).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_rows_that_count(dtype):
    """Long runs of rows that do not count between a few that do, more rows than the kernels' clusters times the rows
    whose operands they read together."""
    rows, v = 40000, 700
    x = torch.randn(rows, v, device="cuda").to(dtype)
    t = torch.randint(v, (rows,), device="cuda")
    old, adv = torch.full((rows,), -6.0, device="cuda"), torch.ones(rows, device="cuda")
    index = torch.randint(v // 4, (rows, 4), device="cuda") + torch.arange(4, device="cuda") * (v // 4)
    teacher = torch.randn(rows, 4, device="cuda")
    full = [cb().policy_loss(x, t, old, adv, weights=torch.ones(rows, device="cuda")),
            cb().distill_loss(x, teacher, index, weights=torch.ones(rows, device="cuda"))]
    for share in (0.0, 0.0005, 0.01, 0.3):
        on = torch.rand(rows, device="cuda") < share
        some = [cb().policy_loss(x, t, old, adv, weights=on), cb().distill_loss(x, teacher, index, weights=on)]
        for f, s in zip(full, some):
            assert torch.equal(s.grad, torch.where(on[:, None], f.grad, torch.zeros_like(f.grad)))
            assert torch.equal(s.row_loss, torch.where(on, f.row_loss, torch.zeros_like(f.row_loss)))
        assert torch.equal(cb().token_logprobs(x, t, on).logprobs,
                           torch.where(on, cb().token_logprobs(x, t).logprobs, torch.zeros((), device="cuda")))
    import ctorch_b200._capi as C
    assert C.wait_timeouts() == 0


@pytest.mark.parametrize("v,dtype", [(5001, torch.float32), (9001, torch.bfloat16)])
def test_few_long_rows_that_count(v, dtype):
    """The same for the log-probabilities of rows that no warp takes whole (5000 of them leave its last wave empty)."""
    rows = 5000
    x = torch.randn(rows, v, device="cuda").to(dtype)
    t, up = torch.randint(v, (rows,), device="cuda"), torch.randn(rows, device="cuda")
    full = cb().token_logprobs(x, t)
    grad = cb().token_logprobs_backward(up, x, t, full.logprobs, full.lse)
    for share in (0.0, 0.0005, 0.01, 0.3):
        on = torch.rand(rows, device="cuda") < share
        r = cb().token_logprobs(x, t, on)
        assert torch.equal(r.logprobs, torch.where(on, full.logprobs, torch.zeros((), device="cuda")))
        g = cb().token_logprobs_backward(up, x, t, r.logprobs, r.lse, on)
        assert torch.equal(g, torch.where(on[:, None], grad, torch.zeros_like(grad)))
    import ctorch_b200._capi as C
    assert C.wait_timeouts() == 0


def test_new_gradients_lie_like_the_logits():
    """A gradient that the call makes has the logits' rows' alignment where that wastes little."""
    w = torch.randn(4, 9, 1001, device="cuda").bfloat16()
    for k, x in enumerate((w[:, :-1], w[1:], w.flatten(0, 1)[1:], w[..., :1000], w[:, ::3], w[:1].expand(4, 9, 1001))):
        t = torch.randint(1000, x.shape[:-1], device="cuda")
        z = torch.zeros(t.shape, device="cuda")
        g = cb().policy_loss(x, t, z, z + 1).grad
        want = cb().policy_loss(x.contiguous(), t, z, z + 1).grad
        # sums of float32 in another order (2^-14 and less apart) may round to neighbouring bfloat16: one step, 2^-7
        assert g.shape == x.shape and ((g.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs()).all()
        if k < 4:  # the others leave most of their memory unused, or broadcast
            assert all((g[i].data_ptr() - x[i].data_ptr()) % 16 == 0 for i in range(len(x)))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("v", [2000, 10824, 32768])
@pytest.mark.parametrize("temperature", [0.8, 1.0, 2.0])
def test_log_probabilities_are_not_off_to_one_side(temperature, v, kind):
    """The mean error over many rows, which a sequence's sum adds up. The hardware's 2^t is corrected by 5.0e-8, its
    mean; over [-1, 0] alone that is 2.1e-8 too much. Roundings average out: of a row's error (1.5e-7) the mean of 4000
    keeps 2.4e-9, three times which is 7e-9."""
    rows = 4000
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    x = 2 * torch.randn(rows, v, generator=g, device="cuda")
    x.scatter_add_(1, torch.randint(v, (rows, 3), generator=g, device="cuda"), 9 + 3 * torch.rand(rows, 3, generator=g, device="cuda"))
    x = x.to(KIND[kind])
    t = x.argmax(1)
    z = torch.cat([x[i:i + 500].double() / temperature for i in range(0, rows, 500)])
    want = torch.log_softmax(z, -1).gather(1, t[:, None])[:, 0]
    old = want.float()
    for got in (cb().token_logprobs(x, t, temperature=temperature).logprobs,
                cb().policy_loss(x, t, old, old, temperature=temperature).logprobs):
        assert abs((got.double() - want).mean().item()) < 2.9e-8


def test_rows_far_apart():
    """Row offsets beyond 2^31 elements."""
    v, step = 1000, (1 << 31) // 2 + 8
    big = torch.empty(3 * step, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((4, v), (step - 1000, 1))
    y = torch.randn(4, v, device="cuda").to(torch.bfloat16)
    x.copy_(y)
    t = torch.tensor([1, 2, 3, 999], device="cuda")
    assert torch.equal(cb().token_logprobs(x, t).logprobs, cb().token_logprobs(y, t).logprobs)
    old, adv = torch.zeros(4, device="cuda") - 7, torch.ones(4, device="cuda")
    want = cb().policy_loss(y, t, old, adv).grad
    cb().policy_loss(x, t, old, adv, out_grad=x)
    assert torch.equal(x, want)
