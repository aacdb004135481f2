"""GPU checks of what stands around the losses (the norm and its backward pass, the projection with its cross entropy, the
balance loss) against 64 bits (tests/model_oracle.py), within the bounds derived there."""
import math

import pytest
import torch

import model_oracle as O

pytestmark = pytest.mark.gpu

KIND = {"f32": torch.float32, "bf16": torch.bfloat16}
NAN = float("nan")


def cb():
    import ctorch_b200

    return ctorch_b200


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * std).to(dtype)


def near(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN positions differ"
    off = (got - value).abs() - bound
    off = torch.where(torch.isnan(value), -1.0, off)
    if off.numel() and off.max() > 0:
        k = int(off.argmax())
        at = torch.broadcast_to(torch.as_tensor(bound, device=value.device), value.shape).reshape(-1)[k]
        raise AssertionError(f"{what}: {float(got.reshape(-1)[k])!r} for {float(value.reshape(-1)[k])!r}, allowed {float(at):.3g}")


def layout(x, how):
    """The same [rows, columns] values in other memory."""
    n, v = x.shape
    if how == "contiguous":
        return x.contiguous()
    if how == "pitched":  # 16-byte rows with a gap that holds NaN
        w = torch.full((n, (v + 15) // 8 * 8 + 8), NAN, dtype=x.dtype, device=x.device)
        w[:, :v] = x
        return w[:, :v]
    if how == "offset":  # rows that start anywhere
        w = torch.full((n * (v + 3) + 5,), NAN, dtype=x.dtype, device=x.device)
        y = w[5:].view(n, v + 3)[:, 1:v + 1]
        y.copy_(x)
        return y
    if how == "columns":
        return x.t().contiguous().t()
    raise ValueError(how)


LAYOUTS = ["contiguous", "pitched", "offset", "columns"]

# ------------------------------------------------------------------------------------- norm

NORM_SHAPES = [(1, 1), (3, 2), (2, 7), (5, 100), (4, 128), (33, 129), (3, 640), (700, 64), (300, 1000), (5, 4096), (2, 5003), (3, 8192),
               (2, 16384), (3, 20008), (2, 40001)]


def check_norm(r, x, res, w, eps, quant, type_):
    s = x if res is None else r.summed
    if res is not None:
        exact = x.double() + res.double()
        # the sum in float32, then in its type: half a step, and what the first rounding may move
        near(r.summed, (exact, exact.abs() * (O.half(type_) + 2 * O.U)), "summed")
    y, rstd, bound = O.norm(s, None, w, eps)
    near(r.rstd, (rstd[..., 0], rstd[..., 0] * ((x.shape[-1] / 32 + 8) / 2 + 6) * O.U), "rstd")
    if quant is None:
        near(r.out, (y, bound + O.half(type_) * y.abs() + 1e-38), "out")
        return
    one, scale = O.scales(y, quant)
    c = (bound / y.abs().clamp_min(1e-300)).max().item() + 2 * O.U
    near(r.scales, (one[..., 0] if quant == "row" else one, (one[..., 0] if quant == "row" else one) * c), "scales")
    assert r.out.dtype == torch.float8_e4m3fn
    # half a step of e4m3 (2^-4; 2^-10 below its normal numbers), of a value off by its own bound and two roundings
    near(r.out.float().double() * scale, (y, y.abs() * (2.0 ** -4 + 4 * c) + scale * (2.0 ** -10 + 1e-6)), "out")


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("quant", [None, "row", "block"])
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm(rows, dim, kind, quant, how):
    g, t = gen(rows * dim), KIND[kind]
    x, res = layout(normal(g, rows, dim, dtype=t), how), layout(normal(g, rows, dim, std=2.0, dtype=t), how)
    w = (1 + 0.3 * normal(g, dim)).to(t if rows % 2 else torch.float32)
    check_norm(cb().rms_norm(x, w, residual=res, quant=quant), x, res, w, 1e-6, quant, t)
    plain = cb().rms_norm(x, w, eps=1e-3, quant=quant)
    assert plain.summed is x
    check_norm(plain, x, None, w, 1e-3, quant, t)


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm_backward(rows, dim, how, kind):
    g, t = gen(rows + dim), KIND[kind]
    x, up, passed = (layout(normal(g, rows, dim, dtype=t), how) for _ in range(3))
    w = (1 + 0.3 * normal(g, dim)).to(t if rows % 2 else torch.float32)
    f = cb().rms_norm(x, w, eps=1e-5)
    for extra in (None, passed):
        r = cb().rms_norm_backward(up, x, w, f.rstd, grad_summed=extra)
        gx, bx, gw, bw = O.norm_grad(up, x, w, 1e-5, extra)
        near(r.grad_x, (gx, bx + O.half(t) * gx.abs() + 1e-38), "grad_x")
        near(r.grad_weight, (gw, bw + O.half(w.dtype) * gw.abs() + 1e-38), "grad_weight")
        assert r.grad_weight.dtype == w.dtype


def test_norm_gradient_against_differences():
    g = gen(5)
    x, w, up = normal(g, 3, 24, dtype=torch.float64), 1 + 0.2 * normal(g, 24, dtype=torch.float64), normal(g, 3, 24, dtype=torch.float64)
    f = lambda y, v: (O.norm(y, None, v, 1e-3)[0] * up).sum()
    gx, _, gw, _ = O.norm_grad(up, x, w, 1e-3, None)
    for at, grad, call in ((x, gx, lambda y: f(y, w)), (w, gw, lambda v: f(x, v))):
        for k in range(0, at.numel(), 5):
            step = torch.zeros_like(at).view(-1)
            step[k] = 1e-5
            step = step.view(at.shape)
            # h^2 / 6 of a third derivative below 100, and 1e-15 / h of rounding
            assert abs((call(at + step) - call(at - step)) / 2e-5 - grad.reshape(-1)[k]) < 1e-8


@pytest.mark.parametrize("rows,dim", [(64, 1024), (3, 5003)])
@pytest.mark.parametrize("kind", list(KIND))
def test_norm_in_place_and_extremes(kind, rows, dim):
    g, t = gen(11), KIND[kind]
    x, res, w = normal(g, rows, dim, dtype=t), normal(g, rows, dim, dtype=t), normal(g, dim, dtype=t)
    w[0] = 0.0
    want = cb().rms_norm(x, w, residual=res)
    x2, res2 = x.clone(), res.clone()
    r = cb().rms_norm(x2, w, residual=res2, out_summed=res2)
    assert r.summed is res2 and torch.equal(r.out, want.out) and torch.equal(res2, want.summed) and torch.equal(x2, x)
    r = cb().rms_norm(x2, w, residual=res, out=x2)
    assert torch.equal(x2, want.out) and torch.equal(r.summed, want.summed)
    up, passed = normal(g, rows, dim, dtype=t), normal(g, rows, dim, dtype=t)
    want_b = cb().rms_norm_backward(up, want.summed, w, want.rstd, grad_summed=passed)
    for k in range(3):
        a = [up.clone(), want.summed.clone(), passed.clone()]
        b = cb().rms_norm_backward(a[0], a[1], w, want.rstd, grad_summed=a[2], out=a[k])
        assert torch.equal(a[k], want_b.grad_x) and torch.equal(b.grad_weight, want_b.grad_weight)
    # a row of zeros, one with NaN, one with an infinity; the others are as before
    y = x.clone()
    y[0], y[1, 2], y[2, 3] = 0.0, NAN, float("inf")
    r, before = cb().rms_norm(y, w), cb().rms_norm(x, w)
    assert (r.out[0] == 0).all() and torch.isnan(r.out[1]).all()
    assert torch.isnan(r.out[2, 3]) and (r.out[2].nan_to_num() == 0).all()  # 1 / inf of all but inf / inf
    assert torch.equal(r.out[3:], before.out[3:])
    for quant in ("row", "block"):
        q = cb().rms_norm(y, w, quant=quant)
        assert (q.scales[0] == 1).all() and (q.out[0].float() == 0).all() and torch.isnan(q.out[1].float()).all()


def test_norm_leading_dims_and_nothing():
    g = gen(3)
    big = normal(g, 3, 4, 5, 100)
    x = big.transpose(0, 1)[:, :, ::2]
    w = normal(g, 100)
    check_norm(cb().rms_norm(x, w, residual=x), x, x, w, 1e-6, None, torch.float32)
    q = cb().rms_norm(x, w, quant="block")
    assert q.scales.shape == (4, 3, 3, 1)
    r = cb().rms_norm(x[:0], w, residual=x[:0])
    assert r.out.shape == (0, 3, 3, 100)
    b = cb().rms_norm_backward(x[:0], x[:0], w, r.rstd)
    assert (b.grad_weight == 0).all()


def test_norm_many_rows_are_repeatable():
    g = gen(8)
    x, up, w = normal(g, 20000, 257, dtype=torch.bfloat16), normal(g, 20000, 257, dtype=torch.bfloat16), normal(g, 257)
    f = cb().rms_norm(x, w)
    a, b = (cb().rms_norm_backward(up, x, w, f.rstd) for _ in range(2))
    assert torch.equal(a.grad_x, b.grad_x) and torch.equal(a.grad_weight, b.grad_weight)
    gx, bx, gw, bw = O.norm_grad(up, x, w, 1e-6, None)
    near(a.grad_weight, (gw, bw + O.half(w.dtype) * gw.abs()), "grad_weight")


# ------------------------------------------------------------------------------------- head


def head_inputs(g, rows, dim, vocab, kind, how="contiguous"):
    t = KIND[kind]
    w = layout(normal(g, vocab, dim, std=2 / math.sqrt(dim), dtype=t), how)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    lean = 3 * torch.rand(rows, 1, generator=g, device="cuda", dtype=torch.float64)
    h = layout((normal(g, rows, dim, dtype=torch.float64) + lean * w[targets].double()).to(t), how)
    return h, w, targets


def check_head(r, want, kind):
    for k in (k for k in want if not k.startswith("unit") and k != "alike"):
        near(getattr(r, k), want[k], k)
    # and as a whole: a gradient's rounding and that of the logits' gradients before it are 2^-8 / sqrt 3 / 1.47 = 0.0015
    # each on average; float32 sums of up to some thousand terms err by a few times 2^-24 of their terms' root. A row's
    # sum of exponentials is a float32 of at least 1, so p - 1 of a target errs by 2^-24 and more however small it is:
    # 2^-22 of the terms that a p - 1 of 1 would give is allowed beside
    for k in ("grad_hidden", "grad_weight"):
        if k in want:
            value, unit = want[k][0], want["unit_" + k]
            off = float((getattr(r, k).double() - value).norm())
            each = 3e-3 * want["alike"] ** 0.5 if kind == "bf16" else 4e-6
            assert off <= each * float(value.norm()) + 2.0 ** -22 * unit, k


HEAD_SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (2, 64, 256), (64, 64, 300), (129, 100, 257), (128, 72, 1000), (255, 130, 511),
               (257, 256, 2049), (300, 40, 5003), (1, 512, 32768), (17, 1024, 10007), (520, 328, 777), (1000, 64, 513)]


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim,vocab", HEAD_SHAPES)
def test_head(rows, dim, vocab, kind):
    g = gen(rows * dim + vocab)
    h, w, t = head_inputs(g, rows, dim, vocab, kind)
    r = cb().linear_cross_entropy(h, w, t)
    check_head(r, O.head(h, w, t, None), kind)
    only = cb().linear_cross_entropy(h, w, t, grad=False)
    assert only.grad_hidden is None and only.grad_weight is None
    assert torch.equal(only.row_loss, r.row_loss) and torch.equal(only.lse, r.lse) and torch.equal(only.loss, r.loss)
    keep = (torch.rand(rows, generator=g, device="cuda") < 0.6).float()
    keep[0] = 1
    share = keep / keep.sum()
    h2 = torch.where(keep[:, None] != 0, h, NAN).to(h.dtype)  # what does not count may hold anything
    t2 = torch.where(keep != 0, t, -1)
    check_head(cb().linear_cross_entropy(h2, w, t2, weights=share, z_coef=0.01, temperature=1.3),
               O.head(h, w, t, share, 0.01, 1.3), kind)


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim,vocab", [(70, 96, 515), (300, 33, 1030)])
def test_head_layouts(rows, dim, vocab, kind, how):
    g = gen(rows)
    h, w, t = head_inputs(g, rows, dim, vocab, kind, how)
    want = O.head(h, w, t, None)
    check_head(cb().linear_cross_entropy(h, w, t.int()), want, kind)
    gh, gw = layout(torch.zeros_like(h), how), layout(torch.zeros_like(w), how)
    share = torch.rand(rows, generator=g, device="cuda")
    r = cb().linear_cross_entropy(h, w, t, weights=share, out_grad_hidden=gh, out_grad_weight=gw)
    assert r.grad_hidden is gh and r.grad_weight is gw
    check_head(r, O.head(h, w, t, share), kind)


@pytest.mark.parametrize("kind", list(KIND))
def test_head_leading_dims(kind):
    g = gen(2)
    h, w, t = head_inputs(g, 60, 48, 301, kind)
    x, tt = h.view(3, 20, 48), t.view(3, 20)
    mask = torch.rand(3, 20, generator=g, device="cuda") < 0.5
    mask[0, 0] = True
    whole = cb().linear_cross_entropy(x, w, tt, weights=mask)
    check_head(whole, O.head(x, w, tt, mask), kind)
    # every other position of a batch laid out positions first
    y = x.transpose(0, 1).contiguous().transpose(0, 1)[:, ::2]
    check_head(cb().linear_cross_entropy(y, w, tt[:, ::2]), O.head(y, w, tt[:, ::2], None), kind)
    row = torch.rand(3, 1, generator=g, device="cuda", dtype=torch.float64)
    check_head(cb().linear_cross_entropy(x, w, tt, weights=row), O.head(x, w, tt, row), kind)
    # one hidden state for many targets
    z = x[:, :1].expand(3, 20, 48)
    check_head(cb().linear_cross_entropy(z, w, tt), O.head(z, w, tt, None, alike=20), kind)


@pytest.mark.parametrize("kind", list(KIND))
def test_head_without_rows_or_without_counted_ones(kind):
    g = gen(4)
    h, w, t = head_inputs(g, 40, 64, 300, kind)
    empty = cb().linear_cross_entropy(h[:0], w, t[:0])
    assert float(empty.loss) == 0 and empty.grad_hidden.shape == (0, 64) and (empty.grad_weight == 0).all()
    h[:] = NAN
    none = cb().linear_cross_entropy(h, w, t, weights=torch.zeros(40, device="cuda"))
    assert float(none.loss) == 0 and (none.row_loss == 0).all() and (none.lse == 0).all()
    assert (none.grad_hidden == 0).all() and (none.grad_weight == 0).all()


@pytest.mark.parametrize("kind", list(KIND))
def test_head_bad_targets_and_values(kind):
    g = gen(6)
    h, w, t = head_inputs(g, 50, 64, 300, kind)
    good = cb().linear_cross_entropy(h, w, t)
    bad = t.clone()
    bad[7] = 300
    status = cb().index_status()
    r = cb().linear_cross_entropy(h, w, bad, status=status)
    others = torch.arange(50, device="cuda") != 7
    for a, b in ((r.row_loss, good.row_loss), (r.lse, good.lse), (r.grad_hidden, good.grad_hidden)):
        assert torch.isnan(a[7]).all() and torch.equal(a[others], b[others])
    assert torch.isnan(r.loss) and torch.isnan(r.grad_weight).all()
    with pytest.raises(cb().ShapeError, match="300"):
        cb().check_index_status(status)
    x = h.clone()
    x[3, 5] = NAN
    r = cb().linear_cross_entropy(x, w, t)
    others = torch.arange(50, device="cuda") != 3
    assert torch.isnan(r.row_loss[3]) and torch.equal(r.row_loss[others], good.row_loss[others])
    assert torch.isnan(r.grad_hidden[3]).all() and torch.equal(r.grad_hidden[others], good.grad_hidden[others])
    # logits far apart: the likeliest one has all of the mass, and a far target its whole distance
    far = (40 * h.float()).to(h.dtype)
    check_head(cb().linear_cross_entropy(far, w, t), O.head(far, w, t, None), kind)


@pytest.mark.parametrize("kind", list(KIND))
def test_head_weights_of_any_size(kind):
    """float64 weights far below float32's numbers count, and add nothing that a float32 could hold."""
    g = gen(14)
    h, w, t = head_inputs(g, 90, 64, 301, kind)
    tiny = torch.full((90,), 1e-50, dtype=torch.float64, device="cuda")
    r = cb().linear_cross_entropy(h, w, t, weights=tiny)
    assert float(r.loss) == 0 and (r.grad_hidden == 0).all() and (r.grad_weight == 0).all() and torch.isfinite(r.row_loss).all()
    tiny[::3] = 0.5
    check_head(cb().linear_cross_entropy(h, w, t, weights=tiny), O.head(h, w, t, tiny), kind)
    signs = torch.where(torch.arange(90, device="cuda") % 2 == 0, 1.0, -0.25)
    check_head(cb().linear_cross_entropy(h, w, t, weights=signs), O.head(h, w, t, signs), kind)


@pytest.mark.parametrize("kind", list(KIND))
def test_a_single_row_without_leading_dims(kind):
    g = gen(15)
    h, w, t = head_inputs(g, 1, 72, 301, kind)
    r = cb().linear_cross_entropy(h[0], w, t[0])
    assert r.row_loss.shape == () and r.grad_hidden.shape == (72,)
    check_head(r, O.head(h[0], w, t[0], None), kind)
    for quant in (None, "row", "block"):
        n = cb().rms_norm(h[0], w[0], residual=w[1], quant=quant)
        assert n.rstd.shape == () and n.out.shape == (72,)
        check_norm(n, h[0], w[1], w[0], 1e-6, quant, KIND[kind])
    one = cb().balance_loss(h[0], torch.tensor([3, 5], device="cuda"))
    check_balance(one, O.balance(h, torch.tensor([[3, 5]], device="cuda"), None, 1, 0.01, 0.0) | {"grad": tuple(
        v[0] for v in O.balance(h, torch.tensor([[3, 5]], device="cuda"), None, 1, 0.01, 0.0)["grad"])})


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim", [(2000, 255), (700, 1001), (300, 4093), (40, 8191), (30, 16383)])
def test_norm_every_row_of_odd_ones(rows, dim, kind):
    """Rows that start anywhere, many to a group of threads, next to rows of NaN: packs of memory that two rows share."""
    g, t = gen(rows), KIND[kind]
    x, res, up, passed = (normal(g, rows, dim, dtype=t) for _ in range(4))
    w = (1 + 0.3 * normal(g, dim)).to(t)
    x[5::7] = NAN
    fine = ~torch.isnan(x[:, 0])
    for quant in (None, "row", "block"):
        r = cb().rms_norm(x, w, residual=res, quant=quant)
        assert torch.isnan(r.out[~fine].float()).all() and torch.isnan(r.rstd[~fine]).all()
        check_norm(type(r)(r.out[fine], r.summed[fine], r.rstd[fine], None if quant is None else r.scales[fine]), x[fine], res[fine], w,
                   1e-6, quant, t)
    x = torch.where(fine[:, None], x, 1.0).to(t)
    f = cb().rms_norm(x, w)
    b = cb().rms_norm_backward(up, x, w, f.rstd, grad_summed=passed)
    gx, bx, gw, bw = O.norm_grad(up, x, w, 1e-6, passed)
    near(b.grad_x, (gx, bx + O.half(t) * gx.abs() + 1e-38), "grad_x")
    near(b.grad_weight, (gw, bw + O.half(w.dtype) * gw.abs() + 1e-38), "grad_weight")


def test_head_against_differences():
    g = gen(9)
    h, w, t = normal(g, 5, 6, dtype=torch.float64), normal(g, 11, 6, dtype=torch.float64), torch.tensor([0, 10, 3, 3, 7], device="cuda")
    share = torch.tensor([0.3, 0.0, 1.0, -0.5, 0.2], device="cuda", dtype=torch.float64)
    want = O.head(h, w, t, share, 0.02, 1.4)
    for at, name, call in ((h, "grad_hidden", lambda y: O.head(y, w, t, share, 0.02, 1.4, False)["loss"][0]),
                           (w, "grad_weight", lambda y: O.head(h, y, t, share, 0.02, 1.4, False)["loss"][0])):
        for k in range(at.numel()):
            step = torch.zeros_like(at).view(-1)
            step[k] = 1e-5
            step = step.view(at.shape)
            assert abs((call(at + step) - call(at - step)) / 2e-5 - want[name][0].reshape(-1)[k]) < 1e-8


@pytest.mark.parametrize("kind", list(KIND))
def test_head_blocks_of_rows(kind):
    """More rows than one block holds: gradients of the weight add up over the blocks."""
    g = gen(12)
    vocab, rows = (1 << 21, 600) if kind == "bf16" else (1 << 20, 700)
    h, w, t = head_inputs(g, rows, 8, vocab, kind)
    keep = torch.rand(rows, generator=g, device="cuda") < 0.95
    keep[0] = True
    for weights in (None, keep.float() / keep.sum(), (torch.arange(rows, device="cuda") < 200).float()):
        r = cb().linear_cross_entropy(h, w, t, weights=weights)
        parts = [O.head(h[i:i + 100], w, t[i:i + 100], torch.full((min(100, rows - i),), 1 / rows, device="cuda", dtype=torch.float64)
                        if weights is None else weights[i:i + 100]) for i in range(0, rows, 100)]
        near(r.row_loss, tuple(torch.cat([p["row_loss"][k] for p in parts]) for k in (0, 1)), "row_loss")
        near(r.grad_hidden, tuple(torch.cat([p["grad_hidden"][k] for p in parts]) for k in (0, 1)), "grad_hidden")
        value, bound = (sum(p["grad_weight"][k] for p in parts) for k in (0, 1))
        near(r.grad_weight, (value, bound), "grad_weight")


def test_head_is_repeatable():
    g = gen(13)
    h, w, t = head_inputs(g, 1500, 512, 20001, "bf16")
    share = torch.rand(1500, generator=g, device="cuda")
    a = cb().linear_cross_entropy(h, w, t, weights=share)
    for _ in range(3):
        b = cb().linear_cross_entropy(h, w, t, weights=share)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------- balance


def balance_inputs(g, rows, experts, k, t):
    x = normal(g, rows, experts, dtype=t)
    return x, torch.topk(x.float(), k, dim=-1).indices


def check_balance(r, want):
    assert torch.equal(r.counts, want["counts"][0])
    for name in ("loss", "probs", "grad"):
        near(getattr(r, name), want[name], name)


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,experts,k,groups", [(1, 1, 1, 1), (3, 2, 1, 3), (64, 8, 2, 1), (60, 7, 7, 4), (1000, 33, 5, 10),
                                                   (5000, 64, 6, 1), (4096, 60, 4, 16), (999, 256, 8, 3), (300, 512, 8, 1),
                                                   (130, 1025, 40, 2), (40, 4096, 3, 1), (100000, 16, 2, 1)])
def test_balance(rows, experts, k, groups, kind):
    g, t = gen(rows + experts), KIND[kind]
    x, chosen = balance_inputs(g, rows, experts, k, t)
    check_balance(cb().balance_loss(x, chosen, groups=groups), O.balance(x, chosen, None, groups, 0.01, 0.0))
    mask = torch.rand(rows, generator=g, device="cuda") < 0.5
    want = O.balance(x, chosen, mask, groups, 0.3, 0.02)
    y = torch.where(mask[:, None], x, NAN).to(t)
    c = torch.where(mask[:, None], chosen, -5).int()
    r = cb().balance_loss(y, c, mask=mask, groups=groups, coef=0.3, z_coef=0.02)
    check_balance(r, want)
    none = cb().balance_loss(y, c, mask=mask, groups=groups, coef=0.3, z_coef=0.02, grad=False)
    assert none.grad is None and torch.equal(none.loss, r.loss) and torch.equal(none.counts, r.counts)
    again = cb().balance_loss(y, c, mask=mask, groups=groups, coef=0.3, z_coef=0.02, out_grad=y)
    assert again.grad is y and torch.equal(y, r.grad)  # in place


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
def test_balance_layouts(kind, how):
    g, t = gen(1), KIND[kind]
    x, chosen = balance_inputs(g, 200, 40, 4, t)
    y = layout(x, how)
    out = layout(torch.zeros_like(x), how)
    r = cb().balance_loss(y, layout(chosen.double(), how).long() if how != "columns" else chosen.t().contiguous().t(), groups=4, out_grad=out)
    check_balance(r, O.balance(x, chosen, None, 4, 0.01, 0.0))
    z = y.view(4, 50, 40) if how == "contiguous" else y.unflatten(0, (4, 50))
    mask = torch.rand(50, generator=g, device="cuda") < 0.7
    r = cb().balance_loss(z, chosen.view(4, 50, 4), mask=mask, groups=4)
    check_balance(r, O.balance(z, chosen.view(4, 50, 4), mask.expand(4, 50), 4, 0.01, 0.0))


def test_balance_extremes():
    g = gen(7)
    x, chosen = balance_inputs(g, 90, 10, 2, torch.float32)
    x[:, 4] = -float("inf")  # an expert that is switched off
    x[5] = torch.finfo(torch.float32).min  # a uniform row
    want = O.balance(x, chosen, None, 3, 0.1, 0.0)
    got = cb().balance_loss(x, chosen, groups=3, coef=0.1)
    assert torch.equal(got.counts, want["counts"][0])
    near(got.probs, want["probs"], "probs")
    assert (got.grad[torch.arange(90) != 5, 4] == 0).all() and torch.isfinite(got.grad).all()
    same = torch.zeros(90, 2, dtype=torch.int64, device="cuda")  # the same expert twice counts twice
    assert cb().balance_loss(x, same).counts[0, 0] == 180
    # an expert that there is none of: its group alone
    chosen[35, 1] = 10
    status = cb().index_status()
    r = cb().balance_loss(x, chosen, groups=3, status=status)
    assert torch.isnan(r.loss) and torch.isnan(r.grad[30:60]).all() and torch.isfinite(r.grad[:30]).all() and torch.isfinite(r.grad[60:]).all()
    assert int(r.counts[1].sum()) == 59
    with pytest.raises(cb().ShapeError, match="10"):
        cb().check_index_status(status)
    mask = torch.ones(90, dtype=torch.bool, device="cuda")
    mask[30:60] = False  # a group without rows
    r = cb().balance_loss(x, chosen, mask=mask, groups=3)
    assert torch.isfinite(r.loss) and (r.counts[1] == 0).all() and (r.probs[1] == 0).all() and (r.grad[30:60] == 0).all()
    e = cb().balance_loss(x[:0], chosen[:0])
    assert float(e.loss) == 0 and (e.counts == 0).all()


def test_balance_gradient_against_differences():
    g = gen(17)
    x = normal(g, 12, 5, dtype=torch.float64)
    chosen = torch.topk(x, 2, dim=-1).indices
    mask = torch.arange(12, device="cuda") % 4 != 1
    f = lambda y: O.balance(y, chosen, mask, 3, 0.4, 0.05)
    want = f(x)["grad"][0]
    for k in range(x.numel()):
        step = torch.zeros_like(x).view(-1)
        step[k] = 1e-5
        step = step.view(x.shape)
        assert abs((f(x + step)["loss"][0] - f(x - step)["loss"][0]) / 2e-5 - want.reshape(-1)[k]) < 1e-8


# ------------------------------------------------------------------------------------- together


def step(h, res, norm_w, w, t, share, router, chosen):
    """The end of a training step: the last norm, the head, its gradients back through the norm, the balance loss."""
    f = cb().rms_norm(h, norm_w, residual=res)
    r = cb().linear_cross_entropy(f.out, w, t, weights=share)
    b = cb().rms_norm_backward(r.grad_hidden, f.summed, norm_w, f.rstd)
    a = cb().balance_loss(router, chosen, mask=share, groups=2)
    return {"loss": r.loss, "total": cb().add(r.loss, a.loss), "grad_x": b.grad_x, "grad_norm": b.grad_weight, "grad_weight": r.grad_weight,
            "grad_router": a.grad}


@pytest.mark.parametrize("kind", list(KIND))
def test_a_step(kind):
    g, t = gen(21), KIND[kind]
    rows, dim, vocab = 384, 256, 3001
    h, res, w = normal(g, rows, dim, dtype=t), normal(g, rows, dim, dtype=t), normal(g, vocab, dim, std=2 / 16, dtype=t)
    norm_w = (1 + 0.2 * normal(g, dim)).to(t)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    keep = (torch.rand(rows, generator=g, device="cuda") < 0.8).float()
    share = keep / keep.sum()
    router, chosen = balance_inputs(g, rows, 16, 2, t)
    args = (h, res, norm_w, w, targets, share, router, chosen)
    got = step(*args)
    # the same by differentiation in 64 bits
    hx, nw, ww = (h.double() + res.double()).requires_grad_(), norm_w.double().requires_grad_(), w.double().requires_grad_()
    y = hx / torch.sqrt((hx * hx).mean(1, keepdim=True) + 1e-6) * nw
    loss = (torch.nn.functional.cross_entropy(y @ ww.T, targets, reduction="none") * share.double()).sum()
    loss.backward()
    rel = lambda a, b: float((a.double() - b.detach()).norm() / b.detach().norm())
    # three roundings of bfloat16 (sum, norm, gradient) and those of the head: 2^-9 each on average at most; float32 sums
    tol = 8e-3 if kind == "bf16" else 1e-5
    assert rel(got["loss"], loss) < (1e-3 if kind == "bf16" else 1e-6)
    assert rel(got["grad_x"], hx.grad) < tol and rel(got["grad_norm"], nw.grad) < tol and rel(got["grad_weight"], ww.grad) < tol
    assert not got["grad_x"][share == 0].any()
    # captured into a graph and replayed on other values, with an eager call between
    static = [a.clone() for a in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for a in static[:4]:
        a.normal_()
    other = step(*static)
    graph.replay()
    for k in out:
        assert torch.equal(out[k], other[k]), k
    for a, b in zip(static, args):
        a.copy_(b)
    graph.replay()
    for k in out:
        assert torch.equal(out[k], got[k]), k


def test_python_front_refusals():
    c = cb()
    g = gen(40)
    x, w = normal(g, 6, 16), normal(g, 16)
    W, t = normal(g, 9, 16), torch.zeros(6, dtype=torch.int64, device="cuda")
    for error, f in ((c.DTypeError, lambda: c.rms_norm(x.double(), w)), (c.DTypeError, lambda: c.rms_norm(x.int(), w)),
                     (c.ShapeError, lambda: c.rms_norm(x[0, 0], w)), (ValueError, lambda: c.rms_norm(x, w, quant="rows")),
                     (ValueError, lambda: c.rms_norm(x, w, out_summed=x)), (ValueError, lambda: c.rms_norm(x, w, quant="row", out=x)),
                     (c.AliasError, lambda: c.rms_norm(x[:, :8], w[:8], out=x[:, 4:12])), (c.AliasError, lambda: c.rms_norm(x, w, residual=W[:6], out=W[:6])),
                     (c.DeviceError, lambda: c.rms_norm(x, w.cpu())), (c.DTypeError, lambda: c.linear_cross_entropy(x, W.bfloat16(), t)),
                     (c.AliasError, lambda: c.linear_cross_entropy(x, W, t, out_grad_hidden=x)),
                     (c.AliasError, lambda: c.linear_cross_entropy(x, W, t, out_grad_weight=W)),
                     (c.ShapeError, lambda: c.linear_cross_entropy(x, W, t, out_grad_weight=W[:8].clone())),
                     (c.ShapeError, lambda: c.linear_cross_entropy(x, W[:, :8], t)), (ValueError, lambda: c.linear_cross_entropy(x, W, t, temperature=0.0)),
                     (c.ShapeError, lambda: c.balance_loss(x, t[:, None], groups=4)), (ValueError, lambda: c.balance_loss(x, t[:, None], groups=0)),
                     (c.DTypeError, lambda: c.balance_loss(x, t[:, None].float())), (c.AliasError, lambda: c.balance_loss(x[:, :8], t[:, None], out_grad=x[:, 4:12])),
                     (c.DTypeError, lambda: c.add(c.rms_norm(x, w, quant="row").out, x)), (TypeError, lambda: c.rms_norm(x, 1.0))):
        with pytest.raises(error):
            f()


def test_streams():
    """Calls on two streams at once, each with its own scratch."""
    g = gen(30)
    sets = [head_inputs(g, 600, 256, 9001, "bf16") for _ in range(2)]
    want = [cb().linear_cross_entropy(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(cb().linear_cross_entropy(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[k]))
