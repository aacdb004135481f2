"""GPU checks of what stands around the losses where it can go wrong without the bounds of test_gpu_model.py seeing it: logits
that are exact and long sums, quotients to 8 bits, what the norm returns of x, scores without gradients, weights without a
value, calls of no rows and refused ones."""
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


def whole(g, low, high, *shape):
    return torch.randint(low, high + 1, shape, generator=g, device="cuda").double()


def check_exact_logits(h, w, t, dtype):
    """Every product and every partial sum of the logits is a float32, so only the softmax errs: an exponential by 2^-22, its
    argument's two roundings (2^-24 of at most 40, in powers of 2, before the exponential vanishes against the sum) and the
    sum's additions (32 of a tile's quarter, the tiles by fours and lanes) by 2^-24 each; then a log's result is rounded."""
    z = h @ w.T
    lse = torch.logsumexp(z, 1)
    loss = lse - z.gather(1, t[:, None])[:, 0]
    r = cb().linear_cross_entropy(h.to(dtype), w.to(dtype), t, grad=False)
    bound = (4 + 2 * 40 + 64) * O.U
    for name, got, want in (("lse", r.lse, lse), ("row_loss", r.row_loss, loss)):
        off = (got.double() - want).abs() - (bound + 2 * O.U * want.abs())
        k = int(off.argmax())
        assert off[k] <= 0, (name, float(got[k]), float(want[k]))


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("dim", [64, 100, 768, 4096, 16384])
def test_logits_of_one_column_are_exact(dim, kind):
    """Rows with one entry that is not 0, in the first column, the last one and others."""
    g = gen(dim)
    rows, vocab = 70, 600
    w = whole(g, -64, 64, vocab, dim)
    at = torch.randint(dim, (rows,), generator=g, device="cuda")
    at[0], at[1], at[2], at[3] = 0, dim - 1, min(dim - 1, 767), min(dim - 1, 768)
    h = torch.zeros(rows, dim, dtype=torch.float64, device="cuda").scatter_(1, at[:, None], 1.0)
    check_exact_logits(h, w, torch.randint(vocab, (rows,), generator=g, device="cuda"), KIND[kind])


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("dim", [64, 1000, 4096, 16384])
def test_logits_of_whole_numbers_are_exact(dim, kind):
    """Sums of whole numbers below 2^24."""
    g = gen(dim + 1)
    rows, vocab = 70, 600
    check_exact_logits(whole(g, -2, 2, rows, dim), whole(g, -8, 8, vocab, dim), torch.randint(vocab, (rows,), generator=g, device="cuda"), KIND[kind])


@pytest.mark.parametrize("rows,dim,vocab", [(64, 256, 70000), (40000, 256, 64)])
def test_gradients_of_long_sums(rows, dim, vocab):
    """One way sums of many terms, along the vocabulary and along the rows: what truncated sums lose shows in their mean. The
    results' rounding to bfloat16 (2^-8 at most, independent) averages to 2^-8 / sqrt(3 n) over n of them, six of which are
    allowed, beside what a stretch loses (below 2e-5) and the truth's own share of G's rounding, likewise averaged."""
    g = gen(rows)
    h = (1 + torch.rand(rows, dim, generator=g, device="cuda")).bfloat16()
    w = (torch.rand(vocab, dim, generator=g, device="cuda") / dim).bfloat16()
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    r = cb().linear_cross_entropy(h, w, t)
    want = O.head(h, w, t, None)
    for name, got in (("grad_hidden", r.grad_hidden), ("grad_weight", r.grad_weight[1:])):
        value = want[name][0] if name == "grad_hidden" else want[name][0][1:]
        big = value.abs() > 0.1 * value.abs().mean()
        n = int(big.sum())
        bias = float((got.double() / value - 1)[big].mean())
        terms = vocab if name == "grad_hidden" else rows
        assert abs(bias) <= 6 * 2.0 ** -8 * (1 / (3 * n)) ** 0.5 + 6 * 2.0 ** -8 * (1 / (3 * terms)) ** 0.5 + 2e-5, (name, bias)


# ------------------------------------------------------------------------------------- 8 bits


@pytest.mark.parametrize("quant", ["row", "block"])
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim", [(1, 1), (64, 64), (40, 129), (300, 4096), (37, 5003), (5, 20008), (3, 40000), (400, 640)])
def test_8_bits_are_the_quotients_rounded_to_nearest(rows, dim, kind, quant):
    """y and its largest are the float32 numbers that the kernel has too (the rows' own rstd, two products), so the scale and
    the quotient rounded to 8 bits are known to the bit. Whole numbers and weights of few bits bring many quotients next to a
    tie."""
    g, t = gen(rows + dim), KIND[kind]
    x = whole(g, -60, 60, rows, dim).to(t)
    w = (whole(g, 1, 8, dim) / 4).to(t)
    for view in (x, torch.cat([x, x[:, :1]], 1)[:, :dim], x.t().contiguous().t()):  # packs, rows that start anywhere, columns
        r = cb().rms_norm(view, w, quant=quant)
        y = x.float() * r.rstd[:, None] * w.float()
        width = dim if quant == "row" else O.BLOCK
        top = torch.stack([p.abs().amax(-1) for p in y.split(width, -1)], -1)
        scale = torch.where(top == 0, 1.0, top / torch.tensor(448.0, device="cuda"))
        assert torch.equal(r.scales, scale[:, 0] if quant == "row" else scale)
        want = (y / scale.repeat_interleave(width, -1)[:, :dim]).to(torch.float8_e4m3fn)
        assert torch.equal(r.out.view(torch.uint8), want.view(torch.uint8))


# ------------------------------------------------------------------------------------- the norm's summed


@pytest.mark.parametrize("kind", list(KIND))
def test_norm_in_the_place_of_x_has_no_summed(kind):
    """Without a residual the backward pass needs x, which an out in its place has written over."""
    g, t = gen(5), KIND[kind]
    x, up, w = whole(g, -9, 9, 6, 40).to(t), whole(g, -9, 9, 6, 40).to(t), torch.ones(40, device="cuda")
    want = cb().rms_norm(x, w)
    assert want.summed is x
    apart = cb().rms_norm(x, w, out=torch.empty_like(x))
    assert apart.summed is x and torch.equal(apart.out, want.out)
    for y in (x.clone(), x.clone().view(2, 3, 40)):
        r = cb().rms_norm(y, w, out=y.view(y.shape))
        assert r.summed is None and torch.equal(r.out.view(6, 40), want.out)
        with pytest.raises(ValueError, match="summed"):
            cb().rms_norm_backward(up.view(y.shape), r.summed, w, r.rstd)
    y = x.clone()
    r = cb().rms_norm(y, w, residual=up, out=y)  # with a residual the sum is kept apart
    b = cb().rms_norm_backward(up, r.summed, w, r.rstd)
    gx, bx, _, _ = O.norm_grad(up, (x.double() + up.double()).to(t), w, 1e-6, None)
    assert ((b.grad_x.double() - gx).abs() <= bx + O.half(t) * gx.abs()).all()


# ------------------------------------------------------------------------------------- a projection without gradients


def test_scores_of_many_rows():
    """More rows than a block of statistics holds, in little memory; the same numbers as with gradients."""
    g = gen(33)
    rows, dim, vocab = 33_000, 8, 131_072
    h, w = torch.randn(rows, dim, generator=g, device="cuda").bfloat16(), torch.randn(vocab, dim, generator=g, device="cuda").bfloat16()
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    share = (torch.rand(rows, generator=g, device="cuda") < 0.99).float()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for weights in (None, share):
        r = cb().linear_cross_entropy(h, w, t, weights=weights, grad=False)
        assert torch.cuda.max_memory_allocated() - before < 300 << 20
        for s in (slice(0, 300), slice(32_700, 33_000)):
            some = cb().linear_cross_entropy(h[s], w, t[s], weights=None if weights is None else weights[s])
            assert torch.equal(r.row_loss[s], some.row_loss) and torch.equal(r.lse[s], some.lse)
        total = (r.row_loss.double() * (1 / rows if weights is None else weights.double())).sum()
        assert abs(float(r.loss) - float(total)) <= 4 * O.U * float(total)
        del some
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()


# ------------------------------------------------------------------------------------- weights without a value


@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("odd", [float("inf"), -float("inf"), NAN, 1e300])
def test_a_weight_without_a_value_spoils_its_own_row_alone(odd, kind):
    g, t = gen(44), KIND[kind]
    h, w = torch.randn(50, 64, generator=g, device="cuda").to(t), torch.randn(300, 64, generator=g, device="cuda").to(t)
    targets = torch.randint(300, (50,), generator=g, device="cuda")
    share = (torch.rand(50, generator=g, device="cuda") + 0.5).double()
    share[5] = share[6] = share.max()  # the largest stays when the odd row's is gone
    share[9] = 0
    usual = cb().linear_cross_entropy(h, w, targets, weights=share)
    share[5] = odd
    r = cb().linear_cross_entropy(h, w, targets, weights=share)
    others = torch.arange(50, device="cuda") != 5
    assert torch.equal(r.row_loss, usual.row_loss) and torch.equal(r.lse, usual.lse)
    assert torch.equal(r.grad_hidden[others], usual.grad_hidden[others])
    assert not torch.isfinite(r.grad_hidden[5]).any() and not torch.isfinite(r.loss)
    alone = cb().linear_cross_entropy(h[5:6], w, targets[5:6], weights=share[5:6])
    assert not torch.isfinite(alone.grad_hidden).any() and torch.equal(alone.row_loss, usual.row_loss[5:6])


# ------------------------------------------------------------------------------------- calls refused, and not


def test_outputs_of_no_rows_overlap_nothing():
    c, none = cb(), lambda *shape: torch.empty(shape, device="cuda")
    w, W, t = torch.ones(16, device="cuda"), torch.ones(9, 16, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    out, summed = none(0, 16), none(0, 16)
    r = c.rms_norm(none(0, 16), w, residual=none(0, 16), out=out, out_summed=summed)
    assert r.out is out and r.summed is summed
    b = c.rms_norm_backward(none(0, 16), none(0, 16), w, none(0), out=none(0, 16))
    assert b.grad_x.shape == (0, 16) and not b.grad_weight.any()
    gw = torch.ones(9, 16, device="cuda")
    h = c.linear_cross_entropy(none(0, 16), W, t, out_grad_hidden=none(0, 16), out_grad_weight=gw)
    assert h.grad_weight is gw and not gw.any() and float(h.loss) == 0
    a = c.balance_loss(none(0, 16), t[:, None], out_grad=none(0, 16))
    assert a.grad.shape == (0, 16) and float(a.loss) == 0


def test_groups_are_refused_before_their_tables_are_made():
    x, e = torch.randn(6, 4096, device="cuda"), torch.zeros(6, 1, dtype=torch.int64, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for error, groups in ((ValueError, 0), (ValueError, (1 << 20) + 1), (ValueError, 1 << 50), (cb().ShapeError, 1 << 20), (cb().ShapeError, 4)):
        with pytest.raises(error):
            cb().balance_loss(x, e, groups=groups, grad=False)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 40])
def test_a_few_rows_losses(rows):
    """Rows that lean towards their targets: losses far below the logits. What a row's loss errs by: its log-sum-exp and its
    target's logit, each within a stretch's truncation (2^-23 of the partial sums that one of 16 products at most reaches, by a
    step, one way), which a stretch of 4 stages holds to 16 steps and one of 12 to 48; as a mean square over the rows."""
    g = gen(rows)
    dim, vocab = 2048, 20_000
    w = (torch.randn(vocab, dim, generator=g, device="cuda") * (2 / dim ** 0.5)).bfloat16()
    steps = 16 if rows <= 8 else 48
    for _ in range(4):
        t = torch.randint(vocab, (rows,), generator=g, device="cuda")
        h = (torch.randn(rows, dim, generator=g, device="cuda") + 2 * w[t].float()).bfloat16()
        z = h.double() @ w.double().T
        lse = torch.logsumexp(z, 1)
        zt = z.gather(1, t[:, None])[:, 0]
        r = cb().linear_cross_entropy(h, w, t, grad=False)
        # a logit's partial sums stay below its own size and six deviations of a sum of such products, 2 |h| / sqrt(dim)
        reach = zt.abs() + 6 * 2 * h.double().norm(dim=1) / dim ** 0.5
        bound = 2 * steps * 2 * O.U * reach + 60 * O.U + 2 * O.U * lse.abs()
        assert ((r.row_loss.double() - (lse - zt)).abs() <= bound).all()
        assert ((r.lse.double() - lse).abs() <= bound).all()


@pytest.mark.parametrize("quant", ["row", "block"])
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("dim", [300, 640, 5003, 40000])
def test_8_bits_beside_infinities_and_the_smallest_numbers(dim, kind, quant):
    """By an infinite scale: 0, and NaN of the infinity; scales that would be below float32's normal numbers stay at the least."""
    g, t = gen(dim), KIND[kind]
    x = whole(g, 1, 60, 6, dim).to(t)
    x[4] = 0.0
    w = torch.ones(dim, device="cuda")
    w[200] = float("inf")
    r = cb().rms_norm(x, w, quant=quant)
    rows = [0, 1, 2, 3, 5]
    hit = torch.zeros(dim, dtype=torch.bool, device="cuda")
    hit[slice(None) if quant == "row" else slice(128, 256)] = True
    out = r.out.float()
    assert torch.isnan(out[:, 200]).all()  # infinity over infinity, and 0 times infinity
    hit[200] = False
    assert (out[rows][:, hit] == 0).all() and torch.isnan(out[4, hit]).all()
    assert torch.isfinite(out[:, ~hit & (torch.arange(dim, device="cuda") != 200)]).all()
    small = cb().rms_norm(x, torch.full((dim,), 2.0 ** -126, device="cuda"), quant=quant)
    assert torch.isfinite(small.out.float()).all() and (small.scales[rows] == 2.0 ** -126).all() and (small.scales[4] == 1).all()
