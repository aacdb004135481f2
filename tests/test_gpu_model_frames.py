"""GPU checks that the norm, the projection and the balance loss write their outputs and nothing else: outputs inside larger
buffers, with gaps between rows, rows that start anywhere, and in the place of operands. What lies around them stays as it was
to the bit. Values go by the bounds of tests/model_oracle.py."""
import pytest
import torch

import model_oracle as O
from test_gpu_model import KIND, balance_inputs, cb, check_balance, check_head, check_norm, gen, head_inputs, near, normal

pytestmark = pytest.mark.gpu

BITS = {torch.float32: torch.int32, torch.bfloat16: torch.int16}
FRAMES = [(0, 0), (8, 0), (8, 3), (1, 0), (3, 5), (16, 8)]  # (elements between rows, elements before the first)


class Frame:
    """[rows, columns] values inside a larger buffer of other numbers."""

    def __init__(self, x, frame):
        gap, before = frame
        rows, cols = x.shape
        self.flat = torch.randn(before + rows * (cols + gap) + 40, device="cuda").to(x.dtype)
        self.mask = torch.ones(self.flat.shape, dtype=torch.bool, device="cuda")
        at = ((rows, cols), (cols + gap, 1), before)
        self.view = self.flat.as_strided(*at)
        self.view.copy_(x)
        self.mask.as_strided(*at).fill_(False)
        self.old = self.flat.view(BITS[x.dtype]).clone()

    def check(self):
        assert torch.equal(self.flat.view(self.old.dtype)[self.mask], self.old[self.mask]), "written outside the output"

    def unchanged(self):
        assert torch.equal(self.flat.view(self.old.dtype), self.old), "an operand was written"


@pytest.mark.parametrize("frame", FRAMES)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim", [(40, 3), (41, 7), (33, 9), (300, 100), (50, 257), (90, 1001), (20, 4099), (3, 16400), (4, 20011)])
def test_norm_writes_its_outputs_alone(rows, dim, kind, frame):
    g, t = gen(rows + dim), KIND[kind]
    x, res, w = normal(g, rows, dim, dtype=t), normal(g, rows, dim, std=2.0, dtype=t), (1 + 0.3 * normal(g, dim)).to(t)
    fx, fr, fo, fs = (Frame(v, frame) for v in (x, res, torch.zeros_like(x), torch.zeros_like(x)))
    r = cb().rms_norm(fx.view, w, residual=fr.view, out=fo.view, out_summed=fs.view)
    check_norm(r, x, res, w, 1e-6, None, t)
    fx.unchanged(), fr.unchanged(), fo.check(), fs.check()
    for quant in ("row", "block"):
        q = cb().rms_norm(fx.view, w, residual=fr.view, quant=quant, out_summed=fs.view)
        check_norm(q, x, res, w, 1e-6, quant, t)
        fx.unchanged(), fr.unchanged(), fs.check()
    want = r.out.clone(), r.summed.clone()
    r = cb().rms_norm(fx.view, w, residual=fr.view, out=fx.view, out_summed=fr.view)  # each in an operand's place
    assert torch.equal(r.out, want[0]) and torch.equal(r.summed, want[1])
    fx.check(), fr.check()
    alone = Frame(x, frame)
    check_norm(cb().rms_norm(alone.view, w, out=alone.view), x, None, w, 1e-6, None, t)
    alone.check()


@pytest.mark.parametrize("frame", FRAMES)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim", [(40, 3), (41, 7), (33, 9), (300, 100), (50, 257), (90, 1001), (20, 4099), (3, 16400), (4, 20011)])
def test_norm_backward_writes_its_output_alone(rows, dim, kind, frame):
    g, t = gen(rows * dim), KIND[kind]
    x, up, passed, w = *(normal(g, rows, dim, dtype=t) for _ in range(3)), (1 + 0.3 * normal(g, dim)).to(t)
    rstd = cb().rms_norm(x, w).rstd
    for extra in (None, passed):
        gx, bx, gw, bw = O.norm_grad(up, x, w, 1e-6, extra)
        fu, fx, fo = Frame(up, frame), Frame(x, frame), Frame(torch.zeros_like(x), frame)
        fp = None if extra is None else Frame(extra, frame)
        p = None if extra is None else fp.view
        operands = [f for f in (fu, fx, fp) if f is not None]

        def check(r):
            near(r.grad_x, (gx, bx + O.half(t) * gx.abs() + 1e-38), "grad_x")
            near(r.grad_weight, (gw, bw + O.half(t) * gw.abs() + 1e-38), "grad_weight")

        check(cb().rms_norm_backward(fu.view, fx.view, w, rstd, grad_summed=p, out=fo.view))
        fo.check()
        for f in operands:
            f.unchanged()
        for place in operands:  # in the place of each
            again = [Frame(v, frame) for v in (up, x, extra) if v is not None]
            where = again[operands.index(place)]
            check(cb().rms_norm_backward(again[0].view, again[1].view, w, rstd, grad_summed=again[2].view if len(again) > 2 else None, out=where.view))
            for f in again:
                f.check() if f is where else f.unchanged()


@pytest.mark.parametrize("frame", FRAMES)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,dim,vocab", [(1, 9, 5), (70, 96, 515), (130, 33, 300), (257, 264, 129)])
def test_projection_writes_its_gradients_alone(rows, dim, vocab, kind, frame):
    g = gen(rows + vocab)
    h, w, t = head_inputs(g, rows, dim, vocab, kind)
    share = torch.rand(rows, generator=g, device="cuda") + 0.1
    share[rows // 2 + 1:: 3] = 0
    for weights in (None, share):
        fh, fw, gh, gw = Frame(h, frame), Frame(w, frame), Frame(torch.ones_like(h), frame), Frame(torch.ones_like(w), frame)
        r = cb().linear_cross_entropy(fh.view, fw.view, t, weights=weights, out_grad_hidden=gh.view, out_grad_weight=gw.view)
        check_head(r, O.head(h, w, t, weights), kind)
        fh.unchanged(), fw.unchanged(), gh.check(), gw.check()


@pytest.mark.parametrize("frame", FRAMES)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("rows,experts,k,groups", [(6, 3, 1, 2), (64, 8, 2, 1), (300, 60, 4, 3), (40, 257, 3, 2), (33, 1028, 5, 1), (20, 4096, 2, 1)])
def test_balance_loss_writes_its_gradient_alone(rows, experts, k, groups, kind, frame):
    g, t = gen(rows + experts), KIND[kind]
    x, chosen = balance_inputs(g, rows, experts, k, t)
    mask = torch.rand(rows, generator=g, device="cuda") < 0.7
    want = O.balance(x, chosen, mask, groups, 0.3, 0.02)
    fx, fo = Frame(x, frame), Frame(torch.ones_like(x), frame)
    check_balance(cb().balance_loss(fx.view, chosen, mask=mask, groups=groups, coef=0.3, z_coef=0.02, out_grad=fo.view), want)
    fx.unchanged(), fo.check()
    check_balance(cb().balance_loss(fx.view, chosen, mask=mask, groups=groups, coef=0.3, z_coef=0.02, out_grad=fx.view), want)
    fx.check()


def test_weight_gradient_of_rows_far_out():
    """More than 2^31 elements, rows that start anywhere: grad_weight of a backward pass over all of them."""
    rows, dim = 530_000, 4097
    g = gen(1)
    x = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    up = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.ones(dim, device="cuda") * 1.5
    b = cb().rms_norm_backward(up, x, w, cb().rms_norm(x, w).rstd)
    total, size = torch.zeros(dim, dtype=torch.float64, device="cuda"), torch.zeros(dim, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 20_000):
        s = x[i:i + 20_000].double()
        terms = up[i:i + 20_000].double() * s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6)
        total += terms.sum(0)
        size += terms.abs().sum(0)
    # a thread adds at most every 144th row (a CTA an SM, whole eights of them), of terms that rstd's roundings and a product's move
    near(b.grad_weight, (total, size * (rows / 144 + dim / 64 + 30) * O.U + O.U * total.abs()), "grad_weight")
