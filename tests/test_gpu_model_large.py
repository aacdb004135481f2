"""GPU checks of the norm, the projection and the balance loss on matrices of more than 2^31 elements: the last rows, which only
64-bit offsets reach, against the same rows by themselves."""
import pytest
import torch

import model_oracle as O

pytestmark = pytest.mark.gpu


def filled(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty((rows, cols), dtype=dtype, device="cuda").normal_(generator=g)


def test_norm_rows_far_out():
    import ctorch_b200 as cb

    rows, dim = 530_000, 4097  # 2.17e9 elements, rows that start anywhere
    x, res = filled(rows, dim, torch.bfloat16, 1), filled(rows, dim, torch.bfloat16, 2)
    w = torch.ones(dim, device="cuda") * 1.5
    r = cb.rms_norm(x, w, residual=res)
    q = cb.rms_norm(x, w, residual=res, quant="block")
    b = cb.rms_norm_backward(x, r.summed, w, r.rstd, grad_summed=res)
    for k in (0, rows // 2, rows - 3):
        s = slice(k, k + 3)
        y, rstd, bound = O.norm(x[s], res[s], w, 1e-6)
        assert ((r.out[s].double() - y).abs() <= bound + O.half(torch.bfloat16) * y.abs()).all()
        one, scale = O.scales(y, "block")
        # half a step of e4m3 and what the sum's and the scale's roundings move
        assert ((q.out[s].float().double() * scale - y).abs() <= y.abs() * (2.0 ** -4 + 1e-4) + scale * 2.0 ** -10 * 1.01).all()
        gx, bx, _, _ = O.norm_grad(x[s], r.summed[s], w, 1e-6, res[s])
        assert ((b.grad_x[s].double() - gx).abs() <= bx + O.half(torch.bfloat16) * gx.abs()).all()


def test_head_of_a_weight_far_out():
    import ctorch_b200 as cb

    vocab, dim, rows = 530_000, 4096, 5
    w = filled(vocab, dim, torch.bfloat16, 3)
    h = filled(rows, dim, torch.bfloat16, 4) * 0.05
    t = torch.tensor([0, vocab - 1, vocab - 2, vocab // 2, vocab - 1], device="cuda")
    r = cb.linear_cross_entropy(h, w, t)
    z = torch.cat([h.double() @ w[i:i + 50_000].double().T for i in range(0, vocab, 50_000)], 1)
    lse = torch.logsumexp(z, 1)
    # a logit errs by 4 u a step of 16 products of what Cauchy and Schwarz allow
    dz = (dim / 16 + 1) * 4 * O.U * h.double().norm(dim=1) * w[:1000].double().norm(dim=1).max() * 1.2
    assert ((r.lse.double() - lse).abs() <= dz + 300 * O.U + 2 * O.U * lse).all()
    g = torch.exp(z - lse[:, None])
    g[torch.arange(rows), t] -= 1
    g /= rows
    for k in (0, vocab // 2, vocab - 600):
        want = g[:, k:k + 600].T @ h.double()
        off = (r.grad_weight[k:k + 600].double() - want).norm()
        assert off <= 4e-3 * want.norm()  # two roundings of 2^-8 / sqrt 3 / 1.47, five rows alone to average them
    gh = sum(g[:, i:i + 50_000] @ w[i:i + 50_000].double() for i in range(0, vocab, 50_000))
    assert (r.grad_hidden.double() - gh).norm() <= 4e-3 * gh.norm()


def test_balance_rows_far_out():
    import ctorch_b200 as cb

    rows, experts = 8_600_000, 256  # 2.2e9 logits
    x = filled(rows, experts, torch.bfloat16, 5)
    chosen = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
    chosen[-1] = 255
    r = cb.balance_loss(x, chosen, groups=2, coef=1.0)
    assert r.counts[0].tolist() == [rows // 2] + [0] * 255 and r.counts[1, 0] == rows // 2 - 1 and r.counts[1, 255] == 1
    tail = slice(rows - 3, rows)
    p = torch.softmax(x[tail].double(), 1)
    a = 256 * r.counts[1].double() / (rows // 2)
    want = p * (a - (a * p).sum(1, keepdim=True)) / rows
    assert ((r.grad[tail].double() - want).abs() <= O.half(torch.bfloat16) * want.abs() + 1e-4 * (p * (a + (a * p).sum(1, keepdim=True))) / rows).all()
