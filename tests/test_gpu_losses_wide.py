"""GPU checks of the distillation loss on slices of which three fit an SM's shared memory: the two list warps and the
consumers hand every stage from one row to the next, at the last rows of a cluster and around rows that do not count."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,share", [(1, 1.0), (37, 1.0), (200, 1.0), (2600, 0.02), (2600, 0.2), (2600, 0.9)])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("v,dtype", [(131072, torch.bfloat16), (16384, torch.float32), (15003, torch.float32)])
def test_rows_of_three_stages(v, dtype, tail, rows, share):
    import ctorch_b200 as cb
    from ctorch_b200 import _capi as C

    rows *= 4 if dtype == torch.float32 else 1  # a CTA has a row where four share one of 131072
    top = 100
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    x = torch.randn(rows, v, generator=g, device="cuda", dtype=dtype)
    index = torch.randint(v // top, (rows, top), generator=g, device="cuda") + torch.arange(top, device="cuda") * (v // top)
    teacher = torch.randn(rows, top, generator=g, device="cuda")
    lse = teacher.logsumexp(1) + 0.3 if tail else None
    on = torch.rand(rows, generator=g, device="cuda") < share
    got = cb.distill_loss(x, teacher, index, lse, on)
    again = cb.distill_loss(x, teacher, index, lse, on)
    assert torch.equal(got.grad, again.grad) and torch.equal(got.row_loss, again.row_loss)
    assert C.wait_timeouts() == 0
    for i in range(0, rows, 200):
        b = slice(i, i + 200)
        p = torch.softmax(x[b].double(), -1)
        p_named = p.gather(1, index[b])
        if tail:
            q = (teacher[b].double() - lse[b, None].double()).exp()
            q_rest, p_rest = 1 - q.sum(1), 1 - p_named.sum(1)  # both far from 0 here
            want = p * (1 - q_rest / p_rest)[:, None]
        else:
            q, want = teacher[b].double().softmax(1), p.clone()
        want.scatter_(1, index[b], p_named - q)
        want *= on[b, None]
        # 2^-15: 64 roundings of float32 and more (losses_oracle); on an element that the teacher names p - q may cancel,
        # and with a tail 1 - q'/p' does: their terms' own errors count. Half a step of bfloat16 is 2^-8 of the value.
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -15 * p * on[b, None] + 1e-30
        bound.scatter_add_(1, index[b], 2.0 ** -20 * q)
        assert ((got.grad[b].double() - want).abs() <= bound).all()
