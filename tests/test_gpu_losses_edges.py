"""GPU checks of the losses over logits rows at the edges of what they promise, against float64."""
import numpy as np
import pytest
import torch

import losses_oracle as O
from test_gpu_losses import KIND, LAYOUTS, cb, check, dev, host, layouts

pytestmark = pytest.mark.gpu


def distill_apart(x, teacher, index, tlse, temperature, kind):
    """Distillation with a tail, each row's weight 1, the columns outside the entries by their own log-sum-exp: row losses
    and gradient with their bounds (losses_oracle's counts; the entries' share of the loss also carries q's rounding
    to float32 and one for the reference that x is taken from)."""
    n, v = x.shape
    u = O.EPS["f64" if kind == "f64" else "f32"]
    whole = O.Row(x, temperature, kind)
    loss, loss_tol, grad, grad_tol = np.zeros(n), np.zeros(n), np.zeros((n, v)), np.zeros((n, v))
    for i in range(n):
        k = index[i]
        others = np.delete(np.arange(v), k)
        rest = O.Row(x[i : i + 1, others], temperature, kind)
        log_q = teacher[i] / temperature - tlse[i]
        q = np.exp(log_q)
        q_rest = 1.0 - q.sum()
        big = q.sum() + q_rest
        log_p_rest = rest.lse[0] - whole.lse[i]
        loss[i] = (q * (log_q - whole.logp[i, k])).sum() + q_rest * (np.log(q_rest) - log_p_rest)
        far = np.abs(x[i, k] - x[i, k].max()) / temperature
        loss_tol[i] = whole.s_rel[i] + q_rest * rest.s_rel[0] + 2 * u * (q * (1 + far)).sum() + 4 * u * np.abs(loss[i])
        # q, its own log and log q' in float64
        loss_tol[i] += 2.0 ** -50 * (1 + abs(log_p_rest)) * (q * (np.abs(log_q) + np.abs(teacher[i] / temperature) + 4)).sum()
        p, share = whole.p[i], rest.p[0]
        grad[i, k] = big * p[k] - q
        grad_tol[i, k] = big * p[k] * (whole.p_rel[i, k] + 8 * u) + 6 * u * q
        grad[i, others] = big * p[others] - q_rest * share
        grad_tol[i, others] = big * p[others] * (whole.p_rel[i, others] + 8 * u) + q_rest * share * (rest.p_rel[0] + 8 * u)
    return (loss, loss_tol), (grad, grad_tol + O.EPS[kind] * (np.abs(grad) + grad_tol) + 1e-37)


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("v,top", [(700, 6), (5003, 300), (40000, 6)])
@pytest.mark.parametrize("gap,temperature", [(30.0, 1.0), (100.0, 1.0), (1000.0, 1.0), (50.0, 0.05), ("lowest", 1.0), (-100.0, 1.0)])
def test_a_student_far_from_certain_of_the_rest(gap, temperature, v, top, kind, how):
    """The columns outside the entries far below them (or far above): their share is less than the smallest float32, and
    its logarithm and the gradient there are ordinary numbers all the same."""
    rng = np.random.default_rng(v + top)
    n = 3
    x = rng.normal(size=(n, v)) * temperature
    index = np.stack([rng.permutation(v)[:top] for _ in range(n)])
    if gap == "lowest":
        named = np.take_along_axis(x, index, 1)
        x[:] = torch.finfo(KIND[kind]).min
    else:
        named = np.take_along_axis(x, index, 1) + gap
    np.put_along_axis(x, index, named, 1)
    y = dev(x, torch.float64).to(KIND[kind])
    teacher = rng.normal(size=(n, top)).astype(np.float32).astype(np.float64)
    tlse = (np.log(np.exp(teacher / temperature).sum(1)) + 0.4).astype(np.float32).astype(np.float64)
    row_loss, grad = distill_apart(host(y), teacher, index, tlse, temperature, kind)
    scale = 1.0 / temperature
    got = cb().distill_loss(layouts(y, how), dev(teacher, torch.float32), dev(index), dev(tlse, torch.float32),
                            torch.ones(n, device="cuda"), temperature)
    check(got.row_loss, row_loss, "row_loss")
    check(got.grad, (grad[0] * scale, grad[1] * scale * (1 + 2.0 ** -20)), "grad")


@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("kind", list(KIND))
@pytest.mark.parametrize("v", [5, 700, 20000])
@pytest.mark.parametrize("offsets", [[0, 5, 3], [2, 4, 3, 6, 7], [0, 5, 10 ** 6], [-1, 5, 9], [8, 4, 0], [0, 0, -3]])
def test_bad_offsets_make_every_result_nan(offsets, v, kind, how):
    """Rows between, before and behind the sequences, masked or not: nothing in the results looks like a number."""
    rows, pairs = 9, (len(offsets) - 1) // 2
    rng = np.random.default_rng(v)
    x = dev(rng.normal(size=(rows, v)), torch.float64).to(KIND[kind])
    t = rng.integers(0, v, rows)
    t[8] = -100
    mask = rng.random(rows) < 0.6
    for m in (None, mask):
        got = cb().preference_loss(layouts(x, how), dev(t), pairs, mask=None if m is None else dev(m), offsets=dev(np.array(offsets)))
        for name in ("loss", "pair_loss", "rewards", "logprobs", "grad"):
            assert torch.isnan(getattr(got, name)).all(), name


@pytest.mark.parametrize("kind", list(KIND))
def test_results_keep_no_scratch_alive(kind):
    """A program may keep the scalar of every step, or its row losses, and save them: their storage holds them and little
    else (8 KiB of scratch at most, or as much as they take themselves), whatever the call needed."""
    rows, v = 600, 300
    x = torch.randn(rows, v, device="cuda").to(KIND[kind])
    t = torch.randint(v, (rows,), device="cuda")
    z = torch.zeros(rows, device="cuda")
    index = torch.stack([torch.randperm(v, device="cuda")[:100] for _ in range(rows)])
    calls = [lambda n: cb().policy_loss(x[:n], t[:n], z[:n], z[:n], weights=z[:n] + 1)]
    for top in (1, 100):
        calls.append(lambda n, top=top: cb().distill_loss(x[:n], index[:n, :top].float(), index[:n, :top], weights=z[:n] + 1))
    calls.append(lambda n: cb().preference_loss(x[:n], t[:n], 2))
    for call in calls:
        for n in (4, 600):
            r = call(n)
            size = r.loss.element_size()
            assert r.loss.shape == () and r.loss.untyped_storage().nbytes() == size
            for name, a in zip(r._fields, r):
                if name not in ("loss", "grad"):
                    assert a.untyped_storage().nbytes() <= 8192 + 3 * n * size + 64, name
            assert r.grad.untyped_storage().nbytes() <= 2 * r.grad.nbytes
