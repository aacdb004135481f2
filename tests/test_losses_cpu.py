"""CPU checks of the losses over logits rows: the oracle's gradients against differences of its own
losses, and every refusal of the C ABI and of the Python front (all made before any launch)."""
import ctypes

import numpy as np
import pytest
import torch

import losses_oracle as O
from test_capi_cpu import _lib, view

F32, F64, I32, I64, BOOL, BF16 = range(6)


def differences(f, x, h=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


@pytest.mark.parametrize("what", ["policy", "distill", "distill_tail", "preference"])
def test_oracle_gradient_against_differences(what):
    rng = np.random.default_rng(3)
    n, v = 6, 9
    x, t = rng.normal(size=(n, v)), rng.integers(0, v, n)
    w = np.array([0.3, 0.0, 1.0, 0.2, 0.5, 0.1])
    if what == "policy":
        old = O.token(x, t, w != 0, 1.5, "f64")[0] + 0.3 * rng.normal(size=n)
        f = lambda y: O.policy(y, t, old, rng2, ref, w, 0.2, 0.3, 0.1, 1.5, "f64")
        rng2, ref = rng.normal(size=n), old + 0.2
    elif what == "preference":
        ref, mask = -rng.random(n), np.array([1, 1, 0, 1, 1, 1], bool)
        f = lambda y: O.preference(y, t, [0, 3, 6], ref, mask, np.array([0.7]), 0.5, 0.1, True, "f64")
    else:
        index = np.stack([rng.permutation(v)[:4] for _ in range(n)])
        teacher = rng.normal(size=(n, 4))
        lse = np.log(np.exp(teacher / 1.5).sum(1)) + 0.4 if what == "distill_tail" else None
        f = lambda y: O.distill(y, teacher, index, lse, w, 1.5, "f64")
    got = f(x)["grad"][0]
    # central differences at h: h^2/6 times the third derivative (below 10 here) and 1e-16 / h of rounding
    assert np.abs(got - differences(lambda y: f(y)["loss"][0], x)).max() < 1e-9


def P(v):
    return ctypes.byref(v) if v is not None else None


def base(C, **over):
    """A valid policy call's views over [2, 3] rows of 8 logits; the addresses are never followed."""
    d = dict(logits=view(C, [2, 3, 8]), targets=view(C, [2, 3], dtype=I64), old=view(C, [2, 3]), adv=view(C, [2, 1]),
             ref=None, weights=None, loss=view(C, []), row=view(C, [2, 3]), logp=view(C, [2, 3]), kl=None,
             grad=view(C, [2, 3, 8]), scale=1.0, lo=0.2, hi=0.2, klc=0.0, temp=1.0, status=None, scratch=4096,
             nbytes=1 << 20)
    d.update(over)
    return d


def policy(C, **over):
    d = base(C, **over)
    return C.lib.ctb_policy_loss(P(d["logits"]), P(d["targets"]), P(d["old"]), P(d["adv"]), P(d["ref"]), P(d["weights"]),
                                 d["scale"], d["lo"], d["hi"], d["klc"], d["temp"], P(d["loss"]), P(d["row"]),
                                 P(d["logp"]), P(d["kl"]), P(d["grad"]), d["status"], d["scratch"], d["nbytes"], None)


REFUSED_POLICY = [
    (dict(logits=lambda C: view(C, [2, 3, 8], dtype=I32)), "ERR_DTYPE"),
    (dict(logits=lambda C: view(C, [])), "ERR_SHAPE"),
    (dict(logits=lambda C: view(C, [2, 3, 0])), "ERR_SHAPE"),
    (dict(logits=None), "ERR_ARGUMENT"),
    (dict(logits=lambda C: view(C, [2, 3, 8], data=None)), "ERR_ARGUMENT"),
    (dict(targets=lambda C: view(C, [2, 3], dtype=F32)), "ERR_DTYPE"),
    (dict(targets=lambda C: view(C, [2, 4], dtype=I64)), "ERR_SHAPE"),
    (dict(targets=None), "ERR_ARGUMENT"),
    (dict(old=lambda C: view(C, [2, 3], dtype=BF16)), "ERR_DTYPE"),
    (dict(adv=lambda C: view(C, [1, 2, 3])), "ERR_SHAPE"),
    (dict(weights=lambda C: view(C, [2, 3], dtype=I32)), "ERR_DTYPE"),
    (dict(ref=lambda C: view(C, [3, 3])), "ERR_SHAPE"),
    (dict(klc=0.1), "ERR_ARGUMENT"),
    (dict(klc=-0.1, ref=lambda C: view(C, [2, 3])), "ERR_ARGUMENT"),
    (dict(klc=float("nan"), ref=lambda C: view(C, [2, 3])), "ERR_ARGUMENT"),
    (dict(lo=1.5), "ERR_ARGUMENT"),
    (dict(lo=float("nan")), "ERR_ARGUMENT"),
    (dict(hi=-0.1), "ERR_ARGUMENT"),
    (dict(temp=0.0), "ERR_ARGUMENT"),
    (dict(temp=-1.0), "ERR_ARGUMENT"),
    (dict(temp=float("nan")), "ERR_ARGUMENT"),
    (dict(temp=float("inf")), "ERR_ARGUMENT"),
    (dict(loss=lambda C: view(C, [2])), "ERR_SHAPE"),
    (dict(loss=lambda C: view(C, [], dtype=F64)), "ERR_DTYPE"),
    (dict(row=lambda C: view(C, [2, 1])), "ERR_SHAPE"),
    (dict(row=lambda C: view(C, [2, 3], [0, 1])), "ERR_ARGUMENT"),
    (dict(logp=lambda C: view(C, [2, 3], dtype=F64)), "ERR_DTYPE"),
    (dict(grad=lambda C: view(C, [2, 3, 8], dtype=BF16)), "ERR_DTYPE"),
    (dict(grad=lambda C: view(C, [2, 3, 7])), "ERR_SHAPE"),
    (dict(grad=lambda C: view(C, [6, 8])), "ERR_SHAPE"),
    (dict(grad=lambda C: view(C, [2, 3, 8], [0, 8, 1])), "ERR_ARGUMENT"),
    (dict(grad=lambda C: view(C, [2, 3, 8], [24, 8, 0])), "ERR_ARGUMENT"),
    (dict(scratch=None), "ERR_SCRATCH"),
    (dict(nbytes=8), "ERR_SCRATCH"),
    (dict(scratch=4100), "ERR_ARGUMENT"),
    (dict(status=4100), "ERR_ARGUMENT"),
]


@pytest.mark.parametrize("k", range(len(REFUSED_POLICY)))
def test_policy_refusals(k):
    C = _lib()
    over, code = REFUSED_POLICY[k]
    over = {n: f(C) if callable(f) else f for n, f in over.items()}
    assert policy(C, **over) == getattr(C, code), C.last_error()
    assert C.last_error()


def distill(C, logits=None, teacher=None, index=None, lse=None, temp=1.0, scratch=4096, grad=None):
    logits = logits or view(C, [6, 8])
    return C.lib.ctb_distill_loss(P(logits), P(teacher or view(C, [6, 3])), P(index or view(C, [6, 3], dtype=I64)), P(lse),
                                  None, 1.0, temp, P(view(C, [])), None, P(grad), None, scratch, 1 << 20, None)


def test_distill_refusals():
    C = _lib()
    assert distill(C, index=view(C, [6, 4], dtype=I64)) == C.ERR_SHAPE
    assert distill(C, index=view(C, [6, 3], dtype=F32)) == C.ERR_DTYPE
    assert distill(C, index=view(C, [5, 3], dtype=I64)) == C.ERR_SHAPE
    assert distill(C, teacher=view(C, [6, 3], dtype=I64)) == C.ERR_DTYPE
    assert distill(C, teacher=view(C, []), index=view(C, [], dtype=I64)) == C.ERR_SHAPE
    assert distill(C, teacher=view(C, [6, 0]), index=view(C, [6, 0], dtype=I64)) == C.ERR_SHAPE
    assert distill(C, teacher=view(C, [6, 2049]), index=view(C, [6, 2049], dtype=I64)) == C.ERR_SHAPE
    assert distill(C, logits=view(C, [6, (1 << 20) + 1])) == C.ERR_SHAPE
    assert distill(C, lse=view(C, [6], dtype=BF16)) == C.ERR_DTYPE
    assert distill(C, lse=view(C, [5])) == C.ERR_SHAPE
    assert distill(C, grad=view(C, [6, 9])) == C.ERR_SHAPE
    assert distill(C, scratch=None) == C.ERR_SCRATCH


def preference(C, logits=None, pairs=3, offsets=None, beta=0.1, eps=0.0, weights=None, pair_loss=None, rewards=None,
               nbytes=1 << 20, targets=None):
    logits = logits or view(C, [6, 8])
    lead = list(logits.shape[: logits.ndim - 1])
    return C.lib.ctb_preference_loss(P(logits), P(targets or view(C, lead, dtype=I64)), pairs, P(offsets), None, None,
                                     P(weights), 1.0, beta, eps, 0, P(view(C, [])), P(pair_loss), P(rewards), None, None,
                                     None, 4096, nbytes, None)


def test_preference_refusals():
    C = _lib()
    assert preference(C, pairs=0) == C.ERR_ARGUMENT
    assert preference(C, pairs=2) == C.ERR_SHAPE  # 6 rows, 4 sequences
    assert preference(C, offsets=view(C, [6], dtype=I64)) == C.ERR_SHAPE
    assert preference(C, offsets=view(C, [7], dtype=F32)) == C.ERR_DTYPE
    assert preference(C, logits=view(C, [6, 1, 8]), offsets=view(C, [7], dtype=I32)) == C.ERR_SHAPE
    assert preference(C, beta=0.0) == C.ERR_ARGUMENT
    assert preference(C, beta=float("inf")) == C.ERR_ARGUMENT
    assert preference(C, eps=0.5) == C.ERR_ARGUMENT
    assert preference(C, eps=-0.1) == C.ERR_ARGUMENT
    assert preference(C, weights=view(C, [4])) == C.ERR_SHAPE
    assert preference(C, weights=view(C, [3], dtype=I32)) == C.ERR_DTYPE
    assert preference(C, pair_loss=view(C, [6])) == C.ERR_SHAPE
    assert preference(C, rewards=view(C, [6], dtype=F64)) == C.ERR_DTYPE
    assert preference(C, rewards=view(C, [6], [0])) == C.ERR_ARGUMENT
    assert preference(C, nbytes=(3 * 6 + 3) * 8 - 1) == C.ERR_SCRATCH


def test_token_refusals():
    C = _lib()
    x, t, o = view(C, [6, 8]), view(C, [6], dtype=I64), view(C, [6])
    fwd = lambda x=x, t=t, m=None, lp=o, lse=None: C.lib.ctb_token_logprobs(P(x), P(t), P(m), 1.0, P(lp), P(lse), None, None)
    assert fwd(lp=None) == C.ERR_ARGUMENT
    assert fwd(lp=view(C, [6, 1])) == C.ERR_SHAPE
    assert fwd(lse=view(C, [6], dtype=F64)) == C.ERR_DTYPE
    assert fwd(m=view(C, [6], dtype=I32)) == C.ERR_DTYPE
    assert fwd(x=view(C, [6, 1 << 31])) == C.ERR_SHAPE
    deep = view(C, [1] * 16)
    deep.ndim = 17
    assert fwd(x=deep) == C.ERR_SHAPE
    bwd = lambda up=o, lse=o, g=view(C, [6, 8]): C.lib.ctb_token_logprobs_backward(
        P(up), P(x), P(t), P(o), P(lse), None, 1.0, P(g), None, None)
    assert bwd(up=view(C, [6], dtype=BF16)) == C.ERR_DTYPE
    assert bwd(up=None) == C.ERR_ARGUMENT
    assert bwd(lse=None) == C.ERR_ARGUMENT
    assert bwd(g=None) == C.ERR_ARGUMENT
    assert bwd(g=view(C, [6, 8], dtype=F64)) == C.ERR_DTYPE


def test_scratch_bytes():
    C = _lib()
    need = C.lib.ctb_loss_scratch_bytes
    assert need(P(view(C, [2, 3, 8])), 0, 0) == 6 * 8
    assert need(P(view(C, [10 ** 6, 8])), 0, 0) <= 148 * 16 * 8
    assert need(P(view(C, [6, 8])), 3, 0) == (3 * 6 + 3) * 8
    assert need(P(view(C, [6, 8])), 0, 5) == 6 * 8 + 6 * (24 + 5 * 8)
    assert need(P(view(C, [0, 8])), 0, 0) == 0
    assert need(None, 0, 0) == 0


def test_python_front_refuses_cpu_tensors_and_types():
    import ctorch_b200 as cb

    x, t, r = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: cb.token_logprobs(x, t), lambda: cb.token_logprobs_backward(r, x, t, r, r),
                 lambda: cb.distill_loss(x, x[:, :2], t[:, None].expand(2, 2)), lambda: cb.policy_loss(x, t, r, r),
                 lambda: cb.preference_loss(x, t, 1)):
        with pytest.raises(cb.DeviceError):
            call()
