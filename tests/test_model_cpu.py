"""CPU checks of what stands around the losses: every refusal of the C ABI and of the Python front (all made before any
launch), and the oracle's gradients against differences of its own values."""
import ctypes

import pytest
import torch

import model_oracle as O
from test_capi_cpu import _lib, view

F32, F64, I32, I64, BOOL, BF16, F8 = range(7)


def P(v):
    return ctypes.byref(v) if v is not None else None


def call(C, fn, base, over):
    d = dict(base(C))
    d.update({n: f(C) if callable(f) else f for n, f in over.items()})
    return fn(C, d)


def norm_base(C):
    return dict(x=view(C, [2, 3, 8]), w=view(C, [8]), res=view(C, [2, 3, 8]), eps=1e-6, quant=0, out=view(C, [2, 3, 8]),
                summed=view(C, [2, 3, 8]), rstd=view(C, [2, 3]), scales=None)


def norm(C, d):
    return C.lib.ctb_rms_norm(P(d["x"]), P(d["w"]), P(d["res"]), d["eps"], d["quant"], P(d["out"]), P(d["summed"]), P(d["rstd"]),
                              P(d["scales"]), None)


def grad_base(C):
    return dict(up=view(C, [6, 8]), s=view(C, [6, 8]), w=view(C, [8]), rstd=view(C, [6]), passed=None, gx=view(C, [6, 8]),
                gw=view(C, [8]), scratch=4096, nbytes=1 << 20)


def grad(C, d):
    return C.lib.ctb_rms_norm_backward(P(d["up"]), P(d["s"]), P(d["w"]), P(d["rstd"]), P(d["passed"]), P(d["gx"]), P(d["gw"]),
                                       d["scratch"], d["nbytes"], None)


def head_base(C):
    return dict(h=view(C, [2, 3, 8]), w=view(C, [11, 8]), t=view(C, [2, 3], dtype=I64), weights=None, scale=1.0, temp=1.0, z=0.0,
                loss=view(C, []), row=view(C, [2, 3]), lse=None, gh=view(C, [2, 3, 8]), gw=view(C, [11, 8]), status=None,
                scratch=4096, nbytes=1 << 30)


def head(C, d):
    return C.lib.ctb_linear_cross_entropy(P(d["h"]), P(d["w"]), P(d["t"]), P(d["weights"]), d["scale"], d["temp"], d["z"], P(d["loss"]),
                                          P(d["row"]), P(d["lse"]), P(d["gh"]), P(d["gw"]), d["status"], d["scratch"], d["nbytes"], None)


def balance_base(C):
    return dict(x=view(C, [4, 3, 8]), e=view(C, [4, 3, 2], dtype=I64), mask=None, groups=4, coef=0.1, z=0.0, loss=view(C, []),
                counts=view(C, [4, 8], dtype=I64), probs=view(C, [4, 8]), g=view(C, [4, 3, 8]), status=None, scratch=4096, nbytes=1 << 20)


def balance(C, d):
    return C.lib.ctb_balance_loss(P(d["x"]), P(d["e"]), P(d["mask"]), d["groups"], d["coef"], d["z"], P(d["loss"]), P(d["counts"]),
                                  P(d["probs"]), P(d["g"]), d["status"], d["scratch"], d["nbytes"], None)


NAN, INF = float("nan"), float("inf")
REFUSED = {
    "norm": (norm, norm_base, [
        (dict(x=None), "ERR_ARGUMENT"),
        (dict(x=lambda C: view(C, [2, 3, 8], data=None)), "ERR_ARGUMENT"),
        (dict(x=lambda C: view(C, [2, 3, 8], dtype=F64)), "ERR_DTYPE"),
        (dict(x=lambda C: view(C, [2, 3, 8], dtype=F8)), "ERR_DTYPE"),
        (dict(x=lambda C: view(C, [])), "ERR_SHAPE"),
        (dict(x=lambda C: view(C, [2, 3, 0])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [7])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [1, 8])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [8], dtype=F64)), "ERR_DTYPE"),
        (dict(w=None), "ERR_ARGUMENT"),
        (dict(res=lambda C: view(C, [2, 3, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(res=lambda C: view(C, [6, 8])), "ERR_SHAPE"),
        (dict(res=lambda C: view(C, [1, 3, 8])), "ERR_SHAPE"),
        (dict(res=None), "ERR_ARGUMENT"),
        (dict(summed=None), "ERR_ARGUMENT"),
        (dict(summed=lambda C: view(C, [2, 3, 8], [0, 8, 1])), "ERR_ARGUMENT"),
        (dict(out=lambda C: view(C, [2, 3, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(out=lambda C: view(C, [2, 3, 8], [24, 8, 0])), "ERR_ARGUMENT"),
        (dict(out=None), "ERR_ARGUMENT"),
        (dict(rstd=lambda C: view(C, [2, 1])), "ERR_SHAPE"),
        (dict(rstd=lambda C: view(C, [2, 3], dtype=F64)), "ERR_DTYPE"),
        (dict(scales=lambda C: view(C, [2, 3])), "ERR_ARGUMENT"),
        (dict(quant=3), "ERR_ARGUMENT"),
        (dict(quant=1), "ERR_DTYPE"),
        (dict(quant=1, out=lambda C: view(C, [2, 3, 8], dtype=F8)), "ERR_ARGUMENT"),
        (dict(quant=1, out=lambda C: view(C, [2, 3, 8], dtype=F8), scales=lambda C: view(C, [2, 3, 1])), "ERR_SHAPE"),
        (dict(quant=2, out=lambda C: view(C, [2, 3, 8], dtype=F8), scales=lambda C: view(C, [2, 3])), "ERR_SHAPE"),
        (dict(quant=2, out=lambda C: view(C, [2, 3, 8], dtype=F8), scales=lambda C: view(C, [2, 3, 2])), "ERR_SHAPE"),
        (dict(eps=-1.0), "ERR_ARGUMENT"),
        (dict(eps=NAN), "ERR_ARGUMENT"),
        (dict(eps=INF), "ERR_ARGUMENT"),
    ]),
    "norm backward": (grad, grad_base, [
        (dict(up=lambda C: view(C, [6, 8], dtype=F64)), "ERR_DTYPE"),
        (dict(s=lambda C: view(C, [6, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(s=lambda C: view(C, [6, 7])), "ERR_SHAPE"),
        (dict(rstd=lambda C: view(C, [5])), "ERR_SHAPE"),
        (dict(rstd=None), "ERR_ARGUMENT"),
        (dict(passed=lambda C: view(C, [8])), "ERR_SHAPE"),
        (dict(gx=None), "ERR_ARGUMENT"),
        (dict(gx=lambda C: view(C, [6, 8], [0, 1])), "ERR_ARGUMENT"),
        (dict(gw=lambda C: view(C, [8], dtype=BF16)), "ERR_DTYPE"),
        (dict(gw=lambda C: view(C, [8], [0])), "ERR_ARGUMENT"),
        (dict(scratch=None), "ERR_SCRATCH"),
        (dict(nbytes=8), "ERR_SCRATCH"),
        (dict(scratch=4104), "ERR_ARGUMENT"),
    ]),
    "head": (head, head_base, [
        (dict(h=lambda C: view(C, [2, 3, 8], dtype=F64)), "ERR_DTYPE"),
        (dict(h=lambda C: view(C, [2, 3, 0])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [11, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(w=lambda C: view(C, [11, 7])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [0, 8])), "ERR_SHAPE"),
        (dict(w=lambda C: view(C, [1, 11, 8])), "ERR_SHAPE"),
        (dict(w=None), "ERR_ARGUMENT"),
        (dict(t=lambda C: view(C, [2, 3], dtype=F32)), "ERR_DTYPE"),
        (dict(t=lambda C: view(C, [2, 4], dtype=I64)), "ERR_SHAPE"),
        (dict(t=None), "ERR_ARGUMENT"),
        (dict(weights=lambda C: view(C, [2, 3], dtype=I32)), "ERR_DTYPE"),
        (dict(weights=lambda C: view(C, [3, 3])), "ERR_SHAPE"),
        (dict(scale=INF), "ERR_ARGUMENT"),
        (dict(temp=0.0), "ERR_ARGUMENT"),
        (dict(temp=NAN), "ERR_ARGUMENT"),
        (dict(z=-0.1), "ERR_ARGUMENT"),
        (dict(z=NAN), "ERR_ARGUMENT"),
        (dict(loss=lambda C: view(C, [2])), "ERR_SHAPE"),
        (dict(loss=lambda C: view(C, [], dtype=F64)), "ERR_DTYPE"),
        (dict(row=lambda C: view(C, [2, 3], [0, 1])), "ERR_ARGUMENT"),
        (dict(lse=lambda C: view(C, [6])), "ERR_SHAPE"),
        (dict(gh=None), "ERR_ARGUMENT"),
        (dict(gw=None), "ERR_ARGUMENT"),
        (dict(gh=lambda C: view(C, [2, 3, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(gh=lambda C: view(C, [2, 3, 8], [0, 8, 1])), "ERR_ARGUMENT"),
        (dict(gw=lambda C: view(C, [11, 9])), "ERR_SHAPE"),
        (dict(gw=lambda C: view(C, [11, 8], [0, 1])), "ERR_ARGUMENT"),
        (dict(status=4100), "ERR_ARGUMENT"),
        (dict(scratch=None), "ERR_SCRATCH"),
        (dict(nbytes=64), "ERR_SCRATCH"),
        (dict(scratch=4096 + 128), "ERR_ARGUMENT"),
    ]),
    "balance": (balance, balance_base, [
        (dict(x=lambda C: view(C, [4, 3, 8], dtype=F64)), "ERR_DTYPE"),
        (dict(x=lambda C: view(C, [4, 3, 4097])), "ERR_SHAPE"),
        (dict(e=lambda C: view(C, [4, 3, 2], dtype=F32)), "ERR_DTYPE"),
        (dict(e=lambda C: view(C, [4, 3, 0], dtype=I64)), "ERR_SHAPE"),
        (dict(e=lambda C: view(C, [12, 2], dtype=I64)), "ERR_SHAPE"),
        (dict(e=None), "ERR_ARGUMENT"),
        (dict(mask=lambda C: view(C, [4, 3], dtype=I64)), "ERR_DTYPE"),
        (dict(groups=0), "ERR_ARGUMENT"),
        (dict(groups=5), "ERR_SHAPE"),
        (dict(coef=NAN), "ERR_ARGUMENT"),
        (dict(z=INF), "ERR_ARGUMENT"),
        (dict(counts=lambda C: view(C, [4, 8], dtype=I32)), "ERR_DTYPE"),
        (dict(counts=lambda C: view(C, [8], dtype=I64)), "ERR_SHAPE"),
        (dict(probs=lambda C: view(C, [4, 8], [0, 1])), "ERR_ARGUMENT"),
        (dict(g=lambda C: view(C, [4, 3, 8], dtype=BF16)), "ERR_DTYPE"),
        (dict(loss=lambda C: view(C, [4])), "ERR_SHAPE"),
        (dict(scratch=None), "ERR_SCRATCH"),
        (dict(scratch=4100), "ERR_ARGUMENT"),
        (dict(status=4100), "ERR_ARGUMENT"),
    ]),
}


@pytest.mark.parametrize("what,k", [(w, k) for w in REFUSED for k in range(len(REFUSED[w][2]))])
def test_refusals(what, k):
    C = _lib()
    fn, base, cases = REFUSED[what]
    over, code = cases[k]
    assert call(C, fn, base, over) == getattr(C, code), C.last_error()
    assert C.last_error()


def test_other_operators_refuse_8_bits():
    C = _lib()
    a = view(C, [4], dtype=F8)
    assert C.lib.ctb_binary(C.ADD, a, a, a, None) != C.OK
    assert C.lib.ctb_unary(C.NEG, a, a, None) != C.OK
    assert C.lib.ctb_cast(a, view(C, [4]), None) != C.OK
    assert C.lib.ctb_reduce(C.SUM, a, view(C, []), 1, None, 0, None) != C.OK
    assert C.lib.ctb_token_logprobs(P(view(C, [2, 4], dtype=F8)), P(view(C, [2], dtype=I64)), None, 1.0, P(view(C, [2])), None, None,
                                    None) != C.OK


def test_scratch_bytes():
    C = _lib()
    need = C.lib.ctb_linear_loss_scratch_bytes
    x, w = view(C, [8192, 4096], dtype=BF16), view(C, [131072, 4096], dtype=BF16)
    held = 8192 * 131072 * 2
    assert held <= need(P(x), P(w), 0, 0) < 1.1 * held  # nothing is copied
    assert held <= need(P(x), P(w), 1, 1) < 1.3 * held
    # more rows than a block: the held part stays, what is added up over blocks joins it
    big = view(C, [1 << 20, 4096], dtype=BF16)
    assert need(P(big), P(w), 0, 0) < 1.2 * held
    assert need(P(x), P(view(C, [131072, 8], dtype=BF16)), 0, 1) == 0  # refused
    assert need(P(view(C, [0, 4096], dtype=BF16)), P(w), 0, 1) == 0
    assert need(None, P(w), 0, 1) == 0
    assert C.lib.ctb_balance_loss_scratch_bytes(P(view(C, [6, 8])), 0) == 0
    assert C.lib.ctb_balance_loss_scratch_bytes(P(view(C, [6, 8])), 2) > 0
    assert C.lib.ctb_rms_norm_backward_scratch_bytes(None) == 0


def test_python_front_refuses_cpu_tensors():
    import ctorch_b200 as cb

    x, w, t = torch.zeros(2, 4), torch.zeros(5, 4), torch.zeros(2, dtype=torch.int64)
    for f in (lambda: cb.rms_norm(x, x[0]), lambda: cb.rms_norm_backward(x, x, x[0], x[:, 0]),
              lambda: cb.linear_cross_entropy(x, w, t), lambda: cb.balance_loss(x, t[:, None])):
        with pytest.raises(cb.DeviceError):
            f()


def differences(f, x, h=1e-5):
    g = torch.zeros_like(x)
    for k in range(x.numel()):
        step = torch.zeros_like(x).view(-1)
        step[k] = h
        step = step.view(x.shape)
        g.view(-1)[k] = (f(x + step) - f(x - step)) / (2 * h)
    return g


def test_oracle_against_differences():
    """Central differences at 1e-5: h^2 / 6 of third derivatives below 100, and 1e-15 / h of rounding."""
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w, up = n(3, 7), 1 + 0.2 * n(7), n(3, 7)
    gx, _, gw, _ = O.norm_grad(up, x, w, 1e-3, None)
    assert (differences(lambda y: (O.norm(y, None, w, 1e-3)[0] * up).sum(), x) - gx).abs().max() < 1e-8
    assert (differences(lambda v: (O.norm(x, None, v, 1e-3)[0] * up).sum(), w) - gw).abs().max() < 1e-8
    h, v, t, share = n(5, 6), n(11, 6), torch.tensor([0, 10, 3, 3, 7]), torch.tensor([0.3, 0.0, 1.0, -0.5, 0.2], dtype=torch.float64)
    want = O.head(h, v, t, share, 0.02, 1.4)
    assert (differences(lambda y: O.head(y, v, t, share, 0.02, 1.4, False)["loss"][0], h) - want["grad_hidden"][0]).abs().max() < 1e-8
    assert (differences(lambda y: O.head(h, y, t, share, 0.02, 1.4, False)["loss"][0], v) - want["grad_weight"][0]).abs().max() < 1e-8
    r = n(12, 5)
    chosen, mask = torch.topk(r, 2, dim=-1).indices, torch.arange(12) % 4 != 1
    f = lambda y: O.balance(y, chosen, mask, 3, 0.4, 0.05)
    assert (differences(lambda y: f(y)["loss"][0], r) - f(r)["grad"][0]).abs().max() < 1e-8
