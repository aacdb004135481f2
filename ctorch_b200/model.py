"""What a language model's step has around the losses over logits rows (include/ctb/ctb.h, "around the losses"): the
root-mean-square norm with the residual's addition and its backward pass, the projection to the vocabulary with its
cross entropy and both gradients, and the balance loss of routed experts. ctorch has none of them; they follow the
losses' conventions (losses.py): CUDA tensors only, the current stream, no host synchronisation, gradients returned
beside the value instead of autograd, rows that do not count left alone, `status` for bad indices.

Matrices are [..., columns] in float32 or bfloat16, any leading dims and strides; a row is one position of the
leading dims. Results a row are float32.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _capi as C
from .errors import AliasError, DTypeError, ShapeError
from .losses import _PACK, _VIEW0, _check, _run, _scale, _status, _view
from .ops import _cuda, _same_view, may_overlap

RmsNorm = namedtuple("RmsNorm", ["out", "summed", "rstd", "scales"])
RmsNormGrad = namedtuple("RmsNormGrad", ["grad_x", "grad_weight"])
LinearCrossEntropy = namedtuple("LinearCrossEntropy", ["loss", "row_loss", "lse", "grad_hidden", "grad_weight"])
BalanceLoss = namedtuple("BalanceLoss", ["loss", "counts", "probs", "grad"])

SCALE_BLOCK = 128  # columns that share a scale with quant="block"
MAX_GROUPS = 1 << 20  # of the balance loss
_QUANT = {None: 0, "row": 1, "block": 2}
_MATRIX = (torch.float32, torch.bfloat16)
_FLOAT8 = torch.float8_e4m3fn


def _new(shape, dtype, dev):
    """torch.empty() by way of torch.empty_strided(), which takes half the time (1.5 us against 3)."""
    n = len(shape)
    strides = (1,) if n == 1 else (shape[1] or 1, 1) if n == 2 else ()
    if n > 2:
        step, strides = 1, [0] * n
        for d in range(n - 1, -1, -1):
            strides[d] = step
            step *= shape[d] or 1
    return torch.empty_strided(shape, strides, dtype=dtype, device=dev)


def _scratch(need, dev):
    return torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev)


def _matrices(name, first, *others):
    """The checks of losses._check for a matrix and further operands, without float64 matrices."""
    if isinstance(first, torch.Tensor) and first.device.type == "cuda":
        if first.dtype not in _MATRIX:
            raise DTypeError(f"ctorch::{name}: float32 and bfloat16 are supported (got {first.dtype})")
        if first.dim() == 0:
            raise ShapeError(f"ctorch::{name}: at least one dim is needed (the columns, last)")
    return _check(name, first, *others)


def _overlap(a, b):
    """Nothing overlaps a tensor of no elements (whose storage may have no address, like another's)."""
    return a.numel() > 0 and b.numel() > 0 and may_overlap(a, b)


def _output(name, what, out, like, dev, same=(), apart=()):
    """A new tensor like `like`, or `out` checked: `same` are operands whose own view it may be, `apart` those that it
    must not overlap."""
    if out is None:
        return _new(like.shape, like.dtype, dev)
    _cuda(name, like, out)
    if out.dtype != like.dtype or out.shape != like.shape:
        raise (DTypeError if out.dtype != like.dtype else ShapeError)(
            f"ctorch::{name}: {what} must be {like.dtype} {list(like.shape)}")
    for t in same:
        if t is not None and _overlap(out, t) and not _same_view(out, t):
            raise AliasError(f"ctorch::{name}: {what} overlaps an operand without being the same view")
    for t in apart:
        if t is not None and _overlap(out, t):
            raise AliasError(f"ctorch::{name}: {what} overlaps an operand")
    return out


def _view8(t):
    """The view of a float8 output, a type that no other operator takes."""
    shape = t.shape
    if len(shape) > C.MAX_DIMS:
        raise ShapeError(f"ctorch: tensor rank exceeds kMaxRank (got {len(shape)})")
    return _PACK[len(shape)](t.data_ptr(), C.F8E4M3, len(shape), *shape, *t.stride())


def rms_norm(x, weight, residual=None, eps: float = 1e-6, quant: str | None = None, out=None,
             out_summed=None) -> RmsNorm:
    """The root-mean-square norm of x's rows, with the residual's addition in the same pass:

        summed = x + residual (in their type; x itself without a residual)
        rstd = 1 / sqrt(mean(summed ** 2) + eps),    out = summed * rstd * weight

    With quant="row" or "block", out is float8_e4m3fn and stands for out * scales: a float32 scale a row, or one for
    every 128 columns ([..., ceil(columns / 128)]). scales is None without quant. `out` (not with quant) and
    `out_summed` may be given; out may be x's own view, out_summed x's or the residual's. Without a residual an out in
    x's place leaves nothing of x to differentiate: summed is None then."""
    name = "rms_norm"
    dev = _matrices(name, x, weight, residual)
    if quant not in _QUANT:
        raise ValueError(f"ctorch::{name}: quant must be None, 'row' or 'block'")
    shape, rows = x.shape, x.shape[:-1]
    summed = vsum = scales = vscales = None
    if residual is None and out_summed is not None:
        raise ValueError(f"ctorch::{name}: out_summed goes with a residual")
    if residual is not None:
        summed = _new(shape, x.dtype, dev) if out_summed is None else \
            _output(name, "out_summed", out_summed, x, dev, same=(x, residual), apart=(weight,))
        vsum = _view(summed)
    if quant is None:
        y = _new(shape, x.dtype, dev) if out is None else \
            _output(name, "out", out, x, dev, same=(x,), apart=(weight, residual))
        if out is not None and summed is not None and _overlap(out, summed):
            raise AliasError(f"ctorch::{name}: out overlaps summed")
        vout = _view(y)
    else:
        if out is not None:
            raise ValueError(f"ctorch::{name}: out cannot be given with quant")
        y = _new(shape, _FLOAT8, dev)
        vout = _view8(y)
        scales = _new(rows if quant == "row" else (*rows, -(-shape[-1] // SCALE_BLOCK)), torch.float32, dev)
        vscales = _view(scales)
    rstd = _new(rows, torch.float32, dev)
    _run(name, dev, C.lib.ctb_rms_norm, _view(x), _view(weight), _view(residual), eps, _QUANT[quant], vout, vsum,
         _view(rstd), vscales)
    if summed is None and (out is None or not _overlap(out, x)):
        summed = x
    return RmsNorm(y, summed, rstd, scales)


def rms_norm_backward(grad_out, summed, weight, rstd, grad_summed=None, out=None) -> RmsNormGrad:
    """The gradients of rms_norm for what comes back to out (grad_out) and, from elsewhere, to summed (grad_summed):
    grad_x, of x and of the residual alike, and grad_weight in weight's type. summed and rstd are rms_norm's. grad_x
    is written to `out` when given, which may be the view of grad_out, summed or grad_summed."""
    name = "rms_norm_backward"
    if summed is None:
        raise ValueError(f"ctorch::{name}: summed is needed (rms_norm wrote over x where out was x's own view)")
    dev = _matrices(name, grad_out, summed, weight, rstd, grad_summed)
    grad_x = _new(grad_out.shape, grad_out.dtype, dev) if out is None else \
        _output(name, "out", out, grad_out, dev, same=(grad_out, summed, grad_summed), apart=(weight, rstd))
    grad_weight = _new(weight.shape, weight.dtype, dev)
    vs = _view(summed)
    need = C.lib.ctb_rms_norm_backward_scratch_bytes(vs)
    scratch = _scratch(need, dev)
    _run(name, dev, C.lib.ctb_rms_norm_backward, _view(grad_out), vs, _view(weight), _view(rstd), _view(grad_summed),
         _view(grad_x), _view(grad_weight), scratch.data_ptr(), need)
    return RmsNormGrad(grad_x, grad_weight)


def linear_cross_entropy(hidden, weight, targets, weights=None, temperature: float = 1.0, z_coef: float = 0.0,
                         grad: bool = True, out_grad_hidden=None, out_grad_weight=None, status=None) -> LinearCrossEntropy:
    """Cross entropy of the projection of hidden [..., D] to a vocabulary, weight [V, D], without keeping the logits
    z = hidden @ weight.T / temperature. With lse = log sum exp z of a row,

        row_loss = lse - z[target] + z_coef * lse ** 2

    loss = sum(weights * row_loss), or the mean of the rows when weights is None; grad_hidden and grad_weight are the
    gradients of loss in their operands' types, None when grad=False. A row whose weight is 0 does not count (and
    costs no product); a target outside [0, V) in a row that counts makes that row's results NaN, and grad_weight."""
    name = "linear_cross_entropy"
    dev = _matrices(name, hidden, weight, targets, weights)
    if hidden.dtype != weight.dtype:
        raise DTypeError(f"ctorch::{name}: weight's dtype must equal hidden's")
    rows = hidden.shape[:-1]
    grad = grad or out_grad_hidden is not None or out_grad_weight is not None
    gh = gw = None
    if grad:
        operands = (hidden, weight, targets, weights)
        gh = _output(name, "out_grad_hidden", out_grad_hidden, hidden, dev, apart=operands)
        gw = _output(name, "out_grad_weight", out_grad_weight, weight, dev, apart=(*operands, out_grad_hidden))
    vh, vw = _view(hidden), _view(weight)
    if grad:
        need = C.lib.ctb_linear_loss_scratch_bytes(vh, vw, weights is not None, True)
    else:
        need = C.lib.ctb_linear_loss_forward_scratch_bytes(vh, vw, weights is not None)
    scratch = _scratch(need, dev)
    row_loss, lse = _new(rows, torch.float32, dev), _new(rows, torch.float32, dev)
    loss = _new((), torch.float32, dev)
    _run(name, dev, C.lib.ctb_linear_cross_entropy, vh, vw, _view(targets), _view(weights), _scale(weights, rows),
         temperature, z_coef, _VIEW0(loss.data_ptr(), C.F32, 0), _view(row_loss), _view(lse), _view(gh), _view(gw),
         _status(name, status, dev), scratch.data_ptr(), need)
    return LinearCrossEntropy(loss, row_loss, lse, gh, gw)


def balance_loss(logits, experts, mask=None, groups: int = 1, coef: float = 0.01, z_coef: float = 0.0, grad: bool = True,
                 out_grad=None, status=None) -> BalanceLoss:
    """The balance loss of routed experts: logits [..., E] of the router, experts [..., k] the ones chosen for each
    row (by any rule). The rows are `groups` equal shares in their order (sequences; 1: the whole batch). In a group
    of which n rows count, with p = softmax(logits) and lse = log sum exp of a row,

        counts[e] = times e was chosen,  f = counts / (n k),  probs = mean of p
        group loss = coef * E * sum(f * probs) + z_coef * mean(lse ** 2)

    loss = the mean of the groups' losses; counts [groups, E] int64; probs [groups, E]; grad = the gradient of the
    logits, None when grad=False (written to out_grad when given, which may be the logits' own view)."""
    name = "balance_loss"
    dev = _matrices(name, logits, experts, mask)
    g = None
    if grad or out_grad is not None:
        g = _output(name, "out_grad", out_grad, logits, dev, same=(logits,), apart=(experts, mask))
    n = logits.shape[-1]
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"ctorch::{name}: groups must be 1 to {MAX_GROUPS}")
    if n and logits.numel() // n % groups:  # before anything a group is allocated
        raise ShapeError(f"ctorch::{name}: the rows do not divide into {groups} groups")
    vx = _view(logits)
    need = C.lib.ctb_balance_loss_scratch_bytes(vx, groups)
    scratch = _scratch(need, dev)
    counts = _new((groups, n), torch.int64, dev)
    probs = _new((groups, n), torch.float32, dev)
    loss = _new((), torch.float32, dev)
    _run(name, dev, C.lib.ctb_balance_loss, vx, _view(experts), _view(mask), groups, coef, z_coef,
         _VIEW0(loss.data_ptr(), C.F32, 0), _view(counts), _view(probs), _view(g), _status(name, status, dev),
         scratch.data_ptr(), need)
    return BalanceLoss(loss, counts, probs, g)
