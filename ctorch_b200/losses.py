"""Losses over the rows of a logits matrix, with their gradients (the "losses" section of
include/ctb/ctb.h): log-probabilities of chosen tokens, distillation from a teacher's top entries, the
clipped policy loss and the preference loss on pairs of sequences. ctorch has no losses; these follow
its front-doors' conventions (eager, explicit outputs, the same exception types) and, like every op of
this package, run on CUDA tensors only, on the current stream, without a host synchronisation.

There is no autograd here: a loss returns the gradient of its logits beside its value. That is what lets
policy_loss and distill_loss read the logits once and write the gradient from the same pass.

Logits are [..., V] (float32, float64 or bfloat16, any strides), a row is one position of the leading
dims. Numbers a row (targets, weights, ...) broadcast to the leading dims. A row whose mask or weight is
0 does not count: nothing of it is looked at, its results and its gradient are 0. Results a row are
float32 (float64 for float64 logits).

An index outside [0, V) in a row that counts makes that row's results NaN. To be told of it by an
exception instead, pass a `status` (index_status()) to the calls and look at it when a host
synchronisation is affordable (check_index_status()).
"""
from __future__ import annotations

import struct
from collections import namedtuple
from math import prod

import torch

from . import _capi as C
from .errors import AliasError, DTypeError, ShapeError
from .ops import _call, _cuda, _same_view, may_overlap

TokenLogprobs = namedtuple("TokenLogprobs", ["logprobs", "lse"])
DistillLoss = namedtuple("DistillLoss", ["loss", "row_loss", "grad"])
PolicyLoss = namedtuple("PolicyLoss", ["loss", "row_loss", "logprobs", "kl", "grad"])
PreferenceLoss = namedtuple("PreferenceLoss", ["loss", "pair_loss", "rewards", "logprobs", "grad"])

_SIZE = {torch.float32: 4, torch.float64: 8, torch.bfloat16: 2}
# of a row's results, by the logits' type: dtype, its code, bytes
_RESULT = {torch.float32: (torch.float32, C.F32, 4), torch.bfloat16: (torch.float32, C.F32, 4),
           torch.float64: (torch.float64, C.F64, 8)}

# A loss of a few rows takes the GPU less time than it takes Python to describe its operands, so the views
# are packed in one go (ctb_view as bytes) and the results a row share one allocation, with the scratch where
# that is small. The scalar loss has storage of its own: a program may keep it for every step, for its log.
_VIEW = [struct.Struct(f"<Qii{n}q{8 * (C.MAX_DIMS - n)}x{n}q{8 * (C.MAX_DIMS - n)}x") for n in range(C.MAX_DIMS + 1)]


_VIEW0, _VIEW1 = _VIEW[0].pack, _VIEW[1].pack
_PACK = [v.pack for v in _VIEW]
_CODE = C.CODE_OF_TORCH
_SMALL = 8192  # bytes of scratch that the results a row carry along; more only where it is less than they are


def _view(t):
    if t is None:
        return None
    shape = t.shape
    n = len(shape)
    if n > C.MAX_DIMS:
        raise ShapeError(f"ctorch: tensor rank exceeds kMaxRank (got {n})")
    return _PACK[n](t.data_ptr(), _CODE[t.dtype], n, *shape, *t.stride())


def _check(name, logits, *others):
    """Device and dtype checks shared by the losses; returns the device."""
    if not isinstance(logits, torch.Tensor) or logits.device.type != "cuda":
        _cuda(name, logits)  # raises
    dev = logits.device
    if logits.dtype not in _SIZE:
        raise DTypeError(f"ctorch::{name}: logits must be float32, float64 or bfloat16 (got {logits.dtype})")
    for t in others:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"ctorch::{name}: expected a tensor")
        if t.device != dev:
            _cuda(name, logits, t)  # raises
        if t.dtype not in _CODE:
            raise DTypeError(f"ctorch::{name}: {t.dtype} is not supported")
    if logits.dim() == 0:
        raise ShapeError(f"ctorch::{name}: logits must have at least one dim (the vocabulary, last)")
    return dev


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _run(name, dev, fn, *args):
    """fn(*args, stream) on the current stream of the operands' device."""
    if dev.index == _current_device():
        _call(fn(*args, C.raw_stream(dev)), name)
    else:
        with torch.cuda.device(dev):
            _call(fn(*args, C.raw_stream(dev)), name)


def _results(logits, dev, rows, per_row, others=(), scratch=0, scalar=True):
    """Tensors for `per_row` results of the leading shape `rows`, vectors of `others` elements, and the scalar loss.
    Returns the address of the scratch (bytes) and what keeps it, the results and their packed views."""
    dtype, code, size = _RESULT[logits.dtype]
    n = prod(rows)
    apart = scratch > _SMALL and scratch > per_row * n * size
    sizes = [n] * per_row
    sizes += others
    lead = 0 if apart else -(-scratch // size)
    if lead:
        sizes.insert(0, lead)
    keep = flat = torch.empty(sum(sizes), dtype=dtype, device=dev)
    base = at = flat.data_ptr()
    if apart:
        keep = torch.empty(scratch, dtype=torch.uint8, device=dev)
        base = keep.data_ptr()
    out = list(torch.unsafe_split_with_sizes(flat, sizes))  # nothing here is differentiated, so nothing needs tracking
    views = []
    for n in sizes:
        views.append(_VIEW1(at, code, 1, n, 1))
        at += n * size
    if lead:
        del out[0], views[0]
    if len(rows) != 1:
        for i in range(per_row):
            out[i] = out[i].view(rows)
            views[i] = _view(out[i])
    if scalar:
        loss = torch.empty_strided((), (), dtype=dtype, device=dev)
        out.append(loss)
        views.append(_VIEW0(loss.data_ptr(), code, 0))
    return (base, keep), out, views


def _grad_for(name, logits, out, dev):
    """The gradient's tensor: `out` (checked), or a new one. Rows of the two that are aligned alike modulo 16
    bytes move in 16-byte pieces, so the new one's rows lie like the logits' rows: where those all start
    on 16 bytes although V elements are not a multiple of it (a vocabulary padded in memory), so do the
    new one's; where they start anywhere, it takes the logits' strides if that wastes little."""
    if out is not None:
        _cuda(name, logits, out)
        if out.dtype != logits.dtype:
            raise DTypeError(f"ctorch::{name}: the gradient's dtype must equal the logits'")
        if out.shape != logits.shape:
            raise ShapeError(f"ctorch::{name}: the gradient's shape must equal the logits'")
        if may_overlap(out, logits) and not _same_view(out, logits):
            raise AliasError(f"ctorch::{name}: the gradient overlaps the logits without being the same view")
        return out
    if logits.is_contiguous() and logits.data_ptr() % 16 == 0:
        return torch.empty_like(logits)
    shape, strides, size = logits.shape, logits.stride(), _SIZE[logits.dtype]
    lead, v = logits.data_ptr() % 16 // size, shape[-1]
    if logits.numel() == 0:
        return torch.empty(shape, dtype=logits.dtype, device=dev)
    if lead == 0 and all(st * size % 16 == 0 for s, st in zip(shape[:-1], strides) if s > 1):
        if v * size % 16 and logits.dim() > 1:
            pitch = -(-v * size // 128) * 128 // size
            return torch.empty((*shape[:-1], pitch), dtype=logits.dtype, device=dev)[..., :v]
    elif strides[-1] == 1:
        span = 1  # elements from the first to the last, if the dims nest
        for st, s in sorted((st, s) for s, st in zip(shape, strides) if s > 1):
            span = span + (s - 1) * st if st >= span else 0
            if not span:
                break
        if 0 < span <= logits.numel() * 5 // 4:
            return torch.empty(lead + span, dtype=logits.dtype, device=dev).as_strided(shape, strides, lead)
    return torch.empty(shape, dtype=logits.dtype, device=dev)


def index_status(device="cuda") -> torch.Tensor:
    """A cleared status for the losses' `status` argument; one serves any number of calls on a device."""
    return torch.zeros(2, dtype=torch.int64, device=device)


def check_index_status(status: torch.Tensor) -> None:
    """Synchronises and raises ShapeError if a call that was given `status` met a bad index since it
    was made (or cleared with zero_())."""
    flag, index = status.tolist()
    if flag & 0xFFFFFFFF:
        raise ShapeError(f"ctorch::losses: index {index} out of range, named twice in one row, or an offset "
                         "that falls")


def _status(name, status, dev):
    if status is None:
        return None
    if not isinstance(status, torch.Tensor) or status.dtype != torch.int64 or status.numel() != 2 or \
            not status.is_contiguous() or status.device != dev:
        raise ValueError(f"ctorch::{name}: status must come from index_status() on the logits' device")
    return status.data_ptr()


def token_logprobs(logits, targets, mask=None, temperature: float = 1.0, status=None) -> TokenLogprobs:
    """log p[target] and log-sum-exp of each row, with p = softmax(logits / temperature). Forward only:
    token_logprobs_backward() pulls a gradient back through it."""
    name = "token_logprobs"
    dev = _check(name, logits, targets, mask)
    _, (logp, lse), (v_logp, v_lse) = _results(logits, dev, logits.shape[:-1], 2, scalar=False)
    _run(name, dev, C.lib.ctb_token_logprobs, _view(logits), _view(targets), _view(mask), temperature, v_logp, v_lse,
         _status(name, status, dev))
    return TokenLogprobs(logp, lse)


def token_logprobs_backward(grad_logprobs, logits, targets, logprobs, lse, mask=None, temperature: float = 1.0,
                            out=None, status=None) -> torch.Tensor:
    """The gradient of sum(grad_logprobs * logprobs) with respect to the logits; logprobs and lse are
    token_logprobs' results for the same logits, targets, mask and temperature. Written to `out` when
    given, which may be the logits themselves."""
    name = "token_logprobs_backward"
    dev = _check(name, logits, grad_logprobs, targets, logprobs, lse, mask)
    grad = _grad_for(name, logits, out, dev)
    _run(name, dev, C.lib.ctb_token_logprobs_backward, _view(grad_logprobs), _view(logits), _view(targets),
         _view(logprobs), _view(lse), _view(mask), temperature, _view(grad), _status(name, status, dev))
    return grad


def _scale(weights, rows):
    return 1.0 if weights is not None else 1.0 / max(prod(rows), 1)


def distill_loss(logits, teacher_logits, teacher_indices, teacher_lse=None, weights=None, temperature: float = 1.0,
                 grad: bool = True, out_grad=None, status=None) -> DistillLoss:
    """Distillation from the K entries a row that a teacher finds likeliest: teacher_logits [..., K] at
    vocabulary indices teacher_indices [..., K] (all different; an entry of -inf is padding). Without
    teacher_lse the entries are renormalised; with teacher_lse [...] (the log-sum-exp of the teacher's
    whole row of logits / temperature) the mass outside them is one more event.

    row_loss = KL(teacher || student) of each row at `temperature` (not multiplied by its square);
    loss = sum(weights * row_loss), or the mean of the rows when weights is None; grad = the gradient of
    loss, None when grad=False. Fastest with up to 186 entries, in rows of unit stride of up to 262144 logits
    (float32: 131072)."""
    name = "distill_loss"
    dev = _check(name, logits, teacher_logits, teacher_indices, teacher_lse, weights)
    rows = logits.shape[:-1]
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    vx = _view(logits)
    need = C.lib.ctb_loss_scratch_bytes(vx, 0, teacher_logits.shape[-1] if teacher_logits.dim() else 0)
    (scratch, _keep), (row_loss, loss), (v_row, v_loss) = _results(logits, dev, rows, 1, scratch=need)
    _run(name, dev, C.lib.ctb_distill_loss, vx, _view(teacher_logits), _view(teacher_indices), _view(teacher_lse),
         _view(weights), _scale(weights, rows), temperature, v_loss, v_row, _view(g), _status(name, status, dev),
         scratch, need)
    return DistillLoss(loss, row_loss, g)


def policy_loss(logits, targets, old_logprobs, advantages, ref_logprobs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, grad: bool = True,
                out_grad=None, status=None) -> PolicyLoss:
    """The clipped policy loss with a KL term, a row a sampled token. With logp = log p[target],
    r = exp(logp - old_logprobs), A = advantages and d = ref_logprobs - logp:

        row_loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * kl,   kl = exp(d) - 1 - d

    loss = sum(weights * row_loss), or the mean of the rows when weights is None; logprobs = logp; kl is 0
    without ref_logprobs; grad = the gradient of loss, None when grad=False. Fastest in rows of unit stride of up
    to 262144 logits (float32: 131072)."""
    name = "policy_loss"
    dev = _check(name, logits, targets, old_logprobs, advantages, ref_logprobs, weights)
    rows = logits.shape[:-1]
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    vx = _view(logits)
    need = C.lib.ctb_loss_scratch_bytes(vx, 0, 0)
    (scratch, _keep), (row_loss, logp, kl, loss), (v_row, v_logp, v_kl, v_loss) = _results(logits, dev, rows, 3, scratch=need)
    _run(name, dev, C.lib.ctb_policy_loss, vx, _view(targets), _view(old_logprobs), _view(advantages),
         _view(ref_logprobs), _view(weights), _scale(weights, rows), clip_low, clip_high, kl_coef, temperature,
         v_loss, v_row, v_logp, v_kl, _view(g), _status(name, status, dev), scratch, need)
    return PolicyLoss(loss, row_loss, logp, kl, g)


def preference_loss(logits, targets, pairs: int, ref_logprobs=None, mask=None, offsets=None, weights=None,
                    beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False, grad: bool = True,
                    out_grad=None, status=None) -> PreferenceLoss:
    """The preference loss on `pairs` pairs of sequences, the chosen ones first: the rows of [2 * pairs,
    length, V] logits (any leading dims that divide evenly), or, with offsets [2 * pairs + 1] on the
    device, rows offsets[s] to offsets[s + 1] of [rows, V] logits. Over a sequence's rows with mask,
    rewards = beta * sum(logp - ref_logprobs) (their mean with average=True), and with h the chosen
    sequence's reward less the rejected one's

        pair_loss = -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)

    loss = sum(weights * pair_loss), or the mean of the pairs when weights is None; logprobs = logp of
    the rows (0 where masked); grad = the gradient of loss, None when grad=False. ref_logprobs are
    token_logprobs() of the reference model. The gradient of a row depends on its whole pair, so the
    logits are read twice."""
    name = "preference_loss"
    dev = _check(name, logits, targets, ref_logprobs, mask, offsets, weights)
    if pairs < 1:
        raise ValueError(f"ctorch::{name}: pairs must be at least 1")
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    vx = _view(logits)
    need = C.lib.ctb_loss_scratch_bytes(vx, pairs, 0)
    (scratch, _keep), (logp, pair_loss, rewards, loss), (v_logp, v_pair, v_rewards, v_loss) = _results(
        logits, dev, logits.shape[:-1], 1, (pairs, 2 * pairs), need)
    _run(name, dev, C.lib.ctb_preference_loss, vx, _view(targets), pairs, _view(offsets), _view(ref_logprobs),
         _view(mask), _view(weights), _scale(weights, (pairs,)), beta, label_smoothing, int(average), v_loss, v_pair,
         v_rewards, v_logp, _view(g), _status(name, status, dev), scratch, need)
    return PreferenceLoss(loss, pair_loss, rewards, logp, g)
