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

from collections import namedtuple

import torch

from . import _capi as C
from .errors import AliasError, DTypeError, ShapeError
from .ops import _call, _cuda, _same_view, _scratch, may_overlap

TokenLogprobs = namedtuple("TokenLogprobs", ["logprobs", "lse"])
DistillLoss = namedtuple("DistillLoss", ["loss", "row_loss", "grad"])
PolicyLoss = namedtuple("PolicyLoss", ["loss", "row_loss", "logprobs", "kl", "grad"])
PreferenceLoss = namedtuple("PreferenceLoss", ["loss", "pair_loss", "rewards", "logprobs", "grad"])

_LOGITS = (torch.float32, torch.float64, torch.bfloat16)


def _check(name, logits, *others):
    """Device and dtype checks shared by the losses; returns the device."""
    dev = _cuda(name, logits, *(t for t in others if t is not None))
    if logits.dtype not in _LOGITS:
        raise DTypeError(f"ctorch::{name}: logits must be float32, float64 or bfloat16 (got {logits.dtype})")
    for t in others:
        if t is not None and t.dtype not in C.CODE_OF_TORCH:
            raise DTypeError(f"ctorch::{name}: {t.dtype} is not supported")
    if logits.dim() == 0:
        raise ShapeError(f"ctorch::{name}: logits must have at least one dim (the vocabulary, last)")
    return dev


def _result_dtype(logits):
    return torch.float64 if logits.dtype == torch.float64 else torch.float32


def _grad_for(name, logits, out, dev):
    """The gradient's tensor: `out` (checked), or a new one whose rows lie like the logits' rows. Where
    those all start on 16 bytes although V elements are not a multiple of it (a vocabulary padded in
    memory), so do the new one's: rows of the two that are aligned alike move in 16-byte pieces."""
    if out is not None:
        _cuda(name, logits, out)
        if out.dtype != logits.dtype:
            raise DTypeError(f"ctorch::{name}: the gradient's dtype must equal the logits'")
        if out.shape != logits.shape:
            raise ShapeError(f"ctorch::{name}: the gradient's shape must equal the logits'")
        if may_overlap(out, logits) and not _same_view(out, logits):
            raise AliasError(f"ctorch::{name}: the gradient overlaps the logits without being the same view")
        return out
    shape, size, v = logits.shape, logits.element_size(), logits.shape[-1]
    if v * size % 16 and logits.dim() > 1 and logits.data_ptr() % 16 == 0 and \
            all(st * size % 16 == 0 for s, st in zip(shape[:-1], logits.stride()) if s > 1):
        pitch = -(-v * size // 128) * 128 // size
        return torch.empty((*shape[:-1], pitch), dtype=logits.dtype, device=dev)[..., :v]
    return torch.empty(shape, dtype=logits.dtype, device=dev)


def _ptr(t):
    return t.data_ptr() if t is not None else None


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
    dev = _check("token_logprobs", logits, targets, mask)
    rows, dt = logits.shape[:-1], _result_dtype(logits)
    logp = torch.empty(rows, dtype=dt, device=dev)
    lse = torch.empty(rows, dtype=dt, device=dev)
    with torch.cuda.device(dev):
        _call(C.lib.ctb_token_logprobs(C.view(logits), C.view(targets), C.view(mask), temperature, C.view(logp),
                                       C.view(lse), _status("token_logprobs", status, dev), C.stream_handle(dev)),
              "token_logprobs")
    return TokenLogprobs(logp, lse)


def token_logprobs_backward(grad_logprobs, logits, targets, logprobs, lse, mask=None, temperature: float = 1.0,
                            out=None, status=None) -> torch.Tensor:
    """The gradient of sum(grad_logprobs * logprobs) with respect to the logits; logprobs and lse are
    token_logprobs' results for the same logits, targets, mask and temperature. Written to `out` when
    given, which may be the logits themselves."""
    name = "token_logprobs_backward"
    dev = _check(name, logits, grad_logprobs, targets, logprobs, lse, mask)
    grad = _grad_for(name, logits, out, dev)
    with torch.cuda.device(dev):
        _call(C.lib.ctb_token_logprobs_backward(C.view(grad_logprobs), C.view(logits), C.view(targets),
                                                C.view(logprobs), C.view(lse), C.view(mask), temperature,
                                                C.view(grad), _status(name, status, dev), C.stream_handle(dev)), name)
    return grad


def _scale(weights, n):
    return 1.0 if weights is not None else 1.0 / max(n, 1)


def _rows(logits):
    return logits.numel() // logits.shape[-1] if logits.shape[-1] else 0


def distill_loss(logits, teacher_logits, teacher_indices, teacher_lse=None, weights=None, temperature: float = 1.0,
                 grad: bool = True, out_grad=None, status=None) -> DistillLoss:
    """Distillation from the K entries a row that a teacher finds likeliest: teacher_logits [..., K] at
    vocabulary indices teacher_indices [..., K] (all different; an entry of -inf is padding). Without
    teacher_lse the entries are renormalised; with teacher_lse [...] (the log-sum-exp of the teacher's
    whole row of logits / temperature) the mass outside them is one more event.

    row_loss = KL(teacher || student) of each row at `temperature` (not multiplied by its square);
    loss = sum(weights * row_loss), or the mean of the rows when weights is None; grad = the gradient of
    loss, None when grad=False."""
    name = "distill_loss"
    dev = _check(name, logits, teacher_logits, teacher_indices, teacher_lse, weights)
    dt = _result_dtype(logits)
    row_loss = torch.empty(logits.shape[:-1], dtype=dt, device=dev)
    loss = torch.empty((), dtype=dt, device=dev)
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    with torch.cuda.device(dev):
        vx = C.view(logits)
        need = C.lib.ctb_loss_scratch_bytes(vx, 0)
        scratch = _scratch(need, dev)
        _call(C.lib.ctb_distill_loss(vx, C.view(teacher_logits), C.view(teacher_indices), C.view(teacher_lse),
                                     C.view(weights), _scale(weights, _rows(logits)), temperature, C.view(loss),
                                     C.view(row_loss), C.view(g), _status(name, status, dev), _ptr(scratch), need,
                                     C.stream_handle(dev)), name)
    return DistillLoss(loss, row_loss, g)


def policy_loss(logits, targets, old_logprobs, advantages, ref_logprobs=None, weights=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, grad: bool = True,
                out_grad=None, status=None) -> PolicyLoss:
    """The clipped policy loss with a KL term, a row a sampled token. With logp = log p[target],
    r = exp(logp - old_logprobs), A = advantages and d = ref_logprobs - logp:

        row_loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * kl,   kl = exp(d) - 1 - d

    loss = sum(weights * row_loss), or the mean of the rows when weights is None; logprobs = logp; kl is 0
    without ref_logprobs; grad = the gradient of loss, None when grad=False."""
    name = "policy_loss"
    dev = _check(name, logits, targets, old_logprobs, advantages, ref_logprobs, weights)
    dt, rows = _result_dtype(logits), logits.shape[:-1]
    row_loss, logp, kl = (torch.empty(rows, dtype=dt, device=dev) for _ in range(3))
    loss = torch.empty((), dtype=dt, device=dev)
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    with torch.cuda.device(dev):
        vx = C.view(logits)
        need = C.lib.ctb_loss_scratch_bytes(vx, 0)
        scratch = _scratch(need, dev)
        _call(C.lib.ctb_policy_loss(vx, C.view(targets), C.view(old_logprobs), C.view(advantages),
                                    C.view(ref_logprobs), C.view(weights), _scale(weights, _rows(logits)), clip_low,
                                    clip_high, kl_coef, temperature, C.view(loss), C.view(row_loss), C.view(logp),
                                    C.view(kl), C.view(g), _status(name, status, dev), _ptr(scratch), need,
                                    C.stream_handle(dev)), name)
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
    dt = _result_dtype(logits)
    if pairs < 1:
        raise ValueError(f"ctorch::{name}: pairs must be at least 1")
    pair_loss = torch.empty(pairs, dtype=dt, device=dev)
    rewards = torch.empty(2 * pairs, dtype=dt, device=dev)
    logp = torch.empty(logits.shape[:-1], dtype=dt, device=dev)
    loss = torch.empty((), dtype=dt, device=dev)
    g = _grad_for(name, logits, out_grad, dev) if grad or out_grad is not None else None
    with torch.cuda.device(dev):
        vx = C.view(logits)
        need = C.lib.ctb_loss_scratch_bytes(vx, pairs)
        scratch = _scratch(need, dev)
        _call(C.lib.ctb_preference_loss(vx, C.view(targets), pairs, C.view(offsets), C.view(ref_logprobs),
                                        C.view(mask), C.view(weights), _scale(weights, pairs), beta, label_smoothing,
                                        int(average), C.view(loss), C.view(pair_loss), C.view(rewards), C.view(logp),
                                        C.view(g), _status(name, status, dev), _ptr(scratch), need,
                                        C.stream_handle(dev)), name)
    return PreferenceLoss(loss, pair_loss, rewards, logp, g)
