"""Losses of class scores by the log-probabilities of their labels
(mfm_label_logprobs_*, mfm_preference_loss_device, mfm_policy_loss_device in the
C ABI).

The softmax models' class scores (``DeviceModel.predict_device`` with n_classes
>= 2, or any (n_tokens, n_classes) matrix) are a policy over the classes. These
calls give the log-probability of each row's label, the paired preference loss
over sequences of rows against a reference, and the clipped policy loss with a
KL term, each with the gradient of the scores; the engine's own losses
(logistic, squared, softmax) exist inside ``fit`` and in ``evaluate``.

All calls take CUDA tensors on one device, run on ``stream`` (a
torch.cuda.Stream, default the current one of that device) and neither
synchronise nor copy to the host, so they can be captured into a CUDA graph.
``logits`` are float64, float32, bfloat16 or float16 with contiguous rows of any
pitch; labels int32 or int64, a label outside ``[0, n_classes)`` masks its row
(log-probability 0, gradient 0), as does a row whose every score is -infinity.
Everything else is in the arithmetic type: float64 for float64 logits, else
float32; sums over rows run in float64 in a fixed order. A row with a NaN or
+infinity among its scores gives NaN, unless its label masks it. The calls are not
part of torch's autograd: results carry no graph, and the gradients are what they
return.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .embedding import _STORAGE, _fail, _hold, _matrix, _on, _one_device, _ptr


class LabelLogprobs(NamedTuple):
    """``logprobs`` and log-sum-exp ``lse`` per row; ``sums`` of the log-probabilities
    per sequence, or None."""
    logprobs: object
    lse: object
    sums: Optional[object]


class PreferenceLoss(NamedTuple):
    """``loss`` (0-dim), ``margins`` (n_pairs), the sequences' ``logprobs`` (2 n_pairs),
    ``grad`` of the logits or None."""
    loss: object
    margins: object
    logprobs: object
    grad: Optional[object]


class PolicyLoss(NamedTuple):
    """``loss``, mean ``kl`` and ``clip_fraction`` (0-dim), ``logprobs`` per row,
    ``grad`` of the logits or None."""
    loss: object
    kl: object
    clip_fraction: object
    logprobs: object
    grad: Optional[object]


def _scores(logits, labels):
    """(dtype code, arithmetic type, pointer, rows, classes, pitch, labels64) of the scores."""
    code = _STORAGE.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float64, float32, bfloat16 or float16")
    p, n, c, ld = _matrix("logits", logits)
    if c < 1:
        raise ValueError("logits must have at least one class")
    kind = labels.dtype
    if kind is not torch.int64 and kind is not torch.int32:
        raise ValueError("labels must be int32 or int64")
    _vector("labels", labels, n, kind)
    wide = torch.float64 if code == _lib.MFM_DTYPE_F64 else torch.float32
    return code, wide, p, n, c, ld, 1 if kind is torch.int64 else 0


def _vector(name, t, n, dtype):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor of {n} values")


def _bounds(indptr):
    """Number of sequences of an indptr."""
    if (indptr.dtype != torch.int64 or indptr.dim() != 1 or not indptr.is_contiguous()
            or indptr.numel() < 1):
        raise ValueError("indptr must be a contiguous 1-D int64 tensor (n_sequences + 1)")
    return indptr.numel() - 1


def label_logprobs(logits, labels, indptr=None, stream=None) -> LabelLogprobs:
    """Log-probability of each row's label, ``logits[t, labels[t]] - lse[t]``, and
    ``lse[t] = log sum exp logits[t]`` (also for masked rows). With ``indptr`` (int64,
    n_sequences + 1) the log-probabilities summed over each sequence's rows too,
    as ``preference_loss`` takes its reference: added in float64 as they are returned
    and rounded to the arithmetic type (in float32 a sum near -8000 has steps of 5e-4)."""
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    n_seq = 0 if indptr is None else _bounds(indptr)
    dev = _one_device(logits, labels, indptr)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, labels, indptr)
    with ctx:
        lp = logits.new_empty(n, dtype=wide)
        lse = logits.new_empty(n, dtype=wide)
        sums = None if indptr is None else logits.new_empty(n_seq, dtype=wide)
    _fail(_lib.lib().mfm_label_logprobs_device(
        code, dev, p, ld, n, c, l64, labels.data_ptr(), _ptr(indptr), n_seq, lp.data_ptr(),
        lse.data_ptr(), sums.data_ptr() if n_seq else None, s))
    return LabelLogprobs(lp, lse, sums)


def label_logprobs_grad(grad, logits, labels, lse, stream=None):
    """Gradient of the logits for the gradient ``grad`` of ``label_logprobs``'
    log-probabilities: ``grad[t] * ([c = labels[t]] - exp(logits[t, c] - lse[t]))``, in
    the logits' type. ``lse`` is the forward's."""
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    _vector("grad", grad, n, wide)
    _vector("lse", lse, n, wide)
    dev = _one_device(logits, labels, grad, lse)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, labels, grad, lse)
    with ctx:
        out = logits.new_empty((n, c))
    _fail(_lib.lib().mfm_label_logprobs_grad_device(
        code, dev, p, ld, n, c, l64, labels.data_ptr(), grad.data_ptr(), lse.data_ptr(),
        out.data_ptr(), c, s))
    return out


def preference_loss(logits, labels, indptr, reference, beta: float = 0.1,
                    label_smoothing: float = 0.0, sample_weight=None, with_grad: bool = True,
                    stream=None) -> PreferenceLoss:
    """Paired preference loss over 2 n_pairs sequences of rows.

    ``indptr`` (int64, 2 n_pairs + 1) bounds the sequences: sequence p is the
    preferred one of pair p, sequence n_pairs + p the other. With S the
    sequences' summed label log-probabilities and R = ``reference`` (2 n_pairs,
    the same sums under the reference, from ``label_logprobs``), the margin is
    ``z = beta * ((S[p] - R[p]) - (S[n_pairs + p] - R[n_pairs + p]))`` and the loss the
    mean, weighted by ``sample_weight`` (n_pairs), of ``-(1 - e) log sigmoid(z) -
    e log sigmoid(-z)`` with e = ``label_smoothing``. Pairs of weight 0 are left
    out; weights that sum to 0 give loss and gradient 0. S is summed from unrounded
    log-probabilities, ``reference`` is in the arithmetic type: against itself a model's
    margins are 0 up to its rounding. An infinite margin (a label whose score is
    -infinity) is taken in the limit: loss 0 on the right side without smoothing.
    """
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    n_seq = _bounds(indptr)
    if n_seq % 2:
        raise ValueError("indptr must bound an even number of sequences")
    n_pairs = n_seq // 2
    _vector("reference", reference, n_seq, wide)
    if sample_weight is not None:
        _vector("sample_weight", sample_weight, n_pairs, wide)
    dev = _one_device(logits, labels, indptr, reference, sample_weight)
    L = _lib.lib()
    nbytes = L.mfm_preference_workspace_bytes(code, n, n_pairs)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, labels, indptr, reference, sample_weight)
    with ctx:
        ws = logits.new_empty(nbytes, dtype=torch.uint8)
        out = logits.new_empty(1 + 3 * n_pairs, dtype=wide)
        grad = logits.new_empty((n, c)) if with_grad else None
    at, size = out.data_ptr(), out.element_size()
    _fail(L.mfm_preference_loss_device(
        code, dev, p, ld, n, c, l64, labels.data_ptr(), indptr.data_ptr(), n_pairs,
        reference.data_ptr(), float(beta), float(label_smoothing), _ptr(sample_weight), at,
        at + size, at + size * (1 + n_pairs), _ptr(grad), c, ws.data_ptr(), nbytes, s))
    loss, margins, logprobs = out.split_with_sizes((1, n_pairs, n_seq))
    return PreferenceLoss(loss.view(()), margins, logprobs, grad)


def policy_loss(logits, labels, old_logprobs, advantages, reference=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, sample_weight=None,
                with_grad: bool = True, stream=None) -> PolicyLoss:
    """Clipped policy loss with a KL term over logged labels.

    Per unmasked row, with lp its label's log-probability, ``r = exp(lp -
    old_logprobs)`` and ``u = reference - lp``: ``-min(r A, clamp(r, 1 - clip_low, 1 +
    clip_high) A) + kl_coef (exp(u) - u - 1)`` with A = ``advantages``; the loss is
    their mean weighted by ``sample_weight`` (rows of weight 0 are left out;
    weights that sum to 0 give 0). ``old_logprobs`` (the policy the labels were
    drawn from), ``advantages``, ``reference`` (None: no KL term) and
    ``sample_weight`` hold one value per row. ``kl`` is the mean of exp(u) - u - 1
    (also with ``kl_coef`` 0, where it is only reported), ``clip_fraction`` the share of
    rows whose clipped term is the smaller one. All means are over the unmasked rows'
    weights, so rows whose every score is -infinity are in none of them.
    """
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    _vector("old_logprobs", old_logprobs, n, wide)
    _vector("advantages", advantages, n, wide)
    if reference is not None:
        _vector("reference", reference, n, wide)
    if sample_weight is not None:
        _vector("sample_weight", sample_weight, n, wide)
    dev = _one_device(logits, labels, old_logprobs, advantages, reference, sample_weight)
    L = _lib.lib()
    nbytes = L.mfm_policy_workspace_bytes(code, n)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, labels, old_logprobs, advantages, reference, sample_weight)
    with ctx:
        ws = logits.new_empty(nbytes, dtype=torch.uint8)
        stats = logits.new_empty(3, dtype=wide)
        lp = logits.new_empty(n, dtype=wide)
        grad = logits.new_empty((n, c)) if with_grad else None
    _fail(L.mfm_policy_loss_device(
        code, dev, p, ld, n, c, l64, labels.data_ptr(), old_logprobs.data_ptr(),
        advantages.data_ptr(), _ptr(reference), float(clip_low), float(clip_high), float(kl_coef),
        _ptr(sample_weight), stats.data_ptr(), lp.data_ptr(), _ptr(grad), c, ws.data_ptr(), nbytes,
        s))
    loss, kl, clipped = stats.unbind(0)
    return PolicyLoss(loss, kl, clipped, lp, grad)
