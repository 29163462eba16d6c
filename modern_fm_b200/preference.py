"""Losses of class scores by the log-probabilities of their labels, and what else a row
of scores says (mfm_label_logprobs_*, mfm_preference_loss_device,
mfm_policy_loss_device, mfm_label_alternatives_* in the C ABI).

The softmax models' class scores (``DeviceModel.predict_device`` with n_classes
>= 2, or any (n_tokens, n_classes) matrix) are a policy over the classes. These
calls give the log-probability of each row's label, the paired preference loss
over sequences of rows against a reference, the clipped policy loss with a KL
term, and the label's rank, the entropy and the best classes, each with the
gradient of the scores; the engine's own losses (logistic, squared, softmax) exist
inside ``fit`` and in ``evaluate``.

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


class LabelAlternatives(NamedTuple):
    """``logprobs`` and ``ranks`` of the labels (None without labels), ``lse`` and
    ``entropy`` per row; ``top_ids`` and ``top_logprobs`` (n_rows, top), or None."""
    logprobs: Optional[object]
    lse: object
    entropy: object
    ranks: Optional[object]
    top_ids: Optional[object]
    top_logprobs: Optional[object]


def _scores(logits, labels):
    """(dtype code, arithmetic type, pointer, rows, classes, pitch, labels64) of the scores;
    labels None: none, with 64-bit ids."""
    code = _STORAGE.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float64, float32, bfloat16 or float16")
    p, n, c, ld = _matrix("logits", logits)
    if c < 1:
        raise ValueError("logits must have at least one class")
    kind = torch.int64 if labels is None else labels.dtype
    if kind is not torch.int64 and kind is not torch.int32:
        raise ValueError("labels must be int32 or int64")
    if labels is not None:
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


def label_alternatives(logits, labels=None, top: int = 0, stream=None) -> LabelAlternatives:
    """What a row of class scores says besides its label's log-probability.

    ``logprobs`` and ``lse`` as ``label_logprobs`` has them, the ``entropy``
    ``-sum p log p``, the label's ``rank`` in the order of falling score (0: the best;
    classes of one score by index), and the first ``top`` classes of that order with
    their log-probabilities, ``top`` at most 32 and the number of classes. ``ranks`` and
    ``top_ids`` have the labels' type (int64 without labels). A class of score
    -infinity has probability 0 and its place in the order. Masked rows have
    log-probabilities and entropy 0, rank and ids -1, and lse 0 (rows whose every score is
    -infinity: lse -infinity); rows with a NaN or +infinity have NaN and -1.
    """
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    top = int(top)
    if not 0 <= top <= min(32, c):
        raise ValueError("top must be between 0 and 32, and at most the number of classes")
    dev = _one_device(logits, labels)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, labels)
    some, kind = (0, torch.int64) if labels is None else (n, labels.dtype)
    lps = ranks = ids = None
    with ctx:
        values = logits.new_empty(some + n * (2 + top), dtype=wide)
        if labels is not None:
            ranks = torch.empty_like(labels)
        if top:
            ids = logits.new_empty((n, top), dtype=kind)
    at, size = values.data_ptr(), values.element_size()
    _fail(_lib.lib().mfm_label_alternatives_device(
        code, dev, p, ld, n, c, l64, _ptr(labels), top, at if some else None, at + size * some,
        at + size * (some + n), _ptr(ranks), _ptr(ids), at + size * (some + 2 * n) if top else None,
        s))
    if top:
        lp, lse, entropy, lps = values.split_with_sizes((some, n, n, n * top))
        lps = lps.view(n, top)
    else:
        lp, lse, entropy = values.split_with_sizes((some, n, n))
    return LabelAlternatives(None if labels is None else lp, lse, entropy, ranks, ids, lps)


def label_alternatives_grad(logits, lse, entropy=None, labels=None, grad_logprobs=None,
                            grad_entropy=None, top_ids=None, grad_top=None, stream=None):
    """Gradient of the logits, in their type, for the gradients of ``label_alternatives``'
    log-probabilities, entropy and best classes' log-probabilities, each of which may be
    None: ``[sum of the log-probabilities' gradients at class c] - p[c] (their sum over
    the row + grad_entropy (log p[c] + entropy))``. ``lse``, ``entropy`` and ``top_ids`` are
    the forward's; ids outside the classes have no part in it, a class named twice has the
    sum."""
    code, wide, p, n, c, ld, l64 = _scores(logits, labels)
    _vector("lse", lse, n, wide)
    if grad_logprobs is not None:
        if labels is None:
            raise ValueError("grad_logprobs needs labels")
        _vector("grad_logprobs", grad_logprobs, n, wide)
    if grad_entropy is not None:
        if entropy is None:
            raise ValueError("grad_entropy needs entropy")
        _vector("entropy", entropy, n, wide)
        _vector("grad_entropy", grad_entropy, n, wide)
    top = 0
    if (top_ids is None) != (grad_top is None):
        raise ValueError("top_ids and grad_top go together")
    if top_ids is not None:
        kind = torch.int64 if l64 else torch.int32
        top = top_ids.shape[-1] if top_ids.dim() == 2 else -1
        if not 0 <= top <= 32 or top_ids.dtype != kind or tuple(top_ids.shape) != (n, top) \
                or not top_ids.is_contiguous():
            raise ValueError(f"top_ids must be a contiguous {kind} matrix of one row per row of "
                             "logits and at most 32 columns")
        if grad_top.dtype != wide or grad_top.shape != top_ids.shape or not grad_top.is_contiguous():
            raise ValueError(f"grad_top must be contiguous, {wide} and have the shape of top_ids")
    dev = _one_device(logits, lse, entropy, labels, grad_logprobs, grad_entropy, top_ids, grad_top)
    s, ctx = _on(stream, dev)
    _hold(stream, logits, lse, entropy, labels, grad_logprobs, grad_entropy, top_ids, grad_top)
    with ctx:
        out = logits.new_empty((n, c))
    _fail(_lib.lib().mfm_label_alternatives_grad_device(
        code, dev, p, ld, n, c, l64, _ptr(labels), lse.data_ptr(), _ptr(entropy),
        _ptr(grad_logprobs), _ptr(grad_entropy), top, _ptr(top_ids), _ptr(grad_top),
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
