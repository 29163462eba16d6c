"""AdamW over many tensors at once (mfm_adamw_* in the C ABI).

``embedding_grad``, ``embedding_grad_rows`` and the class-score losses return
gradients; this steps the parameters they belong to, in one launch for all tensors
of a type (the engine's own optimizers step its models inside ``fit``). Tables of
latent rows may be stepped by the rows that a batch touched, each with a step count
of its own, as the engine's lazy Adam does (rust/src/optimizer.rs:68-85).

All tensors are CUDA tensors on one device. A step runs on ``stream`` (a
torch.cuda.Stream, default the current one of that device) and neither synchronises
nor copies to the host, and the step count lives on the device, so a step can be
captured into a CUDA graph. Parameters are written in place, without a trace in
torch's autograd. Every sum has a fixed order: results are bitwise reproducible. An
``AdamW`` and its state are made on the current stream, and stepped by one thread and
on one stream at a time.
"""

from __future__ import annotations

import ctypes as ct
from operator import attrgetter
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import _lib
from .embedding import _STORAGE, EmbeddingRows, _fail, _hold, _matrix, _on, _ptr

_HALVES = (torch.bfloat16, torch.float16)
_BLOCK = 32  # values that share an exponent; every tensor's moments begin at a multiple of it


class AdamWState(NamedTuple):
    """What a step changes besides the parameters, to be kept in a checkpoint and handed to
    a new ``AdamW``: the 0-dim int64 ``step`` count; the moments ``m`` and ``v`` of all
    tensors behind each other (``AdamW.view`` gives one tensor's), float32 or float64, or
    codes of 8 bits with one exponent byte for each 32 in ``m_exp`` and ``v_exp``;
    ``master`` weights (float32) of the 16-bit parameters; ``row_steps`` (int32) of the
    tables that are stepped by rows. None where there are none."""
    step: object
    m: object
    v: object
    m_exp: Optional[object] = None
    v_exp: Optional[object] = None
    master: Optional[object] = None
    row_steps: Optional[object] = None


def _each(name, value, n, kind):
    """`value` for each of n tensors."""
    if isinstance(value, (list, tuple)):
        if len(value) != n:
            raise ValueError(f"{name} must have one value per parameter")
        return [kind(v) for v in value]
    return [kind(value)] * n


class AdamW:
    """One step per call of ``step``, in float32 for 16- and 32-bit parameters, in float64
    for float64 ones, with t the number of the step and s the gradients' factor:

        g = s * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p -= lr weight_decay p + lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

    ``params``: contiguous float32, bfloat16 or float16 tensors, or all float64, none of
    them overlapping; ``weight_decay`` one number or one per parameter. ``state_bits`` 8
    keeps the moments in 8 bits (not for float64): blocks of 32 values share an exponent,
    a value has 3 bits of mantissa and 15 (m) or 31 (v) octaves below its block's largest;
    m is rounded to nearest, v up or down at random in proportion, by bits that ``seed``, the
    step and the value's place give: the average is kept where steps of a thousandth are below the
    code's. ``master`` keeps float32 copies of the 16-bit parameters and steps those.
    ``by_rows`` (one truth value, or one per parameter) marks matrices with contiguous
    rows of any pitch that are stepped by touched rows: their gradient is an
    ``EmbeddingRows``, t is the row's own count, rows that are not touched stay as they
    are, without decay, and their 8-bit blocks end with the row. ``state`` is that of an
    ``AdamW`` of the same parameters and options, used in place.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay=0.01, state_bits: int = 32, master: bool = False, by_rows=False,
                 seed: int = 0, state: Optional[AdamWState] = None):
        self.params = list(params)
        n = len(self.params)
        if n < 1:
            raise ValueError("there must be at least one parameter")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 32 or 8")
        b1, b2 = (float(b) for b in betas)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError("betas must be in [0, 1)")
        if not eps >= 1.2e-38:
            raise ValueError("eps must be at least 2^-126")
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError("seed must be in [0, 2^32)")
        decay = _each("weight_decay", weight_decay, n, float)
        rows = self._by_rows = _each("by_rows", by_rows, n, bool)
        self.lr, self._bits = float(lr), int(state_bits)
        self._kinds, self._shapes = [p.dtype for p in self.params], [p.shape for p in self.params]
        table = self._table = np.zeros(n, _lib.ADAMW_TENSOR)
        self._at, self._dims, self._master_at = [], [], []
        size = master_size = n_steps = 0
        for i, p in enumerate(self.params):
            code = _STORAGE.get(p.dtype)
            if code is None:
                raise ValueError("parameters must be float64, float32, bfloat16 or float16")
            if not p.is_cuda or p.get_device() != self.params[0].get_device():
                raise ValueError("every parameter must be a CUDA tensor on one device")
            if rows[i]:
                at, n_rows, d, ld = _matrix(f"parameter {i}", p)
                if n_rows >= 1 << 31 or d >= 1 << 31:
                    raise ValueError("a table has at most 2^31 - 1 rows and columns")
            elif not p.is_contiguous():
                raise ValueError(f"parameter {i} must be contiguous")
            else:
                at, n_rows, d, ld = p.data_ptr(), 1, p.numel(), p.numel()
            pitch = -(-d // _BLOCK) * _BLOCK if state_bits == 8 else d
            own = -(-n_rows * pitch // _BLOCK) * _BLOCK
            self._at.append(size)
            self._dims.append((n_rows, d, pitch))
            self._master_at.append(master_size)
            t = table[i]
            t["param"], t["n_rows"], t["d"], t["ld"], t["dtype"] = at, n_rows, d, ld, code
            t["grad_dtype"], t["weight_decay"] = code, decay[i]
            size += own
            master_size += own if master and p.dtype in _HALVES else 0
            n_steps += n_rows if rows[i] else 0
        wide = [p.dtype == torch.float64 for p in self.params]
        if any(wide) and not all(wide):
            raise ValueError("float64 parameters are stepped apart from others")
        if wide[0] and state_bits == 8:
            raise ValueError("8-bit moments are for parameters of at most 32 bits")
        self._wide = torch.float64 if wide[0] else torch.float32
        self._device = self.params[0].get_device()
        spans = sorted((int(t["param"]), int(t["param"]) + p.element_size() * int(
            (t["n_rows"] - 1) * t["ld"] + t["d"])) for t, p in zip(table, self.params) if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters must not overlap")
        self._some_by_rows, self._codes = any(rows), table["dtype"].copy()
        self._table_at = table.ctypes.data
        self.state = self._states(size, master_size, n_steps, state, master)
        self._lay_out(master)
        new = self.params[0].new_zeros
        self._work = new(_lib.lib().mfm_adamw_workspace_bytes(), dtype=torch.uint8)
        self._hyper = _lib.AdamW(self.lr, b1, b2, float(eps), 1.0, -1.0, None, None, int(seed),
                                 self._bits)

    def _states(self, size, master_size, n_steps, given, master):
        eight = self._bits == 8
        want = dict(step=((), torch.int64), m=((size,), torch.uint8 if eight else self._wide),
                    v=((size,), torch.uint8 if eight else self._wide),
                    m_exp=((size // _BLOCK,), torch.uint8) if eight else None,
                    v_exp=((size // _BLOCK,), torch.uint8) if eight else None,
                    master=((master_size,), torch.float32) if master_size else None,
                    row_steps=((n_steps,), torch.int32) if n_steps else None)
        if given is None:
            new = self.params[0].new_zeros
            s = AdamWState(**{k: None if w is None else new(w[0], dtype=w[1])
                              for k, w in want.items()})
            if master_size:
                for i, p in enumerate(self.params):
                    if p.dtype in _HALVES:
                        self._view(s.master, self._master_at[i], i).copy_(p.detach())
            return s
        for k, w in want.items():
            t = getattr(given, k)
            if (t is None) != (w is None):
                raise ValueError(f"state.{k} must be {'None' if w is None else 'given'}")
            if t is not None and (tuple(t.shape) != w[0] or t.dtype != w[1] or not t.is_contiguous()
                                  or t.get_device() != self._device or not t.is_cuda):
                raise ValueError(f"state.{k} must be a contiguous {w[1]} tensor of shape {w[0]} on "
                                 f"cuda:{self._device}")
        return given

    def _lay_out(self, master):
        s, table = self.state, self._table
        size, steps = s.m.element_size(), 0
        for i, p in enumerate(self.params):
            t, at = table[i], self._at[i]
            t["m"], t["v"] = s.m.data_ptr() + at * size, s.v.data_ptr() + at * size
            if self._bits == 8:
                t["m_exp"] = s.m_exp.data_ptr() + at // _BLOCK
                t["v_exp"] = s.v_exp.data_ptr() + at // _BLOCK
            if master and p.dtype in _HALVES and s.master is not None:
                t["master"] = s.master.data_ptr() + 4 * self._master_at[i]
            if self._by_rows[i] and s.row_steps is not None:
                t["row_steps"] = s.row_steps.data_ptr() + 4 * steps
                steps += self._dims[i][0]

    def _view(self, flat, at, i):
        n_rows, d, pitch = self._dims[i]
        return flat[at:at + n_rows * pitch].view(n_rows, pitch)[:, :d].view(self._shapes[i]) if (
            pitch == d or n_rows == 1) else flat[at:at + n_rows * pitch].view(n_rows, pitch)[:, :d]

    def view(self, flat, i: int):
        """Parameter i's part of a tensor laid out as the moments are (``moments``,
        ``state.m``), in the parameter's shape."""
        return self._view(flat, self._at[i], i)

    def moments(self, stream=None):
        """(m, v) of all tensors behind each other: the state's own in 32 bits, new bfloat16
        tensors, in which they are exact, for codes of 8 bits."""
        st = self.state
        if self._bits != 8:
            return st.m, st.v
        s, ctx = _on(stream, self._device)
        _hold(stream, st.m, st.v, st.m_exp, st.v_exp)
        with ctx:
            out = [st.m.new_empty(st.m.shape, dtype=torch.bfloat16) for _ in range(2)]
        L = _lib.lib()
        for signed, code, exps, to in ((1, st.m, st.m_exp, out[0]), (0, st.v, st.v_exp, out[1])):
            _fail(L.mfm_adamw_moments_device(self._device, signed, code.data_ptr(), exps.data_ptr(),
                                             code.numel(), to.data_ptr(), s))
        return out[0], out[1]

    def _number(self, name, value):
        """(number, device address or None) of a factor."""
        if not torch.is_tensor(value):
            return float(value), None
        if value.dtype != torch.float64 or value.dim() != 0 or value.get_device() != self._device \
                or not value.is_cuda:
            raise ValueError(f"{name} must be a number or a 0-dim float64 tensor on "
                             f"cuda:{self._device}")
        return 1.0, value.data_ptr()

    def _gradients(self, grads):
        """Writes the gradients' addresses into the table; the tensors to be held."""
        table = self._table
        if not self._some_by_rows:
            # every one a tensor: a few passes over the list instead of a loop's body
            try:
                at = list(map(torch.Tensor.data_ptr, grads))
            except TypeError:
                at = None
            if at is not None:
                if list(map(attrgetter("shape"), grads)) != self._shapes:
                    raise ValueError("every gradient must have its parameter's shape")
                if not all(map(torch.Tensor.is_contiguous, grads)):
                    raise ValueError("gradients must be contiguous")
                if set(map(torch.Tensor.get_device, grads)) != {self._device}:
                    raise ValueError("every gradient must be a CUDA tensor on the parameters' device")
                kinds = list(map(attrgetter("dtype"), grads))
                if kinds != self._kinds:
                    for i, (k, p) in enumerate(zip(kinds, self._kinds)):
                        self._check_kind(i, k, p)
                    table["grad_dtype"] = [_STORAGE[k] for k in kinds]
                else:
                    table["grad_dtype"] = self._codes
                table["grad"] = at
                return grads
        held = []
        for i, g in enumerate(grads):
            t = table[i]
            t["grad"] = 0
            if g is None:
                continue
            if self._by_rows[i]:
                n_rows, d, _ = self._dims[i]
                if not isinstance(g, EmbeddingRows):
                    raise ValueError(f"parameter {i} is stepped by rows: its gradient is an "
                                     "EmbeddingRows")
                keys, rows, count = g.keys, g.rows, g.count
                if (keys.dtype not in (torch.int32, torch.int64) or keys.dim() != 1
                        or not keys.is_contiguous()):
                    raise ValueError("keys must be a contiguous 1-D int32 or int64 tensor")
                if tuple(rows.shape) != (keys.numel(), d) or not rows.is_contiguous():
                    raise ValueError("rows must be contiguous and have one row of the table's "
                                     "width per key")
                if count.dtype != torch.int64 or count.numel() != 1:
                    raise ValueError("count must be one int64 value")
                if keys.numel() >= 1 << 31:
                    raise ValueError("there are at most 2^31 - 1 keys")
                t["keys"], t["count"], t["n_keys"] = keys.data_ptr(), count.data_ptr(), keys.numel()
                t["keys64"] = 1 if keys.dtype == torch.int64 else 0
                held += [keys, count]
                if keys.numel() == 0:
                    continue
                g = rows
            elif not isinstance(g, torch.Tensor):
                raise ValueError("the gradient of a dense parameter is a tensor")
            elif g.shape != self._shapes[i]:
                raise ValueError("every gradient must have its parameter's shape")
            elif not g.is_contiguous():
                raise ValueError("gradients must be contiguous")
            self._check_kind(i, g.dtype, self._kinds[i])
            t["grad"], t["grad_dtype"] = g.data_ptr(), _STORAGE[g.dtype]
            held.append(g)
        if any(h.get_device() != self._device for h in held):
            raise ValueError("every gradient must be a CUDA tensor on the parameters' device")
        return held

    @staticmethod
    def _check_kind(i, kind, param):
        if kind != param and not (param in _HALVES and kind == torch.float32):
            raise ValueError(f"the gradient of parameter {i} must have its type, or float32 for "
                             "bfloat16 and float16")

    def step(self, grads, lr=None, grad_scale=1.0, max_norm: Optional[float] = None, stream=None):
        """One step by ``grads``: for each parameter a contiguous tensor of its shape, in its
        type or float32, an ``EmbeddingRows`` for one that is stepped by rows (of
        distinct ascending ids, as ``embedding_grad_rows`` returns them), or None: it stays
        as it is. ``lr`` (default: the constructor's) and ``grad_scale`` are numbers or 0-dim
        float64 CUDA tensors, which a captured step reads anew each time.

        Every gradient is multiplied by ``grad_scale`` and, with ``max_norm``, by
        ``min(1, max_norm / norm)``, norm being that of all scaled gradients together; it is
        returned (0-dim, in the arithmetic type). A norm that is not finite (or a float64 one
        beyond 1e154, whose squares are not) leaves parameters, state and step count as they
        were. Without ``max_norm`` returns None.
        """
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError("there must be one gradient, or None, per parameter")
        h = self._hyper
        h.learning_rate, h.learning_rate_at = self._number("lr", self.lr if lr is None else lr)
        h.grad_scale, h.grad_scale_at = self._number("grad_scale", grad_scale)
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError("max_norm must be >= 0")
        h.max_norm = -1.0 if max_norm is None else float(max_norm)
        held = self._gradients(grads)
        s, ctx = _on(stream, self._device)
        if stream is not None:
            numbers = [x for x in (lr, grad_scale) if torch.is_tensor(x)]
            _hold(stream, *held, *self.params, *self.state, self._work, *numbers)
        norm = None
        if max_norm is not None:
            with ctx:
                norm = self._work.new_empty((), dtype=self._wide)
        _fail(_lib.lib().mfm_adamw_step_device(
            self._device, self._table_at, len(self.params), ct.byref(h),
            self.state.step.data_ptr(), _ptr(norm), self._work.data_ptr(), self._work.numel(), s))
        return norm
