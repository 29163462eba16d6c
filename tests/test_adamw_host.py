"""CPU checks of the AdamW step: the C ABI's refusals come before any device work, and the
Python class refuses what it cannot step."""

import ctypes as ct

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from modern_fm_b200 import _lib  # noqa: E402
from modern_fm_b200.optim import AdamW  # noqa: E402

F64, F32, BF16, F16 = _lib.MFM_DTYPE_F64, _lib.MFM_DTYPE_F32, _lib.MFM_DTYPE_BF16, _lib.MFM_DTYPE_F16


def _call(hyper=None, ws=256, ws_bytes=1 << 20, step=256, norm=256, **tensor):
    """A step over one tensor whose pointers are never followed: each case fails before."""
    t = np.zeros(1, _lib.ADAMW_TENSOR)
    for k, v in dict(dict(param=256, grad=256, m=256, v=256, n_rows=1, d=4, ld=4, dtype=F32,
                          grad_dtype=F32), **tensor).items():
        t[k] = v
    h = _lib.AdamW(**dict(dict(learning_rate=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-8,
                               grad_scale=1.0, max_norm=-1.0, state_bits=32), **(hyper or {})))
    return _lib.lib().mfm_adamw_step_device(0, t.ctypes.data, 1, ct.byref(h), step, norm, ws,
                                            ws_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(hyper=dict(beta_1=1.0)), "beta_1 and beta_2"),
    (dict(hyper=dict(beta_2=-0.1)), "beta_1 and beta_2"),
    (dict(hyper=dict(beta_2=float("nan"))), "beta_1 and beta_2"),
    (dict(hyper=dict(epsilon=0.0)), "epsilon"),
    (dict(hyper=dict(state_bits=16)), "state_bits"),
    (dict(hyper=dict(max_norm=float("nan"))), "max_norm"),
    (dict(hyper=dict(max_norm=1.0), norm=None), "max_norm needs norm"),
    (dict(ws=None), "workspace of"),
    (dict(ws_bytes=8), "workspace of 8 bytes"),
    (dict(ws=264), "256-byte aligned"),
    (dict(step=None), "step must be provided"),
    (dict(dtype=7), "unknown dtype 7"),
    (dict(grad_dtype=BF16), "grad_dtype must be dtype"),
    (dict(dtype=BF16, grad_dtype=F16), "grad_dtype must be dtype"),
    (dict(d=-1), "must be >= 0"),
    (dict(n_rows=2), "n_rows = 1"),
    (dict(master=256), "16-bit parameters"),
    (dict(m=0), "must be provided"),
    (dict(param=258), "multiple of its element's size"),
    (dict(hyper=dict(state_bits=8)), "must be provided"),
    (dict(hyper=dict(state_bits=8), dtype=F64, grad_dtype=F64), "at most 32 bits"),
    (dict(keys=256, n_rows=5, n_keys=2), "count and row_steps"),
    (dict(keys=256, count=256, row_steps=256, n_rows=5, n_keys=-1), r"\[0, 2\^31\)"),
    (dict(keys=256, count=256, row_steps=256, n_rows=5, n_keys=2, ld=3), "row pitch"),
])
def test_abi_refuses(kw, msg):
    import re
    assert _call(**kw) == _lib.MFM_ERR_INVALID
    assert re.search(msg, _lib.last_error())


def test_tensor_layout_is_the_header_s():
    """Ten pointers, four sizes, a float64 and three ints."""
    assert _lib.ADAMW_TENSOR.itemsize == 8 * 15 + 16
    assert _lib.ADAMW_TENSOR.fields["dtype"][1] == 8 * 15
    assert ct.sizeof(_lib.AdamW) == 8 * 8 + 8


def test_moments_refuses():
    f = _lib.lib().mfm_adamw_moments_device
    assert f(0, 1, 16, 16, -1, 16, None) == _lib.MFM_ERR_INVALID
    assert f(0, 1, None, 16, 4, 16, None) == _lib.MFM_ERR_INVALID
    assert f(0, 1, None, None, 0, None, None) == _lib.MFM_OK


@pytest.mark.parametrize("kw,msg", [
    (dict(params=[]), "at least one parameter"),
    (dict(state_bits=16), "state_bits"),
    (dict(betas=(0.9, 1.0)), "betas"),
    (dict(eps=0.0), "eps"),
    (dict(seed=-1), "seed"),
    (dict(weight_decay=[0.1, 0.1]), "one value per parameter"),
    (dict(by_rows=[True, False]), "one value per parameter"),
    (dict(params=[torch.zeros(3, dtype=torch.int32)]), "parameters must be"),
    (dict(), "must be a CUDA tensor"),
])
def test_constructor_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        AdamW(**dict(dict(params=[torch.zeros(3)]), **kw))
