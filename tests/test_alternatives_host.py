"""CPU checks of the label alternatives: the C ABI's refusals come before any device work."""

import pytest

torch = pytest.importorskip("torch")

from modern_fm_b200 import _lib  # noqa: E402
from modern_fm_b200.preference import label_alternatives, label_alternatives_grad  # noqa: E402


def _forward(dtype=_lib.MFM_DTYPE_F32, logits=256, ld=10, n=3, c=10, labels=256, top=2, lp=256, lse=256,
             entropy=256, ranks=256, ids=256, lps=256):
    return _lib.lib().mfm_label_alternatives_device(dtype, 0, logits, ld, n, c, 1, labels, top, lp, lse, entropy,
                                                    ranks, ids, lps, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "unknown dtype 2"),
    (dict(n=-1), "must be >= 0"),
    (dict(c=0), "n_classes >= 1"),
    (dict(logits=None, labels=None), "must be provided"),
    (dict(ld=9), "row pitch"),
    (dict(top=-1), "top must be"),
    (dict(top=33, c=100, ld=100), "top must be"),
    (dict(top=11), "top must be"),
    (dict(lse=None), "lse and entropy"),
    (dict(entropy=None), "lse and entropy"),
    (dict(labels=None), "go with labels"),
    (dict(lp=None), "go with labels"),
    (dict(ranks=None), "go with labels"),
    (dict(ids=None), "top_ids and top_logprobs"),
])
def test_forward_refuses(kw, msg):
    assert _forward(**kw) == _lib.MFM_ERR_INVALID and msg in _lib.last_error()


def test_too_many_and_none():
    assert _forward(n=2**31) == _lib.MFM_ERR_UNSUPPORTED
    assert _forward(n=0, logits=None, labels=None, lp=None, lse=None, ranks=None) == _lib.MFM_OK


def _backward(ld_out=10, lse=256, entropy=256, g_lp=256, g_h=256, top=2, ids=256, g_top=256, out=256, labels=256):
    return _lib.lib().mfm_label_alternatives_grad_device(_lib.MFM_DTYPE_F32, 0, 256, 10, 3, 10, 1, labels, lse,
                                                         entropy, g_lp, g_h, top, ids, g_top, out, ld_out, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(top=33), "top must be"),
    (dict(lse=None), "lse and d_logits"),
    (dict(out=None), "lse and d_logits"),
    (dict(labels=None), "grad_logprobs needs labels"),
    (dict(entropy=None), "grad_entropy needs entropy"),
    (dict(ids=None), "top_ids and grad_top"),
    (dict(g_top=None), "top_ids and grad_top"),
    (dict(ld_out=9), "row pitch"),
])
def test_gradient_refuses(kw, msg):
    assert _backward(**kw) == _lib.MFM_ERR_INVALID and msg in _lib.last_error()


def test_python_refuses():
    x, y = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    lse = torch.zeros(3)
    for f, msg in [
            (lambda: label_alternatives(x, y, top=33), "top must be"),
            (lambda: label_alternatives(x, y, top=11), "top must be"),
            (lambda: label_alternatives(x, y, top=-1), "top must be"),
            (lambda: label_alternatives(x, y[:2]), "labels must be"),
            (lambda: label_alternatives(x, y.float()), "labels must be"),
            (lambda: label_alternatives(x.int(), y), "logits must be"),
            (lambda: label_alternatives(x, y), "CUDA tensor"),
            (lambda: label_alternatives(x), "CUDA tensor"),
            (lambda: label_alternatives_grad(x, lse[:2]), "lse must be"),
            (lambda: label_alternatives_grad(x, lse, grad_logprobs=lse), "needs labels"),
            (lambda: label_alternatives_grad(x, lse, grad_entropy=lse), "needs entropy"),
            (lambda: label_alternatives_grad(x, lse, lse.double(), grad_entropy=lse), "entropy must be"),
            (lambda: label_alternatives_grad(x, lse, top_ids=y[:, None]), "go together"),
            (lambda: label_alternatives_grad(x, lse, top_ids=y, grad_top=lse), "top_ids must be"),
            (lambda: label_alternatives_grad(x, lse, top_ids=y[:, None].int(), grad_top=lse[:, None]), "top_ids must be"),
            (lambda: label_alternatives_grad(x, lse, top_ids=torch.zeros(3, 33, dtype=torch.int64),
                                             grad_top=torch.zeros(3, 33)), "top_ids must be"),
            (lambda: label_alternatives_grad(x, lse, top_ids=y[:, None], grad_top=torch.zeros(3, 2)), "grad_top must be"),
            (lambda: label_alternatives_grad(x, lse, labels=y, grad_logprobs=lse), "CUDA tensor")]:
        with pytest.raises(ValueError, match=msg):
            f()
