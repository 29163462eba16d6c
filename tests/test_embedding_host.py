"""CPU checks of the embedding and preference calls: argument checks of the
Python wrappers, and host checks of the C ABI before any device work."""

import pytest

torch = pytest.importorskip("torch")

from modern_fm_b200 import _lib, embedding, preference  # noqa: E402

I64 = torch.int64


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("kw,msg", [
    (dict(table=_t(4, 3, dtype=torch.int32)), "table must be"),
    (dict(table=_t(4, 3).t()), "contiguous rows"),
    (dict(table=_t(1, 3).expand(4, 3)), "must not overlap"),
    (dict(table=_t(4, 0)), "width must be >= 1"),
    (dict(ids=_t(5)), "ids must be"),
    (dict(ids=_t(10, dtype=I64)[::2]), "ids must be"),
    (dict(scale=_t(4)), "shape of ids"),
    (dict(scale=_t(5, dtype=torch.float16)), "scale must be torch.float32"),
    (dict(table=_t(4, 3, dtype=torch.bfloat16), scale=_t(5, dtype=torch.float64)),
     "scale must be torch.float32"),
    (dict(indptr=_t(3, dtype=torch.int32)), "indptr must be"),
    (dict(indptr=_t(0, dtype=I64)), "indptr must be"),
    (dict(ids=_t(5, 1, dtype=I64), indptr=_t(3, dtype=I64)), "ids must be 1-D"),
    (dict(), "must be a CUDA tensor"),
])
def test_lookup_refusals(kw, msg):
    a = dict(table=_t(4, 3), ids=_t(5, dtype=I64))
    a.update(kw)
    with pytest.raises(ValueError, match=msg):
        embedding.embedding_lookup(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(grad=_t(5, 3, dtype=torch.int64)), "grad must be"),
    (dict(grad=_t(4, 3)), "one row per id"),
    (dict(grad=_t(5, 3), indptr=_t(3, dtype=I64)), "one row per CSR row"),
    (dict(n_rows=-1), "n_rows must be >= 0"),
    (dict(dtype=torch.float64), "dtype must be grad's"),
    (dict(table=_t(6, 3)), "table must have shape"),
    (dict(table=_t(7, 3, dtype=torch.float64)), "table must have grad's type"),
    (dict(scale=_t(5, dtype=torch.float64)), "scale must be torch.float32"),
    (dict(grad=_t(3, 5).t()), "contiguous rows"),
    (dict(), "must be a CUDA tensor"),
])
@pytest.mark.parametrize("f", [embedding.embedding_grad, embedding.embedding_grad_rows])
def test_gradient_refusals(kw, msg, f):
    a = dict(grad=_t(5, 3), ids=_t(5, dtype=I64), n_rows=7)
    a.update(kw)
    with pytest.raises(ValueError, match=msg):
        f(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=_t(4, 3, dtype=torch.int32)), "logits must be"),
    (dict(logits=_t(4, 0)), "at least one class"),
    (dict(logits=_t(3, 4).t()), "contiguous rows"),
    (dict(labels=_t(4)), "labels must be int32 or int64"),
    (dict(labels=_t(5, dtype=I64)), "labels must be a contiguous 1-D"),
    (dict(labels=_t(8, dtype=I64)[::2]), "labels must be a contiguous 1-D"),
    (dict(), "must be a CUDA tensor"),
])
@pytest.mark.parametrize("f", ["logprobs", "grad", "preference", "policy"])
def test_score_refusals(kw, msg, f):
    a = dict(logits=_t(4, 3), labels=_t(4, dtype=I64))
    a.update(kw)
    z = _t(4)
    with pytest.raises(ValueError, match=msg):
        if f == "logprobs":
            preference.label_logprobs(**a)
        elif f == "grad":
            preference.label_logprobs_grad(z, a["logits"], a["labels"], z)
        elif f == "preference":
            preference.preference_loss(a["logits"], a["labels"], _t(3, dtype=I64), _t(2))
        else:
            preference.policy_loss(a["logits"], a["labels"], z, z)


def test_loss_refusals():
    x, y, z = _t(4, 3), _t(4, dtype=I64), _t(4)
    with pytest.raises(ValueError, match="even number"):
        preference.preference_loss(x, y, _t(4, dtype=I64), _t(3))
    with pytest.raises(ValueError, match="reference must be"):
        preference.preference_loss(x, y, _t(5, dtype=I64), _t(3))
    with pytest.raises(ValueError, match="reference must be"):
        preference.preference_loss(x, y, _t(5, dtype=I64), _t(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="sample_weight must be"):
        preference.preference_loss(x, y, _t(5, dtype=I64), z, sample_weight=z)
    with pytest.raises(ValueError, match="advantages must be"):
        preference.policy_loss(x, y, z, _t(3))
    with pytest.raises(ValueError, match="old_logprobs must be"):
        preference.policy_loss(x.double(), y, z, z)


def _lookup(dtype=1, ids=16, n=4, indptr=None, n_out=4, n_rows=5, d=3, ld=3, out=16, ld_out=3,
            table=16):
    return _lib.lib().mfm_embedding_lookup_device(dtype, 0, 1, ids, n, indptr, n_out, None, 1.0,
                                                  table, n_rows, d, ld, out, ld_out, None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=5), -1, "unknown dtype 5"),
    (dict(dtype=-1), -1, "unknown dtype -1"),
    (dict(n=-1, n_out=-1), -1, "negative embedding size"),
    (dict(d=0), -1, "width must be >= 1"),
    (dict(ids=None), -1, "ids must be provided"),
    (dict(n_out=3), -1, "n_out 3 != n_entries 4"),
    (dict(table=None), -1, "table and out"),
    (dict(out=None), -1, "table and out"),
    (dict(ld=2), -1, "row pitch of table 2 < 3"),
    (dict(ld_out=2), -1, "row pitch of out 2 < 3"),
    (dict(n_rows=2**31), -2, "2^31-1 limit"),
])
def test_lookup_host_checks(kw, code, msg):
    assert _lookup(**kw) == code
    assert msg in _lib.last_error()


def _grad(dtype=1, out_dtype=1, ids=16, n=4, n_rows=5, d=3, grad=16, ld=3, table=None, d_table=256,
          keys=None, rows=None, count=None, d_scale=None):
    return _lib.lib().mfm_embedding_grad_device(
        dtype, out_dtype, 0, 1, ids, n, None, n, None, 1.0, grad, ld, table, 3, n_rows, d, d_table,
        keys, rows, count, d_scale, 256, 1 << 40, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=7), "unknown dtype 7"),
    (dict(d_table=None), "exactly one of"),
    (dict(keys=16), "exactly one of"),
    (dict(d_table=None, keys=16, rows=16), "exactly one of"),
    (dict(out_dtype=0), "out_dtype 0 does not go with dtype 1"),
    (dict(dtype=3, out_dtype=4), "out_dtype 4 does not go with dtype 3"),
    (dict(grad=None), "grad must be provided"),
    (dict(ld=2), "row pitch of grad 2 < 3"),
    (dict(d_scale=16), "table must be provided for d_scale"),
])
def test_gradient_host_checks(kw, msg):
    assert _grad(**kw) == _lib.MFM_ERR_INVALID
    assert msg in _lib.last_error()


def test_gradient_workspace_sizes():
    f = _lib.lib().mfm_embedding_grad_workspace_bytes
    assert f(1, 0, 0, 10, 4) == 0 and f(1, 1, -1, 10, 4) == 0
    assert f(1, 0, 256, 10, 4) == 0  # a few ids need none
    assert 0 < f(1, 0, 257, 10, 4) <= f(0, 0, 257, 10, 4) <= f(0, 0, 100000, 10, 4)
    assert f(1, 1, 100000, 1 << 20, 4) < f(1, 0, 100000, 1 << 20, 4)


def test_score_host_checks():
    L = _lib.lib()
    assert L.mfm_label_logprobs_device(2, 0, 16, 3, 4, 3, 1, 16, None, 0, 16, 16, None, None) == -1
    assert "unknown dtype 2" in _lib.last_error()
    assert L.mfm_label_logprobs_device(1, 0, 16, 2, 4, 3, 1, 16, None, 0, 16, 16, None, None) == -1
    assert "row pitch of logits 2 < 3" in _lib.last_error()
    assert L.mfm_label_logprobs_device(1, 0, 16, 3, 4, 0, 1, 16, None, 0, 16, 16, None, None) == -1
    assert "n_classes >= 1" in _lib.last_error()
    assert L.mfm_label_logprobs_device(1, 0, 16, 3, 4, 3, 1, 16, None, 2, 16, 16, 16, None) == -1
    assert "sums need indptr" in _lib.last_error()

    def pref(eps=0.0, ws=256, nbytes=1 << 40, indptr=16, ld_out=3):
        return L.mfm_preference_loss_device(1, 0, 16, 3, 4, 3, 1, 16, indptr, 1, 16, 0.1, eps, None,
                                            16, 16, 16, 16, ld_out, ws, nbytes, None)

    for kw, msg in ((dict(eps=1.5), "label_smoothing"), (dict(ws=None), "workspace of"),
                    (dict(nbytes=8), "workspace of 8 bytes"), (dict(ws=264), "256-byte aligned"),
                    (dict(indptr=None), "indptr and loss"), (dict(ld_out=1), "row pitch of d_logits")):
        assert pref(**kw) == -1 and msg in _lib.last_error(), msg

    def policy(lo=0.2, hi=0.2, kl=0.0, old=16, ws=256):
        return L.mfm_policy_loss_device(1, 0, 16, 3, 4, 3, 1, 16, old, 16, None, lo, hi, kl, None,
                                        16, 16, None, 3, ws, 1 << 40, None)

    for kw, msg in ((dict(lo=1.5), "clip_low"), (dict(hi=-0.1), "clip_high"),
                    (dict(kl=0.1), "kl_coef needs reference"), (dict(old=None), "old_logprobs"),
                    (dict(ws=None), "workspace of")):
        assert policy(**kw) == -1 and msg in _lib.last_error(), msg


@pytest.mark.parametrize("f", [embedding.embedding_grad, embedding.embedding_grad_rows])
@pytest.mark.parametrize("grad,ids,msg", [
    (_t(3), _t(dtype=I64), "must be a CUDA tensor"),  # one id without an axis: passes the shapes
    (_t(2, 4, 3).transpose(0, 1), _t(4, 2, dtype=I64), "must be a CUDA tensor"),
    (_t(2, 4, 0), _t(2, 4, dtype=I64), "width must be >= 1"),
    (_t(3), _t(1, dtype=I64), "matrix with contiguous rows"),
    (_t(2, 5, 3), _t(2, 4, dtype=I64), "one row per id"),
])
def test_gradient_of_ids_of_any_shape(f, grad, ids, msg):
    with pytest.raises(ValueError, match=msg):
        f(grad, ids, 7)


def test_rows_too_long_to_be_summed():
    d = 65536 * 32 + 1  # odd: a value a lane
    got = _lib.lib().mfm_embedding_lookup_device(1, 0, 1, 16, 4, 16, 4, None, 1.0, 16, 5, d, d, 16, d,
                                                 None)
    assert got == -2 and "too long to be summed" in _lib.last_error()


def test_workspace_of_the_most_entries():
    """The sort of the most entries counts digits of 8 bits."""
    f = _lib.lib().mfm_embedding_grad_workspace_bytes
    n, rows = 2**31 - 1, 2**23
    wide, narrow = f(1, 1, n - 2048, rows, 1), f(1, 1, n, rows, 1)
    # 2 passes of 2^20 tiles' 2^12 digits against 3 passes of their 2^8
    assert wide - narrow > (2 * 2**12 - 3 * 2**8) * 2**20 * 4 - 2**20
