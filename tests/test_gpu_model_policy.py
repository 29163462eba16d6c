"""GPU tests of the resident model's factor sums and label log-probabilities, and
of the losses evaluated on it, against float64 NumPy and the oracle's scores.

Tolerances as in the embedding and preference tests: float64 arithmetic 1e-12
relative to the sums of magnitudes, float32 (entries + 4) 2^-24 of them.
"""

import numpy as np
import pytest
import scipy.sparse as sp

from oracle import oracle as O

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200 import preference as P  # noqa: E402
from modern_fm_b200.evaluate import policy_eval_device, preference_eval_device  # noqa: E402
from modern_fm_b200.model import DeviceModel  # noqa: E402


def _case(seed, kind, C, n=240, d=500, k=6, F=5):
    rng = np.random.default_rng(seed)
    X = sp.random(n, d, density=0.02, format="csr", random_state=seed,
                  data_rvs=lambda m: rng.lognormal(0.0, 0.5, size=m))
    X.sort_indices()
    lead = (C,) if C > 1 else ()
    w0 = rng.normal(size=C) if C > 1 else 0.3
    w = rng.normal(size=lead + (d,)) * 0.3
    V = rng.normal(size=lead + ((d, F, k) if kind == "ffm" else (d, k))) * 0.3
    R = rng.uniform(size=lead + (F, F))
    w, V, R = (a.astype(np.float32).astype(np.float64) for a in (w, V, R))
    return X, w0, w, V, R, rng.integers(0, F, size=d), rng


def _model(kind, C, dtype, X, w0, w, V, R, fid):
    m = DeviceModel(kind, X.shape[1], V.shape[-1], 0 if kind == "fm" else int(R.shape[-1]), C,
                    dtype)
    m.set_params(w0, w, V, R if kind == "fwfm" else None, None if kind == "fm" else fid)
    return m


def _csr(X, dtype):
    c = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    return (c(X.indptr, torch.int64), c(X.indices, torch.int32),
            c(X.data, torch.float32 if dtype == "float32" else torch.float64))


@pytest.mark.parametrize("kind", ["fm", "ffm", "fwfm"])
@pytest.mark.parametrize("C", [1, 3])
@pytest.mark.parametrize("dtype", ["float32-float64", "float64", "float32"])
def test_factors(kind, C, dtype):
    X, w0, w, V, R, fid, _ = _case(1, kind, C)
    with _model(kind, C, dtype, X, w0, w, V, R, fid) as m:
        got = m.factors_device(*_csr(X, dtype))
        # (C, d, ...) -> (d, ..., C, k): class next to the factors
        T = V if C == 1 else np.moveaxis(V, 0, -2)
        flat = T.reshape(X.shape[1], -1)
        want = (X @ flat).reshape((X.shape[0],) + T.shape[1:])
        size = (abs(X) @ np.abs(flat)).reshape(want.shape)
        assert tuple(got.shape) == want.shape
        tol = 1e-12 if dtype != "float32" else (np.diff(X.indptr).max() + 4) * 2.0**-23
        assert (np.abs(got.cpu().numpy() - want) <= tol * size + 1e-30).all()


@pytest.mark.parametrize("dtype,rtol", [("float32-float64", 1e-9), ("float32", 1e-4)])
def test_losses_of_a_resident_model(dtype, rtol):
    C = 4
    X, w0, w, V, R, fid, rng = _case(2, "fm", C)
    n = X.shape[0]
    logits = np.stack([O.fm_predict_fast_csr(X.indptr.astype(np.int64), X.indices.astype(np.int64),
                                             X.data, X.shape[1], w0[c], w[c], V[c])
                       for c in range(C)], 1)
    lse = np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1)) + logits.max(1)
    y = rng.integers(-1, C, size=n)
    lp = np.where(y >= 0, logits[np.arange(n), np.maximum(y, 0)] - lse, 0.0)
    bounds = np.arange(0, n + 1, 12)
    sums = np.add.reduceat(lp, bounds[:-1])
    ref, old, adv = (rng.normal(size=s) for s in (len(sums), n, n))
    with _model("fm", C, dtype, X, w0, w, V, R, fid) as m:
        csr = _csr(X, dtype)
        wide = csr[2].dtype
        t = lambda a: torch.from_numpy(a).to("cuda", wide)  # noqa: E731
        yt, bt = torch.from_numpy(y).cuda(), torch.from_numpy(bounds).cuda()
        r = m.label_logprobs_device(*csr, yt, bt)
        scale = np.abs(logits).max() * 10
        assert np.abs(r.logprobs.cpu().numpy() - lp).max() <= rtol * scale
        assert np.abs(r.sums.cpu().numpy() - sums).max() <= 12 * rtol * scale
        p = len(sums) // 2
        q = sums - t(ref).cpu().numpy()
        z = 0.2 * (q[:p] - q[p:])
        want = np.mean(np.logaddexp(0, -z) * 0.9 + np.logaddexp(0, z) * 0.1)
        got = preference_eval_device(m, *csr, yt, bt, t(ref), 0.2, 0.1)
        assert got == pytest.approx(want, abs=0.2 * 24 * rtol * scale)
        live = y >= 0
        ratio = np.exp(lp - t(old).cpu().numpy())
        a = t(adv).cpu().numpy()
        want = np.mean(-np.minimum(ratio * a, np.clip(ratio, 0.8, 1.2) * a)[live])
        got = policy_eval_device(m, *csr, yt, t(old), t(adv))
        assert got == pytest.approx(want, abs=rtol * scale * np.abs(ratio * a).max())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        args = (yt, t(old), t(adv))
        side.wait_stream(torch.cuda.current_stream())
        assert got == policy_eval_device(m, *csr, *args, stream=side)
        with pytest.raises(ValueError, match="float"):
            m.factors_device(csr[0], csr[1], csr[2].half())
        with pytest.raises(ValueError, match="labels"):
            m.label_logprobs_device(*csr, yt[:-1])
    with _model("fm", 1, dtype, X, 0.0, w[0], V[0], R, fid) as m:
        with pytest.raises(ValueError, match="n_classes >= 2"):
            m.label_logprobs_device(*csr, yt)
        with pytest.raises(ValueError, match="n_classes >= 2"):
            preference_eval_device(m, *csr, yt, bt, t(ref))


def test_inputs_freed_while_their_stream_still_runs():
    """Scores and factors of another stream read their inputs before the memory is given away."""
    X, w0, w, V, R, fid, _ = _case(3, "fm", 3, n=4000)
    with _model("fm", 3, "float32", X, w0, w, V, R, fid) as m:
        keep = _csr(X, "float32")
        want = m.scores_device(*keep), m.factors_device(*keep)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        for call, expect in ((m.scores_device, want[0]), (m.factors_device, want[1])):
            csr = [t.clone() for t in keep]
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                torch.cuda._sleep(20_000_000)
            got = call(*csr, stream=side)
            del csr
            again = [torch.zeros_like(t) for t in keep]  # would take the same places
            side.synchronize()
            assert torch.equal(got, expect)
            del again
