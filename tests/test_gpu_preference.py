"""GPU tests of the label log-probabilities, the preference loss and the policy
loss against their definitions in float64.

Tolerances, with u = 2^-24 (float32 arithmetic) or 2^-53 (float64), C classes of
magnitude at most X: an exponential is off by 4 u + 2 u |x - m| of itself (ex2.approx:
2^-22; its argument two roundings), so the sum of exponentials by at most
(C / 8 + 32) u of itself (no lane adds more than C / 8 + 16 values in turn, and
|d| exp(d) < 0.4), lse and log-probabilities by e = (C / 8 + 36) u + 4 u X. A gradient
g ([c = y] - p) is off by |g| p (e + 4 u + 2 u |x - lse|) + |dg| + 2 u |g| and its
rounding u_o |result| (float16: 2^-25 below its normal range). Sequences' sums are
off by the number of tokens times e, losses as derived beside them.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.preference import (label_logprobs, label_logprobs_grad,  # noqa: E402
                                       policy_loss, preference_loss)

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16,
         "f16": torch.float16}
SHAPES = [(1, 1), (3, 2), (5, 10), (1000, 10), (33, 31), (17, 33), (9, 100), (70, 1000), (4, 2049),
          (13, 5003), (2, 50001), (1, 120000), (300, 32)]


def _u(wide):
    return 2.0**-53 if wide == torch.float64 else 2.0**-24


def _wide(kind):
    return torch.float64 if kind == "f64" else torch.float32


def _make(seed, n, c, kind, label_type=torch.int64, pad=0.2, std=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, c, generator=g, dtype=torch.float64) * std).to(TYPES[kind]).cuda()
    y = torch.randint(0, c, (n,), generator=g)
    bad = torch.rand(n, generator=g) < pad
    y[bad] = torch.where(torch.rand(n, generator=g) < 0.5, -1, c)[bad]
    return x, y.to(label_type).cuda()


def _define(x, y):
    """float64 (log-probability, lse, probabilities, unmasked)."""
    w = x.double()
    c = x.shape[1]
    lse = torch.logsumexp(w, 1)
    empty = torch.isneginf(lse)
    live = (y >= 0) & (y < c) & ~empty
    at = y.long().clamp(0, c - 1)
    lp = torch.where(live, w.gather(1, at[:, None])[:, 0] - lse, 0.0)
    p = torch.where(empty[:, None], 0.0, torch.exp(w - lse[:, None]))
    return lp, lse, p, live


def _tol(x, wide):
    big = x.double()
    big = float(torch.where(torch.isfinite(big), big, 0.0).abs().max())
    return (x.shape[1] / 8 + 36) * _u(wide) + 4 * _u(wide) * big


def _check_grad(got, x, y, g, dg, wide):
    """got against g ([c = y] - p); dg bounds the error of g."""
    lp, lse, p, live = _define(x, y)
    u, e = _u(wide), _tol(x, wide)
    g = torch.where(live, g, 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, y.long().clamp(0, x.shape[1] - 1)[:, None], 1.0)
    want = g * (hot - p)
    away = torch.where(p > 0, (x.double() - lse[:, None]).abs(), 0.0)
    tol = (g.abs() * (p * (e + 4 * u + 2 * u * away) + 2 * u) + torch.where(live, dg, 0.0)[:, None]
           + torch.finfo(got.dtype).eps / 2 * want.abs()
           + (2.0**-25 if got.dtype == torch.float16 else 1e-37 if wide == torch.float32 else 0.0))
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed"
    assert bool((got[~live] == 0).all())


@pytest.mark.parametrize("n,c", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("label_type", [torch.int32, torch.int64])
def test_label_logprobs(n, c, kind, label_type):
    x, y = _make(1, n, c, kind, label_type)
    wide = _wide(kind)
    r = label_logprobs(x, y)
    lp, lse, p, live = _define(x, y)
    e = _tol(x, wide)
    assert r.logprobs.dtype == r.lse.dtype == wide and r.sums is None
    assert (r.lse.double() - lse).abs().max() <= e
    assert (r.logprobs.double() - lp).abs().max() <= e
    assert bool((r.logprobs[~live] == 0).all())
    g = torch.randn(n, device="cuda", dtype=wide)
    d = label_logprobs_grad(g, x, y, r.lse)
    assert d.dtype == x.dtype
    _check_grad(d, x, y, g.double(), torch.zeros(n, device="cuda", dtype=torch.float64), wide)
    assert torch.equal(d, label_logprobs_grad(g, x, y, label_logprobs(x, y).lse))


@pytest.mark.parametrize("c", [10, 100, 5003])
@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_classes_and_rows(c, kind):
    """-inf and the type's lowest value in places, whole rows of them, NaN and inf in masked
    rows."""
    x, y = _make(2, 12, c, kind, pad=0.0)
    low = torch.finfo(x.dtype).min
    x[0, 1:] = -math.inf
    y[0] = 0  # the only class left: log-probability 0
    x[1] = -math.inf  # nothing left: masked
    x[2] = low  # all alike: uniform
    x[3, ::2] = -math.inf
    y[3] = 1
    x[4, ::2] = low
    y[4] = 1
    x[5] = math.nan
    x[6, 3] = math.inf
    x[7] = -math.inf
    y[5:8] = -1  # masked, whatever is in the row
    x[8, : c // 2] = -math.inf
    y[8] = 0  # a class that is masked out: log-probability -inf
    r = label_logprobs(x, y)
    assert float(r.logprobs[0]) == 0.0
    assert float(r.logprobs[1]) == 0.0 and math.isinf(float(r.lse[1]))
    assert float(r.logprobs[2]) == pytest.approx(-math.log(c), rel=1e-5)
    assert bool((r.logprobs[5:8] == 0).all())
    assert float(r.logprobs[8]) == -math.inf
    rest = torch.tensor([3, 4, 9, 10, 11], device="cuda")
    lp, lse, p, live = _define(x[rest], y[rest])
    assert (r.logprobs[rest].double() - lp).abs().max() <= _tol(x[9:], _wide(kind))
    d = label_logprobs_grad(torch.ones_like(r.lse), x, y, r.lse)
    assert bool((d[[1, 5, 6, 7]] == 0).all())
    assert torch.isfinite(d[[0, 2, 3, 4, 9, 10, 11]].double()).all()
    assert bool((d[3, ::2] == 0).all()) and bool((d[4, ::2] == 0).all())
    # the same through the policy loss
    z = torch.zeros_like(r.lse)
    keep = torch.ones_like(z)
    keep[8] = 0
    q = policy_loss(x, y, z, keep, sample_weight=keep)
    assert torch.isfinite(q.loss) and torch.isfinite(q.grad.double()).all()
    assert bool((q.grad[[1, 5, 6, 7, 8]] == 0).all())


def test_large_scores_do_not_overflow():
    x = torch.tensor([[3e38, -3e38, 0.0], [1e4, 1e4, -1e4], [-1e30, -1e30, -1e30]], device="cuda")
    y = torch.tensor([0, 1, 2], device="cuda")
    r = label_logprobs(x, y)
    assert r.logprobs.tolist() == pytest.approx([0.0, -math.log(2), -math.log(3)], abs=1e-6)
    d = label_logprobs_grad(torch.ones(3, device="cuda"), x, y, r.lse)
    assert torch.isfinite(d).all()


def _sequences(seed, n_pairs, longest, lead=0, tail=0):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, longest + 1, (2 * n_pairs,), generator=g)
    ip = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]) + lead
    return ip.cuda(), int(ip[-1]) + tail


@pytest.mark.parametrize("n_pairs,longest,c", [(1, 1, 2), (3, 5, 10), (200, 12, 10), (5, 90, 1000),
                                               (2, 40, 5003), (4, 3, 50001)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("weighted,eps", [(False, 0.0), (True, 0.2)])
def test_preference_loss(n_pairs, longest, c, kind, weighted, eps):
    ip, n = _sequences(3, n_pairs, longest, lead=2, tail=3)
    x, y = _make(4, n, c, kind)
    wide, beta = _wide(kind), 0.3
    u, e = _u(wide), _tol(x, wide)
    lp, _, _, _ = _define(x, y)
    seq = torch.searchsorted(ip, torch.arange(n, device="cuda"), right=True) - 1
    inside = (seq >= 0) & (seq < 2 * n_pairs)
    s = torch.zeros(2 * n_pairs, dtype=torch.float64, device="cuda")
    s.index_add_(0, seq[inside], lp[inside])
    r = label_logprobs(x, y, ip)
    tol_s = longest * e + u * s.abs()
    assert bool(((r.sums.double() - s).abs() <= tol_s).all())
    ref = (s + torch.randn(2 * n_pairs, device="cuda", dtype=torch.float64)).to(wide)
    w = torch.rand(n_pairs, device="cuda", dtype=wide) if weighted else None
    got = preference_loss(x, y, ip, ref, beta, eps, w)
    q = s - ref.double()
    z = beta * (q[:n_pairs] - q[n_pairs:])
    tol_z = beta * 2 * longest * e + 4 * u * (z.abs() + beta * (s.abs().max() + ref.abs().max()))
    assert bool(((got.margins.double() - z).abs() <= tol_z).all())
    assert bool(((got.logprobs.double() - s).abs() <= tol_s).all())
    ww = w.double() if weighted else torch.ones_like(z)
    each = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
    loss = float((ww * each).sum() / ww.sum())
    assert got.loss.shape == () and got.loss.dtype == wide
    # the loss's slope in z is at most 1
    assert abs(float(got.loss) - loss) <= float(tol_z.max()) + 2 * u * abs(loss)
    slope = -beta * ww / ww.sum() * ((1 - eps) * torch.sigmoid(-z) - eps * torch.sigmoid(z))
    g = torch.zeros(n, dtype=torch.float64, device="cuda")
    g[inside] = torch.cat([slope, -slope])[seq[inside]]
    dg = torch.zeros_like(g)  # sigmoid's slope is at most 1 / 4
    dg[inside] = (torch.cat([tol_z, tol_z]) * beta * torch.cat([ww, ww]) / ww.sum() / 4)[seq[inside]]
    _check_grad(got.grad, x, y, g, dg + 4 * u * g.abs(), wide)
    assert bool((got.grad[~inside] == 0).all())
    only = preference_loss(x, y, ip, ref, beta, eps, w, with_grad=False)
    assert only.grad is None and torch.equal(only.loss, got.loss)
    assert torch.equal(only.margins, got.margins)


@pytest.mark.parametrize("n,c", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("weighted,kl", [(False, 0.0), (True, 0.1)])
def test_policy_loss(n, c, kind, weighted, kl):
    x, y = _make(5, n, c, kind)
    y[0] = 0
    wide = _wide(kind)
    u, e = _u(wide), _tol(x, wide)
    lp, _, _, live = _define(x, y)
    gen = torch.Generator(device="cuda").manual_seed(9)
    step = 0.3 * torch.randn(n, generator=gen, device="cuda", dtype=torch.float64)
    for edge in (math.log(0.9), math.log(1.3)):  # no ratio so near a bound that rounding decides
        step = torch.where((step - edge).abs() < 0.02, edge + 0.04, step)
    old = (lp - step).to(wide)
    ref = (lp + 0.3 * torch.randn(n, generator=gen, device="cuda", dtype=torch.float64)).to(wide)
    adv = torch.randn(n, generator=gen, device="cuda", dtype=wide)
    w = torch.rand(n, generator=gen, device="cuda", dtype=wide) if weighted else None
    got = policy_loss(x, y, old, adv, ref if kl else None, 0.1, 0.3, kl, w)
    a = adv.double()
    ratio = torch.exp(lp - old.double())
    bent = ratio.clamp(0.9, 1.3)
    cut = ratio * a > bent * a
    away = ref.double() - lp if kl else torch.zeros_like(lp)
    k = torch.expm1(away) - away
    ww = torch.where(live, w.double() if weighted else torch.ones_like(lp), 0.0)
    total = ww.sum()
    each = -torch.minimum(ratio * a, bent * a) + kl * k
    want = [float((ww * v).sum() / total) for v in (each, k, cut.double())]
    # a log-probability's error e moves a term by its slope times e
    move = e * (ratio * a.abs() + kl * torch.expm1(away).abs()) + 8 * u * (each.abs() + k + ratio * a.abs())
    tol = float((ww * move).sum() / total) + 4 * u * max(abs(v) for v in want)
    assert abs(float(got.loss) - want[0]) <= tol
    assert abs(float(got.kl) - want[1]) <= float((ww * torch.expm1(away).abs()).sum() / total) * e + 8 * u * want[1] + 8 * u
    assert float(got.clip_fraction) == pytest.approx(want[2], abs=4 * u)
    assert (got.logprobs.double() - lp).abs().max() <= e
    g = ww / total * (torch.where(cut, 0.0, -ratio * a) - kl * torch.expm1(away))
    dg = ww / total * (ratio * a.abs() + kl * torch.exp(away)) * (e + 4 * u) + 4 * u * g.abs()
    _check_grad(got.grad, x, y, g, dg, wide)
    only = policy_loss(x, y, old, adv, ref if kl else None, 0.1, 0.3, kl, w, with_grad=False)
    assert only.grad is None and torch.equal(only.loss, got.loss)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_pitches_and_alignment(kind):
    big, _ = _make(6, 30, 700, kind)
    for lo, c in ((0, 640), (1, 640), (3, 99), (8, 9), (0, 513)):
        x = big[:, lo:lo + c]
        y = torch.randint(-1, c, (30,), device="cuda")
        a, b = label_logprobs(x, y), label_logprobs(x.contiguous(), y)
        e = 2 * _tol(x, torch.float32)
        assert (a.lse - b.lse).abs().max() <= e and (a.logprobs - b.logprobs).abs().max() <= e
        g = torch.randn(30, device="cuda")
        zero = torch.zeros(30, dtype=torch.float64, device="cuda")
        _check_grad(label_logprobs_grad(g, x, y, a.lse), x, y, g.double(), zero, torch.float32)


def test_nothing_to_learn_from():
    """No rows, no pairs, every label masked, weights of 0: loss and gradient 0."""
    x = torch.randn(0, 10, device="cuda")
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    z = torch.zeros(0, device="cuda")
    assert label_logprobs(x, y).logprobs.shape == (0,)
    assert label_logprobs_grad(z, x, y, z).shape == (0, 10)
    assert float(policy_loss(x, y, z, z).loss) == 0.0
    ip = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert float(preference_loss(x, y, ip, z).loss) == 0.0
    ip = torch.zeros(5, dtype=torch.int64, device="cuda")  # two pairs of empty sequences
    r = preference_loss(x, y, ip, torch.zeros(4, device="cuda"))
    assert float(r.loss) == pytest.approx(math.log(2), rel=1e-6)
    x = torch.randn(4, 10, device="cuda")
    y = torch.tensor([-1, 10, -1, 99], device="cuda")
    one = torch.ones(4, device="cuda")
    for weight, labels in ((None, y), (torch.zeros(4, device="cuda"), y.clamp(0, 9))):
        r = policy_loss(x, labels, one, one, one, kl_coef=0.1, sample_weight=weight)
        assert float(r.loss) == float(r.kl) == float(r.clip_fraction) == 0.0
        assert bool((r.grad == 0).all())
    ip = torch.tensor([0, 2, 4], device="cuda")
    r = preference_loss(x, y.clamp(0, 9), ip, torch.zeros(2, device="cuda"),
                        sample_weight=torch.zeros(1, device="cuda"))
    assert float(r.loss) == 0.0 and bool((r.grad == 0).all())


def test_bad_sequence_bounds_stay_inside():
    x, y = _make(7, 20, 10, "f32")
    ip = torch.tensor([-7, 5, 3, 99, 12], device="cuda")
    r = preference_loss(x, y, ip, torch.zeros(4, device="cuda"))
    s = label_logprobs(x, y, ip).sums
    torch.cuda.synchronize()
    assert torch.isfinite(r.loss) and torch.isfinite(s).all()


def test_extreme_margins():
    """Margins far out: loss |z| on the wrong side and 0 on the right one, finite slopes."""
    x = torch.zeros(4, 10, dtype=torch.float64, device="cuda")
    y = torch.zeros(4, dtype=torch.int32, device="cuda")
    ip = torch.tensor([0, 1, 2, 3, 4], device="cuda")
    ref = torch.tensor([1e4, -1e4, 0.0, 0.0], dtype=torch.float64, device="cuda")
    r = preference_loss(x, y, ip, ref, beta=1.0)
    assert r.margins.tolist() == pytest.approx([-1e4, 1e4])
    assert float(r.loss) == pytest.approx(5e3)
    assert float(r.grad[0, 0]) == pytest.approx(-0.5 * 0.9) and float(r.grad[1, 0]) == 0.0


def test_other_stream_and_graph_replay():
    x, y = _make(8, 500, 1000, "bf16")
    ip = torch.arange(0, 501, 50, device="cuda")
    ref = torch.randn(10, device="cuda")
    old, adv = torch.full((500,), -7.0, device="cuda"), torch.randn(500, device="cuda")

    def both(**kw):
        a = preference_loss(x, y, ip, ref, **kw)
        b = policy_loss(x, y, old, adv, old, kl_coef=0.1, **kw)
        return (a.loss, a.margins, a.logprobs, a.grad, b.loss, b.kl, b.clip_fraction, b.logprobs,
                b.grad)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(stream=side)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    x.copy_(x.flip(0))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = both()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_gradient_by_differences(which):
    """Central differences of the loss in float64: error h^2 / 6 of the third derivative
    (at most about 1 here) plus 2^-53 / h of rounding; h = 1e-4."""
    x, y = _make(9, 12, 7, "f64", std=1.0, pad=0.1)
    ip = torch.tensor([0, 3, 6, 6, 12], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    lp = label_logprobs(x, y).logprobs
    step = torch.tensor([0.05, -0.4, 0.4] * 4, device="cuda", dtype=torch.float64)
    adv = torch.randn(12, generator=gen, device="cuda", dtype=torch.float64)

    def run(v, grad):
        if which == "preference":
            return preference_loss(v, y, ip, torch.zeros(4, device="cuda", dtype=torch.float64),
                                   0.5, 0.1, with_grad=grad)
        return policy_loss(v, y, lp - step, adv, lp - 0.3, kl_coef=0.2, with_grad=grad)

    g = run(x, True).grad
    h = 1e-4
    for t in range(12):
        for c in (0, 3, int(y[t].clamp(0, 6))):
            d = torch.zeros_like(x)
            d[t, c] = h
            num = (float(run(x + d, False).loss) - float(run(x - d, False).loss)) / (2 * h)
            assert num == pytest.approx(float(g[t, c]), abs=2e-8)


def test_a_training_step_of_a_linear_policy():
    """The operators together: sparse rows through their latent rows to class scores, a
    reference's log-probabilities, the preference loss, and its gradient back to the
    touched rows: the loss's derivative along the gradient is the gradient's norm."""
    from modern_fm_b200.embedding import embedding_grad, embedding_grad_rows, embedding_lookup

    gen = torch.Generator(device="cuda").manual_seed(2)
    n_features, c, n = 5000, 10, 600
    ids = torch.randint(0, n_features, (n * 9,), generator=gen, device="cuda", dtype=torch.int32)
    val = torch.rand(n * 9, generator=gen, device="cuda", dtype=torch.float64)
    bounds = torch.arange(0, n * 9 + 1, 9, device="cuda")
    w = torch.randn(n_features, c, generator=gen, device="cuda", dtype=torch.float64)
    y = torch.randint(-1, c, (n,), generator=gen, device="cuda", dtype=torch.int32)
    ip = torch.arange(0, n + 1, 30, device="cuda")
    ref = label_logprobs(embedding_lookup(w * 0.9, ids, val, bounds), y, ip).sums

    def loss(table, grad=False):
        return preference_loss(embedding_lookup(table, ids, val, bounds), y, ip, ref, beta=0.2,
                               with_grad=grad)

    d = loss(w, True).grad
    whole = embedding_grad(d, ids, n_features, val, bounds).table
    rows = embedding_grad_rows(d, ids, n_features, val, bounds)
    u = int(rows.count)
    assert torch.equal(whole[rows.keys[:u].long()], rows.rows[:u])
    assert float(whole.abs().sum()) == pytest.approx(float(rows.rows.abs().sum()), rel=1e-12)
    # derivative along the gradient, by a central difference: h^2 of the third derivative
    norm = float((whole * whole).sum())
    direction = whole / norm**0.5
    h = 1e-3
    num = (float(loss(w + h * direction).loss) - float(loss(w - h * direction).loss)) / (2 * h)
    assert num == pytest.approx(norm**0.5, rel=1e-5)


def test_offsets_beyond_32_bits():
    """More than 2^32 scores: a uniform matrix with a few classes raised, in the last row."""
    n, c = 33_000, 131_072
    x = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 2**32
    x[n - 1, c - 1] = 8.0
    y = torch.full((n,), c - 1, device="cuda")
    z = torch.full((n,), -math.log(c), device="cuda")
    tol = _tol(x[-2:], torch.float32)
    r = label_logprobs(x, y)
    last = 8.0 - math.log(c - 1 + math.exp(8.0))
    assert float((r.logprobs[:-1] + math.log(c)).abs().max()) <= tol
    assert abs(float(r.logprobs[-1]) - last) <= tol
    g = label_logprobs_grad(torch.ones(n, device="cuda"), x, y, r.lse)
    assert float(g[n - 1, c - 1]) == pytest.approx(1 - math.exp(last), rel=2.0**-7)
    assert float(g[n - 2, 0]) == pytest.approx(-1 / c, rel=2.0**-7)
    del g
    q = policy_loss(x, y, z, torch.ones(n, device="cuda"), clip_high=1e9)
    # every row's ratio is 1 but the last's
    ratio = math.exp(last + math.log(c))
    assert float(q.loss) == pytest.approx(-(n - 1 + ratio) / n, rel=1e-5)
    assert float(q.grad[n - 1, c - 1]) == pytest.approx(-ratio / n * (1 - math.exp(last)), rel=2.0**-6)


def test_two_streams_at_once():
    x, y = _make(10, 3000, 10, "f32")
    big, yb = _make(11, 40, 30000, "bf16")
    one = torch.full((3000,), -2.0, device="cuda")
    adv = torch.randn(3000, device="cuda")
    ip = torch.arange(0, 41, 10, device="cuda")
    ref = torch.zeros(4, device="cuda")

    def calls(stream):
        p = policy_loss(x, y, one, adv, one, kl_coef=0.1, stream=stream)
        q = policy_loss(big, yb, one[:40], adv[:40], stream=stream)
        r = preference_loss(big, yb, ip, ref, stream=stream)
        return (p.loss, p.grad, p.logprobs, q.loss, q.grad, r.loss, r.grad)

    want = calls(None)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [calls(s) for _ in range(15) for s in (a, b)]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(u, v) for u, v in zip(g, want))
