"""GPU tests of the class-score losses where weights, scores or derivatives are not
finite, rows are empty, or the number of classes meets a limit of a kernel, in
each of the kernels that take rows: up to 32 classes, rows of up to 8 KB, longer
ones. Helpers, and the tolerances that they hold, are those of
test_gpu_preference.
"""

import math
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.preference import (label_logprobs, label_logprobs_grad,  # noqa: E402
                                       policy_loss, preference_loss)

from test_gpu_preference import (TYPES, _check_grad, _define, _make, _tol, _u,  # noqa: E402
                                 _wide)


@pytest.mark.parametrize("c", [10, 32, 100, 9001])
@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_rows_under_a_scale_that_is_not_finite(c, kind):
    """A NaN weight, or weights whose sum is too small to divide by: rows that are masked, of
    no sequence or of a pair of weight 0 keep gradient 0; with the NaN the others get NaN."""
    x, y = _make(1, 70, c, kind, pad=0.4)
    y[0] = y[33] = -1
    y[2] = 0
    wide = _wide(kind)
    ip = torch.tensor([1, 20, 40, 50, 68], device="cuda")  # rows 0, 68, 69: of no sequence
    ref = torch.zeros(4, dtype=wide, device="cuda")
    live = (y >= 0) & (y < c)
    row = torch.arange(70, device="cuda")
    inside = (row >= 1) & (row < 68)
    first = (row < 20) | ((row >= 40) & (row < 50))  # the rows of pair 0
    w = torch.tensor([math.nan, 1.0], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert math.isnan(float(r.loss))
    assert bool((r.grad[~live | ~inside] == 0).all())
    assert torch.isnan(r.grad[live & inside & first].double()).all()
    w = torch.tensor([0.0, math.nan], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert bool((r.grad[~live | ~inside | first] == 0).all())
    # 1 / the sum of the weights is infinite in float64; in float32 the sum's inverse is
    # finite, but the derivatives are 0
    w = torch.tensor([0.0, 5e-324 if kind == "f64" else 1e-45], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert bool((r.grad[~live | ~inside | first] == 0).all())


# 2^22 scores or 65536 rows are where the sum of the weights is found in another way
@pytest.mark.parametrize("n,c", [(1, 3), (40, 10), (40, 32), (300, 100), (3, 2049), (50, 9001),
                                 (70_001, 3), (140_000, 31), (45_000, 100), (2100, 2049),
                                 (470, 9001)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("weighted", [False, True])
def test_policy_mean_without_empty_rows(n, c, kind, weighted):
    """A row whose every score is -infinity is masked as one without a label is: the means
    and the gradient of the others are those without it, also with a NaN for its weight."""
    x, y = _make(2, n, c, kind)
    gen = torch.Generator().manual_seed(3)
    empty = torch.rand(n, generator=gen) < 0.3
    some = min(2, n - 1)
    empty[1:2] = True
    empty[some] = False
    empty = empty.cuda()
    x[empty] = -math.inf
    y[1:2] = c - 1
    y[some] = 0
    wide = _wide(kind)
    u, e = _u(wide), _tol(x, wide)
    lp, _, _, live = _define(x, y)
    assert not bool(live[1:2].any()) and bool(live[some])
    old = (lp + 0.1).to(wide)  # ratios of exp(-0.1): inside the clip's bounds
    ref = (lp - 0.3).to(wide)
    adv = torch.randn(n, generator=gen, dtype=wide).cuda()
    w = (torch.rand(n, generator=gen, dtype=wide) + 0.5).cuda() if weighted else None
    if weighted:
        w[1:2] = math.nan
    got = policy_loss(x, y, old, adv, ref, kl_coef=0.1, sample_weight=w)
    a, away = adv.double(), ref.double() - lp
    ratio = torch.exp(lp - old.double())
    ww = torch.where(live, w.double() if weighted else torch.ones_like(lp), 0.0)
    ww = ww / ww.sum()
    k = torch.expm1(away) - away
    loss, kl = float((ww * (0.1 * k - ratio * a)).sum()), float((ww * k).sum())
    # a log-probability's error e moves a term by its slope times e; exp(u) - u - 1 loses
    # up to 4 u of its terms
    move = (e + 8 * u) * (ratio * a.abs() + 0.1 * (1 + k) + k)
    tol = float((ww * move).sum()) + 4 * u
    assert abs(float(got.loss) - loss) <= tol
    assert abs(float(got.kl) - kl) <= float((ww * (e + 8 * u)).sum()) + 4 * u
    assert float(got.clip_fraction) == 0.0
    assert bool((got.logprobs[~live] == 0).all())
    g = ww * (-ratio * a - 0.1 * torch.expm1(away))
    dg = ww * (ratio * a.abs() + 0.1 * torch.exp(away)) * (e + 8 * u) + 4 * u * g.abs()
    _check_grad(got.grad, x, y, g, dg, wide)
    only = policy_loss(x, y, old, adv, ref, kl_coef=0.1, sample_weight=w, with_grad=False)
    assert torch.equal(only.loss, got.loss) and torch.equal(only.kl, got.kl)
    # the clipped share is of the unmasked rows too
    far = policy_loss(x, y, old - 5, adv.abs() + 0.1, sample_weight=w, with_grad=False)
    assert float(far.clip_fraction) == pytest.approx(1.0, abs=4 * u)


@pytest.mark.parametrize("n,c", [(30, 10), (30, 100), (30, 9001), (70_000, 10), (45_000, 100),
                                 (500, 9001)])
def test_policy_of_empty_rows_alone_and_in_a_graph(n, c):
    """Nothing but empty rows: 0. A captured call whose rows turn empty, and back."""
    x, y = _make(4, n, c, "f32", pad=0.0)
    z = torch.zeros(n, device="cuda")
    r = policy_loss(torch.full_like(x, -math.inf), y, z, z + 1, z, kl_coef=0.1)
    assert float(r.loss) == float(r.kl) == float(r.clip_fraction) == 0.0
    assert bool((r.grad == 0).all())
    some = x.clone()
    some[::3] = -math.inf
    want = [policy_loss(v, y, z - 2, z + 1, z - 2, kl_coef=0.1) for v in (x, some)]
    graph = torch.cuda.CUDAGraph()
    at = x.clone()
    with torch.cuda.graph(graph):
        got = policy_loss(at, y, z - 2, z + 1, z - 2, kl_coef=0.1)
    for v, expect in ((x, want[0]), (some, want[1]), (x, want[0])):
        at.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, expect))


@pytest.mark.parametrize("n,c", [(40, 10), (40, 100), (40, 9001), (70_000, 10), (45_000, 100),
                                 (500, 9001)])
@pytest.mark.parametrize("lo", [0, 1])
def test_policy_weight_of_a_row_with_any_score(n, c, lo):
    """A row with a score somewhere is not empty: its weight counts, whichever score that is
    and whatever its label's score is; also where rows begin off 16 bytes."""
    x = torch.full((n, c + lo), -math.inf, device="cuda", dtype=torch.bfloat16)[:, lo:]
    row = torch.arange(n, device="cuda")
    x[row, row % c] = 1.0
    x[-1] = -math.inf
    y = ((row + 1) % c).int()  # a score of -infinity: ratio 0, no loss, no gradient
    y[::3] = (row % c)[::3].int()  # the only score: log-probability 0
    y[-2] = int(row[-2]) % c
    z = torch.zeros(n, device="cuda")
    r = policy_loss(x, y, z, z + 1)
    mine = (y == row % c) & (row < n - 1)
    # ratios of 1 and 0, advantages of 1: minus the share of the first among n - 1 rows
    assert float(r.loss) == pytest.approx(-int(mine.sum()) / (n - 1), rel=2.0**-22)
    assert bool((r.logprobs[mine] == 0).all()) and bool((r.grad == 0).all())


def _policy_of_classes(c, kind):
    x, y = _make(6, 70, c, kind)
    y[0] = 0
    wide = _wide(kind)
    u, e = _u(wide), _tol(x, wide)
    lp, _, _, live = _define(x, y)
    old = (lp + 0.1).to(wide)  # inside the clip's bounds
    adv = torch.randn(70, generator=torch.Generator().manual_seed(7), dtype=wide).cuda()
    got = policy_loss(x, y, old, adv)
    ratio, share = torch.exp(lp - old.double()), live.double() / live.sum()
    want = float(-(share * ratio * adv.double()).sum())
    move = (share * ratio * adv.double().abs()) * (e + 8 * u)
    assert abs(float(got.loss) - want) <= float(move.sum()) + 4 * u
    _check_grad(got.grad, x, y, -share * ratio * adv.double(), move, wide)


@pytest.mark.parametrize("c", range(1, 35))
@pytest.mark.parametrize("kind", list(TYPES))
def test_policy_of_every_small_number_of_classes(c, kind):
    _policy_of_classes(c, kind)


def test_the_first_call_of_a_process_has_24_float64_classes():
    """Its tiles fill the shared memory that needs no asking, its own arrays go beyond; no call
    before it has asked for more."""
    code = ("import test_gpu_class_loss_limits as t\n"
            "for c in (24, 23, 25, 32): t._policy_of_classes(c, 'f64')\n")
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = " + repr(sys.path) + "\n" + code],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("eps,first", [(0.0, 1), (1.0, 0)])
def test_preference_of_an_infinite_margin(kind, eps, first):
    """A label that cannot be drawn on the side that should lose: the pair's loss is 0 as the
    limit says, and the mean is the other pair's; on the other side the loss is infinite."""
    x, y = _make(8, 8, 10, kind, pad=0.0)
    y[:] = 3
    x[4 * first, 3] = -math.inf  # of pair 0's second sequence, or of its first one
    ip = torch.tensor([0, 2, 4, 6, 8], device="cuda")
    ref = torch.zeros(4, dtype=_wide(kind), device="cuda")
    r = preference_loss(x, y, ip, ref, 0.5, eps)
    assert float(r.margins[0]) == (math.inf if first else -math.inf)
    s = _define(x, y)[0].reshape(4, 2).sum(1)
    z = 0.5 * float(s[1] - s[3])
    e = 0.5 * 4 * _tol(torch.where(torch.isinf(x), 0.0, x), _wide(kind))
    want = math.log1p(math.exp(z if eps else -z)) / 2
    assert float(r.loss) == pytest.approx(want, abs=e + 4 * _u(_wide(kind)))
    assert bool((r.grad[[0, 1, 4, 5]] == 0).all()) and torch.isfinite(r.grad.double()).all()
    half = preference_loss(x, y, ip, ref, 0.5, 0.5)
    assert float(half.loss) == math.inf and torch.isfinite(half.grad.double()).all()


@pytest.mark.parametrize("c", [10, 100, 9001])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("side", ["model", "reference"])
def test_policy_kl_term_without_end(c, kind, side):
    """A label that the model or the reference cannot draw: exp(u) - u - 1 is infinite on both
    sides, and so are the mean and a loss that has the term in it."""
    x, y = _make(9, 20, c, kind, pad=0.0)
    y[:] = 2
    one = torch.ones(20, dtype=_wide(kind), device="cuda")
    ref = -one
    if side == "model":
        x[3, 2] = -math.inf
    else:
        ref[3] = -math.inf
    r = policy_loss(x, y, -2 * one, one, ref, kl_coef=0.1)
    assert float(r.kl) == float(r.loss) == math.inf
    rest = torch.arange(20, device="cuda") != 3
    # a slope of 0.1 exp(u) / 20 beyond float16's 65504 (u > 16.4, lp < -17.4) is infinite there
    assert not torch.isnan(r.grad[rest]).any()
    if side == "reference":  # the term's slope is 1 there
        assert not torch.isnan(r.grad).any()


@pytest.mark.parametrize("c", [10, 100, 9001])
@pytest.mark.parametrize("kind", list(TYPES))
def test_policy_kl_without_a_coefficient(c, kind):
    """With kl_coef 0 the reference only gives the statistic, also where that is infinite: loss
    and gradient are those without a reference."""
    x, y = _make(9, 20, c, kind, pad=0.0)
    y[:] = 2
    x[3, 2] = -math.inf  # log-probability -infinity: an infinite term
    x[4, 2] = -2000.0  # exp(reference - lp) overflows in 64 bits
    one = torch.ones(20, dtype=_wide(kind), device="cuda")
    a = policy_loss(x, y, -2 * one, one, -one)
    b = policy_loss(x, y, -2 * one, one)
    assert float(a.kl) == math.inf and math.isfinite(float(b.loss))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.clip_fraction, b.clip_fraction)
    assert torch.equal(a.grad, b.grad) and torch.isfinite(a.grad.double()).all()


@pytest.mark.parametrize("c", [10, 100, 9001])
@pytest.mark.parametrize("kind", list(TYPES))
def test_policy_ratio_beyond_the_range_without_an_advantage(c, kind):
    """A token without an advantage has no term, however far its ratio is out (exp overflows)."""
    x, y = _make(10, 20, c, kind, pad=0.0)
    one = torch.ones(20, dtype=_wide(kind), device="cuda")
    old, adv = -2 * one, one.clone()
    old[3], adv[3] = -2000.0, 0.0
    r = policy_loss(x, y, old, adv, clip_high=math.inf)
    keep = torch.arange(20, device="cuda") != 3
    want = policy_loss(x[keep], y[keep], old[keep], adv[keep], clip_high=math.inf)
    assert float(r.loss) == pytest.approx(0.95 * float(want.loss), rel=8 * _u(_wide(kind)))
    assert bool((r.grad[3] == 0).all()) and torch.isfinite(r.grad.double()).all()


@pytest.mark.parametrize("c", [10, 100, 9001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,weight", [(3, 2.0**-129), (3, 2.0**-131), (1000, 2.0**120)])
def test_policy_weights_of_any_size(n, c, kind, weight):
    """All weights alike give the loss and the gradient of none at all, also where the inverse of
    their sum is beyond float32 or below its normal range. A product of a weight of 2^-129 and
    a slope is below it too: off by half of 2^-149, which is 2^-21 of the weight."""
    x, y = _make(11, n, c, kind, pad=0.0)
    lp = _define(x, y)[0].float()
    adv = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    args = (x, y, lp + 0.1, adv, lp - 0.2)
    a = policy_loss(*args, kl_coef=0.1)
    b = policy_loss(*args, kl_coef=0.1, sample_weight=torch.full_like(adv, weight))
    lost = 2.0**-150 / weight if weight < 1 else 0.0
    assert abs(float(b.loss) - float(a.loss)) <= 1e-6 * abs(float(a.loss)) + 4 * lost
    # the row's factor moves by that, and by three roundings; the result is rounded in both
    off = (a.grad.double() - b.grad.double()).abs()
    tol = a.grad.double().abs() * (6 * 2.0**-24 + torch.finfo(x.dtype).eps) + lost / n + 1e-37
    assert bool((off <= tol).all())


@pytest.mark.parametrize("c", [10, 100, 9001])
@pytest.mark.parametrize("kind", ["f64", "f32"])
def test_policy_terms_of_one_token_to_the_last_bits(c, kind):
    """One token's ratio and KL term from its own log-probability, so that the differences are
    the only roundings before them. Both inputs of the KL term's u are near, so that u is
    exact; the term by its series (ten or 17 steps, each less than a rounding of the whole) or
    by exp to 2 u and two differences, of at most 1.72 times what is left; the ratio by exp
    of a difference rounded to u |d|."""
    wide = _wide(kind)
    u = _u(wide)
    x = torch.zeros(1, c, dtype=wide, device="cuda")
    y = torch.tensor([1], device="cuda")
    lp = label_logprobs(x, y).logprobs
    one = torch.ones(1, dtype=wide, device="cuda")
    for i in range(-40, 41):
        away = 0.043 * i  # |u| < |lp| / 2 for c = 10 up to 1.15: exact there
        ref = lp + away
        if kind == "f32" and abs(away) * 2 > abs(float(lp)):
            continue
        old = lp + 5 * away
        r = policy_loss(x, y, old, one, ref, clip_high=math.inf, with_grad=False)
        d, a = float(lp) - float(old), float(ref) - float(lp)
        if abs(a) > 1e-6:
            want = math.expm1(a) - a if abs(a) > 0.4 else sum(
                a**k / math.factorial(k) for k in range(2, 24))
            rel = 8 * u + (16 * 2.0**-53 if abs(a) > 0.4 else 0)
            assert float(r.kl) == pytest.approx(want, rel=rel, abs=0), a
        assert float(r.loss) == pytest.approx(-math.exp(d), rel=(4 + abs(d)) * u, abs=0), d


@pytest.mark.parametrize("n,c", [(40, 10), (40, 100), (60, 4097), (30, 9001), (600, 9000)])
@pytest.mark.parametrize("lo", [0, 1, 2, 8])
@pytest.mark.parametrize("kind", list(TYPES))
def test_losses_of_pitched_scores(n, c, lo, kind):
    """Scores inside a wider matrix: their rows and the gradient's begin at other places within
    16 bytes, in every kernel that writes a gradient."""
    big, y = _make(12, n, c + 9 - c % 2, kind)
    x = big[:, lo:lo + c]
    y = torch.where(y >= c, -1, y)
    y[0], y[1], y[2] = 0, c - 1, c // 2
    wide = _wide(kind)
    u, e = _u(wide), _tol(x, wide)
    lp, lse, _, live = _define(x, y)
    zero = torch.zeros(n, dtype=torch.float64, device="cuda")
    r = label_logprobs(x, y)
    assert (r.lse.double() - lse).abs().max() <= e and (r.logprobs.double() - lp).abs().max() <= e
    g = torch.randn(n, generator=torch.Generator().manual_seed(1), dtype=wide).cuda()
    _check_grad(label_logprobs_grad(g, x, y, r.lse), x, y, g.double(), zero, wide)
    # the policy loss, all ratios exp(-0.1), inside the clip's bounds
    old = (lp + 0.1).to(wide)
    ratio, share = torch.exp(lp - old.double()), live.double() / live.sum()
    got = policy_loss(x, y, old, g)
    move = share * ratio * g.double().abs() * (e + 8 * u)
    assert abs(float(got.loss) + float((share * ratio * g.double()).sum())) <= float(move.sum()) + 4 * u
    _check_grad(got.grad, x, y, -share * ratio * g.double(), move, wide)
    # the preference loss of two pairs
    ip = torch.tensor([0, 8, 15, 22, n - 1], device="cuda")
    seq = torch.searchsorted(ip, torch.arange(n, device="cuda"), right=True) - 1
    s = torch.zeros(5, dtype=torch.float64, device="cuda").index_add_(0, seq, lp)[:4]
    ref = s.to(wide)
    q = s - ref.double()
    z = 0.3 * (q[:2] - q[2:])
    got = preference_loss(x, y, ip, ref, 0.3)
    assert float(got.loss) == pytest.approx(float(-torch.nn.functional.logsigmoid(z).mean()),
                                            abs=0.3 * n * e + 8 * u)
    slope = -0.15 * torch.sigmoid(-z)
    d = torch.cat([slope, -slope, torch.zeros(1, device="cuda", dtype=torch.float64)])[seq]
    moved = torch.where(d != 0, 0.15 * 0.3 * n * e / 4, 0.0)  # sigmoid's slope is at most 1 / 4
    _check_grad(got.grad, x, y, d, moved + 4 * u * d.abs(), wide)


@pytest.mark.parametrize("n,c", [(40, 10), (40, 32), (40, 100), (40, 4097), (20, 9001), (600, 9001)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scores_that_are_no_numbers_stay_in_their_rows(n, c, kind, bad):
    """A NaN or +infinity anywhere in a row makes the row NaN, masked rows keep their zeros, and
    no other row changes."""
    x, y = _make(13, n, c, kind, pad=0.0)
    rows = torch.arange(0, n, 3, device="cuda")
    x2, y2 = x.clone(), y.clone()
    x2[rows, (rows * 7919) % c] = bad
    y2[::6] = -1
    y[::6] = -1
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[rows] = True
    masked = y2 < 0
    one = torch.ones(n, dtype=_wide(kind), device="cuda")
    a, b = label_logprobs(x, y), label_logprobs(x2, y2)
    assert torch.equal(a.logprobs[~hit], b.logprobs[~hit]) and torch.equal(a.lse[~hit], b.lse[~hit])
    assert torch.isnan(b.lse[hit]).all() and torch.isnan(b.logprobs[hit & ~masked]).all()
    assert bool((b.logprobs[masked] == 0).all())
    g = label_logprobs_grad(one, x2, y2, b.lse)
    assert torch.isnan(g[hit & ~masked].double()).all() and bool((g[masked] == 0).all())
    assert torch.equal(g[~hit], label_logprobs_grad(one, x, y, a.lse)[~hit])
    w = (~hit).to(one.dtype)  # rows of weight 0 are left out, whatever is in them
    p, q = (policy_loss(v, l, -2 * one, one, -one, kl_coef=0.1, sample_weight=w)
            for v, l in ((x, y), (x2, y2)))
    assert torch.equal(p.loss, q.loss) and torch.equal(p.grad, q.grad)
    q = policy_loss(x2, y2, -2 * one, one)
    assert math.isnan(float(q.loss)) and bool((q.grad[masked] == 0).all())
    assert torch.equal(q.grad[~hit], policy_loss(x, y, -2 * one, one).grad[~hit])
