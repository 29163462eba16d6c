"""GPU tests of the label alternatives and their gradient against their definitions in
float64.

Tolerances, with u = 2^-24 (float32 arithmetic) or 2^-53 (float64), C classes of magnitude
at most X: log-probabilities and lse are off by e = (C / 8 + 36) u + 4 u X, as in
test_gpu_preference. With d = x - max, M1 = sum p |d| and M2 = sum p d^2, the entropy log S -
D / S is off by what S is (C / 8 + 32 u of itself: of the logarithm once, of D / S times M1),
by D's own sum (C / 8 + 16 u M1) and terms (an exponential 4 u + 2 u |d| of itself, d and the
product a rounding each: 6 u M1 + 2 u M2) and by four more roundings: eh = u ((C / 8 + 36) + (C / 4 + 58) M1 +
2 M2). A gradient s - p T with T = G + gH (x - lse + H) is off by p (e + 4 u + 2 u |x - lse|) |T|,
by p times T's error (33 u of the magnitudes that G adds, |gH| (e + eh + 4 u (|x - lse| + H))),
by 33 u of the magnitudes of s, 2 u of both parts, and half a step of the result's type.
Ranks and ids are exact.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.preference import (label_alternatives, label_alternatives_grad,  # noqa: E402
                                       label_logprobs)

from test_gpu_preference import TYPES, _make, _tol, _u, _wide  # noqa: E402

SHAPES = [(1, 1), (3, 2), (5, 10), (1000, 10), (33, 31), (300, 32), (17, 33), (9, 100), (70, 1000), (40, 1031), (4, 2049),
          (13, 5003), (2, 50001), (1, 120000), (1, 33), (2500, 100)]


def _define(x, y):
    """float64 (log-probabilities, lse, entropy, bound of its error over u, unmasked rows)."""
    w = x.double()
    c = x.shape[1]
    lse = torch.logsumexp(w, 1)
    live = ~torch.isneginf(lse)
    if y is not None:
        live &= (y >= 0) & (y < c)
    # not w - lse: beside scores of the lowest value the logarithm is lost in lse
    away = w - w.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float64).min)
    lp = away - torch.logsumexp(away, 1, keepdim=True)
    p = torch.where(live[:, None], torch.exp(lp), 0.0)
    lp = torch.where(live[:, None], lp, w)
    entropy = -(p * torch.where(p > 0, lp, 0.0)).sum(1)
    d = torch.where(p > 0, w - w.amax(1, keepdim=True), 0.0)
    m1, m2 = (p * d.abs()).sum(1), (p * d * d).sum(1)
    return lp, lse, entropy, (c / 8 + 36) + (c / 4 + 58) * m1 + 2 * m2, live


def _check(x, y, top, r=None):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    u, e, c = _u(wide), _tol(x, wide), x.shape[1]
    r = label_alternatives(x, y, top=top) if r is None else r
    lp, lse, entropy, eh, live = _define(x, y)
    kind = torch.int64 if y is None else y.dtype
    none = torch.zeros((), device="cuda", dtype=torch.float64)
    masked = torch.zeros_like(live) if y is None else (y < 0) | (y >= c)
    assert r.lse.dtype == r.entropy.dtype == wide
    assert torch.allclose(r.lse.double(), torch.where(masked, none, lse), rtol=0, atol=e)
    assert bool(((r.entropy.double() - torch.where(live, entropy, none)).abs() <= eh * u).all())
    assert bool((r.entropy >= 0).all())
    order = x.double().sort(dim=1, descending=True, stable=True).indices
    if y is None:
        assert r.logprobs is None and r.ranks is None
    else:
        at = y.long().clamp(0, c - 1)[:, None]
        want = torch.where(live, lp.gather(1, at)[:, 0], none)
        inf = torch.isneginf(want)
        assert torch.equal(inf, torch.isneginf(r.logprobs))
        assert bool(((r.logprobs.double() - want)[~inf].abs() <= e).all())
        place = (order == at).int().argmax(1)
        assert r.ranks.dtype == kind and torch.equal(r.ranks.long(), torch.where(live, place, -1))
    if not top:
        assert r.top_ids is None and r.top_logprobs is None
        return r
    assert r.top_ids.dtype == kind and r.top_ids.shape == r.top_logprobs.shape == (x.shape[0], top)
    assert torch.equal(r.top_ids.long(), torch.where(live[:, None], order[:, :top], -1))
    want = torch.where(live[:, None], lp.gather(1, order[:, :top]), none)
    inf = torch.isneginf(want)
    assert torch.equal(inf, torch.isneginf(r.top_logprobs))
    assert bool(((r.top_logprobs.double() - want)[~inf].abs() <= e).all())
    return r


def _check_grad(got, x, y, r, g_lp, g_h, ids, g_top):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    u, e, c = _u(wide), _tol(x, wide), x.shape[1]
    lp, lse, entropy, eh, live = _define(x, y)
    zero = torch.zeros(x.shape[0], device="cuda", dtype=torch.float64)
    gl = zero if g_lp is None else torch.where(live, g_lp.double(), 0.0)
    gh = zero if g_h is None else torch.where(live, g_h.double(), 0.0)
    s, size = torch.zeros(x.shape, device="cuda", dtype=torch.float64), torch.zeros(x.shape, device="cuda", dtype=torch.float64)
    total, mass = gl.clone(), gl.abs()
    if y is not None:
        at = y.long().clamp(0, c - 1)[:, None]
        s.scatter_add_(1, at, gl[:, None])
        size.scatter_add_(1, at, gl.abs()[:, None])
    if ids is not None:
        ok = (ids >= 0) & (ids < c) & live[:, None]
        gt = torch.where(ok, g_top.double(), 0.0)
        s.scatter_add_(1, ids.long().clamp(0, c - 1), gt)
        size.scatter_add_(1, ids.long().clamp(0, c - 1), gt.abs())
        total, mass = total + gt.sum(1), mass + gt.abs().sum(1)
    p = torch.where(live[:, None], torch.exp(lp), 0.0)
    z = torch.where(p > 0, lp, 0.0)
    t = total[:, None] + gh[:, None] * (z + torch.where(live, entropy, 0.0)[:, None])
    want = s - p * t
    ghn = gh.abs()[:, None]
    off_t = 33 * u * mass[:, None] + ghn * (e + (eh * u)[:, None] + 4 * u * (z.abs() + entropy[:, None].nan_to_num()))
    # a probability of less than 2^-126 is 0 in 32 bits
    tiny = (2.0**-25 if x.dtype == torch.float16 else 1e-37 if wide == torch.float32 else 0.0)
    tol = (p * (e + 4 * u + 2 * u * z.abs()) * t.abs() + p * off_t + 33 * u * size + 2 * u * (s.abs() + (p * t).abs())
           + torch.finfo(got.dtype).eps / 2 * want.abs() + tiny * (1 + t.abs() * 100))
    off = (got.double() - want).abs()
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed"
    assert bool((got[~live] == 0).all())


def _grads(x, top, seed=5):
    g = torch.Generator().manual_seed(seed)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    n = x.shape[0]
    return [torch.randn(s, generator=g, dtype=torch.float64).to(wide).cuda() for s in ((n,), (n,), (n, top))]


@pytest.mark.parametrize("n,c", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("label_type", [torch.int32, torch.int64])
def test_against_the_definition(n, c, kind, label_type):
    x, y = _make(1, n, c, kind, label_type)
    for top in sorted({0, 1, min(5, c), min(20, c), min(32, c)}):
        r = _check(x, y, top)
        g_lp, g_h, g_top = _grads(x, top)
        if top:
            g_top[:, 0] = 0.0
        d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top if top else None)
        _check_grad(d, x, y, r, g_lp, g_h, r.top_ids, g_top)
        again = label_alternatives(x, y, top=top)
        assert all(a is None or torch.equal(a, b) for a, b in zip(r, again))
    same = label_logprobs(x, y)
    assert (same.logprobs - r.logprobs).abs().max() <= 2 * _tol(x, _wide(kind))


@pytest.mark.parametrize("n,c", [(5, 10), (33, 100), (70, 1000), (3, 50001)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_parts_that_are_left_out(n, c, kind):
    x, y = _make(2, n, c, kind)
    top = min(7, c)
    r = _check(x, None, top)
    _check(x, None, 0)
    g_lp, g_h, g_top = _grads(x, top)
    _check_grad(label_alternatives_grad(x, r.lse, r.entropy, None, None, g_h, r.top_ids, g_top), x, None, r, None, g_h,
                r.top_ids, g_top)
    _check_grad(label_alternatives_grad(x, r.lse, grad_top=g_top, top_ids=r.top_ids), x, None, r, None, None, r.top_ids, g_top)
    assert bool((label_alternatives_grad(x, r.lse) == 0).all())
    r = _check(x, y, 0)
    _check_grad(label_alternatives_grad(x, r.lse, labels=y, grad_logprobs=g_lp), x, y, r, g_lp, None, None, None)
    _check_grad(label_alternatives_grad(x, r.lse, r.entropy, y, grad_entropy=g_h), x, y, r, None, g_h, None, None)
    # gradients that add up to 0, ids of no class, and a class named twice and by the label
    r = _check(x, y, top)
    ids = r.top_ids.clone()
    ids[:, 0], ids[:, -1] = y.clamp(0, c - 1), -1
    if top > 3:
        ids[:, 2], ids[:, 3] = ids[:, 1], c
    _check_grad(label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, ids, g_top), x, y, r, g_lp, g_h, ids, g_top)
    level = -g_lp[:, None] * torch.tensor([1.0] + [0.0] * (top - 1), device="cuda", dtype=g_lp.dtype)
    _check_grad(label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, None, r.top_ids, level), x, y, r, g_lp, None,
                r.top_ids, level)


@pytest.mark.parametrize("n,c", [(40, 10), (30, 32), (20, 100), (12, 1000), (12, 5003), (3, 50001), (3, 120000), (1300, 20000)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_ties_and_masked_classes(n, c, kind):
    """Few values, one value, few classes left, the lowest value in places: order by index."""
    x, y = _make(3, n, c, kind, pad=0.1)
    x = x.double().round().to(x.dtype)
    x[0] = 1.5
    x[1, :] = -math.inf
    x[1, c // 2] = 0.25
    x[1, c - 1] = 0.25
    y[1] = c - 1
    x[2, ::2] = torch.finfo(x.dtype).min
    if n > 3:
        x[3] = torch.finfo(x.dtype).min
        x[4] = -math.inf
        x[5, 1:] = -math.inf
        y[5] = c - 1  # of a class that is masked out
        x[6] = torch.where(torch.rand(c, device="cuda") < 0.5, 0.0, -0.0).to(x.dtype)
        x[7, c // 3:] = -math.inf
    for top in sorted({1, min(5, c), min(32, c)}):
        r = _check(x, y, top)
        _check(x, None, top)
        g_lp, g_h, g_top = _grads(x, top)
        if n > 5:
            g_lp[5] = 0.0
        d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
        _check_grad(d, x, y, r, g_lp, g_h, r.top_ids, g_top)


@pytest.mark.parametrize("n,c", [(3, 120000), (1300, 60000), (40, 3000)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f64"])
@pytest.mark.parametrize("offset", [0, 1])
def test_best_classes_in_the_hands_of_few_threads(n, c, kind, offset):
    """Every 32nd, 128th or 256th vector of 16 bytes holds the large values, rising or not, and the
    row's order among them is random: more of them than are listed as candidates."""
    g = torch.Generator().manual_seed(c)
    v = 128 // torch.finfo(TYPES[kind]).bits
    for lanes in (128, 256, 32):
        i = torch.arange(c)
        big = (((i + offset) // v) % lanes == 0) & (i > 200)
        x = torch.where(big, 50.0 + torch.rand(n, c, generator=g) * 8, torch.randn(n, c, generator=g)).to(TYPES[kind]).cuda()
        _check(x, None, 32)
        _check(torch.where(big.cuda(), i.cuda().to(x.dtype) / c + 50, x).to(x.dtype), None, 7)
        if n > 100:
            break


@pytest.mark.parametrize("c", [520, 1000, 2040])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("share", [4, 16])
def test_best_classes_in_the_hands_of_few_lanes(c, kind, share):
    """Rows that lanes hold in registers: 4 or 16 of 32 lanes have all large values, more than
    are listed as candidates, or less; some of them equal."""
    g = torch.Generator().manual_seed(c + share)
    v = 128 // torch.finfo(TYPES[kind]).bits
    big = (torch.arange(c) // v) % 32 < share
    x = torch.where(big, 50.0 + torch.rand(20, c, generator=g) * 8, torch.randn(20, c, generator=g))
    x[10:] = x[10:].round()
    x = x.to(TYPES[kind]).cuda()
    y = torch.randint(0, c, (20,), generator=g).cuda()
    for top in (1, 7, 16, 17, 32):
        _check(x, y, top)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vectors", [16, 30, 62, 125])
@pytest.mark.parametrize("share,lanes", [(1, 4), (3, 8), (6, 16)])
def test_best_classes_in_the_hands_of_few_lanes_of_a_group(vectors, kind, share, lanes):
    """The same of rows that share a warp, beside rows without: what a group lists may run over in
    some of them, among all values or among those above the ties."""
    g = torch.Generator().manual_seed(vectors + share)
    v = 128 // torch.finfo(TYPES[kind]).bits
    c = vectors * v
    big = (torch.arange(c) // v) % lanes < share
    x = torch.where(big, 50.0 + torch.rand(41, c, generator=g) * 8, torch.randn(41, c, generator=g))
    x[10:20] = x[10:20].round()
    x[20:24] = torch.where(big, 9.0, 4.0)
    x[24:28, ~big] = -math.inf
    x[1::3] = torch.randn(14, c, generator=g)
    x = x.to(TYPES[kind]).cuda()
    y = torch.randint(0, c, (41,), generator=g).cuda()
    for top in (1, 5, 10, 12, 20, 24, 32):
        _check(x, y, top)


@pytest.mark.parametrize("c", [33, 39, 64, 65, 100, 127, 128, 135, 200, 256, 263])
@pytest.mark.parametrize("kind", list(TYPES))
def test_short_rows_of_every_kind_beside_each_other(c, kind):
    """Several rows share a warp, each in a way of its own: plain, with ties, all equal, with few
    classes or none left, masked by their label, with signed zeros; at every place within 16 bytes."""
    g = torch.Generator().manual_seed(c)
    x = torch.randn(96, c, generator=g) * 2.5
    for i in range(0, 96, 2):  # neighbours differ
        what = i // 2 % 8
        if what == 0:
            x[i] = x[i].round()
        elif what == 1:
            x[i] = float(x[i, 0])
        elif what == 2:
            x[i, torch.randperm(c, generator=g)[3:]] = -math.inf
        elif what == 3:
            x[i] = -math.inf
        elif what == 4:
            x[i, ::2] = -math.inf
        elif what == 5:
            x[i] = torch.where(x[i] > 1.5, x[i], torch.where(x[i] > 0, 0.0, -0.0))
        elif what == 6:
            x[i] = torch.finfo(torch.float16).min
        else:
            x[i, :8] += 20
    y = torch.randint(0, c, (96,), generator=g)
    y[5::17] = -100
    pitch = c + 1
    flat = torch.full((96 * pitch,), 99.0, dtype=TYPES[kind], device="cuda")
    rows = flat.as_strided((96, c), (pitch, 1))
    rows.copy_(x.to(TYPES[kind]))
    for top in (1, 4, 5, 8, 9, 10, 11, 16, 17, 20, 24, 25, 32):
        _check(rows, y.cuda(), top)


@pytest.mark.parametrize("c", [10, 32, 100, 1000, 5003, 50001])
@pytest.mark.parametrize("kind", list(TYPES))
def test_not_finite(c, kind):
    x, y = _make(4, 8, c, kind, pad=0.0)
    x[1, c // 2] = math.nan
    x[2, 1] = math.inf
    x[3] = math.nan
    x[4, 0] = math.inf
    y[3:5] = -1
    top = min(5, c)
    r = label_alternatives(x, y, top=top)
    for t in (1, 2):
        for v in (r.logprobs[t], r.lse[t], r.entropy[t], r.top_logprobs[t]):
            assert bool(torch.isnan(v).all())
        assert int(r.ranks[t]) == -1 and bool((r.top_ids[t] == -1).all())
    for t in (3, 4):
        for v in (r.logprobs[t], r.lse[t], r.entropy[t], r.top_logprobs[t]):
            assert bool((v == 0).all())
        assert int(r.ranks[t]) == -1 and bool((r.top_ids[t] == -1).all())
    rest = [0, 5, 6, 7]
    pick = type(r)(*[v[rest] for v in r])
    _check(x[rest], y[rest], top, pick)
    g_lp, g_h, g_top = _grads(x, top)
    d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
    assert torch.isnan(d[1:3].double()).all() and bool((d[3:5] == 0).all())
    _check_grad(d[rest], x[rest], y[rest], pick, g_lp[rest], g_h[rest], pick.top_ids, g_top[rest])
    quiet = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp * 0, g_h * 0, r.top_ids, g_top * 0)
    assert bool((quiet == 0).all())
    # one NaN gradient stays in its row
    g_lp[0], g_h[5] = math.nan, math.nan
    d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
    assert torch.isnan(d[[0, 5]].double()).all() and torch.isfinite(d[6:].double()).all()


@pytest.mark.parametrize("n,c,pitch,first", [(30, 10, 13, 1), (30, 100, 131, 3), (30, 1000, 1001, 0), (30, 1000, 1017, 5), (9, 5003, 5009, 2), (3, 40000, 40003, 7), (50, 32, 40, 8)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_inside_a_wider_matrix(n, c, pitch, first, kind):
    whole, y = _make(5, n, pitch, kind)
    y = torch.where(y < c, y, c)
    x = whole[:, first:first + c]
    top = min(9, c)
    r = _check(x, y, top)
    g_lp, g_h, g_top = _grads(x, top)
    d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
    _check_grad(d, x, y, r, g_lp, g_h, r.top_ids, g_top)


@pytest.mark.parametrize("c", [7, 60, 700, 9001])
def test_gradient_against_differences(c):
    """Central differences of the operator in float64: with steps of h = 2^-17 the third
    derivative leaves 2 h^2 of the values' scale (a few units), rounding 2^-52 / h of it."""
    x, y = _make(6, 3, c, "f64", pad=0.0, std=1.0)
    top = min(4, c)
    g_lp, g_h, g_top = _grads(x, top)
    r = label_alternatives(x, y, top=top)

    def value(z):
        q = label_alternatives(z, y, top=top)
        best = torch.log_softmax(z, 1).gather(1, r.top_ids)  # of the same classes
        assert torch.equal(q.top_ids, r.top_ids)
        return (q.logprobs * g_lp + q.entropy * g_h).sum(), (best * g_top).sum()

    d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
    g = torch.Generator().manual_seed(1)
    h = 2.0**-17
    for _ in range(4):
        e = torch.randn(3, c, generator=g, dtype=torch.float64).cuda()
        gap = x.sort(1).values
        e *= min(1.0, float(gap.diff(dim=1)[:, -top:].min()) / h / 100)  # the order of the best stays
        up, down = value(x + h * e), value(x - h * e)
        rise = sum(float(a - b) for a, b in zip(up, down)) / (2 * h)
        scale = float((g_lp.abs() + g_h.abs() * 10 + g_top.abs().sum(1)).sum()) * float(e.abs().max()) ** 3
        assert abs(rise - float((d * e).sum())) <= scale * (20 * h * h + 2.0**-44 / h / max(1e-3, float(e.abs().max()) ** 2))


def test_offsets_beyond_32_bits():
    n, c = 70_001, 32_768
    x = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16)
    y = torch.full((n,), -1, device="cuda")
    gen = torch.Generator().manual_seed(0)
    rows = [0, 65_537, n - 2, n - 1]
    for t in rows:
        x[t] = torch.randn(c, generator=gen).bfloat16()
        y[t] = 17
    r = label_alternatives(x, y, top=20)
    pick = type(r)(*[v[rows] for v in r])
    _check(x[rows], y[rows], 20, pick)
    assert int((r.ranks >= 0).sum()) <= 4
    g_lp, g_h, g_top = _grads(x, 20)
    d = label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top)
    _check_grad(d[rows], x[rows], y[rows], pick, g_lp[rows], g_h[rows], pick.top_ids, g_top[rows])
    assert int((d != 0).any(1).sum()) == 4


def test_no_rows():
    x = torch.empty(0, 10, device="cuda")
    y = torch.empty(0, device="cuda", dtype=torch.int32)
    r = label_alternatives(x, y, top=3)
    assert r.top_ids.shape == (0, 3) and r.lse.shape == (0,)
    assert label_alternatives_grad(x, r.lse, r.entropy, y, r.logprobs, r.entropy, r.top_ids, r.top_logprobs).shape == (0, 10)


@pytest.mark.parametrize("n,c", [(500, 10), (100, 1000), (4, 50001)])
def test_streams_and_graphs(n, c):
    x, y = _make(7, n, c, "bf16")
    g_lp, g_h, g_top = _grads(x, 5)

    def both(stream=None):
        r = label_alternatives(x, y, top=5, stream=stream)
        return list(r) + [label_alternatives_grad(x, r.lse, r.entropy, y, g_lp, g_h, r.top_ids, g_top, stream=stream)]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = both()
        graphs.append((graph, out))
    x.copy_(_make(8, n, c, "bf16")[0])
    want = both()
    for graph, out in graphs:
        graph.replay()
    for graph, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("dtype", ["float32-float64", "float64", "float32"])
def test_resident_model(dtype):
    """The alternatives of a resident model's own scores."""
    from test_gpu_model_policy import _case, _csr, _model

    X, w0, w, V, R, fid, rng = _case(3, "fm", 7)
    labels = torch.from_numpy(rng.integers(-1, 7, size=X.shape[0])).cuda()
    with _model("fm", 7, dtype, X, w0, w, V, R, fid) as m:
        csr = _csr(X, dtype)
        _check(m.scores_device(*csr), labels, 4, m.label_alternatives_device(*csr, labels, top=4))
        _check(m.scores_device(*csr), None, 0, m.label_alternatives_device(*csr))
    X, w0, w, V, R, fid, rng = _case(3, "fm", 1)
    with _model("fm", 1, dtype, X, w0, w, V, R, fid) as m, pytest.raises(ValueError, match="n_classes >= 2"):
        m.label_alternatives_device(*_csr(X, dtype))
