"""GPU tests of the AdamW step against its formulas in float64, a step at a time from the
state that the step before left.

Tolerances, with u = 2^-24 (2^-53 for float64 parameters): m is off by at most 6 u of its two
terms' magnitudes (a rounding each for the scaled gradient's two factors, the constant, the
product and the sum), v, whose gradient is squared, by 8 u of itself. The move m i1 / (sqrt(v
i2) + eps) is off by what m is off, divided by the denominator, and 16 u of itself (v's 8 u
halved by the root, i1 and i2 with 6 u each, of which i2's is halved, four roundings). p is
off by lr times that, 4 u of lr times the move, 4 u of itself and of its decay, and half a
step of its type. A norm is off by 32 u (8 squares added in 32 bits, a rounding to 32 bits).
The formulas in float64 make the same roundings: against them a float64 result may be off by
twice that (1 - b^t is expm1 there too: the difference would lose log2(1 / (1 - b^t)) of its
53 bits, 8 at the third step).
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.embedding import EmbeddingRows  # noqa: E402
from modern_fm_b200.optim import AdamW, AdamWState  # noqa: E402

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16,
         "f16": torch.float16}
SIZES = [1, 31, 32, 33, 100, 255, 2047, 2048, 2049, 10007]
B1, B2 = 0.9, 0.999


def _u(t):
    return 2.0**-53 if t == torch.float64 else 2.0**-24


def _tensors(sizes, kind, seed=0, std=0.3, off=0):
    """Contiguous tensors that begin `off` values into their memory."""
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n + off, generator=g, dtype=torch.float64) * std).to(TYPES[kind]).cuda()[off:]
            for n in sizes]


def _want(p, g, m, v, t, lr, wd, eps, scale=1.0):
    """float64 (p, m, v) and the bounds of p, m and v's errors; all inputs float64."""
    g = g * scale
    m1, v1 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    i1, i2 = (-1 / torch.expm1(torch.as_tensor(t, dtype=torch.float64) * math.log(b)).to(p.device) for b in (B1, B2))
    den = torch.sqrt(v1 * i2) + eps
    move = m1 * i1 / den
    p1 = p - lr * wd * p - lr * move
    em = 6 * ((B1 * m).abs() + ((1 - B1) * g).abs())
    ep = lr * (em * i1 / den + 20 * move.abs()) + 4 * p.abs() * (1 + lr * wd)
    return (p1, m1, v1), (ep, em, 8 * v1)


def _near(got, want, bound, u, what):
    half = torch.finfo(got.dtype).eps / 2 * want.abs() if got.dtype in (torch.bfloat16, torch.float16) else 0.0
    tiny = 2.0**-25 if got.dtype == torch.float16 else 0.0
    off = (got.double() - want).abs()
    tol = bound * u * (2 if got.dtype == torch.float64 else 1 + 1e-3) + half * (1 + 1e-3) + tiny + 1e-37
    assert bool((off <= tol).all()), f"{what}: off by {float((off - tol).max())} more than allowed"


def _check(opt, before, grads, lr, wd, eps=1e-8, scale=1.0, which=None):
    """The tensors of `opt` after a step against the step from `before` = (p, m, v, t) each."""
    for i in range(len(opt.params)) if which is None else which:
        p, m, v, t = before[i]
        u = _u(opt.params[i].dtype)
        want, bound = _want(p, grads[i].double(), m, v, t, lr, wd[i], eps, scale)
        master = opt.state.master is not None and opt.params[i].dtype in (torch.bfloat16, torch.float16)
        _near(opt.params[i], want[0], bound[0], u, f"parameter {i}")
        if master:
            at = opt._master_at[i]
            _near(opt.state.master[at:at + p.numel()].view_as(p), want[0], bound[0], u, f"master {i}")
        if opt._bits == 32:
            _near(opt.view(opt.state.m, i), want[1], bound[1], u, f"m {i}")
            _near(opt.view(opt.state.v, i), want[2], bound[2], u, f"v {i}")


def _now(opt, t):
    """(p, m, v, t) of every tensor in float64; p from the master weights where there are any."""
    m, v = opt.moments()
    out = []
    for i, p in enumerate(opt.params):
        if opt.state.master is not None and p.dtype in (torch.bfloat16, torch.float16):
            at = opt._master_at[i]
            p = opt.state.master[at:at + p.numel()].view_as(p)
        out.append((p.double().clone(), opt.view(m, i).double().clone(), opt.view(v, i).double().clone(), t))
    return out


@pytest.mark.parametrize("kind,grad", [("f64", "f64"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("off", [0, 1, 4])
@pytest.mark.parametrize("master", [False, True])
def test_dense(kind, grad, off, master):
    if master and kind in ("f64", "f32"):
        pytest.skip("no master weights of these")
    ps = _tensors(SIZES, kind, 1, off=off)
    wd = [0.1 * (i % 3) for i in range(len(SIZES))]
    opt = AdamW(ps, lr=1e-2, weight_decay=wd, master=master)
    for t in range(1, 4):
        gs = _tensors(SIZES, grad, 10 + t, 0.02, off)
        before = _now(opt, t)
        assert opt.step(gs) is None
        assert int(opt.state.step) == t
        _check(opt, before, gs, 1e-2, wd)


def test_hundreds_of_tensors_and_types_and_missing_gradients():
    sizes = [1 + (i * 37) % 3000 for i in range(900)]
    ps = _tensors(sizes[:450], "f32", 2) + _tensors(sizes[450:], "bf16", 3)
    ps = [p for pair in zip(ps[:450], ps[450:]) for p in pair]
    opt = AdamW(ps, lr=1e-3, weight_decay=0.01)
    gs = [torch.randn_like(p) for p in ps]
    before = _now(opt, 1)
    norm = opt.step(gs, max_norm=1e9)
    _check(opt, before, gs, 1e-3, [0.01] * 900)
    whole = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert float(norm) == pytest.approx(whole, rel=32 * 2.0**-24)
    missing = {0, 5, 899}
    some = [None if i in missing else g for i, g in enumerate(gs)]
    before = _now(opt, 2)
    opt.step(some)
    _check(opt, before, gs, 1e-3, [0.01] * 900, which=[i for i in range(900) if i not in missing])
    for i in missing:
        assert torch.equal(opt.params[i].double(), before[i][0])
    opt.step([None] * 900)
    assert int(opt.state.step) == 3


@pytest.mark.parametrize("kind", list(TYPES))
def test_clip(kind):
    wide = torch.float64 if kind == "f64" else torch.float32
    ps, gs = _tensors(SIZES, kind, 4), _tensors(SIZES, kind, 5, 0.5)
    opt = AdamW(ps, lr=1e-2, weight_decay=0.0)
    whole = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    for t, (scale, most) in enumerate([(1.0, whole / 7), (0.25, whole), (2.0, whole / 3), (1.0, math.inf),
                                       (-1.0, whole / 2), (1.0, 0.0)], 1):
        before = _now(opt, t)
        norm = opt.step(gs, grad_scale=scale, max_norm=most)
        assert norm.dtype == wide and norm.dim() == 0
        assert float(norm) == pytest.approx(abs(scale) * whole, rel=32 * _u(wide))
        # the factor is off by what the norm is: more than the formula's bounds have for it
        factor = scale * min(1.0, most / (abs(scale) * whole))
        for i, p in enumerate(opt.params):
            want, bound = _want(before[i][0], gs[i].double(), before[i][1], before[i][2], t, 1e-2, 0.0, 1e-8, factor)
            grown = [b + 40 * (1 - B1) * (gs[i].double() * factor).abs() for b in bound[:2]]
            den = torch.sqrt(want[2] / (1 - B2**t)) + 1e-8
            grown[0] = bound[0] + 1e-2 * (40 * (1 - B1) * (gs[i].double() * factor).abs() / (1 - B1**t) / den
                                          + 40 * (want[1] / (1 - B1**t) / den).abs())
            _near(p, want[0], grown[0], _u(wide), f"parameter {i}")
            _near(opt.view(opt.state.m, i), want[1], grown[1], _u(wide), f"m {i}")
            _near(opt.view(opt.state.v, i), want[2], bound[2] + 80 * want[2], _u(wide), f"v {i}")


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_that_is_not_finite_changes_nothing(kind, bits):
    if kind == "f64" and bits == 8:
        pytest.skip("not offered")
    ps, gs = _tensors([33, 5000], kind, 6), _tensors([33, 5000], kind, 7)
    table = _tensors([70], kind, 8)[0].view(10, 7)
    rows = EmbeddingRows(torch.tensor([1, 4, -1], device="cuda"), torch.ones(3, 7, device="cuda", dtype=TYPES[kind]),
                         torch.tensor(2, device="cuda"), None)
    opt = AdamW(ps + [table], by_rows=[False, False, True], state_bits=bits)
    opt.step(gs + [rows], max_norm=1.0)
    kept = [x.clone() for x in opt.params] + [x.clone() for x in opt.state if x is not None]
    for bad in (math.inf, -math.inf, math.nan):
        for where in ((0, 0), (1, 4999)):
            worse = [g.clone() for g in gs]
            worse[where[0]][where[1]] = bad
            norm = opt.step(worse + [rows], max_norm=1.0)
            assert not math.isfinite(float(norm))
        worse = rows._replace(rows=rows.rows.clone())
        worse.rows[1, 6] = bad
        assert not math.isfinite(float(opt.step(gs + [worse], max_norm=1.0)))
        now = list(opt.params) + [x for x in opt.state if x is not None]
        assert all(torch.equal(a, b) for a, b in zip(kept, now))
    # behind the count anything may stand
    worse = rows._replace(rows=rows.rows.clone())
    worse.rows[2] = math.nan
    assert math.isfinite(float(opt.step(gs + [worse], max_norm=1.0)))
    assert int(opt.state.step) == 2


def test_norms_beyond_the_squares_range():
    for size in (1e-30, 1e-22, 1e25, 3e38):
        g = torch.full((3000,), size, device="cuda")
        norm = AdamW([torch.zeros(3000, device="cuda")]).step([g], max_norm=1.0)
        assert float(norm) == pytest.approx(min(size * math.sqrt(3000), math.inf), rel=1e-6) or size == 3e38
    assert float(AdamW([torch.zeros(5, device="cuda")]).step([torch.zeros(5, device="cuda")], max_norm=1.0)) == 0.0


# ------------------------------------------------------------------ 8 bits --


def _grid(x, up):
    """x >= 0 rounded down or up to 3 bits of mantissa, float64."""
    f, e = torch.frexp(x)
    k = f * 16
    k = torch.ceil(k) if up else torch.floor(k)
    return torch.where(x > 0, torch.ldexp(k, e - 4), 0.0)


@pytest.mark.parametrize("kind,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("master", [False, True])
def test_moments_in_8_bits(kind, grad, off, master):
    """Each moment is one of its two neighbours among the values of 3 bits of mantissa (m: the
    nearer one, up to m's error), or below the block's reach: 0 or the smallest for m, the smallest for v."""
    if master and kind == "f32":
        pytest.skip("no master weights of these")
    u = 2.0**-24
    ps = _tensors(SIZES, kind, 11, off=off)
    opt = AdamW(ps, lr=1e-3, weight_decay=0.1, state_bits=8, master=master, seed=7)
    for t in range(1, 5):
        gs = _tensors(SIZES, grad, 20 + t, 0.02, off)
        for g in gs:  # a wide range within a block
            g.mul_(10.0 ** (torch.arange(g.numel(), device="cuda") % 9 - 6).to(g.dtype))
        before = _now(opt, t)
        opt.step(gs)
        _check(opt, before, gs, 1e-3, [0.1] * len(SIZES))
        m, v = opt.moments()
        for i in range(len(SIZES)):
            p0, m0, v0, _ = before[i]
            want, bound = _want(p0, gs[i].double(), m0, v0, t, 1e-3, 0.1, 1e-8)
            for got, x, e, octaves in ((opt.view(m, i).double(), want[1], bound[1] * u, 15),
                                       (opt.view(v, i).double(), want[2], bound[2] * u, 31)):
                a, s = x.abs(), torch.sign(x)
                n = -(-x.numel() // 32) * 32
                top = torch.nn.functional.pad(a + e, (0, n - x.numel())).view(-1, 32).amax(1)
                # the block's least value: 2^-octaves of the largest's power of two, or less
                least = torch.ldexp(torch.ones_like(top), torch.frexp(top)[1] - octaves).repeat_interleave(32)[:x.numel()]
                low, high = _grid((a - e).clamp(min=0), False), _grid(a + e, True)
                fits = (got.abs() >= low) & (got.abs() <= high) & ((got == 0) | (torch.sign(got) == s) | (a <= e))
                small = (a <= 2 * least) & (got.abs() <= 2 * least)
                if octaves == 31:
                    small &= (got > 0) | (a <= e)
                    assert bool((got[a > 0] > 0).all())
                else:
                    near = (got.abs() - a).abs() <= (high - low).abs() * (0.5 + 2.0**-13) + e
                    fits &= near
                assert bool((fits | small).all())


@pytest.mark.parametrize("kind,master", [("bf16", False), ("f32", False), ("f16", True)])
def test_large_tensors_in_8_bits(kind, master):
    """More than a block's share of chunks, in several tensors that end anywhere: parameters to
    their bounds, moments to a step of their codes and 2^-14 of their block's largest."""
    sizes = [17_000_003, 40, 9_000_031, 1 << 20]
    ps = _tensors(sizes, kind, 13)
    opt = AdamW(ps, lr=1e-3, weight_decay=0.1, state_bits=8, master=master)
    for t in (1, 2):
        gs = [torch.randn_like(p) * 0.02 for p in ps]
        before = _now(opt, t)
        opt.step(gs)
        _check(opt, before, gs, 1e-3, [0.1] * 4)
        m, v = opt.moments()
        for i, n in enumerate(sizes):
            want, _ = _want(before[i][0], gs[i].double(), before[i][1], before[i][2], t, 1e-3, 0.1, 1e-8)
            for flat, x in ((m, want[1]), (v, want[2])):
                whole = torch.nn.functional.pad(x.abs(), (0, -n % 32)).view(-1, 32).amax(1).repeat_interleave(32)[:n]
                assert bool(((opt.view(flat, i).double() - x).abs() <= x.abs() / 8 + 2.0**-14 * whole).all())
        del before, m, v


def test_rounding_of_v_keeps_its_average():
    """A thousand steps' worth of values, each moved by less than half a step of its code: their
    mean moves as v does. v's values after one step lie on two codes a step h apart, up with
    probability f: the mean of n independent ones is off by h sqrt(f (1 - f) / n), here at
    most six times that; and the neighbours' choices are independent."""
    n = 1 << 20
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1.0, device="cuda")
    opt = AdamW([p], lr=0.0, state_bits=8, betas=(B1, B2), seed=3)
    opt.step([g])  # v = 0.001 everywhere, rounded to the codes next to it
    for step in range(4):
        v0 = opt.moments()[1].double()
        opt.step([g * (1 + step)])
        v = opt.moments()[1].double()
        want = B2 * v0 + (1 - B2) * (1.0 + step) ** 2
        low, high = _grid(want, False), _grid(want, True)
        assert bool(((v == low) | (v == high)).all())
        f = torch.where(high > low, (want - low) / (high - low), 0.0)
        spread = math.sqrt(float(((high - low) ** 2 * f * (1 - f)).sum()))
        assert abs(float((v - want).sum())) <= 6 * spread
        up = ((v - want) / (high - low).clamp(min=1e-30))
        pairs = (up[1:] * up[:-1]).sum() / (up * up).sum()
        assert abs(float(pairs)) <= 6 / math.sqrt(n)
    others = [AdamW([p], lr=0.0, state_bits=8, seed=seed) for seed in (3, 3, 4)]
    for o in others:
        o.step([g])
    assert torch.equal(others[0].state.v, others[1].state.v) and not torch.equal(others[0].state.v, others[2].state.v)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-3, 1.0, 3.0, 1000.0, 3e4, 7e4, 1e10, 1e17])
def test_codes_at_every_scale(scale, off):
    """b1 = b2 = 0: m is the gradient to 1 / 16 of itself (half a step; 2^-13 more for where
    ties go), v its square to 1 / 8, if they are within the codes' reach of 15 and 31 octaves.
    Below 2^-126 float32 values, and codes, have steps of one size: 2^-129 with 3 bits, of which half
    (and 2^-13) is lost, and all of a value below half."""
    g = torch.Generator().manual_seed(1)
    size = torch.exp2(-12 * torch.rand(4096 + off, generator=g)) * torch.where(torch.rand(4096 + off, generator=g) < 0.5, -1, 1)
    x = (size * scale).cuda()[off:]
    opt = AdamW([torch.zeros(4096 + off, device="cuda")[off:]], state_bits=8, betas=(0.0, 0.0), lr=0.0)
    opt.step([x])
    m, v = (t.double() for t in opt.moments())
    x = x.double()
    assert bool(((m - x).abs() <= x.abs() * (1 / 16 + 2.0**-13) + 2.0**-130 * (1 + 2.0**-12)).all())
    if 1e-18 < scale:
        assert bool(((v - x * x).abs() <= x * x * (1 / 8 + 2.0**-20)).all())
    assert bool((torch.sign(m) == torch.sign(x))[x.abs() >= 2.0**-129].all())


def test_codes_of_extreme_values():
    """Zero, infinity and NaN, and magnitudes from the smallest to the largest float32."""
    x = torch.tensor([0.0, -0.0, 1.0, -1.0, 1.9999999, 3.4028235e38, -3.4028235e38, 1e-38, 1e-45, 1.17e-38] + [0.0] * 22,
                     device="cuda")
    for first in (None, 2, 5, 7, 8):
        g = torch.zeros(64, device="cuda")
        g[:32] = x if first is None else torch.where(torch.arange(32, device="cuda") == first, x, 0.0)
        opt = AdamW([torch.zeros(64, device="cuda")], state_bits=8, betas=(0.0, 0.0), lr=0.0)
        opt.step([g])
        m, v = (t.float() for t in opt.moments())
        assert bool((m[g == 0] == 0).all()) and bool((v[g == 0] == 0).all())
        assert bool(torch.isfinite(m).all())
        big = g.abs() == g.abs().max()
        if float(g.abs().max()) > 1.2e-38:
            assert bool(((m[big] - g[big]).abs() <= g[big].abs() / 15).all())
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.full((64,), 0.5, device="cuda")
        g[5] = bad
        opt = AdamW([torch.zeros(64, device="cuda")], state_bits=8, lr=0.0)
        opt.step([g])
        m, v = (t.float() for t in opt.moments())
        rest = torch.arange(64, device="cuda") != 5
        assert bool(torch.isfinite(m[rest]).all()) and bool(torch.isfinite(v[rest]).all())
        assert (math.isnan(float(m[5])) if math.isnan(bad) else float(m[5]) == bad)
        assert not math.isfinite(float(v[5]))


# ------------------------------------------------------------------- rows --


@pytest.mark.parametrize("kind,grad", [("f64", "f64"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,d,pitch", [(7, 1, 1), (40, 16, 16), (40, 17, 20), (100, 33, 33), (300, 8, 8), (50, 300, 304), (60, 24, 24), (30, 40, 48),
                                       (20, 256, 256), (9, 1000, 1000), (30, 104, 104)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_rows(kind, grad, n, d, pitch, bits, ids):
    if kind == "f64" and bits == 8:
        pytest.skip("not offered")
    g = torch.Generator().manual_seed(n * d)
    store = (torch.randn(n, pitch, generator=g, dtype=torch.float64) * 0.3).to(TYPES[kind]).cuda()
    outside = store[:, d:].clone()
    table = store[:, :d]
    other = _tensors([77], kind, 3)[0]
    opt = AdamW([table, other], lr=1e-2, weight_decay=0.05, state_bits=bits, by_rows=[True, False])
    steps = torch.zeros(n, dtype=torch.float64)
    for t in range(1, 5):
        some = torch.randperm(n, generator=g)[: max(1, n // 3)].sort().values
        cap = some.numel() + 3
        keys = torch.full((cap,), -1, dtype=ids)
        keys[:some.numel()] = some.to(ids)
        rows = torch.randn(cap, d, generator=g, dtype=torch.float64).to(TYPES[grad]).cuda() * 0.02
        grads = EmbeddingRows(keys.cuda(), rows, torch.tensor(some.numel(), device="cuda"), None)
        og = torch.randn(77, generator=g, dtype=torch.float64).to(TYPES[kind]).cuda()
        before = _now(opt, t)
        opt.step([grads, og])
        steps[some] += 1
        assert torch.equal(opt.state.row_steps.cpu().double(), steps)
        p0, m0, v0, _ = before[0]
        full = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        full[some.cuda()] = rows[:some.numel()].double()
        touched = torch.zeros(n, dtype=torch.bool, device="cuda")
        touched[some.cuda()] = True
        tt = steps.clamp(min=1)[:, None].cuda()
        want, bound = _want(p0, full, m0, v0, tt, 1e-2, 0.05, 1e-8)
        m, v = opt.moments()
        u = _u(table.dtype)
        _near(table[touched], want[0][touched], bound[0][touched], u, "rows")
        assert torch.equal(table[~touched].double(), p0[~touched])
        for flat, old, x, e in ((m, m0, want[1], bound[1]), (v, v0, want[2], bound[2])):
            now = opt.view(flat, 0)
            assert torch.equal(now[~touched].double(), old[~touched])
            if bits == 32:
                _near(now[touched], x[touched], e[touched], u, "moments")
            else:
                off = (now.double() - x).abs()[touched]
                top = x.abs().amax(1, keepdim=True)[touched]
                assert bool((off <= x.abs()[touched] / 8 + 2.0**-14 * top).all())
        assert torch.equal(store[:, d:], outside)
        _check(opt, before, [None, og], 1e-2, [0, 0.05], which=[1])


def test_rows_left_out():
    """Keys outside the table, behind the count, or not above the one before."""
    table = torch.randn(10, 4, device="cuda")
    kept = table.clone()
    opt = AdamW([table], by_rows=True, lr=0.1)
    keys = torch.tensor([-3, 2, 2, 5, 4, 7, 10, 9], device="cuda")
    rows = torch.ones(8, 4, device="cuda")
    opt.step([EmbeddingRows(keys, rows, torch.tensor(7, device="cuda"), None)])
    assert opt.state.row_steps.tolist() == [0, 0, 1, 0, 0, 1, 0, 1, 0, 0]
    moved = (table != kept).any(1)
    assert moved.nonzero()[:, 0].tolist() == [2, 5, 7]
    for count in (0, -5):
        kept = table.clone()
        opt.step([EmbeddingRows(keys, rows, torch.tensor(count, device="cuda"), None)])
        assert torch.equal(table, kept)
    opt.step([EmbeddingRows(keys, rows, torch.tensor(10**12, device="cuda"), None)])
    assert opt.state.row_steps.tolist() == [0, 0, 2, 0, 0, 2, 0, 2, 0, 0]  # 9 is not above 10
    opt.step([EmbeddingRows(keys[:0], rows[:0], torch.tensor(0, device="cuda"), None)])
    opt.step([None])
    assert int(opt.state.step) == 6


def test_offsets_beyond_32_bits():
    """The last rows of a table of more than 2^32 bytes of codes; a dense tensor of 2^31 + 5 values."""
    n, d = (1 << 22) + 3, 1100
    table = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    opt = AdamW([table], by_rows=True, state_bits=8, lr=0.5, weight_decay=0.0)
    keys = torch.tensor([0, n - 2, n - 1], device="cuda")
    rows = torch.ones(3, d, device="cuda", dtype=torch.bfloat16) * torch.tensor([[1.0], [2.0], [-1.0]], device="cuda").bfloat16()
    opt.step([EmbeddingRows(keys, rows, torch.tensor(3, device="cuda"), None)])
    assert bool((table[0] == -0.5).all()) and bool((table[n - 2] == -0.5).all()) and bool((table[n - 1] == 0.5).all())
    assert int((table != 0).sum()) == 3 * d
    m, v = opt.moments()
    assert bool((opt.view(m, 0)[n - 1] < 0).all()) and int((m != 0).sum()) == 3 * d == int((v != 0).sum())
    del table, opt, m, v
    torch.cuda.empty_cache()
    n = (1 << 31) + 5
    p, g = torch.zeros(n, device="cuda", dtype=torch.bfloat16), torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-3:] = 1.0
    g[1 << 30] = -1.0
    opt = AdamW([p], state_bits=8, lr=0.5, weight_decay=0.0)
    norm = opt.step([g], max_norm=10.0)
    assert float(norm) == 2.0
    at = (p != 0).nonzero()[:, 0].tolist()
    assert at == [1 << 30, n - 3, n - 2, n - 1] and float(p[-1]) == -0.5


# ---------------------------------------------------------- how it is used --


def _model(kind="bf16", bits=8, master=True):
    ps = _tensors(SIZES, kind, 30)
    table = _tensors([64 * 20], kind, 31)[0].view(64, 20)
    return AdamW(ps + [table], lr=1e-2, state_bits=bits, master=master, by_rows=[False] * len(ps) + [True])


def _grads(kind, seed):
    rows = EmbeddingRows(torch.tensor([1, 5, 63, -1], device="cuda"), _tensors([80], kind, seed + 1)[0].view(4, 20),
                         torch.tensor(3, device="cuda"), None)
    return _tensors(SIZES, kind, seed) + [rows]


def _all(opt):
    return [p.clone() for p in opt.params] + [s.clone() for s in opt.state if s is not None]


@pytest.mark.parametrize("kind,bits,master", [("bf16", 8, True), ("f32", 32, False), ("f16", 8, False)])
def test_state_is_handed_on_and_steps_are_reproducible(kind, bits, master):
    a, b = _model(kind, bits, master), _model(kind, bits, master)
    for t in range(3):
        a.step(_grads(kind, t), max_norm=0.5)
        b.step(_grads(kind, t), max_norm=0.5)
    assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(b)))
    state = AdamWState(*[None if s is None else s.clone() for s in b.state])
    c = AdamW([p.clone() for p in b.params], lr=1e-2, state_bits=bits, master=master,
              by_rows=[False] * len(SIZES) + [True], state=state)
    assert c.state.m is state.m
    for t in range(3, 5):
        a.step(_grads(kind, t), max_norm=0.5)
        c.step(_grads(kind, t), max_norm=0.5)
    assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(c)))


@pytest.mark.parametrize("kind,bits,master", [("bf16", 8, True), ("f32", 32, False)])
def test_captured_step(kind, bits, master):
    """Replays go on counting and read rate and scale anew."""
    a, b = _model(kind, bits, master), _model(kind, bits, master)
    grads = _grads(kind, 1)
    _model(kind, bits, master).step(grads, max_norm=0.3)
    lr, scale = (torch.tensor(x, device="cuda", dtype=torch.float64) for x in (1e-2, 1.0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = b.step(grads, lr=lr, grad_scale=scale, max_norm=0.3)
    assert int(b.state.step) == 0
    for rate, factor in ((1e-2, 1.0), (5e-3, 0.5), (1e-3, 4.0)):
        lr.fill_(rate)
        scale.fill_(factor)
        want = a.step(grads, lr=rate, grad_scale=factor, max_norm=0.3)
        graph.replay()
        assert torch.equal(norm, want)
        assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(b)))
    assert int(b.state.step) == 3


def test_on_another_stream():
    a, b = _model(), _model()
    side = torch.cuda.Stream()
    for t in range(3):
        a.step(_grads("bf16", t), max_norm=1.0)
        grads = _grads("bf16", t)
        side.wait_stream(torch.cuda.current_stream())
        b.step(grads, max_norm=1.0, stream=side)
        m, v = b.moments(stream=side)
        del grads
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(b)))
    assert all(torch.equal(x, y) for x, y in zip((m, v), a.moments()))


def test_two_on_two_streams():
    """Steps of two optimizers in flight at once, and from two threads."""
    import threading

    pairs = [(_model("bf16", 8, True), _model("bf16", 8, True)), (_model("f32", 32, False), _model("f32", 32, False))]
    streams = [torch.cuda.Stream() for _ in pairs]
    grads = [[_grads(kind, t) for t in range(20)] for kind in ("bf16", "f32")]
    torch.cuda.synchronize()
    for (a, _), gs in zip(pairs, grads):
        for g in gs:
            a.step(g, max_norm=0.7)
    torch.cuda.synchronize()

    def run(opt, gs, stream):
        for g in gs:
            opt.step(g, max_norm=0.7, stream=stream)

    threads = [threading.Thread(target=run, args=(b, gs, s)) for (_, b), gs, s in zip(pairs, grads, streams)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for a, b in pairs:
        assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(b)))


def test_empty_tensors():
    ps = [torch.zeros(0, device="cuda"), torch.ones(3, device="cuda"), torch.zeros(0, 5, device="cuda")]
    opt = AdamW(ps, by_rows=[False, False, True])
    none = EmbeddingRows(torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, 5, device="cuda"),
                         torch.tensor(0, device="cuda"), None)
    opt.step([torch.zeros(0, device="cuda"), torch.ones(3, device="cuda"), none], max_norm=1.0)
    assert int(opt.state.step) == 1 and bool((ps[1] < 1).all())
    assert AdamW([torch.zeros(0, device="cuda")]).step([torch.zeros(0, device="cuda")], max_norm=1.0) == 0


def test_refusals():
    f = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
    both = f(10)
    for params, kw, msg in [
            ([f(4, 4).t()[:, 1:]], {}, "contiguous"),
            ([both, both[3:]], {}, "overlap"),
            ([both, both], {}, "overlap"),
            ([f(3), f(3, t=torch.float64)], {}, "float64 parameters"),
            ([f(3, t=torch.float64)], dict(state_bits=8), "at most 32 bits"),
            ([f(3)], dict(by_rows=True), "matrix"),
            ([f(4, 4).t()], dict(by_rows=True), "contiguous rows")]:
        with pytest.raises(ValueError, match=msg):
            AdamW(params, **kw)
    opt = AdamW([f(3, 4), f(5, 4, t=torch.bfloat16)], by_rows=[False, True])
    rows = EmbeddingRows(torch.zeros(2, dtype=torch.int64, device="cuda"), f(2, 4), torch.tensor(1, device="cuda"), None)
    good = [f(3, 4), rows]
    opt.step(good)
    for grads, msg in [
            (good[:1], "one gradient"),
            ([f(4, 3), rows], "shape"),
            ([f(4, 3).t(), rows], "contiguous"),
            ([f(3, 4, t=torch.bfloat16), rows], "must have its type"),
            ([torch.zeros(3, 4), rows], "CUDA tensor"),
            ([f(3, 4), f(5, 4)], "EmbeddingRows"),
            ([rows, rows], "dense parameter is a tensor"),
            ([f(3, 4), rows._replace(rows=f(2, 5))], "width per key"),
            ([f(3, 4), rows._replace(rows=f(3, 4))], "width per key"),
            ([f(3, 4), rows._replace(keys=f(2))], "keys must be"),
            ([f(3, 4), rows._replace(count=torch.tensor(1.0, device="cuda"))], "count must be"),
            ([f(3, 4), rows._replace(count=torch.tensor(1))], "CUDA tensor")]:
        with pytest.raises(ValueError, match=msg):
            opt.step(grads)
    for kw, msg in [(dict(max_norm=-1.0), "max_norm"), (dict(max_norm=math.nan), "max_norm"),
                    (dict(lr=f(())), "lr must be"), (dict(grad_scale=torch.tensor(1.0, dtype=torch.float64)), "grad_scale must be")]:
        with pytest.raises(ValueError, match=msg):
            opt.step(good, **kw)
    assert int(opt.state.step) == 1
    s = opt.state
    for bad in (s._replace(step=None), s._replace(m=s.m[:-1]), s._replace(v=s.v.double()), s._replace(m_exp=s.m), s._replace(row_steps=None)):
        with pytest.raises(ValueError, match="state."):
            AdamW(opt.params, by_rows=[False, True], state=bad)
    dense = AdamW([f(3), f(4)])
    for grads, msg in [([f(3), f(5)], "shape"), ([f(3), f(8)[::2]], "contiguous"), ([f(3), torch.zeros(4)], "CUDA tensor"),
                       ([f(3), f(4, t=torch.float16)], "must have its type")]:
        with pytest.raises(ValueError, match=msg):
            dense.step(grads)
