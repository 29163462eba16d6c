"""GPU tests of the embedding lookup and its gradient (mfm_embedding_*_device)
against their definitions in float64.

Tolerances, with u = 2^-24 (float32 arithmetic) or 2^-53 (float64) and u_o half a
step of the result's type: a sum of m products alpha s x, each rounded twice, is
off by at most (m + 4) u times the sum of |alpha s x| in any order, and its one
rounding to the result adds u_o |result| (float16 results below its normal range:
half its smallest step, 2^-25). Keys, counts and padding are exact.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.embedding import (embedding_grad, embedding_grad_rows,  # noqa: E402
                                      embedding_lookup)

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16,
         "f16": torch.float16}


def _u(wide):
    return 2.0**-53 if wide == torch.float64 else 2.0**-24


def _close(got, want, size, terms, wide):
    """|got - want| within the bound above; size = the sum of the terms' magnitudes."""
    tol = (terms + 4) * _u(wide) * size + torch.finfo(got.dtype).eps / 2 * want.abs() + (
        2.0**-25 if got.dtype == torch.float16 else 1e-40 if wide == torch.float32 else 0.0)
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed"


def _make(seed, n_rows, d, n, kind, scale, indptr, id_type=torch.int64, pad=0.1, hot=0.0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(n_rows, d, generator=g).to(TYPES[kind])
    ids = torch.randint(0, n_rows, (n,), generator=g)
    if n:
        ids[torch.rand(n, generator=g) < hot] = n_rows // 2
        bad = torch.rand(n, generator=g) < pad
        ids[bad] = torch.where(torch.rand(n, generator=g) < 0.5, -3, n_rows)[bad]
    s = None
    if scale:
        s = (torch.randn(n, generator=g, dtype=torch.float64)).to(TYPES[scale])
    ip = None
    if indptr == "rows":  # ragged, with empty rows, all entries in some row
        cuts = torch.randint(0, n + 1, (max(n // 3, 2),), generator=g).sort().values
        ip = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([n])])
    elif indptr == "inside":  # entries before the first row and behind the last
        ip = torch.tensor([n // 4, n // 4, n // 2, max(n - 3, n // 2)])
    return tuple(t.cuda() if t is not None else None
                 for t in (table, ids.to(id_type), s, ip))


def _rows_of(ids, ip):
    n = ids.numel()
    t = torch.arange(n, device="cuda")
    if ip is None:
        return t, torch.ones(n, dtype=torch.bool, device="cuda")
    row = torch.searchsorted(ip, t, right=True) - 1
    ok = (row >= 0) & (row < ip.numel() - 1)
    return row.clamp(0, max(ip.numel() - 2, 0)), ok


def _definition(table, ids, s, ip, alpha):
    """(float64 lookup, sum of magnitudes, longest sum)."""
    n_rows, d = table.shape
    row, ok = _rows_of(ids, ip)
    n_out = ids.numel() if ip is None else ip.numel() - 1
    live = ok & (ids >= 0) & (ids < n_rows)
    v = table.double()[ids.long().clamp(0, n_rows - 1)] * alpha
    if s is not None:
        v = v * s.double()[:, None]
    v = torch.where(live[:, None], v, 0.0)
    out = torch.zeros(n_out, d, dtype=torch.float64, device="cuda").index_add_(0, row, v)
    size = torch.zeros_like(out).index_add_(0, row, v.abs())
    terms = torch.zeros(n_out, dtype=torch.float64, device="cuda").index_add_(
        0, row, live.double())
    return out, size, float(terms.max()) if n_out else 0.0


CASES = [  # n_rows, d, n, table, scale, indptr, ids, hot
    (7, 16, 1, "f32", None, None, torch.int64, 0.0),
    (7, 1, 5, "f64", "f64", None, torch.int32, 0.0),
    (1, 33, 50, "bf16", None, None, torch.int64, 0.0),
    (1000, 16, 400, "f32", "f32", "rows", torch.int32, 0.2),
    (1000, 16, 400, "f32", "f64", "rows", torch.int32, 0.2),
    (333, 7, 1500, "f16", "f32", "rows", torch.int64, 0.9),
    (50000, 20, 9001, "f32", "f32", "rows", torch.int32, 0.3),
    (70000, 8, 20001, "bf16", "f32", "inside", torch.int64, 0.1),
    (257, 250, 3001, "bf16", "f32", None, torch.int64, 0.1),
    (100, 1030, 517, "f64", "f64", "rows", torch.int64, 0.5),
    (5, 512, 64, "f16", None, "rows", torch.int32, 0.0),
    (1 << 17, 4, 500_000, "f32", "f32", "rows", torch.int32, 0.4),
    (40, 64, 33, "bf16", "f32", "inside", torch.int32, 0.0),
    # the sort's paths: one block and tiles (2048 ids), 8-bit digits in one, two and
    # many tiles' passes, 12-bit digits in two and three; runs over many chunks
    (200, 4, 2048, "f32", "f32", None, torch.int64, 0.5),
    (200, 4, 2049, "f32", "f32", None, torch.int64, 0.5),
    (255, 10, 5000, "f32", "f32", "rows", torch.int32, 0.8),
    (60000, 2, 450_000, "f32", None, None, torch.int64, 0.05),
    ((1 << 24) - 1, 1, 30_000, "f32", "f32", None, torch.int32, 0.1),
    (1 << 25, 1, 20_000, "f16", "f32", "rows", torch.int64, 0.1),
    (2000, 300, 9000, "f32", "f32", "rows", torch.int32, 0.9),
    (2000, 6, 40_000, "f64", "f64", None, torch.int64, 0.9),
    (3, 36, 12_000, "f16", "f32", "rows", torch.int32, 0.4),
    # a few ids: one launch
    (300, 20, 256, "f32", "f32", "rows", torch.int32, 0.6),
    (300, 20, 257, "f32", "f32", "rows", torch.int32, 0.6),
    (1 << 20, 5, 100, "bf16", "f32", "inside", torch.int64, 0.3),
    (9, 1500, 200, "f32", "f64", "rows", torch.int32, 0.9),
    (70_000, 64, 3, "f16", None, None, torch.int64, 0.0),
]


@pytest.mark.parametrize("n_rows,d,n,kind,scale,indptr,id_type,hot", CASES)
def test_lookup_matches_definition(n_rows, d, n, kind, scale, indptr, id_type, hot):
    table, ids, s, ip = _make(1, n_rows, d, n, kind, scale, indptr, id_type, hot=hot)
    wide = torch.float64 if "f64" in (kind, scale) else torch.float32
    got = embedding_lookup(table, ids, s, ip, alpha=1.5)
    want, size, terms = _definition(table, ids, s, ip, 1.5)
    assert got.dtype == (torch.float64 if wide == torch.float64 else TYPES[kind])
    _close(got, want, size, terms, wide)
    assert torch.equal(got, embedding_lookup(table, ids, s, ip, alpha=1.5))


@pytest.mark.parametrize("n_rows,d,n,kind,scale,indptr,id_type,hot", CASES)
@pytest.mark.parametrize("rows", [False, True])
def test_gradient_matches_definition(n_rows, d, n, kind, scale, indptr, id_type, hot, rows):
    table, ids, s, ip = _make(2, n_rows, d, n, kind, scale, indptr, id_type, hot=hot)
    wide = torch.float64 if "f64" in (kind, scale) else torch.float32
    kind_g = torch.float64 if wide == torch.float64 else TYPES[kind]
    row, ok = _rows_of(ids, ip)
    n_out = n if ip is None else ip.numel() - 1
    grad = torch.randn(n_out, d, generator=torch.Generator().manual_seed(5)).to("cuda", kind_g)
    live = ok & (ids >= 0) & (ids < n_rows)
    at = ids.long().clamp(0, n_rows - 1)
    v = grad.double()[row] * 0.5
    ds = torch.where(live[:, None], v * table.double()[at], 0.0)
    if s is not None:
        v = v * s.double()[:, None]
    v = torch.where(live[:, None], v, 0.0)
    want = torch.zeros(n_rows, d, dtype=torch.float64, device="cuda").index_add_(0, at, v)
    size = torch.zeros_like(want).index_add_(0, at, v.abs())
    hits = torch.zeros(n_rows, dtype=torch.int64, device="cuda").index_add_(0, at, live.long())
    kinds = [None, torch.float32] if kind in ("bf16", "f16") else [None]
    for dtype in kinds:
        if not rows:
            got = embedding_grad(grad, ids, n_rows, s, ip, alpha=0.5, table=table, dtype=dtype)
            assert got.table.dtype == (dtype or kind_g)
            _close(got.table, want, size, float(hits.max()), wide)
            assert torch.equal(got.table, embedding_grad(grad, ids, n_rows, s, ip, alpha=0.5,
                                                         dtype=dtype).table)
        else:
            got = embedding_grad_rows(grad, ids, n_rows, s, ip, alpha=0.5, table=table,
                                      dtype=dtype)
            keys = hits.nonzero()[:, 0]
            u, cap = keys.numel(), min(n, n_rows)
            assert int(got.count) == u and got.keys.dtype == id_type
            assert got.keys.shape == (cap,) and got.rows.shape == (cap, d)
            assert torch.equal(got.keys[:u].long(), keys)
            assert bool((got.keys[u:] == -1).all()) and bool((got.rows[u:] == 0).all())
            _close(got.rows[:u], want[keys], size[keys], float(hits.max()), wide)
        assert got.scale.shape == ids.shape and got.scale.dtype == wide
        _close(got.scale, ds.sum(1), ds.abs().sum(1), d, wide)
        assert bool((got.scale[~live] == 0).all())


@pytest.mark.parametrize("n", [0, 1])
@pytest.mark.parametrize("n_out", [0, 1, 3])
def test_nothing_to_look_up(n, n_out):
    """No entries, no rows, only padding, an empty table."""
    table = torch.randn(4, 6, device="cuda")
    ids = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    ip = torch.zeros(n_out + 1, dtype=torch.int64, device="cuda")
    ip[-1:] = n if n_out else 0
    out = embedding_lookup(table, ids, None, ip)
    assert out.shape == (n_out, 6) and bool((out == 0).all())
    grad = torch.randn(n_out, 6, device="cuda")
    for rows in (4, 0):
        t = table[:rows]
        r = embedding_grad(grad, ids, rows, None, ip, table=t)
        assert r.table.shape == (rows, 6) and bool((r.table == 0).all())
        assert r.scale.shape == (n,) and bool((r.scale == 0).all())
        r = embedding_grad_rows(grad, ids, rows, None, ip)
        assert int(r.count) == 0 and r.keys.shape == (min(n, rows),) and r.rows.shape[1] == 6
        assert bool((r.keys == -1).all()) and bool((r.rows == 0).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f64"])
def test_pitches_and_alignment(kind):
    """Rows inside a wider matrix, and bases off a 16-byte boundary."""
    big = torch.randn(90, 40, generator=torch.Generator().manual_seed(1)).to("cuda", TYPES[kind])
    ids = torch.randint(-1, 90, (200,), device="cuda")
    for lo, d in ((0, 24), (1, 24), (8, 32), (3, 5)):
        t = big[:, lo:lo + d]
        want = embedding_lookup(t.contiguous(), ids, alpha=2.0)
        assert torch.equal(embedding_lookup(t, ids, alpha=2.0), want)
        out = torch.full((200, 50), 7.0, device="cuda", dtype=TYPES[kind])
        view = out[:, 2:2 + d]
        assert embedding_lookup(t, ids, alpha=2.0, out=view) is view
        assert torch.equal(view, want)
        assert bool((out[:, :2] == 7).all()) and bool((out[:, 2 + d:] == 7).all())
        g = torch.randn(200, 50, device="cuda").to(TYPES[kind])[:, 1:1 + d]
        a = embedding_grad(g, ids, 90, table=t)
        b = embedding_grad(g.contiguous(), ids, 90, table=t.contiguous())
        wide = torch.float64 if kind == "f64" else torch.float32
        tol = 300 * _u(wide) * float(g.abs().double().max()) * float(t.abs().double().max()) * 200
        assert (a.table.double() - b.table.double()).abs().max() <= tol + torch.finfo(
            TYPES[kind]).eps * b.table.double().abs().max()
        assert (a.scale.double() - b.scale.double()).abs().max() <= tol


def test_ids_of_any_shape():
    table = torch.randn(11, 8, device="cuda")
    ids = torch.randint(0, 11, (3, 4, 5), device="cuda", dtype=torch.int32)
    s = torch.rand(3, 4, 5, device="cuda")
    out = embedding_lookup(table, ids, s)
    assert out.shape == (3, 4, 5, 8)
    # one product of float32 values, rounded as torch rounds it
    assert torch.equal(out, table[ids.long()] * s[..., None])
    r = embedding_grad(out, ids, 11, s, table=table)
    assert r.scale.shape == (3, 4, 5) and r.table.shape == (11, 8)


def test_values_that_are_not_finite_stay_where_they_are():
    table = torch.randn(6, 16, device="cuda")
    table[2] = float("nan")
    table[3, 5] = float("inf")
    ids = torch.tensor([0, 2, 6, 3, -1, 1], device="cuda")
    out = embedding_lookup(table, ids, alpha=0.5)
    assert torch.isnan(out[1]).all() and torch.isinf(out[3, 5])
    assert torch.isfinite(out[[0, 2, 4, 5]]).all()
    grad = torch.ones(6, 16, device="cuda")
    grad[2] = float("nan")  # of a padding id: reaches no row
    grad[0, 3] = float("inf")
    g = embedding_grad(grad, ids, 6).table
    assert torch.isinf(g[0, 3]) and int((~torch.isfinite(g)).sum()) == 1
    assert bool((g[[4, 5]] == 0).all())


def test_bad_row_bounds_stay_inside():
    """Bounds that decrease or leave the entries read nothing outside."""
    table = torch.randn(9, 4, device="cuda")
    ids = torch.randint(0, 9, (20,), device="cuda")
    ip = torch.tensor([-5, 3, 1, 40, 18, 25], device="cuda")
    out = embedding_lookup(table, ids, None, ip)
    want = torch.stack([table[ids[0:3]].sum(0), torch.zeros(4, device="cuda"),
                        table[ids[1:20]].sum(0), torch.zeros(4, device="cuda"),
                        table[ids[18:20]].sum(0)])
    assert (out - want).abs().max() < 30 * 2.0**-24 * 20 * float(table.abs().max())
    embedding_grad(torch.randn(5, 4, device="cuda"), ids, 9, None, ip, table=table)
    torch.cuda.synchronize()


def test_other_stream_and_graph_replay():
    """A call on a stream of its own, and two calls captured and replayed with new inputs,
    equal the eager results bit for bit."""
    table, ids, s, ip = _make(3, 5000, 32, 30000, "f32", "f32", "rows", torch.int32, hot=0.2)
    grad = torch.randn(ip.numel() - 1, 32, device="cuda")
    eager = (embedding_lookup(table, ids, s, ip), *embedding_grad(grad, ids, 5000, s, ip, table=table),
             *embedding_grad_rows(grad, ids, 5000, s, ip)[:3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = embedding_lookup(table, ids, s, ip, stream=side)
    b = embedding_grad(grad, ids, 5000, s, ip, table=table, stream=side)
    c = embedding_grad_rows(grad, ids, 5000, s, ip, stream=side)
    side.synchronize()
    for x, y in zip((a, *b, *c[:3]), eager):
        assert torch.equal(x, y)
    graphs, outs = [], []
    st = [t.clone() for t in (ids, s, grad)]
    for _ in range(2):  # two graphs that are replayed at the same time
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((embedding_lookup(table, st[0], st[1], ip),
                         *embedding_grad(st[2], st[0], 5000, st[1], ip, table=table),
                         *embedding_grad_rows(st[2], st[0], 5000, st[1], ip)[:3]))
        graphs.append(g)
    for seed in (1, 2):
        perm = torch.randperm(ids.numel(), device="cuda")
        st[0].copy_(ids[perm])
        st[1].copy_(s * seed)
        st[2].copy_(grad * 0.5)
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = (embedding_lookup(table, st[0], st[1], ip),
                *embedding_grad(st[2], st[0], 5000, st[1], ip, table=table),
                *embedding_grad_rows(st[2], st[0], 5000, st[1], ip)[:3])
        for o in outs:
            for x, y in zip(o, want):
                assert torch.equal(x, y)


def test_gradient_by_differences():
    """The gradients are those of L = <weights, lookup> in float64: L is linear in the
    table and in the scales, so a difference over 2 h is exact up to rounding."""
    table, ids, s, ip = _make(4, 12, 5, 60, "f64", "f64", "rows")
    w = torch.randn(ip.numel() - 1, 5, device="cuda", dtype=torch.float64)
    g = embedding_grad(w, ids, 12, s, ip, alpha=0.7, table=table)

    def loss(t, sc):
        return float((embedding_lookup(t, ids, sc, ip, alpha=0.7) * w).sum())

    rng = np.random.default_rng(0)
    for _ in range(10):
        i, j, e = rng.integers(12), rng.integers(5), rng.integers(60)
        d = torch.zeros_like(table)
        d[i, j] = 0.5
        assert loss(table + d, s) - loss(table - d, s) == pytest.approx(float(g.table[i, j]),
                                                                        abs=1e-11)
        d = torch.zeros_like(s)
        d[e] = 0.5
        assert loss(table, s + d) - loss(table, s - d) == pytest.approx(float(g.scale[e]),
                                                                        abs=1e-11)


def test_offsets_beyond_32_bits():
    """A table and a gradient of more than 2^32 values: the last rows and the first."""
    n_rows, d = 66_000, 65_600
    table = torch.zeros(n_rows, d, device="cuda", dtype=torch.bfloat16)
    assert table.numel() > 2**32
    ids = torch.tensor([n_rows - 1, 0, n_rows - 2, n_rows, n_rows - 1], device="cuda")
    for i in (0, n_rows - 2, n_rows - 1):
        table[i] = torch.randn(d, device="cuda").bfloat16()
    out = embedding_lookup(table, ids)
    assert torch.equal(out[[0, 1, 2, 4]], table[ids[[0, 1, 2, 4]]]) and bool((out[3] == 0).all())
    two = embedding_lookup(table, ids, None, torch.tensor([0, 3, 5], device="cuda"))
    # one rounding of a float32 sum of three bfloat16 values
    want = table[ids[:3]].double().sum(0)
    assert ((two[0].double() - want).abs() <= want.abs() * 2.0**-8 + 2.0**-20).all()
    del out, two
    grad = torch.randn(5, d, device="cuda").bfloat16()
    g = embedding_grad(grad, ids, n_rows, table=table)
    assert torch.equal(g.table[0], grad[1]) and torch.equal(g.table[n_rows - 2], grad[2])
    want = grad[0].double() + grad[4].double()
    assert ((g.table[n_rows - 1].double() - want).abs() <= want.abs() * 2.0**-8).all()
    assert int(g.table[1:n_rows - 2].count_nonzero()) == 0
    assert float(g.scale[3]) == 0.0
    r = embedding_grad_rows(grad, ids, n_rows)
    assert r.keys.tolist() == [0, n_rows - 2, n_rows - 1, -1, -1] and int(r.count) == 3
    assert torch.equal(r.rows[2], g.table[n_rows - 1])
    # and many ids, through the tiled sort and the touched rows' bits
    many = torch.randint(n_rows - 40, n_rows, (3000,), device="cuda")
    g = embedding_grad(torch.ones(3000, d, device="cuda", dtype=torch.bfloat16), many, n_rows)
    want = torch.bincount(many, minlength=n_rows).bfloat16()
    assert torch.equal(g.table[:, -1], want) and torch.equal(g.table[:, 0], want)
    assert int(g.table[:n_rows - 40].count_nonzero()) == 0


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    table, ids, s, ip = _make(6, 3000, 24, 40_000, "f32", "f32", "rows", torch.int32, hot=0.3)
    grad = torch.randn(ip.numel() - 1, 24, device="cuda")
    want = embedding_grad(grad, ids, 3000, s, ip, table=table)
    rows = embedding_grad_rows(grad, ids, 3000, s, ip)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((embedding_grad(grad, ids, 3000, s, ip, table=table, stream=a),
                    embedding_grad_rows(grad, ids, 3000, s, ip, stream=b)))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x.table, want.table) and torch.equal(x.scale, want.scale)
        assert torch.equal(y.rows, rows.rows) and torch.equal(y.keys, rows.keys)


def test_gradient_of_a_view_is_read_by_its_stream():
    """A gradient that needs a copy is copied by the stream that the call runs on, behind the
    work that writes it there; one id without an axis takes its result's shape."""
    ids = torch.randint(0, 50, (64, 32), device="cuda")
    base = torch.randn(32, 64, 24, device="cuda")
    want = embedding_grad(base.transpose(0, 1).contiguous(), ids, 50).table
    late = torch.zeros_like(base)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(base)
    got = embedding_grad(late.transpose(0, 1), ids, 50, stream=side).table
    side.synchronize()
    assert torch.equal(got, want)
    table, one = torch.randn(9, 5, device="cuda"), torch.tensor(4, device="cuda")
    row = embedding_lookup(table, one)
    assert torch.equal(row, table[4])
    g = embedding_grad(row, one, 9).table
    assert torch.equal(g[4], row) and int(g.count_nonzero()) == 5
