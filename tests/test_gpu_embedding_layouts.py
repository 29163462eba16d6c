"""GPU tests of the embedding gradient over rows that begin anywhere: gradients and
tables inside wider matrices, each off 16 bytes by its own amount, every width up
to a few vectors, through each of the sorts (a few ids, one block, tiles). Against
float64 with each sum's own magnitude and number of terms: the helpers and the
bound are those of test_gpu_embedding.
"""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.embedding import embedding_grad, embedding_grad_rows  # noqa: E402
from modern_fm_b200.embedding import embedding_lookup  # noqa: E402

from test_gpu_embedding import TYPES, _close  # noqa: E402


def _inside(gen, n, d, lo, kind):
    """An (n, d) view of random values at column lo of a matrix of odd pitch."""
    big = torch.randn(n, d + lo + 3 - (d + lo) % 2, generator=gen, dtype=torch.float64)
    return big.to("cuda", TYPES[kind])[:, lo:lo + d]


def _check(n, n_rows, d, kind, lo_grad, lo_table, table_kind=None, dtype=None):
    gen = torch.Generator().manual_seed(n + d)
    grad = _inside(gen, n, d, lo_grad, kind)
    table = _inside(gen, n_rows, d, lo_table, table_kind or kind)
    ids = torch.randint(-1, n_rows + 1, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < 0.3] = n_rows // 2  # a run over many chunks
    ids = ids.cuda()
    wide = torch.float64 if kind == "f64" else torch.float32
    s = torch.randn(n, generator=gen, dtype=torch.float64).to("cuda", wide)
    live = (ids >= 0) & (ids < n_rows)
    at = ids.clamp(0, n_rows - 1)
    v = torch.where(live[:, None], grad.double() * 0.5, 0.0)
    ds = v * table.double()[at]
    v = v * s.double()[:, None]
    want = torch.zeros(n_rows, d, dtype=torch.float64, device="cuda").index_add_(0, at, v)
    size = torch.zeros_like(want).index_add_(0, at, v.abs())
    hits = torch.zeros(n_rows, dtype=torch.int64, device="cuda").index_add_(0, at, live.long())
    terms = float(hits.max())
    r = embedding_grad(grad, ids, n_rows, s, alpha=0.5, table=table, dtype=dtype)
    _close(r.table, want, size, terms, wide)
    assert bool((r.table[hits == 0] == 0).all())
    _close(r.scale, ds.sum(1), ds.abs().sum(1), d, wide)
    q = embedding_grad_rows(grad, ids, n_rows, s, alpha=0.5, table=table, dtype=dtype)
    keys = hits.nonzero()[:, 0]
    u = keys.numel()
    assert int(q.count) == u and torch.equal(q.keys[:u], keys)
    assert bool((q.keys[u:] == -1).all()) and bool((q.rows[u:] == 0).all())
    _close(q.rows[:u], want[keys], size[keys], terms, wide)
    assert torch.equal(q.scale, r.scale)


@pytest.mark.parametrize("n", [200, 700, 3000])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d,lo_grad,lo_table", [(24, 1, 1), (24, 0, 1), (24, 1, 0), (24, 4, 2),
                                                (24, 8, 8), (5, 3, 1), (1, 2, 3), (33, 0, 0),
                                                (130, 2, 4), (515, 1, 6)])
def test_rows_that_begin_anywhere(n, kind, d, lo_grad, lo_table):
    _check(n, 90, d, kind, lo_grad, lo_table)


@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("d", [1, 2, 3, 4, 6, 7, 8, 12, 15, 16, 17, 45, 64, 255])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_widths(n, d, kind):
    """Untouched rows between touched ones, of every residue of a vector."""
    _check(n, 4000, d, kind, 0, 0)


@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("d,lo_grad,lo_table", [(24, 0, 0), (24, 2, 1), (7, 1, 2)])
def test_float32_table_with_float64_gradients(n, d, lo_grad, lo_table):
    _check(n, 90, d, "f64", lo_grad, lo_table, table_kind="f32")


@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("d,lo", [(24, 0), (20, 4), (13, 1)])
def test_sums_kept_in_float32(n, kind, d, lo):
    _check(n, 90, d, kind, lo, lo, dtype=torch.float32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d,lo,lo_out", [(24, 1, 2), (24, 4, 4), (130, 3, 1), (515, 6, 0)])
def test_row_sums_between_layouts(kind, d, lo, lo_out):
    gen = torch.Generator().manual_seed(d)
    table = _inside(gen, 90, d, lo, kind)
    ids = torch.randint(-1, 91, (1000,), generator=gen)
    cuts = torch.randint(0, 1001, (40,), generator=gen).sort().values
    ip = torch.cat([torch.tensor([0]), cuts, torch.tensor([1000])]).cuda()
    ids = ids.cuda()
    whole = torch.full((41, d + lo_out + 3), 7.0, device="cuda").to(TYPES[kind])
    out = whole[:, lo_out:lo_out + d]
    assert embedding_lookup(table, ids, None, ip, alpha=1.5, out=out) is out
    live = (ids >= 0) & (ids < 90)
    v = torch.where(live[:, None], table.double()[ids.clamp(0, 89)] * 1.5, 0.0)
    row = torch.searchsorted(ip, torch.arange(1000, device="cuda"), right=True) - 1
    want = torch.zeros(41, d, dtype=torch.float64, device="cuda").index_add_(0, row, v)
    size = torch.zeros_like(want).index_add_(0, row, v.abs())
    _close(out, want, size, float(ip.diff().max()), torch.float64 if kind == "f64" else torch.float32)
    assert bool((whole[:, :lo_out] == 7).all()) and bool((whole[:, lo_out + d:] == 7).all())
