"""GPU test of a training step made of the embedding, alternatives and AdamW calls: a linear
policy over classes on sparse rows, with a bias, its log-probabilities weighted and its
entropy raised, against torch's autograd and the formulas in float64.

Everything runs in float64: each of a step's results is off by a few hundred roundings of
2^-53 at most, three steps of rate 1e-2 carry them on: bounds of 1e-11, relative to 1.
"""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.embedding import embedding_grad_rows, embedding_lookup  # noqa: E402
from modern_fm_b200.optim import AdamW  # noqa: E402
from modern_fm_b200.preference import label_alternatives, label_alternatives_grad  # noqa: E402

N, D, C, RATE, B1, B2, EPS, DECAY, PULL = 300, 2000, 37, 1e-2, 0.9, 0.999, 1e-8, 0.05, 0.02


def _batch(seed, kind):
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, 9, (N,), generator=g)
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    n = int(indptr[-1])
    ids = torch.randint(0, D // 4, (n,), generator=g).int()
    values = torch.randn(n, generator=g, dtype=torch.float64)
    labels = torch.randint(0, C, (N,), generator=g)
    labels[::17] = -1
    weight = torch.randn(N, generator=g, dtype=torch.float64)
    return [t.cuda() for t in (indptr, ids, values.to(kind), labels, weight.to(kind))]


def _parameters(kind):
    g = torch.Generator().manual_seed(0)
    return ((torch.randn(D, C, generator=g, dtype=torch.float64) * 0.3).to(kind).cuda(),
            torch.zeros(C, dtype=kind, device="cuda"))


def _step(opt, batch):
    table, bias = opt.params
    indptr, ids, values, labels, weight = batch
    scores = embedding_lookup(table, ids, values, indptr) + bias
    r = label_alternatives(scores, labels, top=3)
    pull = torch.full_like(weight, -PULL)
    d = label_alternatives_grad(scores, r.lse, r.entropy, labels, -weight, pull)
    rows = embedding_grad_rows(d, ids, D, values, indptr)
    norm = opt.step([rows, d.sum(0)], max_norm=5.0)
    return r, norm


def test_against_autograd():
    table, bias = _parameters(torch.float64)
    opt = AdamW([table, bias], lr=RATE, betas=(B1, B2), eps=EPS, weight_decay=DECAY, by_rows=[True, False])
    p = [table.clone(), bias.clone()]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    steps = torch.zeros(D, 1, device="cuda", dtype=torch.float64)
    for t in range(1, 4):
        batch = _batch(t, torch.float64)
        indptr, ids, values, labels, weight = batch
        before = table.clone()
        r, norm = _step(opt, batch)
        leaves = [x.clone().requires_grad_() for x in p]
        at = torch.repeat_interleave(torch.arange(N, device="cuda"), indptr.diff())
        scores = torch.zeros(N, C, device="cuda", dtype=torch.float64).index_add(
            0, at, leaves[0][ids.long()] * values[:, None]) + leaves[1]
        lp = torch.log_softmax(scores, 1)
        live = labels >= 0
        own = lp.gather(1, labels.clamp(min=0)[:, None])[:, 0]
        entropy = -(lp.exp() * lp).sum(1)
        loss = (torch.where(live, -weight * own - PULL * entropy, 0.0)).sum()
        loss.backward()
        whole = torch.sqrt(sum((x.grad**2).sum() for x in leaves))
        assert torch.allclose(norm, whole, rtol=1e-12)
        assert torch.allclose(r.entropy, torch.where(live, entropy, 0.0).detach(), rtol=0, atol=1e-12)
        best = lp.detach().topk(3).values
        assert torch.allclose(r.top_logprobs, torch.where(live[:, None], best, 0.0), rtol=0, atol=1e-12)
        factor = min(1.0, 5.0 / float(whole))
        touched = torch.zeros(D, 1, dtype=torch.bool, device="cuda")
        touched[ids.long()] = True
        steps += touched
        for i, (x, count, here) in enumerate(zip(leaves, (steps, t), (touched, True))):
            g = x.grad * factor
            m[i] = torch.where(torch.as_tensor(here, device="cuda"), B1 * m[i] + (1 - B1) * g, m[i])
            v[i] = torch.where(torch.as_tensor(here, device="cuda"), B2 * v[i] + (1 - B2) * g * g, v[i])
            c = torch.as_tensor(count, dtype=torch.float64, device="cuda").clamp(min=1)
            move = (m[i] / (1 - B1**c)) / (torch.sqrt(v[i] / (1 - B2**c)) + EPS)
            p[i] = torch.where(torch.as_tensor(here, device="cuda"), p[i] - RATE * (DECAY * p[i] + move), p[i])
        for got, want in zip(opt.params, p):
            assert float((got - want).abs().max()) <= 1e-11
        assert torch.equal(table[~touched[:, 0]], before[~touched[:, 0]])


@pytest.mark.parametrize("kind", [torch.float64, torch.float32])
def test_captured(kind):
    """The whole step as a graph, replayed on new batches of the same shape, gives the eager
    steps' bits."""
    eager, replayed = (AdamW(_parameters(kind), lr=RATE, weight_decay=DECAY, by_rows=[True, False]) for _ in range(2))
    first = _batch(1, kind)
    kept = [p.clone() for p in replayed.params]
    warm = AdamW([p.clone() for p in kept], lr=RATE, weight_decay=DECAY, by_rows=[True, False])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(warm, first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    inputs = [x.clone() for x in first]
    with torch.cuda.graph(graph):
        _, norm = _step(replayed, inputs)
    g = torch.Generator().manual_seed(5)
    for t in range(3):
        batch = [x.clone() for x in first]
        batch[2] = torch.randn(batch[2].shape, generator=g, dtype=torch.float64).to(kind).cuda()
        batch[3] = torch.randint(-1, C, (N,), generator=g).cuda()
        for x, y in zip(inputs, batch):
            x.copy_(y)
        _, want = _step(eager, batch)
        graph.replay()
        assert torch.equal(norm, want)
        assert all(torch.equal(a, b) for a, b in zip(eager.params, replayed.params))
        assert all(a is None or torch.equal(a, b) for a, b in zip(eager.state, replayed.state))
