"""The embedding and preference operators, as a user's program calls them, with their plain forms.

Four operators over the framework's two kinds of device data, sparse rows (ids, values, row
bounds) against a table of latent rows, and one row of class scores per example:

  lookup   embedding_lookup: out[t] = alpha scale[t] table[ids[t]], or summed over the entries of a row
  grad     embedding_grad / embedding_grad_rows: its gradient by sorted ids, the whole table or the
           touched rows only, and the gradient of the scales
  logprobs label_logprobs / label_logprobs_grad: log-softmax of each row's label, and its gradient
  losses   preference_loss (pairs of sequences, log ratios against a reference) and policy_loss
           (clipped ratios with a KL term), each with the gradient of the class scores

Ids outside the table and labels outside the classes are padding.
"""

import math

import numpy as np
import torch

own = False  # set by whoever times this file: the plain forms, or the framework's operators

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one step of serving: the rows of a few tokens, scaled by sqrt(width); only latency counts
        dict(name="lookup_serving", op="lookup", form="tokens", n=32000, d=1024, count=17, table="bf16",
             scale="none", alpha=32.0, pad=0.0, zipf=1.0),
        # a batch of sparse click rows against 2^22 latent rows of 16 float32, summed in float64
        # (the framework's default arithmetic): 13 numeric features of every row, 26 hashed ones
        dict(name="lookup_click_rows", op="lookup", form="rows", n=1 << 22, d=16, count=131072, table="f32",
             scale="f64", alpha=1.0, numeric=13, hashed=26, zipf=1.1),
        # a training batch of tokens, padded, against a wide table in bfloat16
        dict(name="lookup_tokens", op="lookup", form="tokens", n=131072, d=4096, count=32771, table="bf16",
             scale="none", alpha=64.0, pad=0.1, zipf=1.0),
        # a small batch of rows in training: the whole gradient of a small table
        dict(name="grad_small_rows", op="grad", form="rows", n=1003, d=60, count=5, table="f32", scale="f32",
             alpha=1.0, numeric=3, hashed=12, zipf=1.1, result="table", want_scale=True),
        # the same training batch of tokens: the whole table's gradient kept in float32
        dict(name="grad_tokens", op="grad", form="tokens", n=32000, d=2048, count=16384, table="bf16",
             scale="none", alpha=1.0, pad=0.1, zipf=1.0, result="table", out="f32"),
        # one mini-batch of click rows: the touched rows' gradient and the values' (13 ids occur in every row)
        dict(name="grad_click_rows", op="grad", form="rows", n=1 << 22, d=16, count=8192, table="f32", scale="f32",
             alpha=1.0, numeric=13, hashed=26, zipf=1.1, result="rows", want_scale=True),
        # log-probabilities of a batch of tokens under a frozen model, as the losses' references need them
        dict(name="logprobs_tokens", op="logprobs", tokens=8195, classes=32000, type="bf16", pad=0.2, grad=False),
        # the softmax model's ten classes over many rows, forward and gradient
        dict(name="logprobs_classes", op="logprobs", tokens=333333, classes=10, type="f32", pad=0.01, grad=True),
        # short sessions of the softmax model in float64: only latency counts
        dict(name="preference_sessions", op="preference", pairs=16, shortest=0, longest=40, classes=10, type="f64",
             pad=0.1, beta=0.5, smoothing=0.1, weighted=True),
        # pairs of answers over a vocabulary, their prompts masked, and the class scores' gradient
        dict(name="preference_answers", op="preference", pairs=16, shortest=200, longest=800, classes=32000,
             type="bf16", pad=0.3, beta=0.1, smoothing=0.0, weighted=False),
        # logged actions of the softmax model: ten classes, a million rows
        dict(name="policy_classes", op="policy", tokens=1000003, classes=10, type="f32", pad=0.01, kl=0.05,
             weighted=True),
        # sampled tokens over a vocabulary with the KL term against a reference
        dict(name="policy_tokens", op="policy", tokens=4096, classes=65536, type="bf16", pad=0.2, kl=0.05,
             weighted=False),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Widths from 1 to 8192, classes from 2 to 131072, counts from 1 to millions, cut so that a case
    moves no more than about 1.2 GB."""
    op = rng.choice(["lookup", "lookup", "grad", "grad", "logprobs", "preference", "policy"])
    if op in ("lookup", "grad"):
        form = rng.choice(["tokens", "rows"])
        d = _spread(rng, 1, 8192) if form == "tokens" else _spread(rng, 1, 256)
        n = min(_spread(rng, 2, 1 << 22), max(2, (1 << 27) // d))
        table = rng.choice(["f32", "f32", "bf16", "f16", "f64"])
        case = dict(op=op, form=form, n=n, d=d, table=table, zipf=rng.choice([0.0, 1.0, 1.1]),
                    alpha=rng.choice([1.0, round(math.sqrt(d), 3)]))
        if form == "tokens":
            case.update(count=min(_spread(rng, 1, 1 << 20), max(1, (1 << 26) // d)), pad=rng.choice([0.0, 0.1]),
                        scale=rng.choice(["none", "f64" if table == "f64" else "f32"]))
        else:
            case.update(numeric=min(n - 1, rng.randint(0, 13)), hashed=rng.randint(1, 40))
            most = max(1, (1 << 26) // (d * (case["numeric"] + case["hashed"])))
            case.update(count=min(_spread(rng, 1, 1 << 17), most),
                        scale="f64" if table == "f64" else rng.choice(["f32", "f64"] if table == "f32" else ["f32"]))
        if op == "grad":
            case.update(result=rng.choice(["table", "rows"]), want_scale=case["scale"] != "none" and rng.random() < 0.5)
            if table in ("bf16", "f16") and rng.random() < 0.5:
                case["out"] = "f32"
        return case
    kind = rng.choice(["bf16", "f16", "f32", "f64"])
    classes = _spread(rng, 2, 1 << 17)
    tokens = min(_spread(rng, 1, 1 << 20), max(1, (1 << 27) // classes))
    case = dict(op=op, classes=classes, type=kind, pad=rng.choice([0.0, 0.1, 0.5]))
    if op == "preference":
        longest = max(1, min(_spread(rng, 1, 2048), tokens))
        case.update(pairs=max(1, tokens // (longest + 1)), shortest=rng.randint(0, longest), longest=longest,
                    beta=rng.choice([0.05, 0.1, 0.5]), smoothing=rng.choice([0.0, 0.1]), weighted=rng.random() < 0.5)
    else:
        case.update(tokens=tokens)
        if op == "logprobs":
            case.update(grad=rng.random() < 0.5)
        else:
            case.update(kl=rng.choice([0.0, 0.05]), weighted=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------- inputs --


def _ids(g, shape, n, zipf, first=0):
    """Ids in [first, n): popular ones by a power law of their rank, scattered over the table."""
    span = n - first
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    if zipf == 0.0:
        rank = (u * span).long()
    elif zipf == 1.0:
        rank = torch.exp(u * math.log(span + 1)).long() - 1
    else:
        a = 1.0 - zipf
        rank = ((((span + 1) ** a - 1.0) * u + 1.0) ** (1.0 / a)).long() - 1
    return first + (rank.clamp_(0, span - 1) * 2654435761) % span


def _distinct(count, n, zipf):
    """How many of n ids `count` draws of _ids are expected to meet."""
    if zipf == 0.0:
        return n * -math.expm1(count * math.log1p(-1.0 / n)) if n > 1 else 1.0
    edge = np.arange(1, n + 2, dtype=np.float64)
    c = np.log(edge) / math.log(n + 1) if zipf == 1.0 else (edge ** (1 - zipf) - 1) / ((n + 1.0) ** (1 - zipf) - 1)
    return float(-np.expm1(count * np.log1p(-np.minimum(np.diff(c), 1 - 1e-12))).sum())


def _shape_generator(case):
    g = torch.Generator(device="cuda")
    g.manual_seed(case.get("count", 0) + case.get("pairs", 0))
    return g


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return (_prepare_embedding if case["op"] in ("lookup", "grad") else _prepare_scores)(case, g)


def _prepare_embedding(case, g):
    n, d, count, kind = case["n"], case["d"], case["count"], DTYPES[case["table"]]
    st = dict(case=case, indptr=None, scale=None, table=None)
    if case["form"] == "tokens":
        ids = _ids(g, (count,), n, case["zipf"])
        ids[torch.rand(count, generator=g, device="cuda") < case["pad"]] = -1
        st["ids"] = ids
        if case["scale"] != "none":
            st["scale"] = torch.rand(count, generator=g, device="cuda", dtype=DTYPES[case["scale"]]) + 0.5
        lead = count
    else:  # rows of numeric features (ids 0 .. numeric - 1) and hashed ones, some missing, some rows empty
        k = case["numeric"]
        ids = torch.cat([torch.arange(k, device="cuda").expand(count, k),
                         _ids(g, (count, case["hashed"]), n, case["zipf"], k)], 1)
        value = torch.ones(ids.shape, device="cuda", dtype=torch.float64)
        value[:, :k] = torch.log1p(torch.exp(2.0 * torch.randn(count, k, generator=g, device="cuda")))
        shape = _shape_generator(case)  # which values are missing goes by the case: outputs keep their shapes
        keep = torch.rand(ids.shape, generator=shape, device="cuda") < 0.9
        keep[:, :k] = True
        keep &= torch.rand(count, 1, generator=shape, device="cuda") >= 0.01
        ids, order = ids.sort(1)
        value, keep = value.gather(1, order), keep.gather(1, order)
        st["ids"] = ids[keep].int()
        st["scale"] = value[keep].to(DTYPES[case["scale"]])
        st["indptr"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), keep.sum(1).cumsum(0)])
        lead = count
    if case["op"] == "lookup" or case.get("want_scale"):
        st["table"] = _normal(g, (n, d), kind, 0.3)
    if case["op"] == "grad":
        wide = torch.float64 if case["scale"] == "f64" else kind
        st["grad"] = _normal(g, (lead, d), wide, 0.1)
    return st


def _logprob64(x, labels):
    """(log-probability of the label, validity), row blocks in float64."""
    valid = (labels >= 0) & (labels < x.shape[1])
    at = labels.clamp(0, x.shape[1] - 1).long()
    out = torch.empty(x.shape[0], device=x.device, dtype=torch.float64)
    step = max(1, (1 << 26) // x.shape[1])
    for lo in range(0, x.shape[0], step):
        b = x[lo:lo + step].double()
        out[lo:lo + step] = torch.log_softmax(b, 1).gather(1, at[lo:lo + step, None])[:, 0]
    return torch.where(valid, out, 0.0), valid


def _prepare_scores(case, g):
    c, kind = case["classes"], DTYPES[case["type"]]
    side = torch.float64 if kind == torch.float64 else torch.float32
    st = dict(case=case)
    if case["op"] == "preference":
        lengths = torch.randint(case["shortest"], case["longest"] + 1, (2 * case["pairs"],),
                                generator=_shape_generator(case), device="cuda")
        st["indptr"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), lengths.cumsum(0)])
        t = int(st["indptr"][-1])
    else:
        t = case["tokens"]
    x = _normal(g, (t, c), kind, 2.0)
    labels = torch.randint(0, c, (t,), generator=g, device="cuda")
    labels[torch.rand(t, generator=g, device="cuda") < case["pad"]] = -1
    st.update(logits=x, labels=labels.int() if c < 1000 else labels)
    if case["op"] == "logprobs":
        if case["grad"]:
            st["grad"] = _normal(g, (t,), side)
        return st
    logp, valid = _logprob64(x, labels)  # a reference near the model, as training keeps it
    if case["op"] == "preference":
        seq = torch.zeros(2 * case["pairs"], device="cuda", dtype=torch.float64)
        seq.index_add_(0, torch.repeat_interleave(lengths), logp)
        st["reference"] = (seq + 3.0 * torch.randn(seq.shape, generator=g, device="cuda")).to(side)
        if case["weighted"]:
            st["weight"] = torch.rand(case["pairs"], generator=g, device="cuda", dtype=side) + 0.5
        return st
    # old log-probabilities a step away: ratios on both sides of the clip's bounds, none within 1e-3 of one
    step = 0.25 * torch.randn(t, generator=g, device="cuda", dtype=torch.float64)
    for edge in (math.log(0.8), math.log(1.2)):
        step = torch.where((step - edge).abs() < 1e-3, edge + 2e-3, step)
    st["old"] = (logp - step).to(side)
    st["reference"] = (logp + 0.2 * torch.randn(t, generator=g, device="cuda", dtype=torch.float64)).to(side)
    st["advantage"] = torch.randn(t, generator=g, device="cuda", dtype=side) + 0.2
    if case["weighted"]:
        st["weight"] = torch.rand(t, generator=g, device="cuda", dtype=side) + 0.5
    return st


# ------------------------------------------------------------------ runs --


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def _own(st):
    from modern_fm_b200 import embedding, preference

    case, op = st["case"], st["case"]["op"]
    if op == "lookup":
        return embedding.embedding_lookup(st["table"], st["ids"], st["scale"], st["indptr"], alpha=case["alpha"])
    if op == "grad":
        f = embedding.embedding_grad if case["result"] == "table" else embedding.embedding_grad_rows
        r = f(st["grad"], st["ids"], case["n"], st["scale"], st["indptr"], alpha=case["alpha"],
              table=st["table"] if case.get("want_scale") else None,
              dtype=DTYPES[case["out"]] if "out" in case else None)
        return {k: v for k, v in r._asdict().items() if v is not None}
    if op == "logprobs":
        r = preference.label_logprobs(st["logits"], st["labels"])
        out = {"logprobs": r.logprobs, "lse": r.lse}
        if case["grad"]:
            out["grad"] = preference.label_logprobs_grad(st["grad"], st["logits"], st["labels"], r.lse)
        return out
    if op == "preference":
        r = preference.preference_loss(st["logits"], st["labels"], st["indptr"], st["reference"], beta=case["beta"],
                                       label_smoothing=case["smoothing"], sample_weight=st.get("weight"))
    else:
        r = preference.policy_loss(st["logits"], st["labels"], st["old"], st["advantage"], st["reference"],
                                   clip_low=0.2, clip_high=0.2, kl_coef=case["kl"], sample_weight=st.get("weight"))
    return r._asdict()


def _entry_rows(st):
    """For each entry, the row of the sums (or gradients) that it belongs to."""
    count = st["ids"].numel()
    if st["indptr"] is None:
        return torch.arange(count, device="cuda")
    return torch.searchsorted(st["indptr"], torch.arange(count, device="cuda"), right=True) - 1


def _plain_lookup(st):
    case, table = st["case"], st["table"]
    wide = torch.float64 if torch.float64 in (table.dtype, DTYPES.get(case["scale"])) else torch.float32
    ids = st["ids"].long()
    valid = (ids >= 0) & (ids < case["n"])
    got = table[ids.clamp(0, case["n"] - 1)].to(wide) * case["alpha"]
    if st["scale"] is not None:
        got = got * st["scale"].to(wide)[:, None]
    got = torch.where(valid[:, None], got, 0.0)
    if st["indptr"] is not None:
        out = torch.zeros(case["count"], case["d"], device="cuda", dtype=wide)
        got = out.index_add_(0, _entry_rows(st), got)
    return got.to(torch.float64 if wide == torch.float64 else table.dtype)


def _plain_grad(st):
    case, grad, n, count = st["case"], st["grad"], st["case"]["n"], st["ids"].numel()
    wide = torch.float64 if grad.dtype == torch.float64 else torch.float32
    ids = st["ids"].long()
    valid = (ids >= 0) & (ids < n)
    at = ids.clamp(0, n - 1)
    rows = grad[_entry_rows(st)].to(wide) * case["alpha"]
    out = {}
    if case.get("want_scale"):
        out["scale"] = torch.where(valid, (rows * st["table"][at].to(wide)).sum(1), 0.0)
    if st["scale"] is not None:
        rows = rows * st["scale"].to(wide)[:, None]
    rows = torch.where(valid[:, None], rows, 0.0)
    kind = DTYPES[case["out"]] if "out" in case else grad.dtype
    if case["result"] == "table":
        whole = torch.zeros(n, case["d"], device="cuda", dtype=wide).index_add_(0, at, rows)
        return {"table": whole.to(kind), **out}
    # the touched ids in ascending order, -1 behind them, and their rows, 0 behind them
    cap = min(count, n)
    key, order = torch.where(valid, ids, n).sort(stable=True)
    first = torch.ones(count, device="cuda", dtype=torch.bool)
    first[1:] = key[1:] != key[:-1]
    slot = torch.where(key < n, first.cumsum(0) - 1, cap)
    keys = torch.full((cap + 1,), -1, device="cuda", dtype=st["ids"].dtype)
    keys[slot] = key.to(keys.dtype)
    total = torch.zeros(cap + 1, case["d"], device="cuda", dtype=wide).index_add_(0, slot, rows[order])
    return {"keys": keys[:cap], "rows": total[:cap].to(kind), "count": (first & (key < n)).sum(), **out}


def _plain_logprob(x, labels):
    """(log-probability of the label or 0, log-sum-exp, probabilities, validity) in the wide type."""
    w = x.double() if x.dtype == torch.float64 else x.float()
    top = w.max(1).values[:, None]
    e = (w - top).exp()
    total = e.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    valid = (labels >= 0) & (labels < x.shape[1])
    at = labels.clamp(0, x.shape[1] - 1).long()
    logp = torch.where(valid, (w.gather(1, at[:, None]) - top)[:, 0] - total[:, 0].log(), 0.0)
    return logp, lse, e.div_(total), valid


def _plain_score_grad(p, g, labels, valid, kind):
    """g (1[c = label] - p), rounded once; p is used up."""
    g = torch.where(valid, g, 0.0).to(p.dtype)
    p.mul_(-g[:, None])
    p.scatter_add_(1, labels.clamp(0, p.shape[1] - 1).long()[:, None], g[:, None])
    return p.to(kind)


def _plain_logprobs(st):
    logp, lse, p, valid = _plain_logprob(st["logits"], st["labels"])
    out = {"logprobs": logp, "lse": lse}
    if st["case"]["grad"]:
        out["grad"] = _plain_score_grad(p, st["grad"], st["labels"], valid, st["logits"].dtype)
    return out


def _plain_preference(st):
    case, x = st["case"], st["logits"]
    n, side = case["pairs"], st["reference"].dtype
    logp, _, p, valid = _plain_logprob(x, st["labels"])
    seq = torch.searchsorted(st["indptr"], torch.arange(x.shape[0], device="cuda"), right=True) - 1
    total = torch.zeros(2 * n, device="cuda", dtype=torch.float64).index_add_(0, seq, logp.double())
    ratio = total - st["reference"].double()
    z = case["beta"] * (ratio[:n] - ratio[n:])
    w = st["weight"].double() if "weight" in st else torch.ones(n, device="cuda", dtype=torch.float64)
    w = w / w.sum()
    eps = case["smoothing"]
    softplus = torch.log1p(torch.exp(-z.abs()))  # -log sigmoid(z) = max(-z, 0) + log(1 + exp(-|z|))
    loss = (w * (softplus + (1 - eps) * (-z).clamp(min=0) + eps * z.clamp(min=0))).sum()
    up = 1 / (1 + torch.exp(-z))
    slope = -case["beta"] * w * ((1 - eps) * (1 - up) - eps * up)
    g = torch.cat([slope, -slope])[seq]
    return {"loss": loss.to(side), "margins": z.to(side), "logprobs": total.to(side),
            "grad": _plain_score_grad(p, g, st["labels"], valid, x.dtype)}


def _plain_policy(st):
    case, x = st["case"], st["logits"]
    side = st["old"].dtype
    logp, _, p, valid = _plain_logprob(x, st["labels"])
    w = st["weight"].double() if "weight" in st else torch.ones(x.shape[0], device="cuda", dtype=torch.float64)
    w = torch.where(valid, w, 0.0)
    w = w / w.sum().clamp(min=1e-300)
    adv, at = st["advantage"].double(), logp.double()
    ratio = (at - st["old"].double()).exp()
    bent = ratio.clamp(0.8, 1.2) * adv
    clipped = ratio * adv > bent
    away = st["reference"].double() - at
    k = away.exp() - away - 1
    zero = torch.zeros_like(w)
    surrogate = torch.where(valid, -torch.minimum(ratio * adv, bent), zero)
    k = torch.where(valid, k, zero)
    g = w * (torch.where(clipped, zero, -ratio * adv) + case["kl"] * (1 - away.exp()))
    return {"loss": (w * (surrogate + case["kl"] * k)).sum().to(side), "kl": (w * k).sum().to(side),
            "clip_fraction": (w * clipped).sum().to(side), "logprobs": logp,
            "grad": _plain_score_grad(p, g, st["labels"], valid, x.dtype)}


_PLAIN = dict(lookup=_plain_lookup, grad=_plain_grad, logprobs=_plain_logprobs, preference=_plain_preference,
              policy=_plain_policy)


# ----------------------------------------------------------------- exact --


def exact(case, seed):
    """The definitions in 64 bits: sums as products with sparse matrices, softmax by torch's own in row blocks."""
    st = prepare(case, seed)
    return (_exact_embedding if case["op"] in ("lookup", "grad") else _exact_scores)(case, st)


def _sparse(rows, cols, values, shape):
    """A float64 CSR matrix of the entries, no two of them in one place."""
    order = torch.argsort(rows, stable=True)
    bounds = torch.searchsorted(rows[order].contiguous(), torch.arange(shape[0] + 1, device="cuda"))
    return torch.sparse_csr_tensor(bounds, cols[order], values[order], shape)


def _exact_embedding(case, st):
    n, d, ids = case["n"], case["d"], st["ids"].long()
    keep = ((ids >= 0) & (ids < n)).nonzero()[:, 0]
    count = ids.numel()
    if st["indptr"] is None:
        entry = torch.arange(count, device="cuda")
        lead = count
    else:
        entry = torch.repeat_interleave(st["indptr"].diff())
        lead = case["count"]
    value = torch.full((count,), float(case["alpha"]), device="cuda", dtype=torch.float64)
    if st["scale"] is not None:
        value = value * st["scale"].double()
    if case["op"] == "lookup":
        # blocks of rows, each the product of its sparse values and the table
        out = torch.zeros(lead, d, device="cuda", dtype=torch.float64)
        step = max(1, (1 << 25) // d)
        kept = entry[keep]
        for lo in range(0, lead, step):
            a, b = torch.searchsorted(kept, torch.tensor([lo, min(lead, lo + step)], device="cuda")).tolist()
            part = keep[a:b]
            if part.numel():
                size = min(step, lead - lo)
                m = _sparse(entry[part] - lo, torch.arange(b - a, device="cuda"), value[part], (size, b - a))
                out[lo:lo + size] = m @ st["table"][ids[part]].double()
        return out
    touched, at = torch.unique(ids[keep], return_inverse=True)
    grad = st["grad"].double()
    u = touched.numel()
    total = torch.zeros(max(1, u), d, device="cuda", dtype=torch.float64)
    if u:
        total = _sparse(at, torch.arange(keep.numel(), device="cuda"), value[keep], (u, keep.numel())) @ grad[entry[keep]]
    out = {}
    if case["result"] == "table":
        whole = torch.zeros(n, d, device="cuda", dtype=torch.float64)
        whole[touched] = total[:u]
        out["table"] = whole
    else:
        cap = min(count, n)
        rows = torch.zeros(cap, d, device="cuda", dtype=torch.float64)
        rows[:u] = total[:u]
        out.update(keys=None, rows=rows, count=None)
    if case.get("want_scale"):
        ds = torch.zeros(count, device="cuda", dtype=torch.float64)
        step = max(1, (1 << 26) // d)
        for lo in range(0, keep.numel(), step):
            k = keep[lo:lo + step]
            ds[k] = case["alpha"] * torch.einsum("td,td->t", grad[entry[k]], st["table"][ids[k]].double())
        out["scale"] = ds
    return out


def _exact_scores(case, st):
    x, labels, op = st["logits"], st["labels"].long(), case["op"]
    t, c = x.shape
    logp, valid = _logprob64(x, labels)
    lse = torch.cat([torch.logsumexp(b.double(), 1) for b in x.split(max(1, (1 << 26) // c))]) if t else logp
    out, g = {}, None
    if op == "logprobs":
        out = {"logprobs": logp, "lse": lse}
        g = st["grad"].double() if case["grad"] else None
    elif op == "preference":
        n = case["pairs"]
        lengths = st["indptr"].diff()
        total = torch.zeros(2 * n, device="cuda", dtype=torch.float64)
        if t:
            total = (_sparse(torch.repeat_interleave(lengths), torch.arange(t, device="cuda"), torch.ones_like(logp),
                             (2 * n, t)) @ logp[:, None])[:, 0]
        z = (total - st["reference"].double()).requires_grad_()
        w = st["weight"].double() if "weight" in st else torch.ones(n, device="cuda", dtype=torch.float64)
        margin = case["beta"] * (z[:n] - z[n:])
        each = -((1 - case["smoothing"]) * torch.nn.functional.logsigmoid(margin)
                 + case["smoothing"] * torch.nn.functional.logsigmoid(-margin))
        loss = (each * w).sum() / w.sum()
        loss.backward()
        g = torch.repeat_interleave(z.grad, lengths)
        out = {"loss": loss.detach(), "margins": margin.detach(), "logprobs": total}
    else:
        w = st["weight"].double() if "weight" in st else torch.ones_like(logp)
        w = w * valid
        z = logp.clone().requires_grad_()
        ratio = torch.exp(z - st["old"].double())
        adv = st["advantage"].double()
        bent = torch.clamp(ratio, 0.8, 1.2)
        k = torch.expm1(st["reference"].double() - z) - (st["reference"].double() - z)
        norm = w.sum() if float(w.sum()) else 1.0
        kl = (w * k).sum() / norm
        loss = (w * -torch.minimum(ratio * adv, bent * adv)).sum() / norm + case["kl"] * kl
        loss.backward()
        g = z.grad
        cut = (bent * adv < ratio * adv).double()
        out = {"loss": loss.detach(), "kl": kl.detach(), "clip_fraction": (w * cut).sum() / norm, "logprobs": logp}
    if g is not None:
        grad = torch.empty(t, c, device="cuda", dtype=torch.float64)
        step = max(1, (1 << 26) // c)
        for lo in range(0, t, step):
            b = grad[lo:lo + step]
            b.copy_(torch.softmax(x[lo:lo + step].double(), 1))
            gb = (g * valid)[lo:lo + step, None]
            b.mul_(-gb)
            b.scatter_add_(1, labels[lo:lo + step].clamp(0, c - 1)[:, None], gb)
        out["grad"] = grad
    return out


# ------------------------------------------------------------------ work --


def work(case):
    """Bytes: ids, values and bounds once, each distinct table row once, each result once. Operations: one
    multiply and one add per value (an exp counts as one)."""
    size = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}
    if case["op"] in ("lookup", "grad"):
        n, d, s = case["n"], case["d"], size[case["table"]]
        wide = 8 if case["scale"] == "f64" else s
        if case["form"] == "tokens":
            entries, ids = case["count"], 8
            live = entries * (1 - case["pad"])
            distinct = _distinct(live, n, case["zipf"])
        else:
            entries, ids = case["count"] * 0.99 * (case["numeric"] + 0.9 * case["hashed"]), 4
            live = entries
            distinct = case["numeric"] + _distinct(case["count"] * 0.99 * 0.9 * case["hashed"], n - case["numeric"],
                                                   case["zipf"])
        b = entries * (ids + (size[case["scale"]] if case["scale"] != "none" else 0))
        b += 8 * case["count"] if case["form"] == "rows" else 0
        if case["op"] == "lookup":
            return {"bytes": int(b + distinct * d * s + case["count"] * d * wide), "flops": int(2 * live * d)}
        out = size[case["out"]] if "out" in case else wide
        b += (case["count"] if case["form"] == "rows" else live) * d * wide
        b += n * d * out if case["result"] == "table" else min(entries, n) * (d * out + ids)
        if case.get("want_scale"):
            b += distinct * d * s + entries * size[case["scale"]]
        return {"bytes": int(b), "flops": int(2 * live * d * (2 if case.get("want_scale") else 1))}
    c, s = case["classes"], size[case["type"]]
    side = 8 if case["type"] == "f64" else 4
    t = case["pairs"] * (case["shortest"] + case["longest"]) if case["op"] == "preference" else case["tokens"]
    arrays = {"logprobs": 2 + (1 if case.get("grad") else 0), "preference": 0, "policy": 4}[case["op"]]
    grad = case.get("grad", True)
    b = t * (c * s * (2 if grad else 1) + (4 if c < 1000 else 8) + arrays * side)
    return {"bytes": int(b), "flops": int(t * c * (5 if grad else 3))}
