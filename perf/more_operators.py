"""Label alternatives and the AdamW step, as a user's program calls them, with their plain forms.

What a training step over class scores ends with, and what is told of an answer:

  alternatives  label_alternatives: per row of class scores the label's log-probability and rank, the entropy and the
                best classes; label_alternatives_grad: the scores' gradient for the gradients of all of these
  adamw         AdamW.step: one step over many tensors at once, moments in 32 or 8 bits, with the clip of the
                gradients' norm
  rows          AdamW.step of a table of latent rows by the touched rows that embedding_grad_rows gives

Labels outside the classes mask their rows. Moments in 8 bits come back as the values that they stand for.
"""

import math

import torch

own = False  # set by whoever times this file: the plain forms, or the framework's operators

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BETAS, EPS, SEED = (0.9, 0.999), 1e-8, 20977
BLOCK = 32  # values of a moment in 8 bits that share an exponent; every tensor's moments begin at a multiple of it
# Half a step of a code in units of the float32's last place, and 64 more: 0.9 m + 0.1 g of values of few bits often is
# a tie, and goes up whatever the last bits of the 32-bit sum are.
HALF = (1 << 19) + 64


def listed():
    return [
        # one step of serving over a vocabulary: what was answered and the twenty best; only latency counts
        dict(name="alternatives_serving", op="alternatives", tokens=5, classes=65536, type="bf16", top=20, pad=0.0,
             allowed=1.0, grads="none"),
        # a batch of answers under a frozen model, a tenth of the rows with few classes allowed
        dict(name="alternatives_answers", op="alternatives", tokens=8195, classes=32000, type="bf16", top=5, pad=0.1,
             allowed=0.9, grads="none"),
        # the softmax model's ten classes over many rows, the three best of each and the entropy's gradient
        dict(name="alternatives_classes", op="alternatives", tokens=333333, classes=10, type="f32", top=3, pad=0.01,
             allowed=1.0, grads="entropy"),
        # a model of a thousand classes taught its teacher's sixteen best
        dict(name="alternatives_taught", op="alternatives", tokens=20011, classes=1003, type="f16", top=16, pad=0.0,
             allowed=1.0, grads="all"),
        # sampled tokens in training: log-probabilities with an entropy term, and the scores' gradient
        dict(name="alternatives_trained", op="alternatives", tokens=4096, classes=65536, type="bf16", top=0, pad=0.2,
             allowed=1.0, grads="entropy"),
        # a factorization machine's three parameters in a small step: only latency counts
        dict(name="adamw_small", op="adamw", form="tables", width=60, rows=1003, type="f32", grad="f32", bits=32,
             master=False, clip=1.0, decay=0.01, aligned=True, steps=3),
        # hundreds of tensors of odd sizes behind each other, from one value to a million, beginning anywhere
        dict(name="adamw_ragged", op="adamw", form="ragged", count=300, largest=1000003, type="f32", grad="f32", bits=32,
             master=False, clip=0.0, decay=0.01, aligned=False, steps=100),
        # layers of a model in bfloat16 with float32 master weights and moments, its norm clipped
        dict(name="adamw_layers", op="adamw", form="layers", width=1024, depth=12, rows=32000, type="bf16", grad="bf16",
             bits=32, master=True, clip=1.0, decay=0.1, aligned=True, steps=1000),
        # the same layers with moments in 8 bits and no master weights
        dict(name="adamw_layers_8bit", op="adamw", form="layers", width=1024, depth=12, rows=32000, type="bf16",
             grad="bf16", bits=8, master=False, clip=0.0, decay=0.1, aligned=True, steps=1000),
        # the largest float32 model: wide layers, plain float32 moments
        dict(name="adamw_wide", op="adamw", form="layers", width=4096, depth=1, rows=32000, type="f32", grad="f32",
             bits=32, master=False, clip=0.0, decay=0.01, aligned=True, steps=10),
        # the touched rows of one mini-batch of clicks in a table of 2^22 latent rows of 16
        dict(name="rows_clicks", op="rows", n=1 << 22, d=16, entries=302000, zipf=1.1, type="f32", grad="f32", bits=32,
             clip=0.0, decay=0.01, steps=50),
        # the touched rows of a batch of tokens in a wide table, moments in 8 bits
        dict(name="rows_tokens_8bit", op="rows", n=32000, d=1024, entries=65536, zipf=1.0, type="bf16", grad="f32",
             bits=8, clip=1.0, decay=0.0, steps=50),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Classes from 2 to 131072 and rows from 1 to a million, up to 2^27 scores; sets of 1 to 300 tensors of 1 to
    16 million values; tables of up to 2^22 rows of 1 to 4096."""
    op = rng.choice(["alternatives", "alternatives", "alternatives", "adamw", "adamw", "rows"])
    if op == "alternatives":
        classes = _spread(rng, 2, 1 << 17)
        tokens = min(_spread(rng, 1, 1 << 20), max(1, (1 << 27) // classes))
        return dict(op=op, tokens=tokens, classes=classes, type=rng.choice(["bf16", "bf16", "f16", "f32", "f64"]),
                    top=min(classes, rng.choice([0, 1, 5, rng.randint(1, 32)])), pad=rng.choice([0.0, 0.1, 0.5]),
                    allowed=rng.choice([1.0, 1.0, 0.8]), grads=rng.choice(["none", "entropy", "all"]))
    kind, grad = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f64", "f64")])
    bits = 32 if kind == "f64" else rng.choice([32, 8])
    case = dict(op=op, type=kind, grad=grad, bits=bits, clip=rng.choice([0.0, 1.0]), decay=rng.choice([0.0, 0.01, 0.1]),
                steps=_spread(rng, 1, 10000) - 1)
    if op == "rows":
        d = _spread(rng, 1, 4096)
        n = min(_spread(rng, 2, 1 << 22), max(2, (1 << 26) // d))
        case.update(n=n, d=d, entries=min(_spread(rng, 1, 1 << 19), max(1, (1 << 25) // d)), zipf=rng.choice([0.0, 1.0, 1.1]))
        return case
    case.update(master=kind in ("bf16", "f16") and rng.random() < 0.5, aligned=rng.random() < 0.7)
    form = rng.choice(["tables", "ragged", "layers"])
    if form == "tables":
        width = _spread(rng, 1, 256)
        case.update(form=form, width=width, rows=min(_spread(rng, 2, 1 << 20), (1 << 24) // width))
    elif form == "ragged":
        case.update(form=form, count=_spread(rng, 1, 300), largest=_spread(rng, 1, 1 << 19))
    else:
        width = _spread(rng, 8, 1024)
        case.update(form=form, width=width, depth=rng.randint(1, 4), rows=_spread(rng, 2, 8192))
    return case


# ---------------------------------------------------------------- inputs --


def _sizes(case):
    """The numbers of values of the tensors that are stepped."""
    if case["form"] == "tables":
        return [1, case["rows"], case["rows"] * case["width"]]
    if case["form"] == "ragged":
        last = max(1, case["count"] - 1)
        return [max(1, int(round(case["largest"] ** (i / last))) - i % 3) for i in range(case["count"])]
    w = case["width"]
    return [case["rows"] * w] + case["depth"] * [w * w, w * w, w * w, w * w, 4 * w * w, 4 * w * w, w, w]


def _padded(size):
    return (size + BLOCK - 1) // BLOCK * BLOCK


def _normal(g, shape, dtype, std=1.0):
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    return (torch.randn(shape, generator=g, device="cuda", dtype=wide) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return {"alternatives": _prepare_scores, "adamw": _prepare_tensors, "rows": _prepare_rows}[case["op"]](case, g)


def _prepare_scores(case, g):
    t, c, kind = case["tokens"], case["classes"], DTYPES[case["type"]]
    wide = torch.float64 if kind == torch.float64 else torch.float32
    x = _normal(g, (t, c), kind, 2.5)
    labels = torch.empty(t, device="cuda", dtype=torch.int64)
    step = max(1, (1 << 27) // c)
    for lo in range(0, t, step):  # labels drawn from the scores' softmax, in blocks of rows
        b = x[lo:lo + step].float()
        labels[lo:lo + step] = (b - torch.empty_like(b).exponential_(generator=g).log_()).argmax(1)
    if case["allowed"] < 1.0:  # rows with few classes left: their label, and others now and then
        few = (torch.rand(t, generator=g, device="cuda") >= case["allowed"]).nonzero()[:, 0]
        left = torch.rand(few.numel(), c, generator=g, device="cuda") < 12.0 / c
        left.scatter_(1, labels[few, None], True)
        x[few] = torch.where(left, x[few], -math.inf)
    labels[torch.rand(t, generator=g, device="cuda") < case["pad"]] = -1
    st = dict(case=case, logits=x, labels=labels.int() if c < 1000 else labels)
    if case["grads"] != "none":
        st["g_logprobs"] = _normal(g, (t,), wide)
        st["g_entropy"] = _normal(g, (t,), wide, 0.1)
        if case["grads"] == "all" and case["top"]:
            st["g_top"] = _normal(g, (t, case["top"]), wide, 0.3)
    return st


def _prepare_tensors(case, g):
    sizes, kind, wide = _sizes(case), DTYPES[case["type"]], torch.float64 if case["type"] == "f64" else torch.float32
    gaps = [_padded(n) for n in sizes]
    total, whole = sum(sizes), sum(gaps)
    if case["aligned"]:  # parameters and gradients lie as the moments do, with gaps behind odd sizes
        at = torch.tensor([0] + gaps).cumsum(0)[:-1].tolist()
        place, extent = None, whole
    else:  # one value behind the other
        at = torch.tensor([0] + sizes).cumsum(0)[:-1].tolist()
        shift = torch.tensor([0] + [p - n for p, n in zip(gaps, sizes)]).cumsum(0)[:-1]
        place = torch.arange(total, device="cuda") + torch.repeat_interleave(shift.cuda(), torch.tensor(sizes).cuda())
        extent = total
    live = torch.ones(whole, device="cuda", dtype=torch.bool)
    if total < whole:  # the moments' gaps hold zeros
        live.fill_(False)
        live[place if place is not None else torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(at, sizes)])] = True
    keep = live if place is None else torch.ones(1, device="cuda", dtype=torch.bool)
    p, grad = _normal(g, (extent,), kind, 0.3) * keep, _normal(g, (extent,), DTYPES[case["grad"]], 0.02) * keep
    st = dict(case=case, param=p, grad=grad, place=place, step=torch.tensor(case["steps"], device="cuda"),
              params=[p[a:a + n] for a, n in zip(at, sizes)], grads=[grad[a:a + n] for a, n in zip(at, sizes)])
    if case["bits"] == 8:  # the number of each tensor and of each value in it, which the roundings' random bits go by
        number = torch.arange(len(sizes), device="cuda")
        st["tensor"] = torch.repeat_interleave(number, torch.tensor(gaps).cuda()).to(torch.int32)
        st["begin"] = torch.tensor([0] + gaps[:-1]).cumsum(0).cuda()
    _moments(st, g, whole, wide, live)
    if case["master"]:
        near = p.float() + 1e-3 * p.float() * _normal(g, (extent,), torch.float32)
        st["master"] = _spread_out(near, place, whole)
        st["param"].copy_(near)
    return st


def _moments(st, g, whole, wide, live):
    m, v = _normal(g, (whole,), wide, 0.006), 4e-4 * torch.exp(_normal(g, (whole,), wide, 1.5))
    m, v = m * live, v * live
    if st["case"]["bits"] == 8:
        half = torch.full((1,), HALF, device="cuda")
        (st["m"], st["m_exp"]), (st["v"], st["v_exp"]) = _encode(m, half, True), _encode(v, half, False)
    else:
        st["m"], st["v"] = m, v


def _prepare_rows(case, g):
    n, d, kind = case["n"], case["d"], DTYPES[case["type"]]
    wide = torch.float64 if case["type"] == "f64" else torch.float32
    u = torch.rand(case["entries"], generator=_shape_generator(case), device="cuda", dtype=torch.float64)
    if case["zipf"] == 0.0:
        rank = (u * n).long()
    elif case["zipf"] == 1.0:
        rank = torch.exp(u * math.log(n + 1)).long() - 1
    else:
        a = 1.0 - case["zipf"]
        rank = ((((n + 1) ** a - 1.0) * u + 1.0) ** (1.0 / a)).long() - 1
    ids = torch.unique((rank.clamp_(0, n - 1) * 2654435761 + torch.randint(0, n, (1,), generator=g, device="cuda")) % n)
    places, used = min(case["entries"], n), ids.numel()
    pitch = _padded(d) if case["bits"] == 8 else d
    keys = torch.full((places,), -1, device="cuda", dtype=torch.int32)
    keys[:used] = ids.int()
    rows = torch.zeros(places, d, device="cuda", dtype=DTYPES[case["grad"]])
    rows[:used] = _normal(g, (used, d), DTYPES[case["grad"]], 0.02)
    st = dict(case=case, param=_normal(g, (n, d), kind, 0.3), keys=keys, rows=rows,
              count=torch.tensor(used, device="cuda"), used=used, step=torch.tensor(case["steps"], device="cuda"),
              row_steps=torch.randint(0, case["steps"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32))
    live = torch.zeros(_padded(n * pitch), device="cuda", dtype=torch.bool)
    live[:n * pitch] = (torch.arange(pitch, device="cuda") < d).repeat(n) & (st["row_steps"] > 0).repeat_interleave(pitch)
    _moments(st, g, live.numel(), wide, live)
    return st


def _shape_generator(case):
    """Which ids are met goes by the case, but for a shift: the number of touched rows stays."""
    g = torch.Generator(device="cuda")
    g.manual_seed(case["entries"])
    return g


# ------------------------------------------------------------------ runs --


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def _own(st):
    from modern_fm_b200 import optim, preference
    from modern_fm_b200.embedding import EmbeddingRows

    case = st["case"]
    if case["op"] == "alternatives":
        r = preference.label_alternatives(st["logits"], st["labels"], top=case["top"])
        out = {k: v for k, v in r._asdict().items() if v is not None}
        if "g_logprobs" in st:
            out["grad"] = preference.label_alternatives_grad(
                st["logits"], r.lse, r.entropy, st["labels"], st["g_logprobs"], st["g_entropy"],
                r.top_ids if "g_top" in st else None, st.get("g_top"))
        return out
    if "optimizer" not in st:  # kept by a program from step to step; its state is st's own
        state = optim.AdamWState(step=st["step"], m=st["m"], v=st["v"], m_exp=st.get("m_exp"), v_exp=st.get("v_exp"),
                                 master=st.get("master"), row_steps=st.get("row_steps"))
        st["optimizer"] = optim.AdamW(
            st["params"] if case["op"] == "adamw" else [st["param"]], lr=_rate(case), betas=BETAS, eps=EPS,
            weight_decay=case["decay"], state_bits=case["bits"], master=case.get("master", False),
            by_rows=case["op"] == "rows", seed=SEED, state=state)
    opt = st["optimizer"]
    grads = st["grads"] if case["op"] == "adamw" else [EmbeddingRows(st["keys"], st["rows"], st["count"], None)]
    norm = opt.step(grads, max_norm=case["clip"] or None)
    m, v = opt.moments() if case["bits"] == 8 else (st["m"], st["v"])
    return _result(st, norm, m, v)


def _rate(case):
    return 1e-4 if case["bits"] == 8 else 1e-3


def _result(st, norm, m, v):
    out = {"param": st["param"], "m": m, "v": v, "step": st["step"]}
    out.update({k: st[k] for k in ("master", "row_steps") if k in st})
    if norm is not None:
        out["norm"] = norm
    return out


def _plain_alternatives(st):
    case, labels, c = st["case"], st["labels"].long(), st["case"]["classes"]
    x = st["logits"].double() if case["type"] == "f64" else st["logits"].float()
    top = x.max(1, keepdim=True).values
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    logp = (x - top) - total.log()
    p = e.div_(total)
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    valid = (labels >= 0) & (labels < c)
    at = labels.clamp(0, c - 1)[:, None]
    mine = x.gather(1, at)
    before = torch.arange(c, device="cuda") < at
    rank = ((x > mine) | ((x == mine) & before)).sum(1)
    out = {"logprobs": torch.where(valid, logp.gather(1, at)[:, 0], 0.0),
           "lse": torch.where(valid, top[:, 0] + total[:, 0].log(), 0.0),
           "entropy": torch.where(valid, entropy, 0.0),
           "ranks": torch.where(valid, rank, -1).to(st["labels"].dtype)}
    if case["top"]:
        ids = st["logits"].sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_ids"] = torch.where(valid[:, None], ids, -1).to(st["labels"].dtype)
        out["top_logprobs"] = torch.where(valid[:, None], logp.gather(1, ids), 0.0)
    if "g_logprobs" in st:
        # dx = g at each chosen class - p (sum of these g + g_entropy (log p + entropy))
        gl, gh = torch.where(valid, st["g_logprobs"], 0.0)[:, None], torch.where(valid, st["g_entropy"], 0.0)[:, None]
        gt = torch.where(valid[:, None], st["g_top"], 0.0) if "g_top" in st else gl[:, :0]
        d = -p * (gl + gt.sum(1, keepdim=True) + gh * torch.where(p > 0, logp + entropy[:, None], 0.0))
        d.scatter_add_(1, at, gl)
        if "g_top" in st:
            d.scatter_add_(1, ids, gt)
        out["grad"] = d.to(st["logits"].dtype)
    return out


def _mix(x):
    """32 bits, held in 64, that depend on each of the 32 bits of x (two rounds of shift, xor and product)."""
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(st, step):
    """20 random bits for each place of the second moments, by the seed, the tensor's number, the step and the place."""
    if st["case"]["op"] == "rows":
        d, pitch = st["case"]["d"], _padded(st["case"]["d"])
        number = torch.zeros(1, device="cuda", dtype=torch.int64)
        e = st["keys"][:st["used"], None].long() * d + torch.arange(pitch, device="cuda")
        e = e.reshape(-1)
    else:
        number = st["tensor"].long()
        e = torch.arange(number.numel(), device="cuda") - st["begin"][number]
    key = _mix((_mix((_mix(torch.full_like(number[:1], SEED)) + number) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    key = (key + 0x9E3779B9 * (e >> 32)) & 0xFFFFFFFF
    return _mix((e & 0xFFFFFFFF) ^ key) >> 12


def _bits(x):
    return x.view(torch.int32).long()


def _encode(x, random, signed):
    """Codes and shared exponents of float32 values: sign and 7 bits, or 8 bits without a sign. A magnitude's number
    is its upper 11 bits (exponent, 3 bits of mantissa) after adding `random` below them; code = number - 8 exponent."""
    most, reach = (127, 15) if signed else (255, 31)
    size = _bits(x.abs())
    number = ((size + random) >> 20).clamp(max=0x7F7)
    largest = size.view(-1, BLOCK).amax(1)
    shared = ((((largest + (HALF if signed else (1 << 20) - 1)) >> 20).clamp(max=0x7F7) >> 3) - reach).clamp(min=0)
    code = (number.view(-1, BLOCK) - 8 * shared[:, None]).clamp(0 if signed else 1, most).view(-1)
    code = torch.where(size == 0, 0, code)
    return (code + torch.where(x < 0, 128, 0) * (code > 0)).to(torch.uint8) if signed else code.to(torch.uint8), shared.to(torch.uint8)


def _decode(code, shared, signed):
    k = (code & 127 if signed else code).int()
    number = k + 8 * shared.int().repeat_interleave(BLOCK)
    x = torch.where(k == 0, 0, number << 20).view(torch.float32)
    return torch.where(code > 127, -x, x) if signed else x


def _spread_out(x, place, whole):
    if place is None:
        return x
    out = torch.zeros(whole, device="cuda", dtype=x.dtype)
    out[place] = x
    return out


def _step(case, p, g, m, v, t1, t2):
    """New parameters and moments; t1, t2: 1 - beta^t."""
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * (g * g)
    lr = _rate(case)
    return p - lr * case["decay"] * p - lr * ((m / t1) / ((v / t2).sqrt() + EPS)), m, v


def _scaled(case, g, wide):
    """(the gradient in the wide type, clipped to the norm; the norm or None)."""
    g = g.to(wide)
    if not case["clip"]:
        return g, None
    norm = g.double().square().sum().sqrt()
    return g * (case["clip"] / norm).clamp(max=1.0).to(wide), norm.to(wide)


def _plain_adamw(st):
    case, wide, place = st["case"], st["v"].dtype if st["case"]["bits"] == 32 else torch.float32, st["place"]
    whole = st["v"].numel()
    g, norm = _scaled(case, st["grad"], wide)
    g = _spread_out(g, place, whole)
    t = (st["step"] + 1).double()
    t1, t2 = (1 - BETAS[0] ** t).to(wide), (1 - BETAS[1] ** t).to(wide)
    p = st["master"] if case["master"] else _spread_out(st["param"].to(wide), place, whole)
    if case["bits"] == 8:
        p, m, v = _step(case, p, g, _decode(st["m"], st["m_exp"], True), _decode(st["v"], st["v_exp"], False), t1, t2)
        codes = _encode(m, HALF, True) + _encode(v, _random_bits(st, st["step"] + 1), False)
        st["m"], st["m_exp"], st["v"], st["v_exp"] = codes
        m, v = _decode(*codes[:2], True).bfloat16(), _decode(*codes[2:], False).bfloat16()
    else:
        p, m, v = _step(case, p, g, st["m"], st["v"], t1, t2)
        st["m"], st["v"] = m, v
    if case["master"]:
        st["master"] = p
    st["param"] = (p if place is None else p[place]).to(st["param"].dtype)
    st["step"] = st["step"] + 1
    return _result(st, norm, m, v)


def _plain_rows(st):
    case, n, d, used = st["case"], st["case"]["n"], st["case"]["d"], st["used"]
    wide = st["v"].dtype if case["bits"] == 32 else torch.float32
    keys = st["keys"][:used].long()
    g, norm = _scaled(case, st["rows"][:used], wide)
    st["row_steps"][keys] += 1
    t = st["row_steps"][keys, None].double()
    t1, t2 = (1 - BETAS[0] ** t).to(wide), (1 - BETAS[1] ** t).to(wide)
    p = st["param"][keys].to(wide)
    if case["bits"] == 8:
        parts = [st[k].view(n, -1)[keys].view(-1) for k in ("m", "m_exp", "v", "v_exp")]
        m, v = _decode(*parts[:2], True).view(used, -1), _decode(*parts[2:], False).view(used, -1)
        p, m, v = _step(case, p, g, m[:, :d], v[:, :d], t1, t2)
        gap = (0, _padded(d) - d)
        m, v = (torch.nn.functional.pad(x, gap).view(-1) for x in (m, v))
        codes = _encode(m, HALF, True) + _encode(v, _random_bits(st, st["step"] + 1), False)
        for k, x in zip(("m", "m_exp", "v", "v_exp"), codes):
            st[k].view(n, -1)[keys] = x.view(used, -1)
        m, v = (_decode(st[k], st[k + "_exp"], k == "m").bfloat16() for k in ("m", "v"))
    else:
        m, v = st["m"][:n * d].view(n, d), st["v"][:n * d].view(n, d)
        p, m[keys], v[keys] = _step(case, p, g, m[keys], v[keys], t1, t2)
        m, v = st["m"], st["v"]
    st["param"][keys] = p.to(st["param"].dtype)
    st["step"] = st["step"] + 1
    return _result(st, norm, m, v)


_PLAIN = dict(alternatives=_plain_alternatives, adamw=_plain_adamw, rows=_plain_rows)


# ----------------------------------------------------------------- exact --


def exact(case, seed):
    """The definitions in 64 bits: softmax by torch's own in row blocks, its gradient through autograd; the step by
    increments of the moments; codes of 8 bits by exponents and fractions."""
    st = prepare(case, seed)
    return (_exact_alternatives if case["op"] == "alternatives" else _exact_step)(case, st)


def _exact_alternatives(case, st):
    x, labels, c, k = st["logits"], st["labels"].long(), case["classes"], case["top"]
    parts = []
    step = max(1, (1 << 26) // c)
    for lo in range(0, x.shape[0], step):
        b = x[lo:lo + step].double().requires_grad_("g_logprobs" in st)
        y = labels[lo:lo + step]
        live = (y >= 0) & (y < c)
        with torch.set_grad_enabled("g_logprobs" in st):
            lp = torch.log_softmax(b, 1)
            safe = torch.where(torch.isinf(b), 0.0, lp)
            entropy = -(lp.exp() * safe).sum(1)
            mine = torch.gather(safe if b.requires_grad else lp, 1, y.clamp(0, c - 1)[:, None])[:, 0]
            got = {"logprobs": torch.where(live, mine, 0.0), "lse": torch.logsumexp(b.detach(), 1) * live,
                   "entropy": entropy * live, "ranks": None}
            if k:
                best = b.detach().sort(dim=1, descending=True, stable=True).indices[:, :k]
                some = lp.gather(1, best)
                got.update(top_ids=None, top_logprobs=torch.where(live[:, None], some, 0.0))
            if b.requires_grad:
                total = (got["logprobs"] * st["g_logprobs"][lo:lo + step].double()
                         + got["entropy"] * st["g_entropy"][lo:lo + step].double()).sum()
                if "g_top" in st:
                    weight = torch.where(live[:, None], st["g_top"][lo:lo + step].double(), 0.0)
                    gap = torch.isinf(b.detach().gather(1, best))
                    total = total + (safe.gather(1, best) * weight * ~gap).sum()
                total.backward()
                d = torch.where(torch.isfinite(b), b.grad, 0.0)
                if "g_top" in st:  # a best class of score -infinity: the slope of x - lse all the same
                    lost = torch.where(gap, weight, 0.0)
                    d = d.scatter_add(1, best, lost) - torch.softmax(b.detach(), 1) * lost.sum(1, keepdim=True)
                got["grad"] = d
        parts.append({name: None if v is None else v.detach() for name, v in got.items()})
    return {name: None if parts[0][name] is None else torch.cat([q[name] for q in parts]) for name in parts[0]}


def _exact_number(x):
    """The real number whose whole part is a magnitude's exponent and 3 bits of mantissa."""
    fraction, exponent = torch.frexp(x)
    return torch.where(x > 0, 8.0 * (exponent.double() + 126) + 8.0 * (2 * fraction - 1), 0.0)


def _exact_value(number):
    q = torch.floor(number / 8)
    return torch.ldexp(1 + (number - 8 * q) / 8, q - 127)


def _exact_code(x, random, signed):
    number = _exact_number(x.abs())
    top = number.view(-1, BLOCK).amax(1)
    base = 8 * (torch.floor((torch.floor(top + HALF / (1 << 20)) if signed else torch.ceil(top)) / 8) - (15 if signed else 31)).clamp(min=0)
    base = base.repeat_interleave(BLOCK)
    whole = torch.floor(number + (HALF / (1 << 20) if signed else random.double() / (1 << 20)))
    whole = torch.minimum(whole, base + (127 if signed else 255))
    if not signed:
        whole = torch.maximum(whole, base + 1)
    return torch.where((x == 0) | (whole <= base), 0.0, _exact_value(whole) * torch.sign(x))


def _exact_step(case, st):
    rows, d, eight = case["op"] == "rows", case.get("d"), case["bits"] == 8
    used = st.get("used")
    if rows:
        keys = st["keys"][:used].long()
        g, p = st["rows"][:used].double(), st["param"][keys].double()
    else:
        g = _spread_out(st["grad"].double(), st["place"], st["v"].numel())
        p = st["master"].double() if case["master"] else _spread_out(st["param"].double(), st["place"], st["v"].numel())
    norm = torch.linalg.vector_norm(g)
    if case["clip"] and float(norm) > case["clip"]:
        g = g / norm * case["clip"]
    whole = {}
    for k in ("m", "v"):
        whole[k] = _decode(st[k], st[k + "_exp"], k == "m").double() if eight else st[k].double().clone()
    if rows:
        pitch = _padded(d) if eight else d
        m, v = (whole[k][:case["n"] * pitch].view(-1, pitch)[keys, :d] for k in ("m", "v"))
        t = (st["row_steps"][keys] + 1).double()[:, None]
    else:
        m, v, t = whole["m"], whole["v"], (st["step"] + 1).double()
    m, v = torch.lerp(m, g, 1 - BETAS[0]), torch.lerp(v, g.square(), 1 - BETAS[1])
    size = -torch.expm1(t * math.log(BETAS[1]))
    move = m / -torch.expm1(t * math.log(BETAS[0])) / (torch.sqrt(v / size) + EPS) + case["decay"] * p
    p = p - _rate(case) * move
    if eight:
        gap = (0, _padded(d) - d) if rows else (0, 0)
        m, v = (torch.nn.functional.pad(x, gap).reshape(-1) for x in (m, v))
        m, v = _exact_code(m, None, True), _exact_code(v, _random_bits(st, st["step"] + 1), False)
    if rows:
        for k, x in (("m", m), ("v", v)):
            whole[k][:case["n"] * pitch].view(-1, pitch)[keys] = x.reshape(used, pitch)
        table = st["param"].double()
        table[keys] = p
        out = {"param": table, "m": whole["m"], "v": whole["v"], "row_steps": None}
    else:
        out = {"param": p if st["place"] is None else p[st["place"]], "m": m, "v": v}
        if case["master"]:
            out["master"] = p
    out["step"] = None
    if case["clip"]:
        out["norm"] = norm
    return out


# ------------------------------------------------------------------ work --


def work(case):
    """Bytes: each input once, each result once (moments in 8 bits with the values that come back). Operations: one
    multiply and one add per value (an exp counts as one)."""
    size = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "alternatives":
        t, c, s = case["tokens"], case["classes"], size[case["type"]]
        side, ids = 8 if case["type"] == "f64" else 4, 4 if c < 1000 else 8
        live = 1 - case["pad"]
        b = t * (2 * ids + 3 * side + case["top"] * (ids + side)) + t * live * c * s
        grad = case["grads"] != "none"
        if grad:
            b += t * (c * s + 2 * side + (case["top"] * side if case["grads"] == "all" else 0))
        return {"bytes": int(b), "flops": int(t * live * c * (9 if grad else 5))}
    s, gs = size[case["type"]], size[case["grad"]]
    wide = 8 if case["type"] == "f64" else 4
    state = 4 * wide if case["bits"] == 32 else 4 + 4 / BLOCK
    if case["op"] == "rows":
        n, d = case["n"], case["d"]
        if case["zipf"] == 0.0:
            used = n * -math.expm1(case["entries"] * math.log1p(-1 / n))
        else:
            a = 1 - case["zipf"]
            at = lambda r: math.log(r) / math.log(n + 1) if a == 0 else (r**a - 1) / ((n + 1.0) ** a - 1)  # noqa: E731
            used, r = 0.0, 1
            while r <= n:  # ranks of one size of probability at a time
                hi = min(n + 1, r + max(1, r // 16))
                used += (hi - r) * -math.expm1(-case["entries"] * (at(hi) - at(r)) / (hi - r))
                r = hi
        back = 6 * n * _padded(d) if case["bits"] == 8 else 0
        return {"bytes": int(used * (d * (2 * s + gs + state) + 12) + back), "flops": int(14 * used * d)}
    total = sum(_sizes(case))
    back = 6 if case["bits"] == 8 else 0
    return {"bytes": int(total * (2 * s + gs + state + (8 if case["master"] else 0) + back)), "flops": int(14 * total)}
