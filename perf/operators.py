"""What the operators behind learned query adapters are measured on: cases, inputs, plain forms and 64-bit values.

Three operators that are used together, in this order, when retrieval learns from feedback:

* ``adapters``    -- a projection shared by all tenants beside one low-rank adapter per tenant, applied to a batch of
                     query embeddings of many tenants at once (``QueryAdapters.apply``), and its backward pass
                     (``QueryAdapters.backward``)
* ``preference``  -- the preference loss over pairs of table rows with the gradient for the queries
                     (``preference_loss``, ``HvsIndex.preference_loss``)
* ``clip``        -- the global norm of many gradient tensors and the clipped gradients (``clip_grad_norm``)
"""

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one interactive question: the embedding service's fp32 vector on its way into a search
        dict(name="apply_one_query", op="apply", dtype="f32", n=1, d_in=1536, d_out=1536, rank=16, adapters=64),
        # the questions of 40 tenants that wait at the same moment share one call
        dict(name="apply_waiting_requests", op="apply", dtype="bf16", n=40, d_in=1536, d_out=1536, rank=16, adapters=64),
        # nothing is a multiple of anything: an embedding width that is no multiple of 8, a narrower table, an odd rank
        dict(name="apply_odd", op="apply", dtype="f32", n=777, d_in=1001, d_out=770, rank=13, adapters=5),
        # a full batch of questions
        dict(name="apply_batch", op="apply", dtype="bf16", n=4096, d_in=1536, d_out=1536, rank=16, adapters=256),
        # stored rows moved through the projection in bulk, when a table is rewritten into the learned space
        dict(name="apply_bulk", op="apply", dtype="f16", n=65536, d_in=1536, d_out=1536, rank=32, adapters=32),
        # a training step on the feedback of one hour of a small deployment
        dict(name="backward_small", op="backward", dtype="f32", n=96, d_in=768, d_out=768, rank=8, adapters=12),
        # a training step on a full batch
        dict(name="backward_batch", op="backward", dtype="bf16", n=8192, d_in=1536, d_out=1536, rank=16, adapters=64),
        # one question whose answer was rated: the cited chunk against the chunks that were not
        dict(name="preference_one_query", op="preference", queries="f32", rows="f16", dim=1536, n_rows=20000, nq=1,
             max_pairs=16, masked=0.0, reference=True, smoothing=0.0, table="tensor"),
        # fp32 rows, 16-bit queries, no reference policy, smoothed labels, pairs that were withdrawn
        dict(name="preference_ragged", op="preference", queries="bf16", rows="f32", dim=768, n_rows=50000, nq=301,
             max_pairs=9, masked=0.1, reference=False, smoothing=0.1, table="tensor"),
        # a full batch over the table that is being searched
        dict(name="preference_batch", op="preference", queries="f32", rows="f16", dim=1536, n_rows=120000, nq=4096,
             max_pairs=16, masked=0.02, reference=True, smoothing=0.0, table="index"),
        # the gradients of one tenant's adapter
        dict(name="clip_one_adapter", op="clip", tensors=2, smallest=24576, largest=24576, mixed=False, norm="2", share=0.5),
        # the gradients of an embedding model's worth of tensors, several types, one far larger than another
        dict(name="clip_many", op="clip", tensors=60, smallest=64, largest=33554432, mixed=True, norm="2", share=0.1),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["apply", "apply", "backward", "preference", "preference", "clip"])
    if op in ("apply", "backward"):
        n = _spread(rng, 1, 20000)
        width = lambda: rng.choice([256, 768, 1024, 1536, _spread(rng, 33, 2000)])
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), n=n, d_in=width(), d_out=width(),
                    rank=rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)]), adapters=_spread(rng, 1, 300))
    if op == "preference":
        return dict(op=op, queries=rng.choice(["f32", "f16", "bf16"]), rows=rng.choice(["f32", "f16", "bf16"]),
                    dim=rng.choice([256, 768, 1024, 1536, _spread(rng, 9, 4096)]), n_rows=_spread(rng, 50, 50000),
                    nq=_spread(rng, 1, 4096), max_pairs=_spread(rng, 1, 16), masked=rng.choice([0.0, 0.1, 0.5]),
                    reference=rng.random() < 0.6, smoothing=rng.choice([0.0, 0.1]), table=rng.choice(["tensor", "index"]))
    largest = _spread(rng, 1, 4194304)
    return dict(op=op, tensors=_spread(rng, 1, 60), smallest=1 + largest // 1000, largest=largest, mixed=rng.random() < 0.5,
                norm=rng.choice(["2", "2", "inf"]), share=rng.choice([0.01, 0.3, 5.0]))


# -- inputs ----------------------------------------------------------------------------------------------------


def _unit_rows(n, d, gen):
    """Rows of length 1, as embedding services return them."""
    x = torch.randn(n, d, generator=gen, device=DEVICE)
    return x / x.norm(dim=1, keepdim=True).clamp_min(1e-6)


def _adapter_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    n, d_in, d_out, r, s = case["n"], case["d_in"], case["d_out"], case["rank"], case["adapters"]
    t = DTYPES[case["dtype"]]
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)
    uniform = torch.rand(n, generator=gen, device=DEVICE)
    # tenants are not alike: the square puts more requests on the low numbers; one request in 16 has no adapter
    codes = (uniform * uniform * s).to(torch.int32).clamp_(max=s - 1)
    codes[torch.rand(n, generator=gen, device=DEVICE) < 1 / 16] = -1
    inputs = dict(
        x=_unit_rows(n, d_in, gen).to(t),
        codes=codes,
        w=(rnd(d_out, d_in) / math.sqrt(d_in)).to(t),
        a=(rnd(s, r, d_in) / math.sqrt(d_in)).to(t),
        b=(0.3 * rnd(s, d_out, r) / math.sqrt(r)).to(t),
        scale=0.5 + torch.rand(s, generator=gen, device=DEVICE),
    )
    if case["op"] == "backward":
        inputs["grad"] = (0.05 * rnd(n, d_out)).to(t)
        # the hidden values the forward pass returned, in 32 bits
        hidden = torch.zeros(n, r, dtype=torch.float32, device=DEVICE)
        for c in range(s):
            at = (codes == c).nonzero()[:, 0]
            if len(at):
                hidden[at] = (inputs["x"][at].double() @ inputs["a"][c].double().t()).float()
        inputs["hidden"] = hidden
    return inputs


def _preference_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dim, n_rows, nq = case["dim"], case["n_rows"], case["nq"]
    rows = _unit_rows(n_rows, dim, gen).to(DTYPES[case["rows"]])
    # every number of pairs a query from none to max_pairs, in an order of the seed's
    counts = torch.arange(nq, device=DEVICE) % (case["max_pairs"] + 1) if nq > 1 else torch.full((1,), case["max_pairs"], device=DEVICE)
    counts = counts[torch.randperm(nq, generator=gen, device=DEVICE)]
    offsets = torch.zeros(nq + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = counts.cumsum(0)
    pairs = int(offsets[-1])
    chosen = torch.randint(0, n_rows, (pairs,), generator=gen, device=DEVICE)
    rejected = torch.randint(0, n_rows, (pairs,), generator=gen, device=DEVICE)
    chosen[torch.rand(pairs, generator=gen, device=DEVICE) < case["masked"]] = -1
    # a query lies near its first chosen row; the learned query has moved away from the reference by a tenth
    near = torch.zeros(nq, dtype=torch.int64, device=DEVICE)
    if pairs:
        near = chosen[offsets[:-1].clamp(max=pairs - 1)].clamp(min=0)
    base = rows[near].float() + 1.5 * _unit_rows(nq, dim, gen)
    t = DTYPES[case["queries"]]
    return dict(rows=rows, offsets=offsets, chosen=chosen, rejected=rejected, reference=base.to(t) if case["reference"] else None,
                queries=(base + 0.15 * _unit_rows(nq, dim, gen)).to(t), beta=20.0, smoothing=case["smoothing"])


def _clip_inputs(case, seed):
    import random

    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(f"{case['tensors']} {case['smallest']} {case['largest']}")
    grads = []
    for i in range(case["tensors"]):
        # the first tensor is the largest, the others are spread up to it
        n = case["largest"] if i == 0 else _spread(rng, case["smallest"], case["largest"])
        t = [torch.float32, torch.bfloat16, torch.float16][i % 3] if case["mixed"] else torch.float32
        grads.append((0.01 * torch.randn(n, generator=gen, device=DEVICE)).to(t))
    if case["norm"] == "inf":
        full = 0.05
    else:
        full = 0.01 * math.sqrt(sum(g.numel() for g in grads))
    return dict(grads=grads, max_norm=case["share"] * full, norm=float(case["norm"]))


def _inputs(case, seed):
    return {"apply": _adapter_inputs, "backward": _adapter_inputs, "preference": _preference_inputs, "clip": _clip_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    state = dict(op=case["op"], inputs=_inputs(case, seed))
    i = state["inputs"]
    if case["op"] == "clip":
        i["out"] = [torch.empty_like(g) for g in i["grads"]]  # a training loop's own buffers
    if own:
        import hirag_prod_amd as hvs

        state["hvs"] = hvs
        if case["op"] in ("apply", "backward"):
            state["adapters"] = hvs.QueryAdapters(i["w"], i["a"], i["b"], i["scale"])
        if case["op"] == "preference" and case["table"] == "index":
            state["index"] = hvs.HvsIndex(case["dim"], case["rows"], device=0)
            state["index"].add(i["rows"])
            state["index"].sync()
    return state


# -- one pass ---------------------------------------------------------------------------------------------------


def run(state):
    i = state["inputs"]
    if not own:
        return {"apply": _plain_apply, "backward": _plain_backward, "preference": _plain_preference, "clip": _plain_clip}[state["op"]](i)
    if state["op"] == "apply":
        return state["adapters"].apply(i["x"], i["codes"])
    if state["op"] == "backward":
        return state["adapters"].backward(i["grad"], i["x"], i["codes"], i["hidden"])
    if state["op"] == "preference":
        if "index" in state:
            return state["index"].preference_loss(i["queries"], i["chosen"], i["rejected"], i["offsets"], reference=i["reference"],
                                                  beta=i["beta"], label_smoothing=i["smoothing"])
        return state["hvs"].preference_loss(i["queries"], i["rows"], i["chosen"], i["rejected"], i["offsets"], reference=i["reference"],
                                            beta=i["beta"], label_smoothing=i["smoothing"])
    norm = state["hvs"].clip_grad_norm(i["grads"], i["max_norm"], norm_type=i["norm"], out=i["out"])
    return [norm] + i["out"]


def _by_adapter(codes):
    """(rows ordered by adapter, [(adapter, begin, end) within that order])"""
    order = torch.argsort(codes, stable=True)
    present, counts = torch.unique_consecutive(codes[order], return_counts=True)
    spans, begin = [], 0
    for c, m in zip(present.tolist(), counts.tolist()):
        spans.append((c, begin, begin + m))
        begin += m
    return order, spans


def _plain_apply(i):
    x, a, b = i["x"].float(), i["a"], i["b"]
    y = x @ i["w"].float().t()
    if len(x) <= 64:  # few rows: every row takes its own copy of its adapter
        c = i["codes"].clamp(min=0).long()
        u = (a[c].float() * x[:, None, :]).sum(2)
        low = (b[c].float() * u[:, None, :]).sum(2) * i["scale"][c][:, None]
        y = y + low * (i["codes"] >= 0)[:, None]
    else:
        order, spans = _by_adapter(i["codes"])
        xs, low = x[order], torch.zeros_like(y)
        a, b = i["scale"][:, None, None] * a.float(), b.float()
        for c, lo, hi in spans:
            if c >= 0:
                low[lo:hi] = (xs[lo:hi] @ a[c].t()) @ b[c].t()
        y = y.index_add_(0, order, low)
    return y.to(i["x"].dtype)


def _plain_backward(i):
    x, g, hidden = i["x"].float(), i["grad"].float(), i["hidden"]
    a, scale = i["a"].float(), i["scale"][:, None, None]
    b = scale * i["b"].float()
    dx = g @ i["w"].float()
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    order, spans = _by_adapter(i["codes"])
    xs, gs, us, low = x[order], g[order], hidden[order], torch.zeros_like(dx)
    for c, lo, hi in spans:
        if c >= 0:
            v = gs[lo:hi] @ b[c]
            low[lo:hi] = v @ a[c]
            da[c] = v.t() @ xs[lo:hi]
            db[c] = gs[lo:hi].t() @ us[lo:hi]
    return dx.index_add_(0, order, low).to(i["x"].dtype), da, scale * db


def _plain_preference(i):
    offsets, nq = i["offsets"], len(i["queries"])
    pairs = len(i["chosen"])
    q = torch.repeat_interleave(torch.arange(nq, device=offsets.device), offsets[1:] - offsets[:-1], output_size=pairs)
    counted = (i["chosen"] >= 0) & (i["rejected"] >= 0)

    def unit(rows):
        length = rows.norm(dim=1, keepdim=True)
        return torch.where(length > 0, rows / length, torch.zeros_like(rows)), length

    good, _ = unit(i["rows"][i["chosen"].clamp(min=0)].float())
    bad, _ = unit(i["rows"][i["rejected"].clamp(min=0)].float())
    diff = good - bad
    y, length = unit(i["queries"].float())
    cos = (diff * y[q]).sum(1)
    margin = cos
    if i["reference"] is not None:
        ref, _ = unit(i["reference"].float())
        margin = cos - (diff * ref[q]).sum(1)
    margin = torch.where(counted, margin, torch.zeros_like(margin))
    h, e = i["beta"] * margin, i["smoothing"]
    softplus = lambda z: torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))
    loss = torch.where(counted, (1 - e) * softplus(-h) + e * softplus(h), torch.zeros_like(h))
    slope = i["beta"] * (e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h)) / max(pairs, 1)
    slope = torch.where(counted, slope, torch.zeros_like(slope))
    pull = slope[:, None] * (diff - cos[:, None] * y[q])
    grad = torch.zeros_like(y).index_add_(0, q, pull)
    grad = torch.where(length > 0, grad / length, torch.zeros_like(grad))
    return loss, margin, grad.to(i["queries"].dtype)


def _plain_clip(i):
    if i["norm"] == math.inf:
        norm = torch.stack([g.float().abs().max() for g in i["grads"]]).max()
    else:
        norm = torch.stack([(g.double() ** 2).sum() for g in i["grads"]]).sum().sqrt().float()
    coef = torch.clamp(i["max_norm"] / (norm + 1e-6), max=1.0)
    return [norm] + [(g.float() * coef).to(g.dtype) for g in i["grads"]]


# -- the values in 64 bits ---------------------------------------------------------------------------------------


def exact(case, seed):
    i = _inputs(case, seed)
    if case["op"] in ("apply", "backward"):
        x, w = i["x"].double(), i["w"].double()
        codes, scale = i["codes"].tolist(), i["scale"].double()
        rows_of = {}
        for row, c in enumerate(codes):
            if c >= 0:
                rows_of.setdefault(c, []).append(row)
        if case["op"] == "apply":
            y = x.matmul(w.T)
            for c, rows in rows_of.items():
                at = torch.tensor(rows, device=x.device)
                delta = i["b"][c].double().matmul(i["a"][c].double()) * scale[c]  # the adapter as one matrix
                y.index_add_(0, at, x[at].matmul(delta.T))
            return y
        g = i["grad"].double()
        dx = g.matmul(w)
        da = torch.zeros(i["a"].shape, dtype=torch.float64, device=x.device)
        db = torch.zeros(i["b"].shape, dtype=torch.float64, device=x.device)
        for c, rows in rows_of.items():
            at = torch.tensor(rows, device=x.device)
            a, b = i["a"][c].double(), i["b"][c].double()
            dx.index_add_(0, at, g[at].matmul(b.matmul(a) * scale[c]))
            dm = g[at].T.matmul(x[at]) * scale[c]  # the gradient for B A, split by the product rule
            da[c] = b.T.matmul(dm)
            db[c] = dm.matmul(a.T)
        return dx, da, db
    if case["op"] == "preference":
        nq, pairs, e, beta = case["nq"], len(i["chosen"]), i["smoothing"], i["beta"]
        offsets = i["offsets"].tolist()
        loss = torch.zeros(pairs, dtype=torch.float64, device=DEVICE)
        margin = torch.zeros(pairs, dtype=torch.float64, device=DEVICE)
        grad = torch.zeros(nq, case["dim"], dtype=torch.float64, device=DEVICE)
        step = 512  # queries at a time
        for q0 in range(0, nq, step):
            q1 = min(q0 + step, nq)
            lo, hi = offsets[q0], offsets[q1]
            if lo == hi:
                continue
            owner = torch.tensor([k for k in range(q0, q1) for _ in range(offsets[k + 1] - offsets[k])], device=DEVICE)
            c, r = i["chosen"][lo:hi], i["rejected"][lo:hi]
            live = ((c >= 0) & (r >= 0)).double()
            cr = torch.nn.functional.normalize(i["rows"][c.clamp(min=0)].double(), dim=1)
            rr = torch.nn.functional.normalize(i["rows"][r.clamp(min=0)].double(), dim=1)
            y = i["queries"].double()[owner]
            ylen = torch.linalg.vector_norm(y, dim=1)
            cc, rc = (cr * y).sum(1) / ylen, (rr * y).sum(1) / ylen
            m = cc - rc
            if i["reference"] is not None:
                y0 = torch.nn.functional.normalize(i["reference"].double()[owner], dim=1)
                m = m - ((cr * y0).sum(1) - (rr * y0).sum(1))
            m = m * live
            margin[lo:hi] = m
            loss[lo:hi] = live * -((1 - e) * torch.nn.functional.logsigmoid(beta * m) + e * torch.nn.functional.logsigmoid(-beta * m))
            slope = live * beta * (torch.sigmoid(beta * m) - (1 - e)) / pairs
            dcos = (cr - cc[:, None] * (y / ylen[:, None]) - rr + rc[:, None] * (y / ylen[:, None])) / ylen[:, None]
            grad.index_add_(0, owner, slope[:, None] * dcos)
        return loss, margin, grad
    if i["norm"] == math.inf:
        norm = max(float(g.double().abs().max()) for g in i["grads"])
    else:
        norm = math.sqrt(math.fsum(float(g.double().square().sum()) for g in i["grads"]))
    coef = min(1.0, i["max_norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64, device=DEVICE)] + [g.double() * coef for g in i["grads"]]


# -- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    if case["op"] in ("apply", "backward"):
        n, d_in, d_out, r, s, e = case["n"], case["d_in"], case["d_out"], case["rank"], case["adapters"], BYTES[case["dtype"]]
        used = min(n, s)
        moved = e * (n * (d_in + d_out) + d_in * d_out + used * r * (d_in + d_out)) + 4 * n + 4 * used
        flops = 2 * n * d_in * d_out + 2 * n * r * (d_in + d_out)
        if case["op"] == "backward":
            moved += e * n * d_in + 4 * n * r + 4 * s * r * (d_in + d_out)  # dx, hidden, both stacks of gradients
            flops += 2 * n * r * (d_in + d_out)
        return {"bytes": moved, "flops": flops}
    if case["op"] == "preference":
        dim, nq = case["dim"], case["nq"]
        pairs = case["max_pairs"] if nq == 1 else nq * case["max_pairs"] // 2
        rows = min(2 * pairs, case["n_rows"])
        queries = nq * dim * BYTES[case["queries"]] * (3 if case["reference"] else 2)
        return {"bytes": rows * dim * BYTES[case["rows"]] + queries + 24 * pairs + 8 * nq,
                "flops": pairs * dim * (16 if case["reference"] else 12)}
    import random

    rng = random.Random(f"{case['tensors']} {case['smallest']} {case['largest']}")
    moved = total = 0
    for i in range(case["tensors"]):
        n = case["largest"] if i == 0 else _spread(rng, case["smallest"], case["largest"])
        total += n
        moved += 2 * n * ([4, 2, 2][i % 3] if case["mixed"] else 4)
    return {"bytes": moved, "flops": 3 * total}
