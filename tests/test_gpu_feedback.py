"""GPU tier: the preference loss with its gradient, gradient clipping, and a training step through all of them, against float64."""

import math

import numpy as np
import pytest

from oracle import learn_oracle as lo

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


@pytest.fixture(scope="module")
def env():
    import torch

    import hirag_prod_amd as hvs

    class Env:
        pass

    e = Env()
    e.torch, e.hvs, e.dev = torch, hvs, torch.device("cuda", 0)
    return e


def np64(t):
    return t.detach().double().cpu().numpy()


def make(env, qdt, rdt, nq, dim, n_rows, counts, seed=0):
    torch = env.torch
    gen = torch.Generator().manual_seed(seed)
    t = lambda name: getattr(torch, DT[name])
    rows = torch.randn(n_rows, dim, generator=gen).to(env.dev, t(rdt))
    q = torch.randn(nq, dim, generator=gen).to(env.dev, t(qdt))
    ref = (q.float().cpu() + 0.2 * torch.randn(nq, dim, generator=gen)).to(env.dev, t(qdt))
    counts = torch.as_tensor(counts) if counts is not None else torch.randint(0, 7, (nq,), generator=gen)
    offsets = torch.zeros(nq + 1, dtype=torch.int64)
    offsets[1:] = counts.cumsum(0)
    pairs = int(offsets[-1])
    chosen = torch.randint(0, n_rows, (pairs,), generator=gen)
    rejected = torch.randint(0, n_rows, (pairs,), generator=gen)
    return q, ref, rows, chosen.to(env.dev), rejected.to(env.dev), offsets.to(env.dev)


def check(got, want, tol, what):
    got = np64(got)
    assert got.shape == want.shape, what
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN in other places"
    bad = ~(np.abs(got - want) <= tol) & ~nan
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.2f} tolerances at {np.argwhere(bad)[:3].tolist()}"


def check_preference(q, ref, rows, chosen, rejected, offsets, got, qdt, beta, smoothing, weights=None):
    q64, r64 = np64(q), np64(rows)
    ref64 = None if ref is None else np64(ref)
    loss, margin, grad, pull = lo.preference(q64, r64, chosen.cpu().numpy(), rejected.cpu().numpy(), offsets.cpu().numpy(), ref64, beta, smoothing,
                                             None if weights is None else np64(weights))
    dim = q64.shape[1]
    # a cosine is a sum of dim products of norm at most 1, divided by two roots of such sums: relative 2^-22 each at most;
    # a margin holds four of them
    cos_tol = lo.sum_error(1.0, dim) + 8 * 2.0**-24 + 2 * lo.sum_error(1.0, dim)
    margin_tol = 4 * cos_tol
    check(got[1], margin, np.full_like(margin, margin_tol), "margin")
    # |d loss / d margin| <= beta
    check(got[0], loss, beta * margin_tol + 8 * 2.0**-24 * (1 + np.abs(loss)), "loss")
    # the slope changes by at most beta^2 / 4 per unit of margin; every term has length at most 3 pull, element errors of the
    # unit rows 2 cos_tol, and the sum over the pairs rounds once per pair
    pairs_of = np.diff(offsets.cpu().numpy())
    ylen = np.sqrt((q64 * q64).sum(1))
    w = np.full(len(loss), 1.0 / max(len(loss), 1)) if weights is None else np.abs(np64(weights))
    w_sum = np.array([w[a:b].sum() for a, b in zip(offsets.cpu().numpy()[:-1], offsets.cpu().numpy()[1:])])
    inv = np.divide(1.0, ylen, out=np.zeros_like(ylen), where=ylen > 0)
    tol = (inv * w_sum * beta * (beta / 4 * margin_tol * 3 + 3 * cos_tol) + pull * (pairs_of + 8) * 3 * 2.0**-24)[:, None]
    check(got[2], grad, tol + lo.HALF_STEP[qdt] * np.abs(grad) + lo.TINY[qdt], "grad")


@pytest.mark.parametrize("qdt,rdt", [(q, r) for q in DT for r in DT])
@pytest.mark.parametrize("dim", [7, 256, 520, 1536, 2049])
def test_preference(env, qdt, rdt, dim):
    q, ref, rows, c, r, off = make(env, qdt, rdt, 37, dim, 90, None, seed=dim)
    for reference, beta, smoothing in ((ref, 20.0, 0.0), (None, 5.0, 0.1)):
        got = env.hvs.preference_loss(q, rows, c, r, off, reference=reference, beta=beta, label_smoothing=smoothing)
        check_preference(q, reference, rows, c, r, off, got, qdt, beta, smoothing)
        again = env.hvs.preference_loss(q, rows, c, r, off, reference=reference, beta=beta, label_smoothing=smoothing)
        assert all(env.torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dim", [1, 768, 8192, 8193, 16384])
@pytest.mark.parametrize("counts", [[1], [16], [17], [500], [0, 70, 1, 0], [40, 0, 33]])
def test_few_queries_many_pairs(env, dim, counts):
    q, ref, rows, c, r, off = make(env, "f32", "f16", len(counts), dim, 50, counts, seed=dim + len(counts))
    weights = env.torch.rand(len(c), device=env.dev)
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0, weights=weights)
    check_preference(q, ref, rows, c, r, off, got, "f32", 10.0, 0.0, weights)


def test_many_queries(env):
    q, ref, rows, c, r, off = make(env, "bf16", "f32", 700, 100, 300, None, seed=5)
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=20.0)
    check_preference(q, ref, rows, c, r, off, got, "bf16", 20.0, 0.0)


def test_left_out_pairs_and_bad_positions(env):
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f16", 40, 64, 30, None, seed=9)
    n = len(c)
    c[torch.arange(0, n, 3, device=env.dev)] = -1
    r[torch.arange(1, n, 7, device=env.dev)] = -(2**40)
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
    check_preference(q, ref, rows, c, r, off, got, "f32", 20.0, 0.0)
    left = (c < 0) | (r < 0)
    assert not got[0][left].any() and not got[1][left].any()
    c[5], r[8] = 30, 2**40  # one past the last row, and far past it
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
    check_preference(q, ref, rows, c, r, off, got, "f32", 20.0, 0.0)
    c.fill_(-1)
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
    assert not any(t.any() for t in got)


def test_zero_norms_and_same_rows(env):
    torch = env.torch
    for nq in (3, 600):
        q, ref, rows, c, r, off = make(env, "f32", "f32", nq, 40, 20, [4] * nq, seed=2)
        rows[3] = 0
        c[0], r[1] = 3, 3
        c[4] = r[4] = 7  # chosen and rejected alike: margin 0
        q[2] = 0
        ref[0] = 0
        got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=4.0)
        check_preference(q, ref, rows, c, r, off, got, "f32", 4.0, 0.0)
        assert not got[2][2].any() and float(got[1][4]) == 0.0
        assert all(bool(t.isfinite().all()) for t in got)


def test_extreme_margins(env):
    """Losses of thousands and slopes of zero, without overflow."""
    torch = env.torch
    q = torch.tensor([[1.0, 0.0], [1.0, 0.0]], device=env.dev)
    rows = torch.tensor([[1.0, 0.0], [-1.0, 0.0]], device=env.dev)
    off = torch.tensor([0, 1, 2], device=env.dev)
    loss, margin, grad = env.hvs.preference_loss(q, rows, torch.tensor([0, 1], device=env.dev), torch.tensor([1, 0], device=env.dev), off, beta=1000.0)
    assert margin.tolist() == [2.0, -2.0] and loss.tolist() == [0.0, 2000.0]
    assert bool(grad.isfinite().all())


def test_gradient_against_differences(env):
    q, ref, rows, c, r, off = make(env, "f32", "f32", 6, 24, 30, [3, 0, 5, 1, 2, 4], seed=4)
    w = env.torch.rand(len(c), device=env.dev)
    _, _, grad = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=8.0, label_smoothing=0.1, weights=w)
    args = (np64(rows), c.cpu().numpy(), r.cpu().numpy(), off.cpu().numpy(), np64(ref), 8.0, 0.1, np64(w))
    f = lambda x: (lo.preference(x, *args)[0] * args[-1]).sum()
    rng = np.random.default_rng(0)
    q64, g = np64(q), np64(grad)
    for _ in range(6):
        step = rng.standard_normal(q64.shape)
        h = 1e-4
        want = (f(q64 + h * step) - f(q64 - h * step)) / (2 * h)
        # the difference quotient is off by h^2 / 6 times a third derivative of order beta^3, far below 1e-5 of the terms
        assert abs((g * step).sum() - want) <= 1e-4 * np.abs(g * step).sum() + 1e-7


def test_strides(env):
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f16", "f16", 9, 64, 40, None, seed=8)
    want = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
    for left in (8, 3):  # rows that start on 16 bytes, and rows that do not
        wide = lambda t: torch.cat([torch.full_like(t[:, :left], float("nan")), t, torch.full_like(t[:, :left], float("nan"))], 1)[:, left : left + 64]
        got = env.hvs.preference_loss(wide(q), wide(rows), c.int(), r.int(), off.int(), reference=wide(ref))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_table(env):
    """Over the rows of an index: dims that its rows are padded to, after work on the index's own stream, and before."""
    torch = env.torch
    for dtype, dim in (("f16", 100), ("f32", 257), ("bf16", 768)):
        q, ref, rows, c, r, off = make(env, "f32", dtype, 20, dim, 60, None, seed=dim)
        idx = env.hvs.HvsIndex(dim, dtype, device=0)
        idx.add(rows[:30])
        idx.add(rows[30:])
        want = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
        got = idx.preference_loss(q, c, r, off, reference=ref)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = idx.preference_loss(q, c, r, off, reference=ref)
        idx.add(rows)  # grows, and so moves, the table behind the call
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(ValueError):
            idx.preference_loss(q[:, :5], c, r, off)
        graph = torch.cuda.CUDAGraph()
        refused = []
        with torch.cuda.graph(graph):
            try:
                idx.preference_loss(q, c, r, off, reference=ref)
            except env.hvs.HvsError as e:
                refused.append(str(e))
        assert refused and "captured" in refused[0]
        idx.close()


def test_preference_empty_and_refusals(env):
    torch, hvs = env.torch, env.hvs
    q, ref, rows, c, r, off = make(env, "f32", "f32", 4, 16, 10, [1, 2, 0, 1])
    none = torch.zeros(0, dtype=torch.int64, device=env.dev)
    loss, margin, grad = hvs.preference_loss(q, rows, none, none, torch.zeros(5, dtype=torch.int64, device=env.dev))
    assert len(loss) == 0 and len(margin) == 0 and not grad.any()
    loss, margin, grad = hvs.preference_loss(q[:0], rows, none, none, torch.zeros(1, dtype=torch.int64, device=env.dev))
    assert grad.shape == (0, 16)
    nan = hvs.preference_loss(q, rows[:0], c, r, off)
    assert bool(nan[0].isnan().all())
    for kw in (dict(beta=0.0), dict(beta=-1.0), dict(beta=math.nan), dict(beta=math.inf), dict(label_smoothing=-0.1), dict(label_smoothing=0.6)):
        with pytest.raises(hvs.HvsError):
            hvs.preference_loss(q, rows, c, r, off, **kw)
    for args in ((q, rows[:, :8], c, r, off), (q.double(), rows, c, r, off), (q, rows, c[:2], r, off), (q, rows, c, r, off[:-1]), (q, rows.cpu(), c, r, off),
                 (q, rows, c.float(), r, off), (q[0], rows, c, r, off)):
        with pytest.raises(ValueError):
            hvs.preference_loss(*args)
    with pytest.raises(ValueError):
        hvs.preference_loss(q, rows, c, r, off, reference=ref.half())
    with pytest.raises(ValueError):
        hvs.preference_loss(q, rows, c, r, off, weights=torch.ones(3, device=env.dev))


def test_preference_graph(env):
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f16", 5, 128, 60, [30, 2, 0, 50, 1], seed=3)
    call = lambda: env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
    graphs = []
    call()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        graphs.append((graph, outs))
    for turn in range(4):
        q.copy_(torch.randn(5, 128, generator=torch.Generator().manual_seed(turn)).to(env.dev))
        want = call()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(o, w) for o, w in zip(outs, want)), turn


# -- clipping ----------------------------------------------------------------------------------------------------


def check_clip(env, grads, max_norm, infinity, norm, outs):
    g64 = [np64(g) for g in grads]
    want_norm, want = lo.clip(g64, max_norm, infinity)
    # double sums, one rounding to fp32
    assert abs(float(norm) - want_norm) <= 2 * 2.0**-24 * want_norm
    name = {env.torch.float32: "f32", env.torch.float16: "f16", env.torch.bfloat16: "bf16"}
    for g, o, w in zip(grads, outs, want):
        assert o.dtype == g.dtype and o.shape == g.shape
        half = lo.HALF_STEP[name[g.dtype]]
        # the factor and the product in fp32 (four roundings), then one rounding to the type
        assert bool((np.abs(np64(o) - w) <= (4 * 2.0**-24 + half) * np.abs(w) + lo.TINY[name[g.dtype]]).all())


@pytest.mark.parametrize("infinity", [False, True])
@pytest.mark.parametrize("max_norm", [0.0, 0.3, 1e9])
@pytest.mark.parametrize("sizes", [[1], [0], [3, 0, 8191, 8192, 8193], [0, 65000, 535, 1], [65000, 536, 1], [100000, 7], list(range(1, 200))])
def test_clip(env, sizes, max_norm, infinity):
    torch = env.torch
    gen = torch.Generator().manual_seed(len(sizes))
    types = [torch.float32, torch.bfloat16, torch.float16]
    grads = [torch.randn(n, generator=gen).to(env.dev, types[i % 3]) for i, n in enumerate(sizes)]
    kind = math.inf if infinity else 2.0
    outs = [torch.full_like(g, 5.0) for g in grads]
    norm = env.hvs.clip_grad_norm(grads, max_norm, norm_type=kind, out=outs)
    check_clip(env, grads, max_norm, infinity, norm, outs)
    inplace = [g.clone() for g in grads]
    norm2 = env.hvs.clip_grad_norm(inplace, max_norm, norm_type=kind)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(inplace, outs))


def test_clip_unaligned_views_and_neighbours(env):
    torch = env.torch
    for t in (torch.float32, torch.float16, torch.bfloat16):
        base = torch.randn(20001, device=env.dev).to(t)
        want = base.clone()
        out = torch.zeros(20001, device=env.dev, dtype=t)
        view = base[3:20000]
        norm = env.hvs.clip_grad_norm([view], 2.0, out=[out[1:19998]])
        check_clip(env, [view], 2.0, False, norm, [out[1:19998]])
        assert torch.equal(base, want) and float(out[0]) == 0 and float(out[-1]) == 0
        halves = [base[:10000].view(100, 100), base[10000:20000]]
        env.hvs.clip_grad_norm(halves, 1.0)
        assert torch.equal(base[20000], want[20000])


def test_clip_range_and_not_finite(env):
    torch = env.torch
    # squares beyond and below fp32
    for size in (1e25, 1e-30):
        g = torch.full((1000,), size, device=env.dev)
        norm = env.hvs.clip_grad_norm([g], math.inf)
        assert abs(float(norm) - size * math.sqrt(1000)) <= 1e-6 * size * math.sqrt(1000)
        assert bool((g == torch.full((), size, device=env.dev)).all())
    for infinity in (2.0, math.inf):
        g = torch.ones(9000, device=env.dev)
        h = torch.ones(10, device=env.dev, dtype=torch.float16)
        g[8500] = float("nan")
        norm = env.hvs.clip_grad_norm([h, g], 1.0, norm_type=infinity)
        assert math.isnan(float(norm)) and bool(g.isnan().all()) and bool(h.isnan().all())
        g = torch.ones(9000, device=env.dev)
        g[1] = float("-inf")
        norm = env.hvs.clip_grad_norm([g], 1.0, norm_type=infinity)
        assert float(norm) == math.inf and float(g[0]) == 0.0 and math.isnan(float(g[1]))


def test_clip_refusals(env):
    torch, hvs = env.torch, env.hvs
    g = torch.ones(64, device=env.dev)
    for bad in ([], [g.cpu()], [g.double()], [g.view(8, 8).t()], [[1.0]]):
        with pytest.raises(ValueError):
            hvs.clip_grad_norm(bad, 1.0)
    for kw in (dict(norm_type=1.0), dict(out=[]), dict(out=[g.half()]), dict(out=[torch.ones(63, device=env.dev)])):
        with pytest.raises(ValueError):
            hvs.clip_grad_norm([g], 1.0, **kw)
    for bad in (-1.0, math.nan):
        with pytest.raises(hvs.HvsError):
            hvs.clip_grad_norm([g], bad)
    # a tensor named twice would be scaled twice
    with pytest.raises(hvs.HvsError, match="share memory"):
        hvs.clip_grad_norm([g, g], 0.1)
    with pytest.raises(hvs.HvsError, match="share memory"):
        hvs.clip_grad_norm([g[:40], g[30:]], 0.1)
    with pytest.raises(hvs.HvsError, match="overlaps"):
        hvs.clip_grad_norm([g[:40]], 0.1, out=[g[10:50]])
    with pytest.raises(hvs.HvsError, match="share memory"):
        hvs.clip_grad_norm([g[:10], g[20:30]], 0.1, out=[g[20:30], torch.ones(10, device=env.dev)])
    assert bool((g == 1).all())
    # reading one tensor twice is fine
    outs = [torch.zeros_like(g), torch.zeros_like(g)]
    norm = hvs.clip_grad_norm([g, g], 1e9, out=outs)
    assert abs(float(norm) - math.sqrt(128)) < 1e-5 and all(torch.equal(o, g) for o in outs)


def test_clip_graph(env):
    torch = env.torch
    grads = [torch.ones(30000, device=env.dev), torch.ones(77, device=env.dev, dtype=torch.bfloat16)]
    outs = [torch.zeros_like(g) for g in grads]
    env.hvs.clip_grad_norm(grads, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = env.hvs.clip_grad_norm(grads, 1.0, out=outs)
    for turn in range(4):
        for g in grads:
            g.copy_(torch.randn(g.shape, device=env.dev))
        graph.replay()
        torch.cuda.synchronize()
        check_clip(env, grads, 1.0, False, norm, outs)
        want = [torch.zeros_like(g) for g in grads]
        assert torch.equal(norm, env.hvs.clip_grad_norm(grads, 1.0, out=want)) and all(torch.equal(a, b) for a, b in zip(outs, want))


# -- together ----------------------------------------------------------------------------------------------------


def test_training_step_and_search(env):
    """The gradients of a whole step against differences of the float64 loss, and the adapted queries in a search."""
    torch = env.torch
    gen = torch.Generator().manual_seed(1)
    dim, n_rows, nq, s, r = 32, 200, 12, 3, 4
    rows = torch.randn(n_rows, dim, generator=gen)
    idx = env.hvs.HvsIndex(dim, "f32", device=0)
    idx.add(rows.numpy())
    w = torch.eye(dim) + 0.1 * torch.randn(dim, dim, generator=gen)
    a = torch.randn(s, r, dim, generator=gen) / dim**0.5
    b = 0.3 * torch.randn(s, dim, r, generator=gen)
    ad = env.hvs.QueryAdapters(w.to(env.dev), a.to(env.dev), b.to(env.dev), torch.tensor([1.0, 0.5, 2.0], device=env.dev))
    x = torch.randn(nq, dim, generator=gen).to(env.dev)
    codes = torch.tensor([0, 1, 2, -1] * 3, device=env.dev)
    off = torch.arange(0, 3 * nq + 1, 3, device=env.dev)
    c = torch.randint(0, n_rows, (3 * nq,), generator=gen).to(env.dev)
    rej = torch.randint(0, n_rows, (3 * nq,), generator=gen).to(env.dev)
    step = ad.feedback_gradients(idx, x, codes, c, rej, off, beta=6.0)
    tensor_step = ad.feedback_gradients(rows.to(env.dev), x, codes, c, rej, off, beta=6.0)
    assert all(torch.equal(p, q) for p, q in zip(step, tensor_step))
    w64, a64, b64, s64 = np64(ad.projection), np64(ad.a), np64(ad.b), np64(ad.scale)
    x64, cn = np64(x), codes.cpu().numpy()
    ref = x64 @ w64.T
    pref = (rows.double().numpy(), c.cpu().numpy(), rej.cpu().numpy(), off.cpu().numpy(), ref, 6.0, 0.0)
    f = lambda a_, b_: lo.preference(lo.adapters_apply(x64, cn, w64, a_, b_, s64)[0], *pref)[0].mean()
    assert abs(float(step.loss.mean()) - f(a64, b64)) < 1e-5
    rng = np.random.default_rng(0)
    h = 1e-4
    for _ in range(4):
        da, db = rng.standard_normal(a64.shape), rng.standard_normal(b64.shape)
        want = (f(a64 + h * da, b64 + h * db) - f(a64 - h * da, b64 - h * db)) / (2 * h)
        ga, gb = np64(step.grad_a), np64(step.grad_b)
        size = np.abs(ga * da).sum() + np.abs(gb * db).sum()
        assert abs((ga * da).sum() + (gb * db).sum() - want) <= 1e-4 * size
    norm = math.sqrt((np64(step.grad_a) ** 2).sum() + (np64(step.grad_b) ** 2).sum())
    assert abs(float(step.norm) - norm) <= 1e-5 * norm
    clipped = ad.feedback_gradients(idx, x, codes, c, rej, off, beta=6.0, max_norm=norm / 4)
    got = math.sqrt((np64(clipped.grad_a) ** 2).sum() + (np64(clipped.grad_b) ** 2).sum())
    assert abs(got - norm / 4) <= 1e-4 * norm and abs(float(clipped.norm) - norm) <= 1e-5 * norm
    # adapted queries go into a search as they are
    y = ad.apply(x, codes)
    dist, ids, cnt = idx.search(y, k=5)
    y64 = np64(y)
    full = 1 - lo.unit(y64)[0] @ lo.unit(rows.double().numpy())[0].T
    best = np.sort(full, 1)[:, :5]
    assert np.abs(np64(dist) - best).max() < 1e-5
    idx.close()


def test_store_queries_through_adapters(env):
    """Requests of several tenants in flight together, each through its own adapter, on the real index."""
    import asyncio

    import hirag_prod_amd.store as st
    from tests import store_cases

    torch = env.torch
    dim = store_cases.DIM
    gen = torch.Generator().manual_seed(11)
    a = torch.randn(2, 4, dim, generator=gen) / dim**0.5
    b = torch.randn(2, dim, 4, generator=gen) / 2
    ad = env.hvs.QueryAdapters(torch.eye(dim, device=env.dev), a.to(env.dev), b.to(env.dev), torch.ones(2, device=env.dev))
    s = st.HipVectorStore.create(store_cases.make_embedding_func(), vector_type="vector")

    async def scenario():
        tenants = [("ws1", "kb1", 0), ("ws1", "kb2", -1), ("ws2", "kb1", 1)]
        for w, k, _ in tenants:
            props = [store_cases.chunk_props(i, w, k) for i in range(20)]
            await s.upsert_texts([p["text"] for p in props], props, "Chunks")
        s.set_query_adapters(ad, {("ws1", "kb1"): 0, ("ws2", "kb1"): 1})
        asked = [(i, t) for i in range(5) for t in tenants]
        got = await asyncio.gather(*[s.query(f"question {i}", w, k, "Chunks", topk=5, topn=3, distance_threshold=3.0) for i, (w, k, _) in asked])
        for hits, (i, (w, k, c)) in zip(got, asked):
            q = store_cases.embed_text(f"question {i}").astype(np.float32).astype(np.float64)
            y = q if c < 0 else q + np64(b[c]) @ (np64(a[c]) @ q)
            rows = np.stack([store_cases.embed_text(f"text {w} {k} {j}") for j in range(20)])
            dist = 1 - (rows @ y) / np.linalg.norm(rows, axis=1) / np.linalg.norm(y)
            order = np.argsort(dist, kind="stable")[:5]
            store_cases.same_hits([h["documentKey"] for h in hits], [f"chunk-{w}-{k}-{j}" for j in order], dist[order], [h["distance"] for h in hits])

    asyncio.run(scenario())
    s.close()


@pytest.mark.parametrize("nq", [1, 3, 600])
def test_pairs_of_no_query(env, nq):
    """A padded list: pairs before the first query's and after the last one's are left out, the others are what they are alone."""
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f16", nq, 96, 30, [5] * nq, seed=nq)
    pad = lambda t: torch.cat([torch.full((7,), 10**9, device=env.dev), t, torch.full((300,), 3, device=env.dev)])
    weights = torch.rand(len(c), device=env.dev)
    wpad = torch.cat([torch.full((7,), torch.nan, device=env.dev), weights, torch.full((300,), torch.nan, device=env.dev)])
    loss, margin, grad = env.hvs.preference_loss(q, rows, pad(c), pad(r), off + 7, reference=ref, beta=10.0, weights=wpad)
    assert all(not t[:7].any() and not t[7 + len(c) :].any() for t in (loss, margin))
    check_preference(q, ref, rows, c, r, off, (loss[7 : 7 + len(c)], margin[7 : 7 + len(c)], grad), "f32", 10.0, 0.0, weights)


def test_one_query_with_most_pairs(env):
    """Counts that say little about a query: among a few, one has nearly all pairs."""
    for counts in ([0] * 30 + [700], [900] + [1] * 99, [0, 3, 2000, 1], [0] * 300 + [9000]):
        q, ref, rows, c, r, off = make(env, "f32", "bf16", len(counts), 200, 60, counts, seed=len(counts))
        got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0)
        check_preference(q, ref, rows, c, r, off, got, "f32", 10.0, 0.0)


def test_table_read_by_two_streams_then_changed(env):
    """Rows are read as they were when the call was made, whatever the table does next, on two streams in turn."""
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f16", 300, 512, 4000, [60] * 300, seed=3)
    for change in ("update", "compact", "add"):
        idx = env.hvs.HvsIndex(512, "f16", device=0)
        idx.add(rows)
        want = env.hvs.preference_loss(q, rows, c, r, off, reference=ref)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for turn in range(4):
            with torch.cuda.stream(streams[turn % 2]):
                got.append(idx.preference_loss(q, c, r, off, reference=ref))
        if change == "update":
            idx.update(np.arange(4000), np.zeros((4000, 512), dtype=np.float32))
        elif change == "compact":
            idx.set_deleted(np.arange(0, 4000, 2))
            idx.compact()
        else:
            idx.add(rows)
        torch.cuda.synchronize()
        for one in got:
            assert all(torch.equal(a, b) for a, b in zip(one, want)), change
        idx.close()


def test_rows_past_32_bits(env):
    """Positions of rows that lie past 2^31 elements."""
    torch = env.torch
    n, dim = 2_200_000, 1024
    rows = torch.empty(n, dim, dtype=torch.float16, device=env.dev)
    q, ref, some, c, r, off = make(env, "bf16", "f16", 30, dim, 50, None, seed=21)
    at = torch.cat([torch.arange(25), torch.arange(n - 25, n)]).to(env.dev)
    rows[at] = some
    got = env.hvs.preference_loss(q, rows, at[c], at[r], off, reference=ref)
    want = env.hvs.preference_loss(q, some, c, r, off, reference=ref)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_clip_past_32_bits(env):
    torch = env.torch
    n = 2**31 + 4096 + 3
    g = torch.zeros(n, dtype=torch.float16, device=env.dev)
    at = torch.tensor([0, 5, 2**31 - 1, 2**31, n - 1], device=env.dev)
    g[at] = 4.0
    norm = env.hvs.clip_grad_norm([g, torch.zeros(3, device=env.dev)], 1.0)
    want = (5 * 16) ** 0.5
    assert abs(float(norm) - want) <= 2.0**-24 * want
    half = 2.0**-11 + 2.0**-22
    assert bool(((g[at].double() - 4.0 / (want + 1e-6)).abs() <= half * 4 / want).all()) and int((g != 0).sum()) == 5


def test_clip_graph_of_one_launch(env):
    torch = env.torch
    g = torch.ones(500, device=env.dev)
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(g)
    with torch.cuda.graph(graph):
        norm = env.hvs.clip_grad_norm([g], 1.0, out=[out])
    for turn in range(4):
        g.copy_(torch.randn(500, device=env.dev))
        graph.replay()
        torch.cuda.synchronize()
        check_clip(env, [g], 1.0, False, norm, [out])


@pytest.mark.parametrize("qdt", ["f32", "f16"])
@pytest.mark.parametrize("dim,counts", [(1536, [16]), (1536, [3] * 300), (768, [100, 2, 90]), (4000, [5] * 9)])
def test_margins_close_to_the_reference(env, qdt, dim, counts):
    """Queries that have hardly moved, near their chosen rows: the margin's error is a share of the move, not of the cosines."""
    torch = env.torch
    q, _, rows, c, r, off = make(env, qdt, "f16", len(counts), dim, 90, counts, seed=dim + len(counts))
    first = c[off[:-1].clamp(max=len(c) - 1)]
    base = (rows[first].float() + 0.3 * q.float()) * 3.7
    ref = base.to(q.dtype)
    q = (base * 1.3 + 1e-2 * torch.randn(base.shape, device=env.dev)).to(q.dtype)
    _, margin, _ = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0)
    _, want, _, _ = lo.preference(np64(q), np64(rows), c.cpu().numpy(), r.cpu().numpy(), off.cpu().numpy(), np64(ref), 10.0, 0.0)
    # margin = (y^ - y0^) . (c^ - r^): the first factor is right to a few roundings of its own size (and to 2^-45 of the unit
    # vectors), the second to those of the unit rows
    moved = np.linalg.norm(lo.unit(np64(q))[0] - lo.unit(np64(ref))[0], axis=1)
    assert moved.max() < 0.02
    cos_tol = lo.sum_error(1.0, dim) + 8 * 2.0**-24 + 2 * lo.sum_error(1.0, dim)
    check(margin, want, np.repeat(moved, counts) * 4 * cos_tol + 2.0**-45 * dim**0.5, "margin")


def test_norms_at_the_ends_of_the_range(env):
    """Queries of norm 1e30 and 1e-30 are what their unit vectors are; below 1e-38 a norm counts as 0."""
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f16", 12, 64, 30, [4] * 12, seed=2)
    want = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0)
    for size in (2.0**100, 2.0**-100):
        got = env.hvs.preference_loss(q * size, rows, c, r, off, reference=ref * size, beta=10.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool((got[2].double() * size - want[2].double()).abs().max() <= 2.0**-126 * size + 2.0**-22 * want[2].abs().max())
    none = env.hvs.preference_loss(q * 2.0**-140, rows, c, r, off, reference=ref, beta=10.0)
    zero = env.hvs.preference_loss(q * 0.0, rows, c, r, off, reference=ref, beta=10.0)
    assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(none, zero)) and not none[2].any()


@pytest.mark.parametrize("qdt,rdt", [("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("dim", [2056, 4096, 4104, 8200, 12001])
@pytest.mark.parametrize("counts", [[9], [3] * 70, [40] + [1] * 69, [9] * 100, [2] * 300])
def test_wide_rows(env, qdt, rdt, dim, counts):
    """Rows that several waves take together, one block a query and shared."""
    q, ref, rows, c, r, off = make(env, qdt, rdt, len(counts), dim, 30, counts, seed=dim + len(counts))
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0)
    check_preference(q, ref, rows, c, r, off, got, qdt, 10.0, 0.0)


def check_by_terms(q, ref, rows, chosen, rejected, offsets, got, qdt, beta, smoothing, weights=None):
    """Every element against a tolerance made of its own terms (tests/test_adapters_cpu.py shows what that refuses)."""
    args = (np64(q), np64(rows), chosen.cpu().numpy(), rejected.cpu().numpy(), offsets.cpu().numpy(), None if ref is None else np64(ref), beta, smoothing,
            None if weights is None else np64(weights))
    loss, margin, grad, _ = lo.preference(*args)
    loss_tol, margin_tol, grad_tol = lo.preference_tolerance(*args, qdt)
    check(got[1], margin, margin_tol, "margin")
    check(got[0], loss, loss_tol, "loss")
    check(got[2], grad, grad_tol, "grad")


@pytest.mark.parametrize("qdt,rdt", [("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [2, 40, 768, 1536, 2049, 8192, 8193, 16384])
@pytest.mark.parametrize("counts", [[1], [16], [17], [500], [0, 70, 1, 0], [40, 0, 33], [3] * 70])
def test_values_by_their_terms(env, qdt, rdt, dim, counts):
    """Several waves on a pair, shared queries and their join, one block a query."""
    q, ref, rows, c, r, off = make(env, qdt, rdt, len(counts), dim, 50, counts, seed=dim + len(counts))
    weights = env.torch.rand(len(c), device=env.dev)
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0, weights=weights)
    check_by_terms(q, ref, rows, c, r, off, got, qdt, 10.0, 0.0, weights)


@pytest.mark.parametrize("nq,most,dim", [(1, 300, 1536), (100, 16, 768), (250, 12, 1536), (400, 5, 300), (700, 3, 1536)])
def test_values_of_batches_by_their_terms(env, nq, most, dim):
    counts = [(i * 7) % (most + 1) if nq > 1 else most for i in range(nq)]
    for qdt, rdt, reference, smoothing in (("f32", "f16", True, 0.0), ("f16", "bf16", False, 0.1), ("bf16", "f32", True, 0.1)):
        q, ref, rows, c, r, off = make(env, qdt, rdt, nq, dim, 90, counts, seed=nq)
        ref = ref if reference else None
        got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=20.0, label_smoothing=smoothing)
        check_by_terms(q, ref, rows, c, r, off, got, qdt, 20.0, smoothing)


@pytest.mark.parametrize("move", [1e-2, 1e-3])
@pytest.mark.parametrize("qdt", ["f32", "f16"])
@pytest.mark.parametrize("dim,counts", [(1536, [16]), (1536, [3] * 300), (768, [100, 2, 90]), (4000, [5] * 9), (9000, [4] * 5)])
def test_small_moves_by_their_terms(env, move, qdt, dim, counts):
    """Margins next to the reference, to a precision that plain fp32 forms miss (test_margin_tolerance_refuses_plain_forms)."""
    from tests.test_adapters_cpu import near_queries

    torch = env.torch
    rng = np.random.default_rng(dim + len(counts))
    rows = rng.standard_normal((90, dim)).astype(np.float16)
    off = np.concatenate([[0], np.cumsum(counts)])
    c, r = rng.integers(0, 90, off[-1]), rng.integers(0, 90, off[-1])
    q, ref = near_queries(rng, rows.astype(np.float32), c, off, move, {"f32": np.float32, "f16": np.float16}[qdt])
    q, ref, rows, c, r, off = (torch.from_numpy(np.ascontiguousarray(v)).to(env.dev) for v in (q, ref, rows, c, r, off))
    got = env.hvs.preference_loss(q, rows, c, r, off, reference=ref, beta=10.0)
    check_by_terms(q, ref, rows, c, r, off, got, qdt, 10.0, 0.0)


@pytest.mark.parametrize("rdt", ["f32", "bf16"])
@pytest.mark.parametrize("dim,counts", [(64, [4] * 12), (1100, [3] * 20), (1536, [40]), (2049, [9, 1]), (3000, [4] * 130), (9000, [5, 2])])
def test_row_norms_at_the_ends_of_the_range(env, rdt, dim, counts):
    """Rows of fp32's range have squares past it or below it: still only their direction counts, beside ordinary rows and each other,
    down to subnormal elements; an infinite element makes a pair NaN."""
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", rdt, len(counts), dim, 30, counts, seed=dim)
    weights = torch.exp2(torch.arange(len(c), device=env.dev) % 61 - 30.0)
    exponent = torch.tensor([0, 100, -100, 64, -64, -52, 120, -110, 70, -131], device=env.dev).repeat(3)
    sized = (rows.double() * torch.exp2(exponent.double())[:, None]).to(rows.dtype)
    assert bool(sized.isfinite().all()) and bool((sized != 0).any(1).all())
    for w in (None, weights):
        got = env.hvs.preference_loss(q, sized, c, r, off, reference=ref, beta=10.0, weights=w)
        check_by_terms(q, ref, sized, c, r, off, got, "f32", 10.0, 0.0, w)
    sized[4, 5] = torch.inf
    loss, margin, _ = env.hvs.preference_loss(q, sized, c, r, off, reference=ref, beta=10.0)
    touched = (c == 4) | (r == 4)
    assert torch.equal(loss.isnan(), touched) and torch.equal(margin.isnan(), touched)


def table_calls():
    """Calls of a table that return when their work on its stream is done."""
    rng = np.random.default_rng(0)
    q = rng.standard_normal((2, 64)).astype(np.float32)
    rows = rng.standard_normal((5, 64)).astype(np.float32)
    return dict(sync=lambda t: t.sync(), search=lambda t: t.search(q, k=3), range_search=lambda t: t.range_search(q, 0.5), distances=lambda t: t.distances(q),
                filtered=lambda t: t.search(q, k=3, filter=dict(workspace=0)), gather=lambda t: t.gather([1, 2]), kmeans=lambda t: t.kmeans_assign(rows),
                ids=lambda t: t.ids(), export=lambda t: t.export(), set_ids=lambda t: t.set_ids(0, [7, 8]), delete=lambda t: t.set_deleted([3]),
                compact=lambda t: t.compact(), partition=lambda t: t.partition(), add=lambda t: (t.add(rows), t.sync()),
                update=lambda t: (t.update([0], rows[:1]), t.sync()), timer=lambda t: (t.timer_start(), t.timer_stop()))


@pytest.mark.parametrize("call", list(table_calls()))
def test_table_work_runs_after_the_loss(env, call):
    """What is given to a table after a loss over its rows runs after that loss, which waits on its stream behind other work."""
    torch = env.torch
    q, ref, rows, c, r, off = make(env, "f32", "f32", 20, 64, 3000, None, seed=1)
    big = torch.randn(4096, 4096, device=env.dev)
    out = torch.empty_like(big)
    idx = env.hvs.HvsIndex(64, "f32", device=0)
    idx.add(rows.cpu().numpy(), group_codes=np.arange(3000, dtype=np.int32) % 3)
    idx.set_attributes(0, workspace=np.zeros(3000, dtype=np.int32))
    table_calls()[call](idx)  # what the call sets up on its first time
    if call == "compact":
        idx.set_deleted([5])  # without a deleted row it has nothing to do
    want = idx.preference_loss(q, c, r, off, reference=ref)
    side = torch.cuda.Stream()
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(24):  # tens of milliseconds
            torch.mm(big, big, out=out)
        got = idx.preference_loss(q, c, r, off, reference=ref)
    assert not side.query(), "the stream was not busy: the test says nothing"
    table_calls()[call](idx)
    assert side.query(), f"{call} did not wait for the loss"
    if call not in ("compact", "partition", "update", "delete"):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    idx.close()


def test_search_after_a_loss_sees_the_queries_it_was_given(env):
    """Queries made on a stream, a loss on that stream, then a search of the same table by device pointers."""
    import ctypes

    from hirag_prod_amd import _lib

    torch, lib = env.torch, env.hvs.load_library()
    q, ref, rows, c, r, off = make(env, "f32", "f32", 4, 64, 3000, None, seed=2)
    idx = env.hvs.HvsIndex(64, "f32", device=0)
    idx.add(rows)
    want = idx.search(q, k=5)
    late, big = torch.zeros_like(q), torch.randn(4096, 4096, device=env.dev)
    out = torch.empty_like(big)
    outs = torch.empty(4, 5, device=env.dev), torch.empty(4, 5, dtype=torch.int64, device=env.dev), torch.empty(4, dtype=torch.int32, device=env.dev)
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(24):
            torch.mm(big, big, out=out)
        late.copy_(q)
        idx.preference_loss(late, c, r, off, reference=ref)
    assert not side.query()
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())
    _lib.check(lib.hvs_search(idx._h, ptr(late), 4, 1, 5, -1, None, math.inf, 0, -1, *(ptr(t) for t in outs), 1, _lib.HVS_ALGO_AUTO))
    _lib.check(lib.hvs_sync(idx._h))
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    idx.close()


def test_search_captured_while_a_loss_reads_the_table(env):
    """Recording a search neither waits nor fails while a loss is under way; the next call that runs waits for it."""
    import ctypes

    torch, lib = env.torch, env.hvs.load_library()
    q, ref, rows, c, r, off = make(env, "f32", "f32", 4, 64, 3000, None, seed=2)
    stream = torch.cuda.Stream()
    idx = env.hvs.HvsIndex(64, "f32", device=0, stream=stream.cuda_stream)
    idx.add(rows)
    dist, ids, cnt = idx.search(q, k=5)
    outs = torch.empty_like(dist), torch.empty_like(ids), torch.empty_like(cnt)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())
    call = lambda: lib.hvs_search_noalloc(idx._h, ptr(q), 4, 1, 5, -1, None, math.inf, 0, -1, *(ptr(t) for t in outs))
    assert call() == 0
    idx.sync()
    big = torch.randn(4096, 4096, device=env.dev)
    out = torch.empty_like(big)
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.stream(side):
        for _ in range(24):
            torch.mm(big, big, out=out)
        got = idx.preference_loss(q, c, r, off, reference=ref)
        assert not side.query()
    # by hand: torch.cuda.graph waits for the whole GPU first
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="thread_local")
        rc = call()
        with torch.cuda.stream(side):
            try:
                idx.preference_loss(q, c, r, off, reference=ref)
            except env.hvs.HvsError as e:
                refused.append(str(e))
        graph.capture_end()
    assert rc == 0 and refused and "table's stream is being captured" in refused[0]
    assert not side.query()
    idx.sync()
    assert side.query()
    for _ in range(3):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, (dist, ids, cnt)))
    assert all(torch.equal(a, b) for a, b in zip(got, env.hvs.preference_loss(q, rows, c, r, off, reference=ref)))
    del graph
    idx.close()


def step_case(env, dtype, n=4096, pairs_each=16, dim=96, rank=4, tenants=5, seed=0):
    torch = env.torch
    t = getattr(torch, DT[dtype])
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)
    ad = env.hvs.QueryAdapters((torch.eye(dim) + 0.05 * rnd(dim, dim)).to(env.dev, t), (rnd(tenants, rank, dim) / dim**0.5).to(env.dev, t),
                               (0.3 * rnd(tenants, dim, rank)).to(env.dev, t), (0.5 + torch.rand(tenants, generator=gen)).to(env.dev))
    x = rnd(n, dim).to(env.dev, t)
    codes = torch.randint(-1, tenants, (n,), generator=gen).to(env.dev, torch.int32)
    rows = rnd(500, dim).to(env.dev)
    off = torch.arange(0, n * pairs_each + 1, pairs_each, device=env.dev)
    c, r = (torch.randint(0, 500, (n * pairs_each,), generator=gen).to(env.dev) for _ in range(2))
    return ad, x, codes, rows, c, r, off


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("satisfied", [False, True])
@pytest.mark.parametrize("length", [1.0, 40.0])
def test_step_of_many_pairs(env, dtype, satisfied, length):
    """The stack gradients of a whole step over 65 536 pairs, mean loss: against float64 from the adapted queries on.  Satisfied pairs
    (a large margin by weights of the loss's slope) and long queries make the query gradients smaller still."""
    torch = env.torch
    ad, x, codes, rows, c, r, off = step_case(env, dtype)
    x = x * length
    y, hidden = ad.apply(x, codes, return_hidden=True)
    ref = ad.apply(x, torch.full_like(codes, -1))
    weights = torch.full((len(c),), 1e-3 / len(c), device=env.dev) if satisfied else None
    got = ad.feedback_gradients(rows, x, codes, c, r, off, beta=20.0, weights=weights)
    args = (np64(y), np64(rows), c.cpu().numpy(), r.cpu().numpy(), off.cpu().numpy(), np64(ref), 20.0, 0.0, None if weights is None else np64(weights))
    _, _, g, _ = lo.preference(*args)
    _, _, g_tol = lo.preference_tolerance(*args, "f32")
    if dtype != "f32":  # one rounding to the type; fp16: below 2^-14 of a largest element of 2^13 or more, steps of 2^-24
        g_tol += lo.HALF_STEP[dtype] * np.abs(g) + (2.0**-38 * np.abs(g).max() if dtype == "f16" else 0.0)
    cn, x64, u64 = codes.cpu().numpy(), np64(x), np64(hidden)
    a64, b64, s64 = np64(ad.a), np64(ad.b), np64(ad.scale)
    for k in range(ad.n_adapters):
        at = cn == k
        gk, tk, xk, uk = g[at], g_tol[at], x64[at], u64[at]
        rms = lambda p, q: np.sqrt((p * p).T @ (q * q))
        v, v_tol = gk @ b64[k], tk @ np.abs(b64[k]) + lo.sum_error(np.sqrt((gk * gk) @ (b64[k] ** 2)), g.shape[1])
        for what, mine, want, tol in (("grad_a", got.grad_a[k], v.T @ xk, v_tol.T @ np.abs(xk) + lo.sum_error(rms(v, xk), at.sum())),
                                      ("grad_b", got.grad_b[k], gk.T @ uk, tk.T @ np.abs(uk) + lo.sum_error(rms(gk, uk), at.sum()))):
            check(mine, s64[k] * want, s64[k] * tol + 4 * 2.0**-24 * np.abs(s64[k] * want), f"{what} {k}")


def test_half_precision_step_without_a_gradient(env):
    """Every pair left out, and a pair past the last row: zeros, and NaN, as in the other types."""
    torch = env.torch
    ad, x, codes, rows, c, r, off = step_case(env, "f16", n=64, pairs_each=3)
    got = ad.feedback_gradients(rows, x, codes, torch.full_like(c, -1), r, off)
    assert not got.grad_a.any() and not got.grad_b.any() and float(got.norm) == 0.0
    bad = c.clone()
    bad[int(off[int((codes >= 0).nonzero()[0])])] = len(rows)
    got = ad.feedback_gradients(rows, x, codes, bad, r, off)
    assert bool(got.norm.isnan()) and bool(got.loss.isnan().sum() == 1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_step_with_a_code_past_the_last_adapter(env, dtype):
    """Its query's pairs are NaN and add nothing to the gradients of the others."""
    torch = env.torch
    ad, x, codes, rows, c, r, off = step_case(env, dtype, n=64, pairs_each=3)
    left = c.clone()
    left[21:24] = -1  # the pairs of query 7
    want = ad.feedback_gradients(rows, x, codes, left, r, off)
    codes[7] = 5
    got = ad.feedback_gradients(rows, x, codes, c, r, off)
    assert torch.equal(got.loss.isnan().nonzero()[:, 0].cpu(), torch.tensor([21, 22, 23]))
    assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(got[2:], want[2:]))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_step_graph(env, dtype):
    """A whole step captured and replayed, with other work between the replays."""
    torch = env.torch
    ad, x, codes, rows, c, r, off = step_case(env, dtype, n=300, pairs_each=5)
    call = lambda: ad.feedback_gradients(rows, x, codes, c, r, off, max_norm=1e-3)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for turn in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)).to(env.dev, x.dtype))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


@pytest.mark.parametrize("dim", [1, 2])
def test_more_queries_than_a_launch_takes(env, dim):
    """2^24 + 7 queries, most of them without pairs, and pairs of no query behind the last one."""
    torch = env.torch
    nq = 2**24 + 7
    at = torch.tensor([0, 1, 2**22 - 1, 2**22, 2**22 + 1, 2**23, 2**24 - 1, 2**24, nq - 1], device=env.dev)
    counts = torch.zeros(nq, dtype=torch.int64, device=env.dev)
    counts[at] = torch.tensor([3, 0, 2, 5, 1, 4, 2, 1, 3], device=env.dev)
    off = torch.zeros(nq + 1, dtype=torch.int64, device=env.dev)
    off[1:] = counts.cumsum(0)
    _, _, rows, c, r, few_off = make(env, "f32", "f32", len(at), dim, 40, counts[at].cpu(), seed=dim)
    q = torch.randn(nq, dim, device=env.dev)
    ref = q + 0.1
    w = torch.rand(len(c), device=env.dev)
    more = torch.full((5,), 2, device=env.dev)
    loss, margin, grad = env.hvs.preference_loss(q, rows, torch.cat([c, more]), torch.cat([r, more + 1]), off, reference=ref, beta=5.0,
                                                 weights=torch.cat([w, torch.ones(5, device=env.dev)]))
    check_by_terms(q[at], ref[at], rows, c, r, few_off, (loss[:-5], margin[:-5], grad[at]), "f32", 5.0, 0.0, w)
    assert not loss[-5:].any() and not margin[-5:].any()
    grad[at] = 0
    assert not grad.any()


@pytest.mark.parametrize("n", [100, 70000])
def test_clip_without_a_limit_and_an_infinite_norm(env, n):
    """max_norm inf: the data as they are, also next to infinities."""
    torch = env.torch
    for infinity in (2.0, math.inf):
        g = torch.randn(n, device=env.dev)
        g[3], g[4] = torch.inf, -torch.inf
        out = [torch.zeros_like(g)]
        norm = env.hvs.clip_grad_norm([g], math.inf, norm_type=infinity, out=out)
        assert float(norm) == math.inf and torch.equal(out[0], g)
        same = g.clone()
        env.hvs.clip_grad_norm([same], math.inf, norm_type=infinity)
        assert torch.equal(same, g)


def test_lists_and_arrays(env):
    """Codes, positions and offsets as Python lists and numpy arrays, empty ones among them; a step without queries."""
    torch, hvs = env.torch, env.hvs
    q, ref, rows, c, r, off = make(env, "f32", "f32", 4, 16, 10, [1, 2, 0, 1])
    want = hvs.preference_loss(q, rows, c, r, off, reference=ref)
    for kind in (lambda t: t.tolist(), lambda t: t.cpu().numpy(), lambda t: t.int().cpu().numpy()):
        got = hvs.preference_loss(q, rows, kind(c), kind(r), kind(off), reference=ref)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    loss, margin, grad = hvs.preference_loss(q, rows, [], [], [0] * 5)
    assert len(loss) == 0 and len(margin) == 0 and grad.shape == (4, 16) and not grad.any()
    for dtype in DT:
        ad, x, _, table, _, _, _ = step_case(env, dtype, n=3, pairs_each=1)
        assert ad.apply(x[:0], []).shape == (0, 96)
        step = ad.feedback_gradients(table, x[:0], [], [], [], [0])
        assert len(step.loss) == 0 and not step.grad_a.any() and not step.grad_b.any() and float(step.norm) == 0.0
        step = ad.feedback_gradients(table, x, [0, -1, 2], [], [], [0, 0, 0, 0])
        assert len(step.loss) == 0 and not step.grad_a.any() and not step.grad_b.any()
    for bad in ([0.5], np.array([1.0]), ["1"]):
        with pytest.raises((ValueError, TypeError)):
            hvs.preference_loss(q, rows, bad, bad, [0, 1, 1, 1, 1])


def test_training_on_what_a_store_found(env):
    """From a store's hits and keys to a step and back: rows by key, whatever order its table is in, positions among those."""
    import asyncio

    import hirag_prod_amd.store as st
    from tests import store_cases

    torch = env.torch
    dim, tenants = store_cases.DIM, [("ws1", "kb1"), ("ws1", "kb2"), ("ws2", "kb1")]
    ad = env.hvs.QueryAdapters.create(dim, n_adapters=3, rank=4, dtype="f32", seed=3)
    s = st.HipVectorStore.create(store_cases.make_embedding_func(), vector_type="vector")

    async def scenario():
        for i in range(30):  # interleaved, so that a partition moves every row
            for w, k in tenants:
                p = store_cases.chunk_props(i, w, k)
                await s.upsert_texts([p["text"]], [p], "Chunks")
        await s.partition("Chunks")
        s.set_query_adapters(ad, {t: c for c, t in enumerate(tenants)})
        x, codes, pairs, offsets = [], [], [], [0]
        found, place = [], {}
        for c, (w, k) in enumerate(tenants):
            for i in range(4):
                hits = [h["documentKey"] for h in await s.query(f"question {i}", w, k, "Chunks", topk=6, topn=6, distance_threshold=3.0)]
                x.append(store_cases.embed_text(f"question {i}"))
                codes.append(c)
                pairs += [(hits[3], h) for h in hits if h != hits[3]]  # the fourth hit was the useful one
                offsets.append(len(pairs))
            keys = sorted({h for pair in pairs[offsets[4 * c] :] for h in pair})
            for r in await s.query_by_keys(keys, w, k, "Chunks", columns_to_select=["documentKey", "vector"]):
                place[r["documentKey"]] = len(found)
                found.append(r["vector"])
        rows = torch.tensor(found, device=env.dev)
        x = torch.tensor(np.array(x), dtype=torch.float32, device=env.dev)
        chosen, rejected = ([place[p[side]] for p in pairs] for side in (0, 1))
        for key, at in place.items():
            _, w, k, i = key.split("-")
            assert np.array_equal(np64(rows[at]), store_cases.embed_text(f"text {w} {k} {i}").astype(np.float32).astype(np.float64))
        step = ad.feedback_gradients(rows, x, codes, chosen, rejected, offsets, beta=5.0)
        cn, off = np.array(codes), np.array(offsets)
        y, _, u, _ = lo.adapters_apply(np64(x), cn, *(np64(t) for t in (ad.projection, ad.a, ad.b, ad.scale)))
        grad = lo.preference(y, np64(rows), np.array(chosen), np.array(rejected), off, np64(x), 5.0, 0.0)[2]
        _, _, want, _ = lo.adapters_backward(grad, np64(x), cn, u, *(np64(t) for t in (ad.projection, ad.a, ad.b, ad.scale)))
        assert not step.grad_a.any()  # B is zero at the start
        # fp32 sums over 4 queries of 5 pairs; sizes of the terms are at most the norms along the way
        assert np.abs(np64(step.grad_b) - want).max() <= 1e-5 * np.linalg.norm(grad, axis=1).sum() * np.abs(u).max()
        with torch.no_grad():
            ad.b -= 2.0 * step.grad_b
        for (w, k), c in zip(tenants, range(3)):
            q = store_cases.embed_text("question 1").astype(np.float32).astype(np.float64)
            moved = q + np64(ad.b[c]) @ (np64(ad.a[c]) @ q)
            texts = np.stack([store_cases.embed_text(f"text {w} {k} {j}") for j in range(30)])
            dist = 1 - (texts @ moved) / np.linalg.norm(texts, axis=1) / np.linalg.norm(moved)
            order = np.argsort(dist, kind="stable")[:6]
            hits = await s.query("question 1", w, k, "Chunks", topk=6, topn=6, distance_threshold=3.0)
            store_cases.same_hits([h["documentKey"] for h in hits], [f"chunk-{w}-{k}-{j}" for j in order], dist[order], [h["distance"] for h in hits])

    asyncio.run(scenario())
    s.close()
