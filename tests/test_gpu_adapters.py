"""GPU tier: low-rank query adapters (forward, backward) against float64."""

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


def make(env, dtype, n, d_in, d_out, rank, adapters, seed=0, codes=None):
    torch = env.torch
    gen = torch.Generator().manual_seed(seed)
    t = getattr(torch, DT[dtype])
    rnd = lambda *s: torch.randn(*s, generator=gen)
    x = rnd(n, d_in).to(env.dev, t)
    w = (rnd(d_out, d_in) / d_in**0.5).to(env.dev, t)
    a = (rnd(adapters, rank, d_in) / d_in**0.5).to(env.dev, t)
    b = (rnd(adapters, d_out, rank) / rank**0.5).to(env.dev, t)
    scale = (0.5 + torch.rand(adapters, generator=gen)).to(env.dev)
    if codes is None:
        codes = torch.randint(-1, adapters, (n,), generator=gen)
    codes = torch.as_tensor(codes).to(env.dev, torch.int32)
    return env.hvs.QueryAdapters(w, a, b, scale), x, codes, gen


def weights64(ad):
    return np64(ad.projection), np64(ad.a), np64(ad.b), np64(ad.scale)


def check(got, want, tol, what):
    got = np64(got)
    assert got.shape == want.shape, what
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN in other places"
    bad = ~(np.abs(got - want) <= tol) & ~nan
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.2f} tolerances at {np.argwhere(bad)[:3].tolist()}"


def check_apply(env, ad, x, codes, dtype, what="y"):
    y, hidden = ad.apply(x, codes, return_hidden=True)
    cn = codes.cpu().numpy()
    want, tol, u, u_tol = lo.adapters_apply_tolerance(np64(x), cn, *weights64(ad), dtype)
    check(hidden, u, u_tol, "hidden")
    check(y, want, tol, what)
    return y, hidden


SIZES = [
    # n, d_in, d_out, rank, adapters
    (1, 8, 8, 1, 1),
    (1, 1536, 1536, 16, 64),
    (3, 100, 60, 5, 2),
    (16, 64, 16, 16, 3),
    (17, 257, 33, 17, 40),
    (63, 768, 512, 8, 63),
    (64, 1536, 768, 64, 7),
    (65, 64, 64, 8, 3),
    (65, 1, 1, 1, 1),
    (130, 200, 130, 33, 4),
    (300, 1001, 770, 13, 5),
    (1024, 256, 256, 16, 300),
    (1025, 96, 200, 32, 2),
    (2500, 512, 520, 128, 11),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d_in,d_out,rank,adapters", SIZES)
def test_apply(env, dtype, n, d_in, d_out, rank, adapters):
    ad, x, codes, _ = make(env, dtype, n, d_in, d_out, rank, adapters)
    check_apply(env, ad, x, codes, dtype)


def test_apply_largest_tile(env):
    """Enough rows and columns for the 256 x 256 tile."""
    for dtype in ("f16", "bf16"):
        ad, x, codes, _ = make(env, dtype, 8200, 128, 2050, 16, 9)
        check_apply(env, ad, x, codes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d_in,rank,adapters", [(72, 16, 5), (41, 21, 700), (64, 50, 3), (96, 128, 33)])
def test_apply_many_rows(env, dtype, d_in, rank, adapters):
    """Rows enough for the wide form of A x, and more than the grouping counts by itself."""
    ad, x, codes, _ = make(env, dtype, 16500, d_in, 24, rank, adapters)
    check_apply(env, ad, x, codes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [5, 200])
@pytest.mark.parametrize("kind", ["none", "one", "each", "past"])
def test_codes(env, dtype, n, kind):
    codes = {"none": [-1] * n, "one": [2] * n, "each": list(range(n)), "past": [(-3, 0, n, 2**31 - 1)[i % 4] for i in range(n)]}[kind]
    ad, x, codes, _ = make(env, dtype, n, 72, 80, 6, n, codes=codes)
    y, hidden = check_apply(env, ad, x, codes, dtype)
    if kind == "none":
        assert bool((hidden == 0).all())


def test_codes_beyond_32_bits(env):
    torch = env.torch
    ad, x, _, _ = make(env, "f32", 4, 16, 16, 2, 3)
    codes = torch.tensor([0, 2**32, -(2**32), 2**32 + 1], dtype=torch.int64, device=env.dev)
    y = ad.apply(x, codes)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all())
    same = ad.apply(x, torch.tensor([0, -1, -1, -1], dtype=torch.int32, device=env.dev))
    assert torch.equal(y[[0, 2]], same[[0, 2]])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", [10, 150])
def test_strides_and_neighbours(env, dtype, n):
    """Rows inside a wider tensor whose other columns are NaN, unaligned; the output's other columns stay as they were."""
    torch = env.torch
    for d_in, d_out, left in ((64, 64, 8), (100, 40, 4), (99, 41, 3)):
        ad, x, codes, _ = make(env, dtype, n, d_in, d_out, 8, 3)
        wide = torch.full((n, d_in + 2 * left), float("nan"), dtype=x.dtype, device=env.dev)
        wide[:, left : left + d_in] = x
        out = torch.full((n, d_out + 2 * left), 7.0, dtype=x.dtype, device=env.dev)
        ad.apply(wide[:, left : left + d_in], codes, out=out[:, left : left + d_out])
        want = ad.apply(x, codes)
        assert torch.equal(out[:, left : left + d_out], want)
        assert bool((out[:, :left] == 7).all()) and bool((out[:, left + d_out :] == 7).all())
        # a transposed view has no contiguous rows: it is copied
        assert torch.equal(ad.apply(x.t().contiguous().t(), codes), want)
        assert torch.equal(ad.apply(x[:1].expand(n, d_in), codes[:1].expand(n)), ad.apply(x[:1].repeat(n, 1), codes[:1].repeat(n)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [20, 140])
def test_what_is_not_finite_stays_with_its_tenant(env, dtype, n):
    torch = env.torch
    ad, x, codes, _ = make(env, dtype, n, 72, 80, 8, 4, codes=[(i * 7) % 5 - 1 for i in range(n)])
    want = ad.apply(x, codes)
    ad.a[1, 2, 3] = float("nan")
    ad.b[2, 5, 1] = float("inf")
    x[7] = float("inf")
    y = ad.apply(x, codes)
    clean = (codes != 1) & (codes != 2)
    clean[7] = False
    assert torch.equal(y[clean], want[clean])
    assert bool(y[codes == 1].isnan().all()) and bool((~y[7].isfinite()).any())


def test_large_values_in_half_precision(env):
    """A x beyond the largest fp16 number, brought back by B: the middle is held in fp32."""
    torch = env.torch
    for n in (8, 100):
        ad, x, codes, _ = make(env, "f16", n, 64, 64, 16, 2, codes=[i % 2 for i in range(n)])
        ad.a.mul_(512.0)
        x.mul_(1024.0)
        ad.b.mul_(1.0 / 4096.0)
        y, hidden = check_apply(env, ad, x, codes, "f16")
        assert float(hidden.abs().max()) > 65504 and bool(y.isfinite().all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d_in,d_out,rank,adapters", [(1, 8, 8, 1, 1), (2, 100, 60, 5, 3), (64, 256, 128, 16, 5), (96, 768, 768, 8, 12), (333, 257, 130, 33, 7),
                                                       (1030, 200, 96, 16, 40), (3000, 64, 72, 70, 2), (1500, 128, 64, 128, 3)])
def test_backward(env, dtype, n, d_in, d_out, rank, adapters):
    torch = env.torch
    ad, x, codes, gen = make(env, dtype, n, d_in, d_out, rank, adapters)
    g = torch.randn(n, d_out, generator=gen).to(env.dev, x.dtype)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    dx, da, db = ad.backward(g, x, codes, hidden)
    check_backward(ad, g, x, codes, hidden, dtype, dx, da, db)
    # a fixed order of sums: the same bits again, and without grad_x
    dx2, da2, db2 = ad.backward(g, x, codes, hidden)
    assert torch.equal(dx, dx2) and torch.equal(da, da2) and torch.equal(db, db2)
    none, da3, db3 = ad.backward(g, x, codes, hidden, input_grad=False)
    assert none is None and torch.equal(da, da3) and torch.equal(db, db3)


def check_backward(ad, g, x, codes, hidden, dtype, dx, da, db):
    w, a, b, scale = weights64(ad)
    g64, x64, h64, cn = np64(g), np64(x), np64(hidden), codes.cpu().numpy()
    wx, wa, wb, v = lo.adapters_backward(g64, x64, cn, h64, w, a, b, scale)
    # grad_x is the forward with the transposed weights
    _, tol, v_, v_tol = lo.adapters_apply_tolerance(g64, cn, w.T.copy(), b.transpose(0, 2, 1).copy(), a.transpose(0, 2, 1).copy(), scale, dtype)
    check(dx, wx, tol, "grad_x")
    tol_a, tol_b = np.zeros_like(a), np.zeros_like(b)
    for c in range(len(a)):
        at = np.flatnonzero(cn == c)
        m = len(at)
        s = scale[c]
        tol_a[c] = s * (sum_tol(v[at], x64[at], m) + v_tol[at].T @ np.abs(x64[at])) + 2 * 2.0**-24 * np.abs(wa[c])
        tol_b[c] = s * sum_tol(g64[at], h64[at], m) + 2 * 2.0**-24 * np.abs(wb[c])
    check(da, wa, tol_a, "grad_a")
    check(db, wb, tol_b, "grad_b")
    for c in range(len(a)):
        if not (cn == c).any():
            assert not da[c].any() and not db[c].any()


def sum_tol(p, q, count):
    return lo.sum_error(np.sqrt((p * p).T @ (q * q)), max(count, 1)) if count else np.zeros((p.shape[1], q.shape[1]))


def test_gradient_against_differences(env):
    """d sum(G y) / d theta by central differences of the float64 formula the kernels are checked against."""
    ad, x, codes, gen = make(env, "f32", 70, 24, 20, 4, 3)
    g = env.torch.randn(70, 20, generator=gen).to(env.dev)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    dx, da, db = (np64(t) for t in ad.backward(g, x, codes, hidden))
    w, a, b, scale = weights64(ad)
    cn, x64, g64 = codes.cpu().numpy(), np64(x), np64(g)
    f = lambda x_, a_, b_: (lo.adapters_apply(x_, cn, w, a_, b_, scale)[0] * g64).sum()
    rng = np.random.default_rng(0)
    for _ in range(5):
        # the function is bilinear: a central difference along one argument is exact up to float64 rounding
        for k, (arg, grad) in enumerate(((x64, dx), (a, da), (b, db))):
            step = rng.standard_normal(arg.shape)
            args = [x64, a, b]
            hi, lo_ = list(args), list(args)
            hi[k], lo_[k] = arg + step, arg - step
            want, got = (f(*hi) - f(*lo_)) / 2, (grad * step).sum()
            # each of the gradient's elements is off by at most ~70 * 2^-24 of the size of its terms
            assert abs(got - want) <= 1e-5 * np.abs(grad * step).sum() + 1e-9, (k, got, want)


def test_backward_isolates_and_skips(env):
    """Rows without an adapter, or with a code past the last one, add nothing; their inputs may hold anything."""
    torch = env.torch
    n = 200
    codes = [(i * 11) % 6 - 1 for i in range(n)]  # -1 .. 4 over 4 adapters: code 4 is past the last
    ad, x, codes, gen = make(env, "f32", n, 40, 48, 5, 4, codes=codes)
    g = torch.randn(n, 48, generator=gen).to(env.dev)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    _, da, db = ad.backward(g, x, codes, hidden)
    out = (codes < 0) | (codes >= 4)
    x[out] = float("nan")
    g2 = g.clone()
    g2[out] = float("inf")
    dx2, da2, db2 = ad.backward(g2, x, codes, hidden)
    assert torch.equal(da, da2) and torch.equal(db, db2)
    assert bool(dx2[codes >= 4].isnan().all()) and bool(dx2[~out].isfinite().all())


@pytest.mark.parametrize("n", [0, 1])
def test_empty(env, n):
    torch = env.torch
    ad, x, codes, _ = make(env, "f32", n, 16, 12, 3, 2, codes=[-1] * n)
    y, hidden = ad.apply(x, codes, return_hidden=True)
    assert y.shape == (n, 12) and hidden.shape == (n, 3)
    dx, da, db = ad.backward(torch.ones(n, 12, device=env.dev), x, codes, hidden)
    assert dx.shape == (n, 16) and not da.any() and not db.any()


def test_chunks_of_rows(env):
    """More rows than one pass takes (65 536): the same rows give the same results, and gradients add up over the passes."""
    torch = env.torch
    n = 65536 + 700
    ad, x, codes, gen = make(env, "bf16", n, 64, 64, 4, 6)
    y = ad.apply(x, codes)
    assert torch.equal(y[-700:], ad.apply(x[-700:], codes[-700:]))
    assert torch.equal(y[:65536], ad.apply(x[:65536], codes[:65536]))
    g = torch.randn(n, 64, generator=gen).to(env.dev, x.dtype)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    dx, da, db = ad.backward(g, x, codes, hidden)
    g64, x64, cn = g.double(), x.double(), codes
    for c in range(6):
        at = (cn == c).nonzero()[:, 0]
        m = len(at)
        s = float(ad.scale[c])
        v = g64[at] @ ad.b[c].double()
        want_a, want_b = s * (v.t() @ x64[at]), s * (g64[at].t() @ hidden[at].double())
        size_a = ((v * v).t() @ (x64[at] * x64[at])).sqrt()
        size_b = ((g64[at] ** 2).t() @ (hidden[at].double() ** 2)).sqrt()
        assert bool(((da[c] - want_a).abs() <= s * lo.sum_error(1.0, m + 64) * size_a * 2 + 1e-6 * want_a.abs()).all())
        assert bool(((db[c] - want_b).abs() <= s * lo.sum_error(1.0, m) * size_b + 1e-6 * want_b.abs()).all())


def test_many_adapters(env):
    """The largest stack: more bins than one round of the grouping scan, several digits."""
    torch = env.torch
    s = 16382
    gen = torch.Generator().manual_seed(3)
    codes = torch.randint(-1, s + 1, (5000,), generator=gen)
    ad, x, codes, _ = make(env, "f32", 5000, 16, 8, 2, s, codes=codes)
    check_apply(env, ad, x, codes, "f32")
    _, hidden = ad.apply(x, codes, return_hidden=True)
    g = torch.randn(5000, 8, generator=gen).to(env.dev)
    dx, da, db = ad.backward(g, x, codes, hidden)
    check_backward(ad, g, x, codes, hidden, "f32", dx, da, db)


def test_other_stream_and_graph(env):
    """On a stream of the caller's, and captured: every replay gives what the eager call gives, with eager work between."""
    torch = env.torch
    for n in (5, 300):
        ad, x, codes, gen = make(env, "bf16", n, 128, 96, 8, 5)
        g = torch.randn(n, 96, generator=gen).to(env.dev, x.dtype)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y, hidden = ad.apply(x, codes, return_hidden=True)
            grads = ad.backward(g, x, codes, hidden)
        side.synchronize()
        assert torch.equal(y, ad.apply(x, codes))

        def both():
            y_, h_ = ad.apply(x, codes, return_hidden=True)
            return (y_,) + ad.backward(g, x, codes, h_)

        graphs = []
        for _ in range(2):  # two graphs of the same adapters
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = both()
            graphs.append((graph, outs))
        for turn in range(4):
            x.copy_(torch.randn(n, 128, generator=gen).to(env.dev, x.dtype))
            codes.copy_(torch.randint(-1, 5, (n,), generator=gen).to(env.dev, torch.int32))
            want = both()
            for graph, outs in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for graph, outs in graphs:
                assert all(torch.equal(o, w_) for o, w_ in zip(outs, want)), turn
        del grads


def test_weights_changed_in_place_and_numpy(env):
    torch = env.torch
    ad, x, codes, _ = make(env, "f16", 6, 32, 32, 4, 2)
    before = ad.apply(x, codes)
    ad.b.zero_()
    want = ad.apply(x, torch.full_like(codes, -1))
    assert torch.equal(ad.apply(x, codes), want) and not torch.equal(before, want)
    host = ad.apply(x.float().cpu().numpy(), codes.tolist())
    assert host.dtype == np.float32 and np.array_equal(host, want.float().cpu().numpy())
    fresh = env.hvs.QueryAdapters.create(24, 3, rank=4)
    q = torch.randn(5, 24, device=env.dev)
    assert torch.equal(fresh.apply(q, torch.tensor([0, 1, 2, -1, 1], device=env.dev)), q)


def test_refusals(env):
    torch, hvs = env.torch, env.hvs
    ad, x, codes, _ = make(env, "f32", 6, 32, 24, 4, 2)
    hidden = torch.zeros(6, 4, device=env.dev)
    grad = torch.zeros(6, 24, device=env.dev)
    for bad in (x[:, :31], x.half(), x[0], x.cpu()):
        with pytest.raises(ValueError):
            ad.apply(bad, codes)
    for bad in (codes[:5], codes.float(), codes.cpu(), codes[None], [0.5] * 6):
        with pytest.raises(ValueError):
            ad.apply(x, bad)
    square, xs, cs, _ = make(env, "f32", 6, 32, 32, 4, 2)
    with pytest.raises(hvs.HvsError, match="overlaps"):
        square.apply(xs, cs, out=xs)
    with pytest.raises(ValueError):
        ad.apply(x, codes, out=torch.empty(24, 6, device=env.dev).t())
    with pytest.raises(ValueError):
        ad.apply(x, codes, out=torch.empty(6, 24, device=env.dev, dtype=torch.float16))
    for args in ((grad[:, :3], x, codes, hidden), (grad, x, codes, hidden[:, :2]), (grad, x, codes, hidden.double()), (grad[:3], x, codes, hidden)):
        with pytest.raises(ValueError):
            ad.backward(*args)
    w, a, b, s = ad.projection, ad.a, ad.b, ad.scale
    for bad in ((w, a, b, s.double()), (w, a[:1], b, s), (w.t(), a, b, s), (w, a.half(), b, s), (w, a, b[:, :5].contiguous(), s), (w.cpu(), a, b, s), (w.double(), a.double(), b.double(), s)):
        with pytest.raises(ValueError):
            hvs.QueryAdapters(*bad)
    with pytest.raises(ValueError):
        hvs.QueryAdapters.create(16, 2, rank=129)


@pytest.mark.parametrize("adapters", [510, 511, 1022, 1023, 5000, 16382])
def test_grouping_over_many_bins(env, adapters):
    """Rows of the last and of the first adapters, more bins than a round of the grouping takes: each row comes back to its
    place, with its own adapter, and an adapter's gradient holds its rows alone."""
    torch = env.torch
    for n in (1500, 9000):
        gen = torch.Generator().manual_seed(n)
        pick = torch.tensor([-1, 0, 1, adapters - 2, adapters - 1])
        codes = torch.where(torch.rand(n, generator=gen) < 0.5, pick[torch.randint(0, 5, (n,), generator=gen)], torch.randint(0, adapters, (n,), generator=gen))
        ad, x, codes, _ = make(env, "f32", n, 12, 20, 2, adapters, codes=codes)
        y, hidden = check_apply(env, ad, x, codes, "f32")
        g = torch.randn(n, 20, device=env.dev)
        check_backward(ad, g, x, codes, hidden, "f32", *ad.backward(g, x, codes, hidden))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 30, 1100])
def test_hidden_past_the_largest_number(env, dtype, n):
    """A x beyond fp32: the row's outputs are infinite in the sign of B, on every route; the other tenant's are finite."""
    torch = env.torch
    t = getattr(torch, DT[dtype])
    w, a, b = torch.zeros(24, 64, dtype=t, device=env.dev), torch.ones(2, 3, 64, dtype=t, device=env.dev), torch.ones(2, 24, 3, dtype=t, device=env.dev)
    b[:, ::2] = -1
    codes = torch.arange(n, device=env.dev, dtype=torch.int32) % 2
    x = torch.where(codes[:, None] == 0, 3e38, 1.0).expand(n, 64).to(t)
    y, hidden = env.hvs.QueryAdapters(w, a, b, torch.ones(2, device=env.dev)).apply(x.contiguous(), codes, return_hidden=True)
    sign = torch.ones(24, device=env.dev)
    sign[::2] = -1
    assert bool((hidden[0::2] == torch.inf).all()) and bool((hidden[1::2] == 64).all())
    assert torch.equal(y[0::2].float(), (sign * torch.inf).expand(len(y[0::2]), 24)) and torch.equal(y[1::2].float(), (sign * 192).expand(len(y[1::2]), 24))


@pytest.mark.parametrize("n", [3, 2000])
def test_scale_that_is_not_finite_without_rows(env, n):
    """An adapter without rows has zero gradients, whatever its scale is."""
    torch = env.torch
    codes = torch.zeros(n, dtype=torch.int32)
    ad, x, codes, gen = make(env, "f32", n, 40, 24, 4, 3, codes=codes)
    ad.scale[1], ad.scale[2] = torch.nan, torch.inf
    g = torch.randn(n, 24, generator=gen).to(env.dev)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    _, da, db = ad.backward(g, x, codes, hidden)
    assert not da[1:].any() and not db[1:].any() and bool(da[0].isfinite().all()) and bool(db[0].isfinite().all())


@pytest.mark.parametrize("n", [20, 1100])
def test_hidden_near_the_ends_of_the_range(env, n):
    """A x of 2^127.5 and of 2^-100, with weights that bring y back to ordinary size."""
    torch = env.torch
    for big, scale in ((2.0**120, 2.0**-90), (2.0**-100, 2.0**100)):
        x = torch.full((n, 64), big, dtype=torch.bfloat16, device=env.dev)
        a = torch.full((1, 1, 64), 2.82, dtype=torch.bfloat16, device=env.dev)
        b = torch.full((1, 16, 1), 1.5 * 2.0**-40, dtype=torch.bfloat16, device=env.dev) if big > 1 else torch.full((1, 16, 1), 1.5, dtype=torch.bfloat16, device=env.dev)
        w = torch.zeros(16, 64, dtype=torch.bfloat16, device=env.dev)
        y = env.hvs.QueryAdapters(w, a, b, torch.full((1,), scale, device=env.dev)).apply(x, torch.zeros(n, dtype=torch.int32, device=env.dev))
        want = scale * np64(b).max() * 64 * big * np64(a).max()
        assert np.abs(np64(y) - want).max() <= (2.0**-8 + 2.0**-15) * want, (big, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graph_of_many_rows(env, dtype):
    """The grouped routes, captured: counted by the blocks themselves (3000 rows) and by a launch of its own (17 000)."""
    torch = env.torch
    for n, adapters in ((3000, 5), (17000, 600)):
        ad, x, codes, gen = make(env, dtype, n, 48, 40, 4, adapters)
        g = torch.randn(n, 40, generator=gen).to(env.dev, x.dtype)

        def both():
            y_, h_ = ad.apply(x, codes, return_hidden=True)
            return (y_,) + ad.backward(g, x, codes, h_)

        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        for turn in range(4):
            x.copy_(torch.randn(n, 48, generator=gen).to(env.dev, x.dtype))
            codes.copy_(torch.randint(-1, adapters, (n,), generator=gen).to(env.dev, torch.int32))
            want = both()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w_) for o, w_ in zip(outs, want)), turn


def test_two_streams_at_once(env):
    """Calls of one object on two streams, each with scratch memory of its own, give what they give one after the other."""
    torch = env.torch
    ad, x, codes, gen = make(env, "bf16", 6000, 256, 256, 8, 30)
    parts = [(x[:4000], codes[:4000]), (x[1000:], codes[1000:]), (x[:100], codes[:100])]
    g = torch.randn(6000, 256, generator=gen).to(env.dev, x.dtype)

    def step(part):
        xp, cp = part
        y, h = ad.apply(xp, cp, return_hidden=True)
        return (y,) + ad.backward(g[: len(xp)], xp, cp, h)

    want = [step(p) for p in parts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    got = [None] * len(parts)
    for _ in range(5):
        for k, (stream, part) in enumerate(zip(streams, parts)):
            with torch.cuda.stream(stream):
                got[k] = step(part)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_offsets_past_32_bits(env):
    """Rows of a wide tensor, so far apart that the last ones lie past 2^32 bytes and 2^31 elements."""
    torch = env.torch
    n, width = 5000, 450000
    wide = torch.empty(n, width, dtype=torch.float16, device=env.dev)
    ad, x, codes, gen = make(env, "f16", n, 72, 40, 4, 5)
    strided = wide[:, :72]
    strided.copy_(x)
    out = wide[:, -40:]
    assert strided.stride(0) == width and n * width > 2**31
    want, hidden = ad.apply(x, codes, return_hidden=True)
    y, h = ad.apply(strided, codes, return_hidden=True)
    # passes of other sizes may take other routes: both are right to their own last bits
    check_apply(env, ad, x, codes, "f16")
    want64, tol, u, u_tol = lo.adapters_apply_tolerance(np64(x), codes.cpu().numpy(), *weights64(ad), "f16")
    check(y, want64, tol, "y")
    check(h, u, u_tol, "hidden")
    g = torch.randn(n, 40, generator=gen).to(env.dev, x.dtype)
    out.copy_(g)
    check_backward(ad, g, x, codes, hidden, "f16", *ad.backward(out, strided, codes, hidden))
    few = ad.apply(strided[-3:], codes[-3:])
    check(few, want64[-3:], tol[-3:], "last rows")


def test_tensors_that_require_gradients(env):
    """Parameters and views are taken as the numbers they hold; no graph is recorded."""
    torch = env.torch
    ad, x, codes, _ = make(env, "f32", 33, 40, 24, 4, 3)
    par = env.hvs.QueryAdapters(ad.projection, torch.nn.Parameter(ad.a), torch.nn.Parameter(ad.b), ad.scale)
    xp = torch.nn.Parameter(x)
    y = par.apply(xp, codes)
    assert not y.requires_grad and torch.equal(y, ad.apply(x, codes))
    assert torch.equal(par.apply(x.t().contiguous().t(), codes), y) and torch.equal(par.apply(x[:1].expand(33, 40), codes), ad.apply(x[:1].repeat(33, 1), codes))
    assert torch.equal(par.apply(x.flip(0), codes.flip(0)), y.flip(0))


@pytest.mark.parametrize("n", [1, 40, 2000])
def test_columns_of_one_tensor(env, n):
    """Input and output side by side in one tensor are apart; a column in common, or other pitches over the same range, is not."""
    torch = env.torch
    ad, x, codes, gen = make(env, "f32", n, 24, 20, 4, 3)
    want, tol, _, _ = lo.adapters_apply_tolerance(np64(x), codes.cpu().numpy(), *weights64(ad), "f32")
    for x_at, out_at in ((0, 24), (20, 0), (1, 27)):
        wide = torch.zeros(n, 48, device=env.dev)
        wide[:, x_at : x_at + 24] = x
        got = ad.apply(wide[:, x_at : x_at + 24], codes, out=wide[:, out_at : out_at + 20])
        check(got, want, tol, "y")
        assert torch.equal(wide[:, x_at : x_at + 24], x)
        assert not wide[:, max(x_at + 24, out_at + 20) :].any()
    wide = torch.zeros(n + 1, 48, device=env.dev)
    for x_at, out_at in ((0, 23), (19, 0), (4, 4)):
        with pytest.raises(env.hvs.HvsError, match="overlaps"):
            ad.apply(wide[:n, x_at : x_at + 24], codes, out=wide[:n, out_at : out_at + 20])
    if n > 1:
        with pytest.raises(env.hvs.HvsError, match="overlaps"):
            ad.apply(wide[:n, :24], codes, out=wide.view(-1)[24 : 24 + n * 20].view(n, 20))


@pytest.mark.parametrize("dtype,n,d_in,d_out", [("bf16", 300, 90, 3333), ("bf16", 301, 3400, 100), ("f16", 130, 72, 8200), ("f32", 600, 100, 3300), ("f32", 500, 4001, 130),
                                                ("f16", 1024, 64, 900), ("f32", 1024, 64, 1800), ("bf16", 65, 40, 16384)])
def test_routes_by_outputs(env, dtype, n, d_in, d_out):
    """Row counts that one direction takes in arrival order and the other grouped."""
    torch = env.torch
    ad, x, codes, gen = make(env, dtype, n, d_in, d_out, 6, 4)
    _, hidden = check_apply(env, ad, x, codes, dtype)
    g = torch.randn(n, d_out, generator=gen).to(env.dev, x.dtype)
    check_backward(ad, g, x, codes, hidden, dtype, *ad.backward(g, x, codes, hidden))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 30, 1100, 17000])
@pytest.mark.parametrize("rank", [3, 16, 20])
def test_infinite_rows_at_any_rank(env, dtype, n, rank):
    """A row with an infinite element: with positive weights every sum is +inf and none is NaN, whatever the rank is a multiple of;
    the other rows are what they are without it.  The same for a row of the gradient."""
    torch = env.torch
    t = getattr(torch, DT[dtype])
    gen = torch.Generator().manual_seed(n + rank)
    pos = lambda *s: (0.1 + torch.rand(*s, generator=gen)).to(env.dev, t)
    ad = env.hvs.QueryAdapters(pos(40, 64), pos(2, rank, 64), pos(2, 40, rank), torch.ones(2, device=env.dev))
    x, g = pos(n, 64), pos(n, 40)
    codes = torch.arange(n, device=env.dev, dtype=torch.int32) % 2
    y, hidden = ad.apply(x, codes, return_hidden=True)
    dx, _, _ = ad.backward(g, x, codes, hidden)
    bad = n // 2
    x2, g2 = x.clone(), g.clone()
    x2[bad, 5], g2[bad, 7] = torch.inf, torch.inf
    y2, hidden2 = ad.apply(x2, codes, return_hidden=True)
    dx2, _, _ = ad.backward(g2, x, codes, hidden)
    others = torch.arange(n, device=env.dev) != bad
    for got, clean in ((y2, y), (hidden2, hidden), (dx2, dx)):
        assert bool((got[bad] == torch.inf).all())
        assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("d_in,d_out,rank", [(16384, 64, 33), (64, 16384, 65)])
def test_transposed_weights_past_one_launch(env, d_in, d_out, rank):
    """Stacks whose transposed copies take more tiles than a launch has (2^18): 256 for each of 1030 adapters."""
    torch = env.torch
    n, s = 40, 1030
    gen = torch.Generator(device=env.dev).manual_seed(1)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=env.dev, dtype=torch.float32)
    used = torch.tensor([0, 1, 500, 1022, 1023, 1024, 1028, 1029], device=env.dev)
    w = (rnd(d_out, d_in) / d_in**0.5).bfloat16()
    a, b = torch.zeros(s, rank, d_in, dtype=torch.bfloat16, device=env.dev), torch.zeros(s, d_out, rank, dtype=torch.bfloat16, device=env.dev)
    a[used], b[used] = (rnd(len(used), rank, d_in) / d_in**0.5).bfloat16(), (rnd(len(used), d_out, rank) / rank**0.5).bfloat16()
    scale = 0.5 + torch.rand(s, generator=gen, device=env.dev)
    place = torch.arange(n, device=env.dev) % len(used)
    codes, x, g = used[place].to(torch.int32), rnd(n, d_in).bfloat16(), rnd(n, d_out).bfloat16()
    ad = env.hvs.QueryAdapters(w, a, b, scale)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    dx, da, db = ad.backward(g, x, codes, hidden)
    # the same rows over the used adapters alone, which fit one launch
    small = env.hvs.QueryAdapters(w, a[used].contiguous(), b[used].contiguous(), scale[used].contiguous())
    want = small.backward(g, x, place.to(torch.int32), hidden)
    assert torch.equal(dx, want[0]) and torch.equal(da[used], want[1]) and torch.equal(db[used], want[2])
    check_backward(small, g, x, place.to(torch.int32), hidden, "bf16", *want)
    da[used], db[used] = 0, 0
    assert not da.any() and not db.any()


@pytest.mark.parametrize("name", ["projection", "a", "b", "scale"])
def test_weights_put_in_anothers_place(env, name):
    """A tensor like the old one takes its place; one that the kernels would read wrongly, or past its end, is refused."""
    torch = env.torch
    ad, x, codes, gen = make(env, "f32", 30, 24, 24, 24, 24)
    _, hidden = ad.apply(x, codes, return_hidden=True)
    g = torch.randn(30, 24, generator=gen).to(env.dev)
    old = getattr(ad, name)
    setattr(ad, name, old * 2)
    check_apply(env, ad, x, codes, "f32")
    old2 = getattr(ad, name)
    old2.data = old2.data * 0.5
    assert torch.equal(ad.apply(x, codes), env.hvs.QueryAdapters(*[old if k == name else getattr(ad, k) for k in ("projection", "a", "b", "scale")]).apply(x, codes))
    bad = [old.half(), old.bfloat16(), old[:-1], old.cpu(), torch.cat([old, old]), old.double(), None]
    if old.dim() > 1:
        bad += [old.transpose(-1, -2), old.reshape(-1)]
    want = ad.apply(x, codes)
    for t in bad:
        with pytest.raises(ValueError):
            setattr(ad, name, t)
        assert torch.equal(ad.apply(x, codes), want)
    for t in (old.half(), old[:-1].clone(), old.expand(2, *old.shape).reshape(-1)):
        old2.data = t
        with pytest.raises(ValueError, match="must stay"):
            ad.apply(x, codes)
        with pytest.raises(ValueError, match="must stay"):
            ad.backward(g, x, codes, hidden)
    old2.data = old.clone()
    assert torch.equal(ad.apply(x, codes), want)
