"""CPU tier: the learning operators' C ABI (layout, refusals before any GPU call), their oracle against differences, and the
store's use of query adapters."""

import asyncio
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from oracle import learn_oracle as lo
from tests import store_cases
from tests.fake_index import OracleIndex

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structs_match_the_header(tmp_path):
    from hirag_prod_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    structs = {"hvs_adapters": _lib.HvsAdaptersStruct, "hvs_preference": _lib.HvsPreferenceStruct, "hvs_tensor": _lib.HvsTensorStruct}
    body = "".join(f'printf("{n} %zu\\n", sizeof({n}));' + "".join(f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_)
                   for n, s in structs.items())
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "hvs.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")])
    got = dict(line.split() for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines())
    for n, s in structs.items():
        assert int(got[n]) == ctypes.sizeof(s), n
        for f, _ in s._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(s, f).offset, (n, f)
    text = open(os.path.join(ROOT, "include", "hvs.h")).read()
    for name in ("HVS_MAX_ADAPTER_DIM", "HVS_MAX_ADAPTER_RANK", "HVS_MAX_ADAPTERS"):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_lib, name)


# addresses that are never followed: the calls below are refused before anything is launched
P, Q, R, W = 1 << 20, 1 << 24, 1 << 28, 1 << 32


def adapters(**kw):
    from hirag_prod_amd._lib import HvsAdaptersStruct

    fields = dict(projection=P, a=P, b=P, scale=P, dtype=0, d_in=32, d_out=24, rank=4, n_adapters=3)
    fields.update(kw)
    return HvsAdaptersStruct(**fields)


def refused(rc, match):
    import hirag_prod_amd as hvs

    message = hvs.load_library().hvs_last_error().decode()
    assert rc != 0 and re.search(match, message), (rc, message)


@pytest.mark.parametrize("kw,match", [(dict(dtype=7), "dtype"), (dict(d_in=0), "sides"), (dict(d_out=16385), "sides"), (dict(rank=0), "rank"), (dict(rank=129), "rank"),
                                      (dict(n_adapters=0), "adapters"), (dict(n_adapters=16383), "adapters")])
def test_adapters_are_checked(kw, match):
    import hirag_prod_amd as hvs

    lib, ad, need = hvs.load_library(), adapters(**kw), ctypes.c_uint64(0)
    refused(lib.hvs_adapters_workspace(ctypes.byref(ad), 5, 32, 0, ctypes.byref(need)), match)
    refused(lib.hvs_adapters_apply(0, None, ctypes.byref(ad), P, 32, P, 5, Q, 24, None, W, 1 << 30), match)
    refused(lib.hvs_adapters_backward(0, None, ctypes.byref(ad), P, 24, P, 32, P, P, 5, Q, 32, P, P, W, 1 << 30), match)


def test_adapters_calls_are_refused():
    import hirag_prod_amd as hvs

    lib, ad = hvs.load_library(), adapters()
    ref = ctypes.byref(ad)
    ok = dict(x=P, ld_x=32, codes=P, n=5, out=Q, ld_out=24, hidden=None, ws=W, size=1 << 30)

    def apply(ad_ref=ref, **kw):
        a = {**ok, **kw}
        return lib.hvs_adapters_apply(0, None, ad_ref, a["x"], a["ld_x"], a["codes"], a["n"], a["out"], a["ld_out"], a["hidden"], a["ws"], a["size"])

    refused(apply(ad_ref=None), "NULL")
    refused(apply(n=-1), "negative")
    assert apply(n=0, x=None, out=None, codes=None, ws=None, size=0) == 0
    for kw, match in ((dict(x=None), "x is NULL"), (dict(out=None), "out is NULL"), (dict(codes=None), "codes"), (dict(ld_x=31), "pitch"), (dict(ld_out=23), "pitch"),
                      (dict(x=P + 2), "aligned"), (dict(out=Q + 1), "aligned"), (dict(out=P), "overlaps"), (dict(out=P + 32 * 4 * 4), "overlaps"),
                      (dict(ws=None), "workspace"), (dict(ws=W + 8), "workspace"), (dict(size=16), "workspace"), (dict(ld_x=1 << 30), "2 GB")):
        refused(apply(**kw), match)
    for field in ("projection", "a", "b", "scale"):
        refused(apply(ad_ref=ctypes.byref(adapters(**{field: None}))), "weight")
    refused(apply(ad_ref=ctypes.byref(adapters(scale=P + 1))), "aligned")

    ok_b = dict(grad=P, ld_grad=24, x=Q, ld_x=32, codes=P, hidden=P, n=5, gx=R, ld_gx=32, ga=P, gb=P, ws=W, size=1 << 30)

    def backward(**kw):
        a = {**ok_b, **kw}
        return lib.hvs_adapters_backward(0, None, ref, a["grad"], a["ld_grad"], a["x"], a["ld_x"], a["codes"], a["hidden"], a["n"], a["gx"], a["ld_gx"], a["ga"],
                                         a["gb"], a["ws"], a["size"])

    for kw, match in ((dict(n=-1), "negative"), (dict(grad=None), "grad is NULL"), (dict(x=None), "x is NULL"), (dict(hidden=None), "hidden"), (dict(codes=None), "codes"),
                      (dict(ga=None), "grad_a"), (dict(gb=None), "grad_b"), (dict(ga=P + 2), "aligned"), (dict(gx=P), "overlaps"), (dict(gx=Q), "overlaps"),
                      (dict(ld_gx=31), "pitch"), (dict(ws=None), "workspace"), (dict(size=1), "workspace")):
        refused(backward(**kw), match)


def test_workspace_grows_with_the_rows_of_a_pass_only():
    import hirag_prod_amd as hvs

    lib, ad = hvs.load_library(), adapters(d_in=1536, d_out=1536, rank=16)
    size = {}
    for n in (0, 1, 2, 3, 64, 4096, 65536, 10**6, 10**9):
        for backward in (0, 1):
            need = ctypes.c_uint64(0)
            assert lib.hvs_adapters_workspace(ctypes.byref(ad), n, 1536, backward, ctypes.byref(need)) == 0
            size[n, backward] = need.value
    assert size[0, 0] == size[1, 0] == size[2, 0] == 0 < size[3, 0] < size[4096, 0] < size[65536, 0] == size[10**6, 0] == size[10**9, 0]
    assert size[65536, 1] == size[10**9, 1] > size[65536, 0]


def test_preference_calls_are_refused():
    import hirag_prod_amd as hvs
    from hirag_prod_amd._lib import HvsPreferenceStruct

    lib = hvs.load_library()
    ok = dict(queries=P, ld_queries=16, reference=None, ld_reference=0, offsets=P, chosen=P, rejected=P, weights=None, loss=R, margin=R, grad=Q, ld_grad=16, n_queries=4,
              n_pairs=9, query_dtype=0, beta=2.0, label_smoothing=0.0)

    def call(rows=R, dtype=1, dim=16, ld=16, n_rows=50, **kw):
        p = HvsPreferenceStruct(**{**ok, **kw})
        return lib.hvs_preference_loss(0, None, ctypes.byref(p), rows, dtype, dim, ld, n_rows, W, 1 << 30)

    for kw, match in ((dict(dtype=3), "dtype"), (dict(query_dtype=-1), "dtype"), (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(n_queries=-1), "negative"),
                      (dict(n_pairs=-1), "negative"), (dict(beta=0.0), "beta"), (dict(beta=float("nan")), "beta"), (dict(beta=float("inf")), "beta"),
                      (dict(label_smoothing=0.51), "smoothing"), (dict(label_smoothing=float("nan")), "smoothing"), (dict(queries=None), "NULL"), (dict(grad=None), "NULL"),
                      (dict(offsets=None), "NULL"), (dict(chosen=None), "NULL"), (dict(loss=None), "NULL"), (dict(rows=None), "rows"), (dict(n_rows=-1), "rows"),
                      (dict(ld_queries=15), "pitch"), (dict(ld=15), "pitch"), (dict(reference=P, ld_reference=3), "pitch"), (dict(queries=P + 2), "aligned"),
                      (dict(rows=R + 1), "aligned"), (dict(grad=P), "overlaps"), (dict(reference=Q, ld_reference=16), "overlaps"), (dict(n_queries=0), "no query")):
        try:
            refused(call(**kw), match)
        except AssertionError as e:
            raise AssertionError(f"{kw}: {e}") from None
    assert call(n_queries=0, n_pairs=0) == 0
    p = HvsPreferenceStruct(**ok)
    refused(lib.hvs_index_preference_loss(None, None, ctypes.byref(p), None, 0), "NULL")
    refused(lib.hvs_preference_loss(0, None, None, R, 1, 16, 16, 50, None, 0), "NULL")


def test_clip_calls_are_refused():
    import hirag_prod_amd as hvs
    from hirag_prod_amd._lib import HvsTensorStruct

    lib = hvs.load_library()

    def call(entries, max_norm=1.0, norm=R, ws=W, size=1 << 30):
        t = (HvsTensorStruct * max(len(entries), 1))(*entries)
        return lib.hvs_clip_grad_norm(0, None, t, len(entries), max_norm, 0, norm, ws, size)

    one = (P, P, 100, 0)
    for entries, kw, match in (([(P, P, 100, 9)], {}, "dtype"), ([(P, P, -1, 0)], {}, "elements"), ([(None, P, 5, 0)], {}, "NULL"), ([(P, None, 5, 0)], {}, "NULL"),
                               ([(P + 2, P + 2, 5, 0)], {}, "aligned"), ([(P, P + 40, 100, 0)], {}, "overlaps"), ([one, one], {}, "share"),
                               ([one, (P + 396, P + 396, 3, 0)], {}, "share"), ([(P, Q, 100, 0), (Q, Q, 100, 0)], {}, "share"), ([one], dict(max_norm=-0.5), "max_norm"),
                               ([one], dict(max_norm=float("nan")), "max_norm"), ([one], dict(norm=None), "norm"), ([one], dict(ws=None), "workspace"),
                               ([one], dict(ws=W + 4), "workspace"), ([one], dict(size=7), "workspace")):
        refused(call(entries, **kw), match)


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(3)
    n, d_in, d_out, r, s = 7, 6, 5, 2, 3
    x, w = rng.standard_normal((n, d_in)), rng.standard_normal((d_out, d_in))
    a, b, scale = rng.standard_normal((s, r, d_in)), rng.standard_normal((s, d_out, r)), rng.random(s) + 0.5
    codes = np.array([0, 1, 2, -1, 0, 2, 2])
    g = rng.standard_normal((n, d_out))
    f = lambda x_, a_, b_: (lo.adapters_apply(x_, codes, w, a_, b_, scale)[0] * g).sum()
    hidden = lo.adapters_apply(x, codes, w, a, b, scale)[2]
    grads = lo.adapters_backward(g, x, codes, hidden, w, a, b, scale)[:3]
    for k, (arg, grad) in enumerate(zip((x, a, b), grads)):
        step = rng.standard_normal(arg.shape)
        hi, lw = [x, a, b], [x, a, b]
        hi[k], lw[k] = arg + step, arg - step  # bilinear: exact
        assert abs((f(*hi) - f(*lw)) / 2 - (grad * step).sum()) < 1e-10
    q, rows, ref = rng.standard_normal((3, 4)), rng.standard_normal((9, 4)), rng.standard_normal((3, 4))
    c, rej, off = rng.integers(0, 9, 6), rng.integers(0, 9, 6), np.array([0, 2, 2, 6])
    wt = rng.random(6)
    grad = lo.preference(q, rows, c, rej, off, ref, 3.0, 0.2, wt)[2]
    f = lambda q_: (lo.preference(q_, rows, c, rej, off, ref, 3.0, 0.2, wt)[0] * wt).sum()
    step, h = rng.standard_normal(q.shape), 1e-5
    assert abs((f(q + h * step) - f(q - h * step)) / (2 * h) - (grad * step).sum()) < 1e-8


class PlainAdapters:
    """Stands in for QueryAdapters on the CPU: adapter c turns the embedding by c + 1 places."""

    def __init__(self, dim, n_adapters):
        self.d_in, self.n_adapters, self.calls = dim, n_adapters, []

    def apply(self, x, codes):
        assert x.dtype == np.float32 and len(x) == len(codes)
        self.calls.append(list(codes))
        return np.stack([np.roll(v, c + 1) for v, c in zip(x, codes)])


@pytest.mark.parametrize("coalesce", [True, False])
def test_store_sends_queries_through_the_adapters(coalesce):
    import hirag_prod_amd.store as st

    def make():
        return st.HipVectorStore.create(store_cases.make_embedding_func(), vector_type="vector", coalesce_queries=coalesce,
                                        index_factory=lambda dim, dtype, device: OracleIndex(dim, dtype, device))

    async def scenario():
        s = make()
        tenants = [("ws1", "kb1"), ("ws1", "kb2"), ("ws2", "kb1")]
        for w, k in tenants:
            props = [store_cases.chunk_props(i, w, k) for i in range(12)]
            await s.upsert_texts([p["text"] for p in props], props, "Chunks")
        ask = lambda i, w, k: s.query([f"question {i}", f"variant {i}"] if i % 2 else f"question {i}", w, k, "Chunks", topk=6, topn=3, distance_threshold=3.0)
        plain = [await ask(0, w, k) for w, k in tenants]
        ad = PlainAdapters(store_cases.DIM, 2)
        s.set_query_adapters(ad, {("ws1", "kb1"): 0, ("ws2", "kb1"): 1})
        got = await asyncio.gather(*[ask(i, w, k) for i in range(4) for w, k in tenants])
        if coalesce:
            assert len(ad.calls) == 1 and sorted(set(ad.calls[0])) == [-1, 0, 1]  # all tenants' requests in one call
        else:
            assert len(ad.calls) == 12
        shift = {("ws1", "kb1"): 1, ("ws1", "kb2"): 0, ("ws2", "kb1"): 2}
        for n, (i, (w, k)) in enumerate([(i, t) for i in range(4) for t in tenants]):
            texts = [f"question {i}", f"variant {i}"] if i % 2 else [f"question {i}"]
            qs = [np.roll(store_cases.embed_text(t), shift[w, k]) for t in texts]
            rows = [store_cases.embed_text(f"text {w} {k} {j}") for j in range(12)]
            dist = np.array([min(1 - q @ r / np.linalg.norm(q) / np.linalg.norm(r) for q in qs) for r in rows])
            order = np.argsort(dist, kind="stable")[:6]
            store_cases.same_hits([h["documentKey"] for h in got[n]], [f"chunk-{w}-{k}-{j}" for j in order], dist[order], [h["distance"] for h in got[n]])
        s.set_query_adapters(None)
        assert [[h["documentKey"] for h in await ask(0, w, k)] for w, k in tenants] == [[h["documentKey"] for h in p] for p in plain]
        with pytest.raises(ValueError, match="adapter number"):
            s.set_query_adapters(ad, {("ws1", "kb1"): 2})
        s.set_query_adapters(PlainAdapters(5, 1))
        with pytest.raises(ValueError, match="columns"):
            await ask(0, "ws1", "kb1")

    asyncio.run(scenario())


def test_lists_off_their_elements_and_wide_pitches_are_refused():
    import hirag_prod_amd as hvs
    from hirag_prod_amd._lib import HvsPreferenceStruct

    lib, ad, need = hvs.load_library(), adapters(), ctypes.c_uint64(0)
    apply = lambda codes, hidden: lib.hvs_adapters_apply(0, None, ctypes.byref(ad), P, 64, codes, 3, Q, 64, hidden, W, 1 << 30)
    back = lambda codes, hidden: lib.hvs_adapters_backward(0, None, ctypes.byref(ad), P, 64, P, 64, codes, hidden, 3, None, 0, Q, R, W, 1 << 30)
    for call in (apply, back):
        refused(call(R + 2, R), "aligned")
        refused(call(R, R + 1), "aligned")
    for wide in (1 << 31, 1 << 62):
        refused(lib.hvs_adapters_workspace(ctypes.byref(ad), 5, wide, 0, ctypes.byref(need)), "pitch")
    ok = dict(queries=P, ld_queries=16, reference=None, ld_reference=0, offsets=P, chosen=P, rejected=P, weights=P, loss=R, margin=R, grad=Q, ld_grad=16, n_queries=4,
              n_pairs=9, query_dtype=0, beta=2.0, label_smoothing=0.0)
    for name, off in (("offsets", 4), ("chosen", 4), ("rejected", 1), ("weights", 2), ("loss", 2), ("margin", 1)):
        p = HvsPreferenceStruct(**{**ok, name: ok[name] + off})
        refused(lib.hvs_preference_loss(0, None, ctypes.byref(p), R, 1, 16, 16, 50, W, 1 << 30), "aligned")


def preference_case(dim, counts, seed, n_rows=50):
    rng = np.random.default_rng(seed)
    rows = rng.standard_normal((n_rows, dim)).astype(np.float16).astype(np.float64)
    q = rng.standard_normal((len(counts), dim)).astype(np.float32).astype(np.float64)
    ref = (q + 0.2 * rng.standard_normal(q.shape)).astype(np.float32).astype(np.float64)
    off = np.concatenate([[0], np.cumsum(counts)])
    c, r = rng.integers(0, n_rows, off[-1]), rng.integers(0, n_rows, off[-1])
    return q, rows, c, r, off, ref, rng.random(off[-1])


@pytest.mark.parametrize("dim", [2, 768, 8193, 16384])
@pytest.mark.parametrize("counts", [[9], [16], [17], [500], [40, 0, 33], [3] * 70])
def test_gradient_tolerance_refuses_wrong_gradients(dim, counts):
    """The tolerance that the GPU tests hold gradients to is no gradient's size: for every query with a gradient, nothing, the
    negative, half and 1.1 times of it are outside, and so is the gradient without one of the query's pairs."""
    q, rows, c, r, off, ref, w = preference_case(dim, counts, dim + len(counts))
    _, _, grad, _ = lo.preference(q, rows, c, r, off, ref, 10.0, 0.0, w)
    _, _, tol = lo.preference_tolerance(q, rows, c, r, off, ref, 10.0, 0.0, w, "f32")
    c2 = c.copy()
    c2[off[:-1][np.array(counts) > 0]] = -1
    without = lo.preference(q, rows, c2, r, off, ref, 10.0, 0.0, w)[2]
    for k in range(len(counts)):
        if grad[k].any():
            for wrong in (0 * grad[k], -grad[k], 0.5 * grad[k], 1.1 * grad[k], without[k]):
                # (the first pair may name one row twice, and have no gradient)
                assert np.array_equal(wrong, grad[k]) or (np.abs(wrong - grad[k]) > tol[k]).any(), (dim, k)


f4 = np.float32


def tree_dot(a, b):
    """fp32 sum of products over the last axis, added up as the kernel does: 8 elements a lane, 64 lanes, then in pairs."""
    t = a.astype(np.float64) * b.astype(np.float64)  # exact: one rounding at the addition
    t = np.concatenate([t, np.zeros(t.shape[:-1] + ((-t.shape[-1]) % 512,))], -1).reshape(*t.shape[:-1], -1, 64, 8)
    acc = np.zeros(t.shape[:-3] + (64,), f4)
    for c in range(t.shape[-3]):
        for e in range(8):
            acc = (acc + t[..., c, :, e]).astype(f4)
    while acc.shape[-1] > 1:
        acc = acc[..., 0::2] + acc[..., 1::2]
    return acc[..., 0]


def fma(a, b, c):
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(f4)


def margin_forms(q, ref, c, r):
    """The margin in fp32: as the kernel takes it, as two differences of cosines, and from fp32 unit vectors."""
    inv = lambda v: f4(1) / np.sqrt(tree_dot(v, v))[:, None]
    inv64 = lambda v: 1 / np.sqrt((v.astype(np.float64) ** 2).sum(-1, keepdims=True))
    iy, i0 = inv64(q), inv64(ref)
    hy, h0 = iy.astype(f4), i0.astype(f4)
    f = ref * h0
    d = fma(q, hy, -f) + (fma(q, (iy - hy).astype(f4), -fma(ref, h0, -f)) - ref * (i0 - h0).astype(f4))
    kernel = tree_dot(d, fma(c, inv(c), -(r * inv(r))))
    cu, ru, yu, zu = (v * inv(v) for v in (c, r, q, ref))
    return kernel, (tree_dot(yu, cu) - tree_dot(yu, ru)) - (tree_dot(zu, cu) - tree_dot(zu, ru)), tree_dot(yu - zu, cu - ru)


def near_queries(rng, rows, c, off, move, t):
    """A reference near every query's first chosen row, and a query of another length that has moved a little."""
    base = (rows[c[off[:-1]]] + 0.3 * rng.standard_normal((len(off) - 1, rows.shape[1]))) * 3.7
    return (base * 1.3 + move * rng.standard_normal(base.shape)).astype(t), base.astype(t)


@pytest.mark.parametrize("move", [1e-2, 1e-3])
@pytest.mark.parametrize("t", [np.float32, np.float16])
@pytest.mark.parametrize("dim,counts", [(1536, [16]), (1536, [3] * 300), (768, [100, 2, 90]), (4000, [5] * 9), (9000, [4] * 5)])
def test_margin_tolerance_refuses_plain_forms(move, t, dim, counts):
    """What margins next to the reference are held to: the kernel's formula in fp32 stays far within, the plain fp32 forms do not."""
    rng = np.random.default_rng(dim + len(counts))
    rows = rng.standard_normal((90, dim)).astype(np.float16).astype(f4)
    off = np.concatenate([[0], np.cumsum(counts)])
    c, r = rng.integers(0, 90, off[-1]), rng.integers(0, 90, off[-1])
    q, ref = (v.astype(f4) for v in near_queries(rng, rows, c, off, move, t))
    own, apart = np.repeat(np.arange(len(counts)), counts), c != r
    args = (q.astype(float), rows.astype(float), c, r, off, ref.astype(float), 10.0, 0.0, None)
    want, tol = lo.preference(*args)[1], lo.preference_tolerance(*args, "f32")[1]
    kernel, cosines, units = (np.abs(m - want)[apart] / tol[apart] for m in margin_forms(q[own], ref[own], rows[c], rows[r]))
    assert kernel.max() < 0.25 and cosines.max() > 2 and units.max() > 2, (kernel.max(), cosines.max(), units.max())


@pytest.mark.parametrize("weight", ["projection", "a", "b", "scale"])
def test_what_is_written_is_no_weight(weight):
    import hirag_prod_amd as hvs

    lib = hvs.load_library()
    size = dict(projection=32 * 24 * 4, a=3 * 4 * 32 * 4, b=3 * 24 * 4 * 4, scale=12)[weight]
    ad = adapters(**{weight: R})
    apply = lambda out: lib.hvs_adapters_apply(0, None, ctypes.byref(ad), 2 * R, 32, P, 5, out, 24, None, None, 0)
    back = lambda gx: lib.hvs_adapters_backward(0, None, ctypes.byref(ad), 2 * R, 24, 3 * R, 32, P, P, 5, gx, 32, Q, Q, None, 0)
    for call, row in ((apply, 24 * 4), (back, 32 * 4)):
        for at in (R, R + size - 4, R - 5 * row + 4):
            refused(call(at), "overlaps the weights")
        for at in (R + size, R - 5 * row):  # next to it; only the workspace is missing
            refused(call(at), "workspace")
