"""Float64 statements of the learning operators (query adapters, preference loss, clipping) and the error their fp32 sums may
carry.  Test infrastructure: plain loops over adapters, queries and pairs, nothing shared with the kernels."""

from __future__ import annotations

import numpy as np

HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # relative error of one rounding to the type
TINY = {"f32": 2.0**-150, "f16": 2.0**-25, "bf16": 2.0**-134}     # half the spacing of its subnormal numbers


def sum_error(norm_of_terms, count):
    """What an fp32 sum of ``count`` products may be off by, given sqrt(sum of squared terms).  Partial sums of terms of
    mixed signs stay within 4 norms, each of the ``count`` additions rounds by 2^-24 of one, and independent roundings add
    up like sqrt(count); twice that."""
    return 8.0 * np.sqrt(count) * 2.0**-24 * norm_of_terms


def adapters_apply(x, codes, w, a, b, scale):
    """-> (y, norm): y float64 [n, d_out] and the root of the sum of squared terms behind each element."""
    y = x @ w.T
    sq = (x * x) @ (w * w).T
    u = np.zeros((len(x), a.shape[1]))
    u_norm = np.zeros_like(u)
    for i, c in enumerate(codes):
        if c >= len(a):
            y[i] = np.nan
            u[i] = np.nan
        elif c >= 0:
            u[i] = a[c] @ x[i]
            u_norm[i] = np.sqrt((a[c] * a[c]) @ (x[i] * x[i]))
            y[i] += scale[c] * (b[c] @ u[i])
            sq[i] += (scale[c] ** 2) * ((b[c] * b[c]) @ (u[i] * u[i]))
    return y, np.sqrt(sq), u, u_norm


def adapters_apply_tolerance(x, codes, w, a, b, scale, dtype):
    """-> (y, tolerance, u, u tolerance)"""
    y, norm, u, u_norm = adapters_apply(x, codes, w, a, b, scale)
    d_in, r = a.shape[2], a.shape[1]
    u_tol = sum_error(u_norm, d_in) + 2.0**-24 * np.abs(u)
    tol = sum_error(norm, d_in + r) + HALF_STEP[dtype] * np.abs(y) + TINY[dtype]
    split = {"f32": 0.0, "f16": 2.0**-22, "bf16": 2.0**-16}[dtype]  # u as two 16-bit parts
    for i, c in enumerate(codes):
        if 0 <= c < len(a):
            tol[i] += np.abs(scale[c]) * (np.abs(b[c]) @ (u_tol[i] + split * np.abs(u[i]) + split * np.abs(u[i]).max()))
            tol[i] += 4 * 2.0**-24 * norm[i]  # the factor, the product with it
    return y, tol, u, u_tol


def adapters_backward(grad, x, codes, hidden, w, a, b, scale):
    """-> (grad_x, grad_a, grad_b, v): v [n, r] = B^T grad, without scale"""
    grad_x = grad @ w
    grad_a, grad_b, v = np.zeros_like(a), np.zeros_like(b), np.zeros((len(x), a.shape[1]))
    for i, c in enumerate(codes):
        if c >= len(a):
            grad_x[i] = np.nan
        elif c >= 0:
            v[i] = b[c].T @ grad[i]
            grad_x[i] += scale[c] * (a[c].T @ v[i])
            grad_a[c] += scale[c] * np.outer(v[i], x[i])
            grad_b[c] += scale[c] * np.outer(grad[i], hidden[i])
    return grad_x, grad_a, grad_b, v


def unit(rows):
    norm = np.sqrt((rows * rows).sum(-1, keepdims=True))
    return np.divide(rows, norm, out=np.zeros_like(rows), where=norm > 0), norm


def preference(queries, rows, chosen, rejected, offsets, reference, beta, smoothing, weights=None):
    """-> (loss, margin, grad, pull): pull [nq] = sum of |w dL/dmargin| / |y| over a query's pairs, the size of its gradient's terms"""
    pairs = len(chosen)
    loss, margin, grad, pull = np.zeros(pairs), np.zeros(pairs), np.zeros_like(queries), np.zeros(len(queries))
    weights = np.full(pairs, 1.0 / max(pairs, 1)) if weights is None else weights
    for q in range(len(queries)):
        (y,), ylen = unit(queries[q : q + 1])
        (y0,), _ = unit(reference[q : q + 1]) if reference is not None else ((np.zeros_like(y),), None)
        for p in range(offsets[q], offsets[q + 1]):
            if chosen[p] < 0 or rejected[p] < 0:
                continue
            if chosen[p] >= len(rows) or rejected[p] >= len(rows):
                loss[p] = margin[p] = np.nan
                grad[q] = np.nan
                continue
            (c,), _ = unit(rows[chosen[p]][None])
            (r,), _ = unit(rows[rejected[p]][None])
            s = y @ c - y @ r
            m = s - (y0 @ c - y0 @ r)
            h = beta * m
            margin[p] = m
            loss[p] = (1 - smoothing) * np.logaddexp(0, -h) + smoothing * np.logaddexp(0, h)
            slope = beta * (smoothing / (1 + np.exp(-h)) - (1 - smoothing) / (1 + np.exp(h)))
            if ylen[0, 0] > 0:
                grad[q] += weights[p] * slope * (c - r - s * y) / ylen[0, 0]
                pull[q] += abs(weights[p] * slope) / ylen[0, 0]
    return loss, margin, grad, pull


def clip(grads, max_norm, infinity=False):
    if infinity:
        norm = max((np.abs(g).max() for g in grads if g.size), default=0.0)
    else:
        norm = np.sqrt(sum((g * g).sum() for g in grads))
    f = min(1.0, max_norm / (norm + 1e-6))
    return norm, [g * f for g in grads]


def preference_tolerance(queries, rows, chosen, rejected, offsets, reference, beta, smoothing, weights, dtype):
    """What loss, margin and gradient of ``preference`` may be off by when sums are held in fp32: (loss, margin, grad) tolerances
    with the shapes of the values, element by element from the sizes of the terms behind it.

    With c^, r^, y^, y0^ the unit rows and queries, e = c^ - r^ and d = y^ - y0^ (without a reference d = y^), the values come from
    the margin m = d . e, the cosines' difference s = y^ . e and the sum of g (e - s y^) over the pairs, divided by |y|.

    * a row's norm: its squares are added up in a tree at most 48 deep (32 in a lane, 6 in a wave, up to 8 waves), all of one sign:
      relative 24 * 2^-24 of the norm, and 3 roundings more for root, inverse and its product: ``scale_error``, the same factor
      for all elements of a unit row
    * an element of e: 2 roundings of the unit rows' elements; independent of each other, as are those of d (4 of its size) and, below
      both, 2^-45 of the unit queries (their norms are held in double precision)
    * a sum: ``sum_error`` of the root of its squared terms
    * the slope: 12 roundings (smoothing, weight, exponential, its quotient, the products), one of h in its exponential, its
      derivative times the margin's error, and beta 2^-127: past h = 88.7 the exponential is infinite in fp32, and sigma(-h) < 2^-127 is 0
    * the sum over the pairs: every addition rounds by 2^-24 of what is added up, at most the sum of sizes; two additions a pair, and
      20 more in joining teams and blocks and in the last line
    """
    step = 2.0**-24
    dim, pairs = queries.shape[1], len(chosen)
    scale_error = 27 * step
    loss_tol, margin_tol, grad_tol = np.zeros(pairs), np.zeros(pairs), np.zeros_like(queries)
    weights = np.full(pairs, 1.0 / max(pairs, 1)) if weights is None else np.abs(weights)
    y_all, y_len = unit(queries)
    y0_all = unit(reference)[0] if reference is not None else np.zeros_like(y_all)
    rms = lambda *terms: np.sqrt(sum(((a * b) ** 2).sum(1) for a, b in terms))
    grad = np.zeros_like(queries)
    for q in range(len(queries)):
        at = np.arange(offsets[q], offsets[q + 1])
        at = at[(chosen[at] >= 0) & (rejected[at] >= 0) & (chosen[at] < len(rows)) & (rejected[at] < len(rows)) & (chosen[at] != rejected[at])]
        same = [p for p in range(offsets[q], offsets[q + 1]) if chosen[p] == rejected[p]]
        loss_tol[same] = 8 * step
        if not len(at):
            continue
        c, r = unit(rows[chosen[at]])[0], unit(rows[rejected[at]])[0]
        y, d, e = y_all[q][None], (y_all[q] - y0_all[q])[None], c - r

        def dot_error(v):  # of v . e with v right to a few roundings
            products = sum_error(rms((v, e)), dim) + 4 * 2 * step * np.sqrt(rms((v, c)) ** 2 + rms((v, r)) ** 2)
            return products + scale_error * (np.abs((c * v).sum(1)) + np.abs((r * v).sum(1)))

        dm = dot_error(d) + 4 * 4 * step * rms((d, e)) + 2.0**-45 * dim**0.5 + (3 * step * np.abs((e * d).sum(1)) if reference is None else 0.0)
        ds = dot_error(y) + 4 * 4 * step * rms((y, e)) + 3 * step * np.abs((e * y).sum(1))
        m, s = (e * d).sum(1), (e * y).sum(1)
        h = beta * m
        up, down = np.exp(-np.logaddexp(0, -h)), np.exp(-np.logaddexp(0, h))
        slope = beta * (smoothing * up - (1 - smoothing) * down)
        size = beta * (smoothing * up + (1 - smoothing) * down)
        margin_tol[at] = dm + 2 * step * np.abs(m)
        losses = (1 - smoothing) * np.logaddexp(0, -h) + smoothing * np.logaddexp(0, h)
        loss_tol[at] = size * dm + 8 * step * (losses + np.minimum(1.0, np.abs(h)) + 2.0**-10) + 2 * step * np.abs(h)
        if y_len[q, 0] == 0:
            continue
        g = weights[at] * np.abs(slope)
        dg = weights[at] * (beta * beta * up * down * (dm + step * np.abs(m)) + step * np.abs(h) * size + 12 * step * size + beta * 2.0**-127)
        pull = e - s[:, None] * y
        grows = (2 * len(at) + 20) * step
        error = (dg[:, None] * np.abs(pull)).sum(0)
        error += (g[:, None] * (np.abs(c) + np.abs(r))).sum(0) * (scale_error + 3 * step + grows)
        error += ((g * ds).sum() + (g * np.abs(s)).sum() * (grows + 4 * step)) * np.abs(y[0])
        grad[q] = (weights[at, None] * slope[:, None] * pull).sum(0) / y_len[q, 0]
        grad_tol[q] = error / y_len[q, 0] + 4 * step * np.abs(grad[q])
    grad_tol += HALF_STEP[dtype] * np.abs(grad) + TINY[dtype]
    return loss_tol, margin_tol, grad_tol
