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
