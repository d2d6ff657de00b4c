"""Plain float64 forms of the operators that train with a large vocabulary.

TEST INFRASTRUCTURE ONLY -- imported by tests/; never by the product.

  lookup        rows of a table, scaled; zeros for a token outside it
  lookup_grad   the table's gradient: rows added up by token
  dropout       inverted dropout with Philox4x32-10's keep-mask, and a residual
  linear_xent   a projection and its softmax cross-entropy (layers.py:31-37,
                loss.py:17-27), with the gradients of the mean over labelled rows
"""
from __future__ import annotations

import numpy as np

from . import philox


def lookup(w, ids, scale=1.0):
    w = np.asarray(w, np.float64)
    some = (ids >= 0) & (ids < len(w))
    return np.where(some[:, None], w[np.where(some, ids, 0)], 0.0) * scale


def lookup_grad(ids, g, V, scale=1.0):
    """(sum, sum of magnitudes) per table row and column."""
    g = np.asarray(g, np.float64)
    some = (ids >= 0) & (ids < V)
    out = np.zeros((2, V, g.shape[1]))
    np.add.at(out[0], ids[some], g[some])
    np.add.at(out[1], ids[some], np.abs(g[some]))
    return out[0] * scale, out[1] * abs(scale)


def keep(shape, p, seed, offset=0, subsequence=0):
    """The keep-mask of a (rows, cols) array."""
    n = int(np.prod(shape))
    ctr = np.zeros(((n + 3) // 4, 4), np.uint64)
    at = np.arange(len(ctr), dtype=np.uint64) + np.uint64(offset)
    ctr[:, 0], ctr[:, 1], ctr[:, 2] = at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.uint64(subsequence)
    words = philox.philox4x32_10(ctr, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)).reshape(-1)[:n]
    u = (words >> np.uint32(8)).astype(np.float64) * 2.0 ** -24
    return (u > float(np.float32(p))).reshape(shape)


def dropout(x, p, seed, offset=0, residual=None, subsequence=0):
    y = np.where(keep(x.shape, p, seed, offset, subsequence), np.asarray(x, np.float64) / (1.0 - p), 0.0)
    return y if residual is None else np.asarray(residual, np.float64) + y


def linear_xent(x, w, labels, bias=None):
    """dict of z, lse, p, row_loss, loss, dz, dx, dw, db."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    z = x @ w + (0.0 if bias is None else np.asarray(bias, np.float64))
    n, V = z.shape
    m = z.max(1, keepdims=True, initial=-np.inf)
    e = np.exp(z - np.where(m == -np.inf, 0.0, m))
    s = e.sum(1, keepdims=True)
    p = e / np.where(s == 0, 1.0, s)
    with np.errstate(divide="ignore"):
        lse = (m + np.log(s))[:, 0]
    some = (labels >= 0) & (labels < V)
    rows, at = np.nonzero(some)[0], labels[some]
    row_loss = np.zeros(n)
    zy = z[rows, at]
    with np.errstate(invalid="ignore"):
        row_loss[rows] = np.where(zy == -np.inf, np.inf, lse[rows] - zy)
    count = max(1, len(rows))
    dz = p.copy()
    dz[rows, at] -= 1.0
    dz[~some] = 0.0
    dz /= count
    return dict(z=z, lse=lse, p=p, some=some, row_loss=row_loss, loss=row_loss.sum() / count, dz=dz, dx=dz @ w.T, dw=x.T @ dz,
                db=dz.sum(0))
