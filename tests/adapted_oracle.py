"""Plain 64-bit forms of scores_adapted and scores_adapted_grad, for the tests,
and how far 32-bit results may be from them.

Every sum is of products of 32-bit (or shorter) factors in 32 bits: off by at
most its number of additions in half units of the sum of the terms' sizes.
"""
import numpy as np

from tests import answer_oracle

HALF = 2.0 ** -24


def terms(X, A, index, scale):
    """(T, |T|'s sums): rows scale_a A_a x_i, zeros without an adapter."""
    X, A = np.asarray(X, np.float64), np.asarray(A, np.float64)
    n, (count, r, d) = X.shape[0], A.shape
    scale = np.broadcast_to(np.asarray(scale, np.float32).astype(np.float64), (count,))
    T, size = np.zeros((n, r)), np.zeros((n, r))
    for a in np.unique(index[(index >= 0) & (index < count)]):
        rows = index == a
        T[rows] = scale[a] * (X[rows] @ A[a].T)
        size[rows] = abs(scale[a]) * (np.abs(X[rows]) @ np.abs(A[a]).T)
    return T, size * (d + 64) * HALF


def by_rows(T, B, index):
    n, (count, m, r) = T.shape[0], B.shape
    S = np.zeros((n, m))
    for a in np.unique(index[(index >= 0) & (index < count)]):
        rows = index == a
        S[rows] = T[rows] @ np.asarray(B[a], np.float64).T
    return S


def check_scores(got, X, W, sw, A, B, index, scale, half, least):
    q, sx = answer_oracle.quantized(X)
    base = answer_oracle.scores(q, sx, W, sw)
    T, off_T = terms(X, A, index, scale)
    r = T.shape[1]
    more = by_rows(T, B, index)
    off = by_rows(np.abs(T) * (r + 16) * HALF + off_T, np.abs(np.asarray(B, np.float64)), index)
    want = base + more
    bad = (index < -1) | (index >= len(A))
    assert np.isnan(got[bad]).all()
    bound = np.abs(base) * 4 * HALF + off + np.abs(want) * (half * 1.01 + 2 * HALF) + least
    err = np.abs(got.astype(np.float64) - want)
    ok = (err <= bound) | bad[:, None]
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5], bound[~ok][:5])


def grads(G, X, A, B, index, scale):
    """(dA, dB) and their bounds."""
    G, X, B = (np.asarray(v, np.float64) for v in (G, X, B))
    count, r, d = A.shape
    m = B.shape[1]
    T, off_T = terms(X, A, index, scale)
    U, off_U = terms(G, B.transpose(0, 2, 1), index, scale)
    dA, dB = np.zeros((count, r, d)), np.zeros((count, m, r))
    bA, bB = np.zeros_like(dA), np.zeros_like(dB)
    for a in range(count):
        rows = index == a
        k = (rows.sum() + 64) * HALF
        dA[a], dB[a] = U[rows].T @ X[rows], G[rows].T @ T[rows]
        bA[a] = (np.abs(U[rows]) * k + off_U[rows]).T @ np.abs(X[rows])
        bB[a] = np.abs(G[rows]).T @ (np.abs(T[rows]) * k + off_T[rows])
    return (dA, bA), (dB, bB)


def check_grads(got, *args):
    for g, (want, bound), name in zip(got, grads(*args), ("dA", "dB")):
        err = np.abs(g.astype(np.float64) - want)
        ok = err <= bound + 2.0 ** -140
        assert ok.all(), (name, np.argwhere(~ok)[:5], g[~ok][:5], want[~ok][:5], bound[~ok][:5])
