"""Plain 64-bit forms of log_probs and log_probs_grad, for the tests, and how
far 32-bit results may be from them.

An exponent e = s c - ref (c = log2(e) / T) is off by at most 6 half units of
its size: 1 / T, log2(e), their product and the sum are rounded, and a change
of reference rounds twice.  `ref` is one number in the weights and in the
label's exponent, so its own rounding cancels.  A sum of weights, all of one
sign, is off by as many half units as additions follow one another: 32 in a
lane's step, m / 1024 steps at most, 6 exchanges and 16 waves, for the sizes
here under DEPTH, and the two units of each exponential.
"""
import numpy as np

HALF = 2.0 ** -24
DEPTH = 110


def rows(S, T=1.0):
    """(x, p, log p, entropy, log Z, largest) of each row; x = (s - M) / T."""
    S = np.asarray(S, np.float64)
    T = float(np.float32(T))
    M = S.max(axis=1, keepdims=True) if S.shape[1] else None
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = np.where(S == M, 0.0, (S - M) / T)
        w = np.where(M == -np.inf, 0.0, np.exp(x))
        Z = w.sum(axis=1, keepdims=True)
        p = w / Z
        logp = x - np.log(Z)
        plogp = np.where(p > 0, p * logp, 0.0)
    empty = (M == -np.inf)[:, 0] & ~np.isnan(S).any(axis=1)
    bad = np.isnan(S).any(axis=1)
    H = -plogp.sum(axis=1)
    logZ = np.log(np.where(Z > 0, Z, 1.0))[:, 0]
    logZ[empty], H[empty], logp[empty], p[empty], x[empty] = -np.inf, 0.0, -np.inf, 0.0, 0.0
    for v in (H, logZ):
        v[bad] = np.nan
    p[bad], logp[bad], x[bad] = np.nan, np.nan, np.nan
    return x, p, logp, H, logZ, M[:, 0], empty, bad


def spread(x, p):
    """Sums of p |x| and p (x^2 + |x|): what the exponents' errors can make of
    log Z and of the sum of w log w."""
    a = np.where(p > 0, np.abs(x), 0.0)
    return (p * a).sum(axis=1), (p * (a * a + a)).sum(axis=1)


def log_z_error(x, p):
    return HALF * (DEPTH + 4 + 6 * spread(x, p)[0])


def entropy_error(x, p):
    a, b = spread(x, p)
    return 2 * HALF * ((DEPTH + 4) * (1 + a) + 6 * b)


def check(S, labels, T, got_logp, got_H=None, got_stats=None, top=None):
    x, p, logp, H, logZ, M, empty, bad = rows(S, T)
    n, m = x.shape
    ez, eh = log_z_error(x, p), entropy_error(x, p)
    for i in range(n):
        at = f"row {i} of {n} x {m}"
        l = int(labels[i])
        if l == -1:
            assert got_logp[i] == 0, at
        elif not 0 <= l < m or bad[i]:
            assert np.isnan(got_logp[i]), at
        elif logp[i, l] == -np.inf:
            assert got_logp[i] == -np.inf, (at, got_logp[i])
        elif logp[i, l] < -1e30:
            assert got_logp[i] <= logp[i, l] * (1 - 1e-5), (at, got_logp[i], logp[i, l])
        else:
            off = abs(float(got_logp[i]) - logp[i, l])
            assert off <= ez[i] + HALF * (8 * abs(x[i, l]) + 4 * abs(logp[i, l])), (at, got_logp[i], logp[i, l], off)
        if got_H is not None:
            if bad[i]:
                assert np.isnan(got_H[i]), at
            else:
                assert abs(float(got_H[i]) - H[i]) <= eh[i] and got_H[i] >= 0, (at, got_H[i], H[i])
        if got_stats is not None:
            if bad[i]:
                assert np.isnan(got_stats[i, 1]) and np.isnan(got_stats[i, 2]), at
            else:
                assert got_stats[i, 0] == M[i], at
                if empty[i]:
                    assert got_stats[i, 1] == -np.inf and got_stats[i, 2] == 0, at
                else:
                    assert abs(float(got_stats[i, 1]) - logZ[i]) <= ez[i] + HALF * 4 * logZ[i], at
                    assert abs(float(got_stats[i, 2]) - H[i]) <= eh[i], at
    if top:
        lp, at = top
        k = lp.shape[1]
        keys = np.where(np.isnan(S), -np.inf, np.asarray(S, np.float64))
        order = np.argsort(-keys, axis=1, kind="stable")[:, :k]
        for i in range(n):
            want = [j for j in order[i] if keys[i, j] > -np.inf]
            want += [-1] * (k - len(want))
            assert list(at[i]) == want, (i, list(at[i]), want)
            for j, v in zip(want, lp[i]):
                if j < 0:
                    assert v == -np.inf
                elif bad[i]:
                    assert np.isnan(v)
                else:
                    tol = ez[i] + HALF * (8 * abs(x[i, j]) + 4 * abs(logp[i, j]))
                    assert v == logp[i, j] or abs(float(v) - logp[i, j]) <= tol or (v < -1e30 and logp[i, j] < -1e30), (i, j, v, logp[i, j])


def grad(S, labels, g, h, T):
    x, p, logp, H, logZ, M, empty, bad = rows(S, T)
    n, m = x.shape
    T = float(np.float32(T))
    one = np.zeros_like(p)
    labels = np.asarray(labels)
    some = (labels >= 0) & (labels < m)
    one[np.flatnonzero(some), labels[some]] = 1.0
    gg = np.where(labels == -1, 0.0, np.where(some, g, np.nan))[:, None]
    hh = np.zeros((n, 1)) if h is None else np.asarray(h, np.float64)[:, None]
    with np.errstate(invalid="ignore"):
        plogp = np.where(p > 0, p * logp, 0.0)
    D = (gg * (one - p) - hh * (plogp + p * H[:, None])) / T
    D[empty] = np.where(np.isnan(gg[empty]), np.nan, 0.0)
    D[bad] = np.nan
    return D


def check_grad(got, S, labels, g, h, T, half, least):
    """half: half a step of the output's type, least: half its smallest."""
    D = grad(S, labels, g, h, T)
    assert np.array_equal(np.isnan(got), np.isnan(D)), np.argwhere(np.isnan(got) != np.isnan(D))[:5]
    x, p, logp, H, *_ = rows(S, T)
    T = float(np.float32(T))
    ez, eh = log_z_error(x, p)[:, None], entropy_error(x, p)[:, None]
    g = np.abs(np.where(np.asarray(labels) == -1, 0.0, g))[:, None]
    h = np.zeros_like(g) if h is None else np.abs(np.asarray(h, np.float64))[:, None]
    with np.errstate(invalid="ignore"):
        lp = np.where(p > 0, np.abs(logp), 0.0)
        # log p is off by the exponent's rounding, log Z's error, and what the
        # statistics lose when they are kept in 32 bits
        e = ez + HALF * (16 * lp + 8 * np.abs(np.where(p > 0, x, 0.0)) + 8)
        size = g + h * (lp + np.abs(H)[:, None])
        bound = (p * (e + 8 * HALF) * size + p * h * (e + eh + HALF * (lp + np.abs(H)[:, None]) * 4)) / T
        bound += np.abs(D) * (half + 6 * HALF) + 4 * HALF * g / T * (np.abs(D) * T > 0.25 * g) + least + 2.0 ** -126 * (1 + size) / T
        off = np.abs(got.astype(np.float64) - D)
    ok = np.isnan(D) | (off <= bound)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], D[~ok][:5], bound[~ok][:5])
