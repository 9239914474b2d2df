"""Plain 64-bit forms of the answering calls, for the tests."""
import numpy as np

# The weights exp((l - max) / T) are computed in 32 bits: the difference, the
# reciprocal of T and their product are each rounded (2^-24), and what that
# moves the exponent by, at most 3 |x| 2^-24 with |x| < 104 (beyond it the
# weight is 0), is the weight's relative error; expf adds two units.  A sum
# of weights is off by no more than its terms.
EPS = (3 * 104 + 4) * 2.0 ** -24


def quantized(a):
    """(q, scale) of the rows of a float array: the definition itself."""
    a = np.asarray(a).astype(np.float32)
    n, d = a.shape
    q = np.zeros((n, d), np.int8)
    s = np.zeros(n, np.float32)
    for i in range(n):
        if not np.isfinite(a[i]).all():
            s[i] = np.nan
            continue
        s[i] = np.abs(a[i]).max() * np.float32(1 / 127)
        if s[i] > 0:
            q[i] = np.clip(np.rint(a[i] / s[i]), -127, 127).astype(np.int8)
    return q, s


def scores(X, sx, W, sw):
    sums = X.astype(np.int64) @ W.astype(np.int64).T
    return sums * sx.astype(np.float64)[:, None] * sw.astype(np.float64)[None, :]


def check_scores(got, X, sx, W, sw, kind):
    """Three roundings to 24 bits, one to the output's."""
    want = scores(X, sx, W, sw)
    bits, least = {"float32": (24, 2.0 ** -149), "float16": (11, 2.0 ** -25), "bfloat16": (8, 2.0 ** -134)}[kind]
    bound = np.abs(want) * (4 * 2.0 ** -24 + (0 if kind == "float32" else 1.01 * 2.0 ** -bits)) + least
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= bound).all(), (np.argwhere(off > bound)[:5], got[off > bound][:5], want[off > bound][:5])


def check_sample(S, u, T, k, p, q, label, prob, kept):
    """Whether the drawn labels are what the definition in 64 bits allows,
    with the weights' own rounding (EPS) at every cut and at the draw."""
    S = np.asarray(S, np.float64)
    n, m = S.shape
    full = [np.broadcast_to(np.asarray(v, np.float64), (n,)) for v in (T, k, p, q)]
    for r in range(n):
        row = np.where(np.isnan(S[r]), -np.inf, S[r])
        t, kk, pp, qq = (v[r] for v in full)
        at = f"row {r}: T {t} k {kk} p {pp} q {qq} u {u[r]}: got {label[r]}, {prob[r]}, {kept[r]}"
        best = int(np.argmax(row))
        if row[best] == -np.inf:
            assert label[r] == -1 and prob[r] == 0 and kept[r] == 0, at
            continue
        if t == 0:
            assert label[r] == best and prob[r] == 1 and kept[r] == 1, at
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(row == row[best], 1.0, np.exp((row - row[best]) / t))
        order = np.argsort(-row, kind="stable")
        if 0 < kk < m:
            order = order[:int(kk)]
        wo = w[order]
        c = np.cumsum(wo)
        least = most = len(order)
        if pp < 1:
            least = 1 + int(np.searchsorted(c, pp * (1 - EPS) * c[-1]))
            most = min(len(order), 1 + int(np.searchsorted(c, pp * (1 + EPS) * c[-1])))
        low = max(qq * (1 - EPS), 2.0 ** -150)
        high = max(qq * (1 + EPS) if qq < 1 else 1.0, 2.0 ** -148)
        least = min(least, max(1, int((wo >= high).sum())))
        most = min(most, int((wo >= low).sum()))
        assert least <= kept[r] <= most, f"{at}; {least}..{most} can be kept"
        ids = np.sort(order[:int(kept[r])])
        assert label[r] in ids, at
        c = np.cumsum(w[ids])
        j = int(np.searchsorted(ids, label[r]))
        before, after = (c[j - 1] if j else 0.0), c[j]
        assert before <= (u[r] + EPS) * c[-1] and after >= (u[r] - EPS) * c[-1], f"{at}; {before / c[-1]}..{after / c[-1]}"
        assert abs(prob[r] - w[label[r]] / c[-1]) <= 2 * EPS * prob[r] + 1e-40, f"{at}; {w[label[r]] / c[-1]}"
