"""sdca_scores_adapted with adapters and terms at the ends of their types'
ranges, and the digits that terms are held in."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

KINDS = ["float32", "float16", "bfloat16"]
# few, strip, tiles of 64, 128 and 256, in the adapters' order and not
SHAPES = [(1, 512, 90), (2, 600, 300), (40, 77, 100), (80, 700, 900), (300, 300, 500), (1200, 300, 500),
          (3000, 72, 1030), (1024, 64, 14_336)]


def _gen(cuda, seed):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _np(t):
    import torch
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _want(base, X, A, B, index, scale):
    """base (scores without adapters) and the adapters' part, by the formula in
    64 bits."""
    want = base.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        for a in range(len(A)):
            rows = np.flatnonzero(index == a)
            T = np.zeros((len(rows), A.shape[1]))
            for k in range(A.shape[1]):
                T[:, k] = scale[a] * (X[rows].astype(np.float64) * A[a, k].astype(np.float64)).sum(axis=1)
                want[rows] += T[:, k, None] * B[a, :, k].astype(np.float64)
    return want


def _check(got, want, off):
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    far = np.isinf(want)
    assert np.array_equal(got[far], want[far]) and np.isfinite(got[np.isfinite(want)]).all()
    some = np.isfinite(want)
    assert (np.abs(got[some] - want[some]) <= off[some]).all()


def _operands(cuda, n, d, m, r, count, kind, seed):
    """Terms of small whole numbers, which every split holds in its first part."""
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, seed)
    dt = getattr(torch, kind)
    W, sw = sd.quantize_i8(torch.randn((m, d), generator=g, device=cuda) / d ** 0.5)
    X = torch.randint(-1, 2, (n, d), generator=g, device=cuda).to(dt)
    X[:, 0] = 1
    A = torch.zeros((count, r, d), device=cuda)
    A[:, :, :4] = torch.randint(-2, 3, (count, r, 4), generator=g, device=cuda).float()
    B = torch.randn((count, m, r), generator=g, device=cuda)
    index = torch.randint(-1, count, (n,), generator=g, device=cuda)
    index[0] = 1
    return X, W, sw, A, B, index, dt


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("r", [3, 16, 40])
@pytest.mark.parametrize("n,d,m", SHAPES)
def test_infinities_of_an_adapter(cuda, n, d, m, r, kind):
    """An infinity of B by a term is an infinity, by a term of 0 NaN, and the
    other classes keep their scores."""
    import torch
    import libsdca_amd as sd
    print(n, d, m, r, kind, flush=True)
    X, W, sw, A, B, index, dt = _operands(cuda, n, d, m, r, 3, kind, n + r)
    g = _gen(cuda, 5)
    B[1] = torch.where(torch.rand((m, r), generator=g, device=cuda) < 0.02, float("inf"), B[1])
    B[1] = torch.where(torch.rand((m, r), generator=g, device=cuda) < 0.02, -float("inf"), B[1])
    B[2, ::7, r - 1] = float("inf")
    A, B = A.to(dt), B.to(dt)
    base = _np(sd.scores_i8(X, W, sw))
    host = [_np(v) for v in (X, A, B, index)]
    want = _want(base, *host, np.ones(3))
    # the base, r products and their sum: some r half units of their sizes (8 at most)
    off = 2.0 ** -24 * (4 * np.abs(base) + (r + 16) * 8.0 * np.nansum(np.where(np.isinf(host[2]), 0, np.abs(host[2])), axis=2).max())
    _check(_np(sd.scores_adapted(X, W, sw, A, B, index)), want, off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,d,m", SHAPES)
def test_infinite_and_largest_terms(cuda, n, d, m, kind):
    """Infinite terms beside large finite ones, and finite ones that the next
    number of 16 bits is infinite beside."""
    import torch
    import libsdca_amd as sd
    print(n, d, m, kind, flush=True)
    r = 5
    X, W, sw, A, B, index, dt = _operands(cuda, n, d, m, r, 3, kind, n)
    X[:, :3] = torch.tensor([1.0, 100.0, 2.0], device=cuda).to(dt)
    A[:] = 0
    A[:, 3, 0] = 1
    A[1, 0, 0], A[1, 1, 1], A[1, 2, 1] = float("inf"), 60_000, -60_000   # inf, 6e6, -6e6
    A[1, 4, 0] = -3
    A[2, 0, 0] = A[2, 1, 0] = 1
    B[:] = torch.randint(-2, 3, B.shape, generator=_gen(cuda, 7), device=cuda).float()
    A, B = A.to(dt), B.to(dt)
    # (adapter 2's terms: 3.4e38, beyond the largest bfloat16 by less than half its step)
    scale = torch.tensor([1.0, 1.0, 3.4e38], device=cuda)
    B[2] *= 2.0 ** -12
    base = _np(sd.scores_i8(X, W, sw))
    hX, hA, hB, hi = (_np(v) for v in (X, A, B, index))
    # (an infinity in A by a 0 of X would be NaN: here column 0 of X is 1)
    T = np.zeros((n, r))
    s = _np(scale).astype(np.float64)
    with np.errstate(invalid="ignore"):
        for i in np.flatnonzero(hi >= 0):
            A64 = hA[hi[i]].astype(np.float64)
            T[i] = s[hi[i]] * (A64[:, 0] * hX[i, 0] + A64[:, 1] * hX[i, 1])
    want = base.astype(np.float64)
    size = np.abs(want)
    with np.errstate(invalid="ignore"):
        for i in np.flatnonzero(hi >= 0):
            for k in range(r):
                p = T[i, k] * hB[hi[i], :, k].astype(np.float64)
                want[i] += p
                size[i] += np.abs(np.where(np.isfinite(p), p, 0))
    got = _np(sd.scores_adapted(X, W, sw, A, B, index, scale=scale))
    # (the terms' zeros of X times infinity are NaN in both: row 0 of adapter 1 alone)
    _check(got, want, 2.0 ** -24 * 64 * size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,d,m", SHAPES)
def test_terms_have_32_bits(cuda, n, d, m, kind):
    """One term of 24 digits times 1 is the score."""
    import torch
    import libsdca_amd as sd
    dt = getattr(torch, kind)
    g = _gen(cuda, n)
    X = torch.zeros((n, d), device=cuda)
    A = torch.zeros((2, 2, d), device=cuda)
    # eight digits at a time: 1.xxxxxxx + 2^-8 xxxxxxxx + 2^-16 xxxxxxxx
    digits = torch.randint(0, 128, (n, 3), generator=g, device=cuda)
    X[:, 0] = 1 + digits[:, 0] / 128
    X[:, 1], X[:, 2] = digits[:, 1], digits[:, 2] * 2 + 1
    A[:, 0, 0], A[:, 0, 1], A[:, 0, 2] = 1, 2.0 ** -14, 2.0 ** -23
    A[:, 0, 1:3] *= 2.0 ** 9   # (ordinary halves)
    X[:, 1:3] *= 2.0 ** -9
    W = torch.zeros((m, -(-d // 16) * 16), dtype=torch.int8, device=cuda)[:, :d]
    sw = torch.ones(m, device=cuda)
    B = torch.zeros((2, m, 2), device=cuda)
    B[:, :, 0] = 1
    index = torch.arange(n, device=cuda) % 2
    X, A, B = X.to(dt), A.to(dt), B.to(dt)
    T = (X.double() * A[0, 0].double()).sum(dim=1)
    assert torch.equal(T.float().double(), T)
    got = sd.scores_adapted(X, W, sw, A, B, index)
    assert torch.equal(got, T.float()[:, None].expand(n, m))
