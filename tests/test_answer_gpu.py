"""The answering calls (sdca_quantize_i8, sdca_scores_i8, sdca_sample) against
their plain forms in 64 bits (tests/answer_oracle.py)."""
import numpy as np
import pytest

from tests import answer_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float32", "float64", "float16", "bfloat16"]


def _gen(cuda, seed):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _np(t):
    import torch
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _spaced(t, pitch):
    """The same matrix with its rows `pitch` values apart."""
    import torch
    n, d = t.shape
    buf = torch.zeros((n, pitch), dtype=t.dtype, device=t.device)
    if t.dtype == torch.int8:
        buf.fill_(77)  # what lies between the rows counts for nothing
    buf[:, :d] = t
    return buf[:, :d]


# ---------------------------------------------------------------------------
# quantize_i8: equal to the definition, bit for bit.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,d", [(1, 1), (5, 7), (4, 8), (9, 513), (3, 1024), (2, 1025), (7, 4096),
                                 (3, 4100), (2, 12_288), (2, 12_289), (3, 30_001)])
def test_quantize_equals_definition(cuda, kind, n, d):
    import torch
    import libsdca_amd as sd
    a = (torch.randn((n, d), generator=_gen(cuda, n * d), device=cuda) * 3).to(getattr(torch, kind))
    q, s = sd.quantize_i8(a)
    wq, ws = ref.quantized(_np(a))
    assert np.array_equal(_np(s), ws)
    assert np.array_equal(_np(q), wq)
    assert q.stride(0) % 16 == 0
    # rows apart, at odd addresses, and into a given matrix
    out = torch.full((n, d + 3), 99, dtype=torch.int8, device=cuda)
    q2, s2 = sd.quantize_i8(_spaced(a, d + 5), out=out[:, :d])
    assert torch.equal(q2, q) and torch.equal(s2, s)
    assert bool((out[:, d:] == 99).all()), "bytes between the rows were written"


@pytest.mark.parametrize("d", [6, 700, 5000, 20_000])
def test_quantize_special_columns(cuda, d):
    import torch
    import libsdca_amd as sd
    a = torch.randn((10, d), generator=_gen(cuda, d), device=cuda)
    a[0] = 0
    a[1, d // 2] = float("inf")
    a[2, d - 1] = float("nan")
    a[3] *= 1e-38
    a[4] *= 1e-44          # the scale is no 32-bit number above zero
    a[5] *= 1e36
    a[6] = -2.5
    a[7, 0] = -float("inf")
    a[8] *= 3e-43          # subnormal values, a scale of few digits
    a[9, 1:] = 0
    q, s = sd.quantize_i8(a)
    wq, ws = ref.quantized(_np(a))
    assert np.array_equal(_np(s), ws, equal_nan=True)
    assert np.array_equal(_np(q), wq)
    b = torch.full((1, 4), 1e300, dtype=torch.float64, device=cuda)  # no float
    q, s = sd.quantize_i8(b)
    assert bool(torch.isnan(s).all()) and bool((q == 0).all())


@pytest.mark.parametrize("kind", KINDS)
def test_quantize_halves(cuda, kind):
    """Values at and next to halves of a step, where the nearest integer
    hangs on the last bit of the quotient."""
    import torch
    import libsdca_amd as sd
    for top in (127.0, 1.0, 254.0, 96.0, 0.1875):
        half = (torch.arange(-127, 127, device=cuda, dtype=torch.float64) + 0.5) * (top / 127)
        row = torch.cat([torch.tensor([top], device=cuda, dtype=torch.float64), half, half * (1 + 2.0 ** -22),
                         half * (1 - 2.0 ** -22), half * (1 + 2.0 ** -10)])
        a = row.to(getattr(torch, kind)).repeat(3, 1)
        q, s = sd.quantize_i8(a)
        wq, ws = ref.quantized(_np(a))
        assert np.array_equal(_np(s), ws) and np.array_equal(_np(q), wq), top


# ---------------------------------------------------------------------------
# scores_i8
# ---------------------------------------------------------------------------
def _operands(cuda, n, m, d, seed):
    import torch
    g = _gen(cuda, seed)
    X = torch.randint(-127, 128, (n, d), generator=g, device=cuda, dtype=torch.int8)
    W = torch.randint(-127, 128, (m, d), generator=g, device=cuda, dtype=torch.int8)
    return X, 0.01 + torch.rand(n, generator=g, device=cuda), W, 0.01 + torch.rand(m, generator=g, device=cuda)


SHAPES = [(1, 1, 1), (1, 1000, 4096), (2, 3, 16), (3, 65, 100), (4, 1000, 513), (7, 130, 129), (8, 16, 128),
          (15, 100, 640), (16, 137, 513), (17, 137, 1), (31, 300, 2048), (32, 256, 127), (33, 1000, 256),
          (48, 77, 300), (64, 128, 1024), (65, 129, 4096), (100, 513, 384), (128, 1000, 100), (129, 255, 130),
          (200, 700, 512), (257, 257, 1000), (300, 1, 700), (1000, 2000, 64), (513, 1025, 200)]


@pytest.mark.parametrize("n,m,d", SHAPES)
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_scores_of_quantized_examples(cuda, n, m, d, kind):
    import torch
    import libsdca_amd as sd
    print(n, m, d, kind, flush=True)
    X, sx, W, sw = _operands(cuda, n, m, d, n + m + d)
    if kind == "float16":
        sw = sw / 1000  # within the type's range
    dt = getattr(torch, kind)
    S = sd.scores_i8(X, W, sw, x_scales=sx, dtype=dt)
    assert S.dtype == dt and tuple(S.shape) == (n, m)
    ref.check_scores(_np(S), _np(X), _np(sx), _np(W), _np(sw), kind)
    # the same from rows apart, aligned and not, and into a given matrix whose
    # other values stay
    pad = (d + 15) // 16 * 16
    for px, pw, ps in ((pad, pad, m + 1), (d + 1, d + 3, m + 8), (pad + 16, pad + 48, m)):
        out = torch.full((n, ps), -7, dtype=dt, device=cuda)
        got = sd.scores_i8(_spaced(X, px), _spaced(W, pw), sw, x_scales=sx, out=out[:, :m])
        assert torch.equal(got, S), (px, pw, ps)
        assert bool((out[:, m:] == -7).all()), "values between the rows were written"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,m,d", [(1, 1000, 4096), (2, 50, 77), (3, 200, 513), (9, 333, 1024), (33, 100, 4100),
                                   (70, 513, 128), (300, 137, 513)])
def test_scores_of_float_examples(cuda, kind, n, m, d):
    """Equal to the scores of the examples quantised beforehand."""
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, n * m + d)
    X = torch.randn((n, d), generator=g, device=cuda).to(getattr(torch, kind))
    X[n // 2] = 0
    if n > 2:
        X[n - 1, d // 2] = float("nan")
    W, sw = sd.quantize_i8(torch.randn((m, d), generator=g, device=cuda))
    S = sd.scores_i8(X, W, sw)
    q, s = sd.quantize_i8(X)
    assert torch.equal(torch.nan_to_num(S, nan=-3.0), torch.nan_to_num(sd.scores_i8(q, W, sw, x_scales=s), nan=-3.0))
    assert bool((S[n // 2] == 0).all())
    if n > 2:
        assert bool(torch.isnan(S[n - 1]).all()) and not bool(torch.isnan(S[:n - 1]).any())
    # near the scores of the model in floats: both operands are off by half a
    # step at most, |x||w| (1/254 + 1/254 + 1/254^2) sqrt(d) in the mean
    if n <= 2 and d >= 77:
        full = X.double() @ (W.double() * sw.double()[:, None]).T
        bound = s.double()[:, None] * 0.5 * (W.double().abs().sum(dim=1) * sw.double())
        assert bool(((S.double() - full).abs() <= bound * 1.0001 + 1e-30).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_scores_few_classes(cuda, kind, out):
    """Few classes, at the ends of the kernels' units of d, m and n: equal to
    the scores of the examples quantised beforehand, whose kernel is another;
    also from rows apart, with values between that are not to be read, and
    into rows apart, whose values between stay."""
    import torch
    import libsdca_amd as sd
    dt, odt = getattr(torch, kind), getattr(torch, out)
    for i, d in enumerate((1, 7, 8, 9, 15, 63, 64, 65, 127, 200, 511, 512, 513, 520, 767, 1017, 1024, 1025)):
        for m in (1, 15, 32, 33, 96, 137, 256, 257):
            n = (1, 3, 31, 32, 33, 100)[(i + m) % 6]
            print(kind, out, n, m, d, flush=True)
            g = _gen(cuda, n * m + d)
            X = torch.randn((n, d), generator=g, device=cuda).to(dt)
            X[n // 2] = 0
            if n > 3:
                X[n - 1, d - 1] = float("-inf")
                X[1, : d // 2] = 0
            W, sw = sd.quantize_i8(torch.randn((m, d), generator=g, device=cuda))
            q, s = sd.quantize_i8(X)
            want = torch.nan_to_num(sd.scores_i8(q, W, sw, x_scales=s, dtype=odt), nan=-3.0)
            got = torch.nan_to_num(sd.scores_i8(X, W, sw, dtype=odt), nan=-3.0)
            assert torch.equal(got, want)
            wide = torch.full((n, d + 5), float("nan"), dtype=dt, device=cuda)
            wide[:, 1:d + 1] = X
            spare = torch.full((m, (d + 15) // 16 * 16 + 16), 99, dtype=torch.int8, device=cuda)
            spare[:, :d] = W
            S = torch.full((n, m + 3), -7, dtype=odt, device=cuda)
            sd.scores_i8(wide[:, 1:d + 1], spare[:, :d], sw, out=S[:, :m])
            assert torch.equal(torch.nan_to_num(S[:, :m], nan=-3.0), want)
            assert bool((S[:, m:] == -7).all())


@pytest.mark.parametrize("kind", KINDS)
def test_quantize_ends_of_columns(cuda, kind):
    """Every end of a column within a lane's eight values, from rows apart and
    into rows apart."""
    import torch
    import libsdca_amd as sd
    for d in [*range(1, 27), *range(126, 139), 255, 257, 511, 515, 1021, 1030, 2047, 4099]:
        n = 9
        g = _gen(cuda, d)
        wide = torch.full((n, d + 3), float("nan"), dtype=getattr(torch, kind), device=cuda)
        wide[:, 2:d + 2] = torch.randn((n, d), generator=g, device=cuda).to(wide.dtype)
        X = wide[:, 2:d + 2]
        Q = torch.full((n, d + 9), 77, dtype=torch.int8, device=cuda)
        q, s = sd.quantize_i8(X, out=Q[:, :d])
        want_q, want_s = ref.quantized(_np(X.contiguous()))
        assert np.array_equal(_np(q), want_q) and np.array_equal(_np(s), want_s), d
        assert bool((Q[:, d:] == 77).all()), d


@pytest.mark.parametrize("n,m,d,out", [(17_000, 1000, 4096, "float32"), (9000, 8192, 1030, "bfloat16"),
                                       (50_001, 1000, 768, "float16")])
def test_scores_in_two_launches(cuda, n, m, d, out):
    """More examples than whole rounds of the largest tiles: what is left is a
    launch of its own.  The rows next to every multiple of 256 are checked,
    and no row is left out."""
    import torch
    import libsdca_amd as sd
    print(n, m, d, out, flush=True)
    X, sx, W, sw = _operands(cuda, n, m, d, n + d)
    if out == "float16":
        sw = sw / 1000  # within the type's range
    S = torch.full((n, m + 5), float("nan"), dtype=getattr(torch, out), device=cuda)
    sd.scores_i8(X, W, sw, x_scales=sx, out=S[:, :m])
    assert not bool(torch.isnan(S[:, :m]).any()) and bool(torch.isnan(S[:, m:]).all())
    rows = sorted({r for t in range(0, n, 256) for r in (t - 1, t) if r >= 0} | {n - 1})
    cols = sorted({*range(0, m, 61), m - 1})
    ref.check_scores(_np(S[rows][:, cols].contiguous()), _np(X[rows]), _np(sx[rows]), _np(W[cols]), _np(sw[cols]), out)


def test_scores_extreme_sums(cuda):
    """The largest d, every product at its extreme: sums next to 2^31."""
    import torch
    import libsdca_amd as sd
    d = 131_071
    X = torch.full((3, d), -128, dtype=torch.int8, device=cuda)
    W = torch.full((5, d), -128, dtype=torch.int8, device=cuda)
    W[1] = 127
    X[2, ::2] = 127
    one = torch.ones(5, device=cuda)
    S = sd.scores_i8(X, W, one, x_scales=one[:3].contiguous())
    ref.check_scores(_np(S), _np(X), np.ones(3, np.float32), _np(W), np.ones(5, np.float32), "float32")
    with pytest.raises(sd.SdcaError) as e:
        sd.scores_i8(torch.zeros((1, d + 1), dtype=torch.int8, device=cuda),
                     torch.zeros((1, d + 1), dtype=torch.int8, device=cuda), one[:1].contiguous(),
                     x_scales=one[:1].contiguous())
    assert e.value.status == 2


@pytest.mark.parametrize("n,m,d", [(70_000, 32_768, 16), (70_000, 5, 65_536), (3, 70_000, 65_536), (100, 70_000, 65_536)])
def test_scores_offsets_beyond_32_bits(cuda, n, m, d):
    import torch
    import libsdca_amd as sd
    X, sx, W, sw = _operands(cuda, n, m, d, 11)
    S = sd.scores_i8(X, W, sw, x_scales=sx, dtype=torch.bfloat16)
    rows = sorted({0, n // 2, n - 1})
    cols = sorted({0, m // 2, m - 2, m - 1})
    ref.check_scores(_np(S[rows][:, cols]), _np(X[rows]), _np(sx[rows]), _np(W[cols]), _np(sw[cols]), "bfloat16")


# ---------------------------------------------------------------------------
# sample
# ---------------------------------------------------------------------------
def _logits(g, n, m, cuda, kind):
    import torch
    S = torch.randn((n, m), generator=g, device=cuda) * 1.5
    head = max(1, min(200, m // 2))
    at = torch.randint(0, m, (n, head), generator=g, device=cuda)
    S.scatter_(1, at, 12 - 1.2 * torch.arange(1, head + 1, device=cuda).float().log().expand(n, head))
    return S.to(getattr(torch, kind))


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=20), dict(top_p=0.9),
            dict(min_p=0.05), dict(temperature=1.3, top_k=50, top_p=0.95, min_p=0.01), dict(top_k=1),
            dict(temperature=3.0, top_p=0.99), dict(temperature=2.0, top_k=300), dict(top_p=1e-6),
            dict(temperature=0.01, min_p=1.0), dict(temperature=50.0, top_k=700, top_p=0.5)]


def _check(S, u, out, **kw):
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    vals = [_np(v) if hasattr(v, "cpu") else np.float32(v) if name != "top_k" else v for name, v in full.items()]
    label, prob, kept = (_np(v) for v in out)
    ref.check_sample(_np(S), _np(u), *vals, label, prob, kept)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,m", [(3, 1), (4, 2), (5, 63), (7, 100), (9, 1000), (3, 1025), (4, 4097), (3, 9001),
                                 (2, 33_333), (2, 131_075)])
def test_sample_settings(cuda, kind, n, m):
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, n * m)
    S = _logits(g, n, m, cuda, kind)
    for kw in SETTINGS:
        print(kind, n, m, kw, flush=True)
        u = torch.rand(n, generator=g, device=cuda)
        out = sd.sample(S, u, prob=True, kept=True, **kw)
        _check(S, u, out, **kw)
        # the same from rows apart
        for got, want in zip(sd.sample(_spaced(S, m + 7), u, prob=True, kept=True, **kw), out):
            assert torch.equal(got, want)
        assert torch.equal(sd.sample(S, u, **kw), out[0])


@pytest.mark.parametrize("kind,n,m", [("float32", 300, 70_001), ("float16", 300, 70_001), ("bfloat16", 90, 20_000),
                                      ("float32", 70, 32_769), ("float64", 66, 17_000)])
def test_sample_many_long_columns(cuda, kind, n, m):
    """A workgroup to a column that its registers do not hold, or just hold;
    nuclei of a few labels and of very many."""
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, n + m)
    S = _logits(g, n, m, cuda, kind)
    S[: n // 8] = S[: n // 8] / 8  # nearly even
    for kw in (dict(temperature=0.8, top_k=50, top_p=0.9), dict(top_p=0.95), dict(temperature=1.5, top_p=0.97, min_p=1e-5),
               dict(min_p=0.01), dict(top_k=900, top_p=0.99)):
        print(kind, n, m, kw, flush=True)
        u = torch.rand(n, generator=g, device=cuda)
        out = sd.sample(S, u, prob=True, kept=True, **kw)
        _check(S, u, out, **kw)
        # a few of the columns alone go another way, to the same labels
        few = sd.sample(S[:9], u[:9], prob=True, kept=True, **kw)
        for a, b in zip(few, out):
            assert torch.equal(a, b[:9])


@pytest.mark.parametrize("n,m", [(300, 50), (200, 1000), (60, 5000), (12, 40_000)])
def test_sample_settings_of_their_own(cuda, n, m):
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, 3 * n + m)

    def some(values, dtype=torch.float32):
        a = torch.tensor(values, device=cuda, dtype=dtype)
        return a[torch.randint(0, len(a), (n,), generator=g, device=cuda)].contiguous()

    S = _logits(g, n, m, cuda, "float32")
    kw = dict(temperature=some([0.0, 0.5, 1.0, 2.0]), top_k=some([0, 1, 5, 40, m, m + 5], torch.int64),
              top_p=some([0.5, 0.9, 1.0]), min_p=some([0.0, 0.02, 0.3]))
    u = torch.rand(n, generator=g, device=cuda)
    out = sd.sample(S, u, prob=True, kept=True, **kw)
    _check(S, u, out, **kw)
    # a column's label does not hang on its neighbours
    rows = torch.arange(0, n, 3, device=cuda)
    part = sd.sample(S[rows].contiguous(), u[rows].contiguous(), prob=True, kept=True,
                     **{name: v[rows].contiguous() for name, v in kw.items()})
    for a, b in zip(part, out):
        assert torch.equal(a, b[rows])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 70, 1000, 3000, 20_000, 140_000])
def test_sample_masked_rows(cuda, kind, m):
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, m)
    dt = getattr(torch, kind)
    low = torch.finfo(dt).min
    S = _logits(g, 12, m, cuda, kind)
    shut = torch.rand((12, m), generator=g, device=cuda) > 3 / m
    S[1].masked_fill_(shut[1], -float("inf"))
    S[2].masked_fill_(shut[2], low)
    S[3] = -float("inf")
    S[4] = low                      # no label ahead of another: each as likely
    S[5] = float("nan")
    S[6, m // 2] = float("nan")
    S[7, m // 3] = float("inf")
    S[7, m - 1] = float("inf")
    S[8] = 0.0
    S[8, ::2] = -0.0                # one value
    S[9] = float("-inf")
    S[9, m - 1] = low               # a single label, however low
    S[10, : m // 2] = float("-inf")
    S[11] = 1.0
    S[11, 0] = float("nan")
    for kw in SETTINGS:
        u = torch.rand(12, generator=g, device=cuda)
        u[11] = 0.0
        out = sd.sample(S, u, prob=True, kept=True, **kw)
        Sd = S.double()
        if kind == "float64":  # doubles are rounded to float first
            Sd = S.float().double()
        _check(Sd, u, out, **kw)


@pytest.mark.parametrize("m", [64, 1000, 2048, 5000, 50_000])
def test_sample_equal_scores(cuda, m):
    """Equal scores: every sum is a whole number of equal weights, so the
    label is known exactly, and top-k keeps the first k."""
    import torch
    import libsdca_amd as sd
    n = 40
    g = _gen(cuda, m)
    S = torch.full((n, m), -3.25, device=cuda)
    u = torch.rand(n, generator=g, device=cuda)
    for k in (0, 1, 7, m // 2, m - 1):
        count = k if k else m
        label, prob, kept = sd.sample(S, u, top_k=k, prob=True, kept=True)
        assert bool((kept == count).all())
        assert torch.equal(label, torch.floor(u.double() * count).long())
        assert torch.equal(prob, torch.full((n,), 1.0 / count, device=cuda))
    label, kept = sd.sample(S, u, top_p=0.25, kept=True)
    count = -(-m // 4)
    assert bool((kept == count).all()) and torch.equal(label, torch.floor(u.double() * count).long())
    # half of them a step below: top-k cuts inside the lower ones
    S[:, ::2] = -4.25
    k = m // 2 + m // 4
    label, kept = sd.sample(S, u, top_k=k, kept=True)
    assert bool((kept == k).all())
    assert bool(((label % 2 == 1) | (label < 2 * (m // 4))).all())


def test_sample_ends_of_the_interval(cuda):
    import torch
    import libsdca_amd as sd
    S = torch.tensor([[0.0, -float("inf"), 1.0, 2.0, -float("inf")]] * 5, device=cuda)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, float("nan")], device=cuda)
    assert sd.sample(S, u).tolist() == [0, 3, 3, 0, 0]  # what lies outside is brought in
    # settings in device memory outside their ranges
    bad = dict(temperature=torch.tensor([-1.0, float("nan"), 1.0, 1.0, 1.0], device=cuda),
               top_k=torch.tensor([-3, 2 ** 40, 9, -2 ** 62, 1], device=cuda),
               top_p=torch.tensor([2.0, float("nan"), -1.0, 0.0, float("inf")], device=cuda),
               min_p=torch.tensor([-1.0, float("nan"), 0.0, 7.0, float("nan")], device=cuda))
    half = torch.full((5,), 0.5, device=cuda)
    label, kept = sd.sample(S, half, kept=True, **bad)
    assert label.tolist() == [3, 3, 3, 3, 3] and kept.tolist() == [1, 1, 1, 1, 1]
    label, kept = sd.sample(S, half, kept=True, min_p=bad["min_p"], top_p=torch.ones(5, device=cuda))
    assert kept.tolist() == [3, 3, 3, 1, 3]


def test_sample_frequencies(cuda):
    """Over an even grid of random numbers each label comes as often as its
    probability says, to one draw."""
    import torch
    import libsdca_amd as sd
    n, m = 20_000, 37
    row = torch.randn(m, generator=_gen(cuda, 4), device=cuda)
    u = ((torch.arange(n, device=cuda) + 0.5) / n).float()
    label = sd.sample(row.expand(n, m).contiguous(), u, temperature=0.9)
    want = torch.softmax(row.double() / 0.9, 0) * n
    seen = torch.bincount(label, minlength=m).double()
    assert bool(((seen - want).abs() <= 1.01).all())
    assert bool((label[1:] >= label[:-1]).all())


def test_sample_offsets_beyond_32_bits(cuda):
    import torch
    import libsdca_amd as sd
    n, m = 8200, 262_144
    S = torch.full((n, m), -30000.0, dtype=torch.float16, device=cuda)
    at = torch.randint(0, m, (n,), generator=_gen(cuda, 5), device=cuda)
    S[torch.arange(n, device=cuda), at] = 1.0
    u = torch.rand(n, generator=_gen(cuda, 6), device=cuda)
    for kw in (dict(), dict(top_k=3, top_p=0.9), dict(temperature=0.0)):
        assert torch.equal(sd.sample(S, u, **kw), at), kw


# ---------------------------------------------------------------------------
# Streams, captures, host arrays, nothing to do.
# ---------------------------------------------------------------------------
def test_answer_on_another_stream_and_captured(cuda):
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, 8)
    shapes = [(1, 3000, 513), (40, 3000, 513), (300, 9000, 256)]
    data, want = [], []
    for n, m, d in shapes:
        X = torch.randn((n, d), generator=g, device=cuda)
        W, sw = sd.quantize_i8(torch.randn((m, d), generator=g, device=cuda) * 0.2)
        u = torch.rand(n, generator=g, device=cuda)
        data.append((X, W, sw, u))

    def step(X, W, sw, u):
        S = sd.scores_i8(X, W, sw)
        return (S,) + sd.sample(S, u, temperature=0.8, top_k=40, top_p=0.9, prob=True, kept=True)

    for a in data:
        want.append(step(*a))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(2):
        with torch.cuda.stream(side):
            got = [step(*a) for a in data]
        side.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = [step(*a) for a in data]
    for rep in range(4):
        for a in got:
            for t in a:
                t.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), rep
        again = step(*data[rep % 3])  # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(again, want[rep % 3]))
    # new inputs in the captured buffers
    data[0][0].mul_(-1.5)
    eager = step(*data[0])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got[0], eager))


def test_answer_host_arrays(cuda):
    """numpy arrays give what tensors give."""
    import torch
    import libsdca_amd as sd
    rng = np.random.default_rng(9)
    X = rng.standard_normal((20, 77)).astype(np.float32)
    A = rng.standard_normal((50, 80)).astype(np.float16)[:, :77]
    W, sw = sd.quantize_i8(A)
    dW, dsw = sd.quantize_i8(torch.from_numpy(A.copy()).to(cuda))
    assert np.array_equal(W, _np(dW)) and np.array_equal(sw, _np(dsw))
    out = np.full((20, 60), -9, np.float32)
    S = sd.scores_i8(X, W, sw, out=out[:, :50])
    dS = sd.scores_i8(torch.from_numpy(X).to(cuda), dW, dsw)
    assert np.array_equal(S, _np(dS)) and (out[:, 50:] == -9).all()
    u = rng.random(20).astype(np.float32)
    kw = dict(temperature=np.full(20, 0.7, np.float32), top_k=9, top_p=[0.9] * 20, min_p=0.01)
    got = sd.sample(S, u, prob=True, kept=True, **kw)
    want = sd.sample(dS, torch.from_numpy(u).to(cuda), prob=True, kept=True, **kw)
    assert all(np.array_equal(a, _np(b)) for a, b in zip(got, want))


def test_answer_nothing_to_do(cuda):
    import torch
    import libsdca_amd as sd
    W, sw = sd.quantize_i8(torch.ones((5, 32), device=cuda))
    assert tuple(sd.scores_i8(torch.ones((0, 32), device=cuda), W, sw).shape) == (0, 5)
    assert tuple(sd.sample(torch.ones((0, 5), device=cuda), torch.ones(0, device=cuda)).shape) == (0,)
    q, s = sd.quantize_i8(torch.ones((0, 32), device=cuda))
    assert tuple(q.shape) == (0, 32) and tuple(s.shape) == (0,)
