"""sdca_log_probs and sdca_log_probs_grad against their plain forms in 64 bits
(tests/log_probs_oracle.py)."""
import numpy as np
import pytest

from tests import log_probs_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": (2.0 ** -24, 2.0 ** -149), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}
SHAPES = [(1, 1), (3, 2), (5, 63), (4, 64), (7, 65), (2, 255), (9, 257), (3, 1000), (2, 1024), (3, 1025), (2, 2048),
          (3, 2049), (2, 4097), (3, 5000), (2, 8193), (1, 16_385), (2, 32_768), (1, 32_769), (2, 65_537),
          (1, 100_003), (300, 2100), (520, 2100), (257, 33_000), (256, 70_001)]


def _gen(cuda, seed):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _np(t):
    import torch
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _scores(cuda, n, m, kind, seed, scale=3.0):
    import torch
    g = _gen(cuda, seed)
    S = (torch.randn((n, m), generator=g, device=cuda) * scale).to(getattr(torch, kind))
    labels = torch.randint(0, m, (n,), generator=g, device=cuda)
    labels[::5] = S[::5].float().argmax(dim=1)
    if n > 2:
        labels[2] = -1
    return S, labels


def _spaced(t, pitch):
    import torch
    n, d = t.shape
    buf = torch.full((n, pitch), float("nan"), dtype=t.dtype, device=t.device)
    buf[:, :d] = t
    return buf[:, :d]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,m", SHAPES)
def test_log_probs(cuda, n, m, kind):
    import torch
    import libsdca_amd as sd
    print(n, m, kind, flush=True)
    S, labels = _scores(cuda, n, m, kind, n + m)
    few = slice(0, min(n, 40))
    for T, top in ((1.0, 0), (1.0, 1), (0.7, 5), (2.5, 64)):
        res = sd.log_probs(S, labels, temperature=T, top=top, entropy=True, stats=True)
        logp, H, stats = (_np(v) for v in res[:3])
        best = tuple(_np(v)[few] for v in res[3:]) if top else None
        ref.check(_np(S)[few], _np(labels)[few], T, logp[few], H[few], stats[few], best)
        # rows apart, at odd addresses
        far = sd.log_probs(_spaced(S, m + 3), labels, temperature=T, top=top, entropy=True, stats=True)
        ref.check(_np(S)[few], _np(labels)[few], T, *(_np(v)[few] for v in far[:3]), tuple(_np(v)[few] for v in far[3:]) or None)
        if top:
            assert torch.equal(res[4], far[4])
        if n > 40:
            assert torch.equal(logp_of(S, labels, T).isfinite(), res[0].isfinite())
            assert float((logp_of(S, labels, T) - res[0]).abs().max()) < 1e-4
    alone = sd.log_probs(S, labels)
    assert alone.shape == (n,) and alone.dtype == torch.float32


def logp_of(S, labels, T):
    import torch
    lp = torch.log_softmax(S.double() / T, dim=1).gather(1, labels.clamp(min=0)[:, None])[:, 0]
    return torch.where(labels >= 0, lp, 0.0).float()


def _special(cuda, m, kind):
    import torch
    S, labels = _scores(cuda, 16, m, kind, m, 4.0)
    low = torch.finfo(S.dtype).min
    high = torch.finfo(S.dtype).max
    inf = float("inf")
    S[0] = -inf                      # nothing left
    S[1, :] = -inf
    S[1, m // 2] = 1.5               # one left
    S[2] = low                       # equal, at the lowest value
    S[3, ::2] = low
    S[4, 1::2] = -inf
    S[5, m - 1] = float("nan")
    S[6] = float("nan")
    S[7, 0] = inf                    # infinite scores share
    S[7, m - 1] = inf
    S[8] = high
    S[9, m // 3] = high
    S[10] = 0.0
    S[10, 1::2] = -0.0               # equal
    S[11] = -inf
    S[11, m - 1] = low
    S[12] += 1000
    S[13, : max(1, m - 3)] = -inf
    S[14] = torch.linspace(-20, 20, m, device=cuda).to(S.dtype)    # rising
    S[15, 0] = inf
    S[15, m - 1] = float("nan")
    labels[1], labels[7], labels[9], labels[11], labels[13] = m // 2, 0, m // 3, m - 1, m - 1
    return S, labels


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [7, 130, 1000, 3000, 9000, 40_000, 70_000])
@pytest.mark.parametrize("T", [1.0, 0.05, 30.0])
def test_special_rows(cuda, m, kind, T):
    import torch
    import libsdca_amd as sd
    print(m, kind, T, flush=True)
    S, labels = _special(cuda, m, kind)
    for top in (0, 3, 64):
        res = [_np(v) for v in sd.log_probs(S, labels, temperature=T, top=top, entropy=True, stats=True)]
        ref.check(_np(S), _np(labels), T, res[0], res[1], res[2], tuple(res[3:]) or None)
    g = torch.randn(16, generator=_gen(cuda, 3), device=cuda)
    h = torch.randn(16, generator=_gen(cuda, 4), device=cuda)
    stats = sd.log_probs(S, labels, temperature=T, stats=True)[1]
    for hh in (None, h):
        for st in (None, stats):
            D, lp = sd.log_probs_grad(S, labels, g, g_entropy=hh, stats=st, temperature=T, logp=True)
            ref.check_grad(_np(D), _np(S), _np(labels), _np(g).astype(np.float64), None if hh is None else _np(hh), T, *HALF_STEP[kind])
            ref.check(_np(S), _np(labels), T, _np(lp))


@pytest.mark.parametrize("m", [100, 3000, 70_000])
def test_labels_outside(cuda, m):
    import torch
    import libsdca_amd as sd
    S, labels = _scores(cuda, 8, m, "float32", m)
    labels[0], labels[1], labels[2], labels[3] = m, -2, -1, 2 ** 40
    logp = sd.log_probs(S, labels)
    assert bool(torch.isnan(logp[[0, 1, 3]]).all()) and float(logp[2]) == 0 and bool(torch.isfinite(logp[4:]).all())
    g = torch.ones(8, device=cuda)
    for stats in (None, sd.log_probs(S, labels, stats=True)[1]):
        D, lp = sd.log_probs_grad(S, labels, g, stats=stats, logp=True)
        assert bool(torch.isnan(D[[0, 1, 3]]).all()) and bool((D[2] == 0).all()) and bool(torch.isfinite(D[4:]).all())
        assert bool(torch.isnan(lp[[0, 1, 3]]).all()) and float(lp[2]) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [64, 1000, 5000, 33_001])
def test_alternatives_of_equal_and_rising_scores(cuda, m, kind):
    """Every score a candidate: many ties, and rows that rise throughout."""
    import torch
    import libsdca_amd as sd
    dt = getattr(torch, kind)
    g = _gen(cuda, m)
    S = torch.randint(0, 3, (6, m), generator=g, device=cuda).to(dt)
    S[0] = 1
    S[1] = torch.arange(m, device=cuda).to(dt)
    S[2] = -torch.arange(m, device=cuda).float().to(dt)
    S[3, :] = 0
    S[3, m - 1] = 1
    labels = torch.zeros(6, dtype=torch.int64, device=cuda)
    for top in (1, 2, 33, 64):
        res = [_np(v) for v in sd.log_probs(S, labels, top=top)]
        ref.check(_np(S), _np(labels), 1.0, res[0], top=(res[1], res[2]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,m", SHAPES + [(5, 20_000), (2, 140_000)])
def test_gradient(cuda, n, m, kind):
    import torch
    import libsdca_amd as sd
    print(n, m, kind, flush=True)
    S, labels = _scores(cuda, n, m, kind, n * m)
    gen = _gen(cuda, 1)
    g, h = torch.randn(n, generator=gen, device=cuda), torch.randn(n, generator=gen, device=cuda)
    few = slice(0, min(n, 24))
    for T, hh in ((1.0, None), (0.7, h), (1.5, h)):
        logp, stats = sd.log_probs(S, labels, temperature=T, stats=True)
        whole = None
        for st in (None, stats):
            D = sd.log_probs_grad(S, labels, g, g_entropy=hh, stats=st, temperature=T)
            assert D.dtype == S.dtype
            ref.check_grad(_np(D)[few], _np(S)[few], _np(labels)[few], _np(g)[few].astype(np.float64),
                           None if hh is None else _np(hh)[few], T, *HALF_STEP[kind])
            # rows apart, into a given matrix whose other values stay, and in place
            out = torch.full((n, m + 5), 7.0, dtype=S.dtype, device=cuda)
            far, lp = sd.log_probs_grad(_spaced(S, m + 3), labels, g, g_entropy=hh, stats=st, temperature=T,
                                        out=out[:, :m], logp=True)
            ref.check_grad(_np(far)[few], _np(S)[few], _np(labels)[few], _np(g)[few].astype(np.float64),
                           None if hh is None else _np(hh)[few], T, *HALF_STEP[kind])
            assert bool((out[:, m:] == 7).all())
            assert float((lp - logp).abs().max()) <= 1e-5 * (1 + float(logp.abs().max()))
            own = S.clone()
            got, lp2 = sd.log_probs_grad(own, labels, g, g_entropy=hh, stats=st, temperature=T, out=own, logp=True)
            assert got is own and torch.equal(own, D)
            assert float((lp2 - lp).abs().max()) <= 1e-5 * (1 + float(logp.abs().max()))
            if n > 24:
                if whole is not None:
                    assert float((D.float() - whole).abs().max()) <= 2 * HALF_STEP[kind][0] * float(whole.abs().max()) + 1e-5
                whole = D.float()


def test_gradient_sums_to_nothing(cuda):
    """Shifting a row's scores changes nothing, so a gradient sums to zero."""
    import torch
    import libsdca_amd as sd
    S, labels = _scores(cuda, 50, 1000, "float32", 9)
    g = torch.randn(50, generator=_gen(cuda, 2), device=cuda)
    D = sd.log_probs_grad(S, labels, g, g_entropy=g * 0.3)
    # 1000 terms of magnitude |D| in all, each off by ~130 half units
    assert bool((D.double().sum(dim=1).abs() <= 200 * 2.0 ** -24 * (D.double().abs().sum(dim=1) + g.abs())).all())


def test_offsets_beyond_32_bits(cuda):
    import torch
    import libsdca_amd as sd
    n, m = 70_000, 32_768
    if torch.cuda.mem_get_info(cuda)[0] < 24 * 2 ** 30:
        pytest.skip("needs 24 GiB of device memory")
    S = torch.zeros((n, m), dtype=torch.bfloat16, device=cuda)
    S[-3:] = torch.randn((3, m), generator=_gen(cuda, 1), device=cuda).bfloat16()
    labels = torch.arange(n, device=cuda) % m
    g = torch.ones(n, device=cuda)
    logp, at = sd.log_probs(S, labels, top=2)[0::2]
    ref.check(_np(S[-3:]), _np(labels[-3:]), 1.0, _np(logp[-3:]))
    assert float((logp[:-3] + np.log(m)).abs().max()) < 1e-4
    assert bool((at[:-3] == torch.tensor([0, 1], device=cuda)).all())
    stats = sd.log_probs(S, labels, stats=True)[1]
    want = sd.log_probs_grad(S[-3:].clone(), labels[-3:].contiguous(), g[-3:].contiguous())
    for st in (None, stats):
        D = sd.log_probs_grad(S, labels, g, stats=st)
        assert float((D[-3:].float() - want.float()).abs().max()) <= 2.0 ** -7
        assert bool((D[0, 1:] == torch.tensor(-1 / m, device=cuda).bfloat16()).all())
        del D


def test_more_columns_than_a_dispatch(cuda):
    """A wave to a column, 2^25 + 5 of them."""
    import torch
    import libsdca_amd as sd
    n, m = 2 ** 25 + 5, 2
    if torch.cuda.mem_get_info(cuda)[0] < 8 * 2 ** 30:
        pytest.skip("needs 8 GiB of device memory")
    print(n, flush=True)
    S = torch.zeros((n, m), dtype=torch.float16, device=cuda)
    S[:, 1] = (torch.arange(n, device=cuda) % 7).half()
    labels = torch.ones(n, dtype=torch.int64, device=cuda)
    logp, H, best, at = sd.log_probs(S, labels, top=1, entropy=True)
    want = sd.log_probs(S[:7], labels[:7])
    assert torch.equal(logp, want[torch.arange(n, device=cuda) % 7])
    assert torch.equal(at[:, 0], (torch.arange(n, device=cuda) % 7 > 0).long())
    g = torch.ones(n, device=cuda)
    few = sd.log_probs_grad(S[:7], labels[:7], g[:7])
    assert torch.equal(sd.log_probs_grad(S, labels, g), few[torch.arange(n, device=cuda) % 7])


def test_another_stream_and_captured(cuda):
    """On another stream, and replayed from two graphs that were captured on
    one stream and run beside each other."""
    import torch
    import libsdca_amd as sd
    data, want = [], []
    for n, m in ((1, 100_000), (40, 3000), (3, 140_000)):
        S, labels = _scores(cuda, n, m, "float32", n + m)
        data.append((S, labels, torch.randn(n, generator=_gen(cuda, n), device=cuda)))

    def step(S, labels, g):
        res = sd.log_probs(S, labels, top=7, entropy=True, stats=True)
        return res + (sd.log_probs_grad(S, labels, g, g_entropy=g, stats=res[2]), sd.log_probs_grad(S, labels, g))

    for a in data:
        want.append(step(*a))
    torch.cuda.synchronize()
    side, more = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [step(*a) for a in data]
    side.synchronize()
    assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append([step(*a) for a in data])
        graphs.append(graph)
    for rep in range(3):
        for out in outs:
            for a in out:
                for t in a:
                    t.fill_(-5)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(more):
            graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(x, y) for a, b in zip(out, want) for x, y in zip(a, b)), rep
        again = step(*data[rep])  # eager work between the replays
        assert all(torch.equal(x, y) for x, y in zip(again, want[rep]))


def test_host_arrays(cuda):
    import torch
    import libsdca_amd as sd
    for n, m in ((20, 77), (2, 70_000)):
        rng = np.random.default_rng(m)
        wide = rng.standard_normal((n, m + 3)).astype(np.float16)
        S = wide[:, :m]
        labels = rng.integers(0, m, n)
        labels[0] = -1
        g = rng.standard_normal(n).astype(np.float32)
        dS, dl, dg = (torch.from_numpy(v).to(cuda) for v in (wide, labels, g))
        dS = dS[:, :m]  # (sums begin at a multiple of 16 bytes: the same layout, the same bits)
        got = sd.log_probs(S, labels, temperature=0.9, top=4, entropy=True, stats=True)
        want = sd.log_probs(dS, dl, temperature=0.9, top=4, entropy=True, stats=True)
        assert all(np.array_equal(a, _np(b)) for a, b in zip(got, want))
        out = np.full((n, m + 2), 3, np.float16)
        D, lp = sd.log_probs_grad(S, labels, g, g_entropy=g, stats=got[2], temperature=0.9, out=out[:, :m], logp=True)
        dD, dlp = sd.log_probs_grad(dS, dl, dg, g_entropy=dg, stats=want[2], temperature=0.9, logp=True)
        assert np.array_equal(D, _np(dD)) and np.array_equal(lp, _np(dlp)) and (out[:, m:] == 3).all()
        assert np.array_equal(sd.log_probs_grad(S, labels, g), _np(sd.log_probs_grad(dS, dl, dg)))


def test_nothing_to_do(cuda):
    import torch
    import libsdca_amd as sd
    S, l, g = torch.ones((0, 5), device=cuda), torch.ones(0, dtype=torch.int64, device=cuda), torch.ones(0, device=cuda)
    assert [tuple(v.shape) for v in sd.log_probs(S, l, top=2, entropy=True, stats=True)] == [(0,), (0,), (0, 3), (0, 2), (0, 2)]
    assert tuple(sd.log_probs_grad(S, l, g).shape) == (0, 5)


def test_one_label_answers_sample(cuda):
    """The label that `sample` draws from an uncut row has the probability
    that sample gave."""
    import torch
    import libsdca_amd as sd
    S, _ = _scores(cuda, 200, 3000, "float32", 4)
    u = torch.rand(200, generator=_gen(cuda, 5), device=cuda)
    label, prob = sd.sample(S, u, temperature=0.8, prob=True)
    logp = sd.log_probs(S, label, temperature=0.8)
    # each side's sums and exponents are off by some 1e-5 of p at most
    assert bool(((logp.double().exp() - prob.double()).abs() <= 4e-5 * prob.double()).all())
