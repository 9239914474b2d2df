"""sdca_log_probs and sdca_log_probs_grad where scores over the temperature
pass what 32 bits hold to a unit: finite masks, large scores, temperatures near
nothing.  Against the plain forms in 64 bits (tests/log_probs_oracle.py)."""
import numpy as np
import pytest

from tests import log_probs_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": (2.0 ** -24, 2.0 ** -149), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}
MASKS = {"float16": [-3e4, -6e4, -65504.0],
         "float32": [-1e8, -1e9, -5e9, -1e10, -1e12, -1e18, -1e20, -1e25]}
MASKS["bfloat16"] = MASKS["float32"]
# Where M log2(e) / T is 2^24.
EDGE = 2.0 ** 24 * np.log(2)


def _gen(cuda, seed):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _np(t):
    import torch
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _rows(cuda, n, m, kind, T):
    """(S, labels, number of special rows, the first ones)."""
    import torch
    g = _gen(cuda, n + m)
    S = torch.randn((n, m), generator=g, device=cuda) * 4
    labels = torch.randint(0, m, (n,), generator=g, device=cuda)
    most = torch.finfo(getattr(torch, kind)).max
    i = 0
    for v in MASKS[kind]:
        S[i, : m - m // 8 - 1] = v   # whole lanes and waves see masks alone
        labels[i] = m - 1
        S[i + 1, m // 8 + 1:] = v    # masks behind the others
        labels[i + 1] = 0
        S[i + 2] = v                 # nothing but masks
        i += 3
    S[i] = min(1e10, most / 2)
    S[i + 1, m // 3] = min(1e10, most / 2)
    S[i + 2] = (S[i + 2] * 1e9).clamp(-most, most)
    edge = min(EDGE * T, most / 2)
    apart = torch.randint(-20, 21, (2, m), generator=g, device=cuda) * T
    S[i + 3], S[i + 4] = edge + apart[0], -edge + apart[1]
    S[i + 5, ::3] = -2 * edge        # near and far in turn
    S[i + 6] = torch.linspace(-2 * edge, 2 * edge, m, device=cuda)
    S[i + 7] = torch.linspace(2 * edge, -2 * edge, m, device=cuda)
    labels[i + 7] = 0
    return S.to(getattr(torch, kind)), labels, i + 8


def _check(cuda, n, m, kind, T):
    import torch
    import libsdca_amd as sd
    print(n, m, kind, T, flush=True)
    S, labels, some = _rows(cuda, n, m, kind, T)
    few = slice(0, some)
    hS, hl = _np(S[few]), _np(labels[few])
    stats = None
    for top in (0, 3):
        res = sd.log_probs(S, labels, temperature=T, top=top, entropy=True, stats=True)
        stats = res[2]
        host = [_np(v[few]) for v in res]
        ref.check(hS, hl, T, host[0], host[1], host[2], tuple(host[3:]) or None)
    # gradients of the loss in its units: their size does not go with 1 / T
    unit = min(1.0, 1024 * T)
    g = torch.randn(n, generator=_gen(cuda, 3), device=cuda) * unit
    h = torch.randn(n, generator=_gen(cuda, 4), device=cuda) * unit
    for hh, st in ((None, None), (h, None), (h, stats)):
        D, lp = sd.log_probs_grad(S, labels, g, g_entropy=hh, stats=st, temperature=T, logp=True)
        ref.check_grad(_np(D[few]), hS, hl, _np(g[few]).astype(np.float64), None if hh is None else _np(hh[few]), T,
                       *HALF_STEP[kind])
        ref.check(hS, hl, T, _np(lp[few]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [30.0, 1.0, 0.1, 1e-4, 1e-8, 1e-9, 1e-12, 2.0 ** -126])
# a wave to a column, in one vector or four; 4, 16 waves; parts
@pytest.mark.parametrize("m", [60, 900, 3000, 9000, 40_000])
def test_far_scores(cuda, m, T, kind):
    _check(cuda, 32, m, kind, T)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1.0, 1e-9])
# a wave to a longer column; four waves to one, short and long, and the gradient in two passes
@pytest.mark.parametrize("n,m", [(2100, 4000), (300, 5000), (300, 33_000), (520, 40_000)])
def test_far_scores_of_many_columns(cuda, n, m, T, kind):
    _check(cuda, n, m, kind, T)


@pytest.mark.parametrize("n,m", [(1, 2 ** 22), (2, 2 ** 21 + 5)])
def test_sums_of_far_columns_keep_their_digits(cuda, n, m):
    """A long column whose weights come from differences: as few additions
    behind one another as elsewhere (one wave alone would make 2^16)."""
    import torch
    import libsdca_amd as sd
    steps = torch.rand((n, m), generator=_gen(cuda, m), device=cuda)
    S = 3e10 - 2048 * (4 * steps).floor()   # 1e10 is beyond 2^24 at T = 1000
    labels = torch.randint(0, m, (n,), generator=_gen(cuda, 1), device=cuda)
    res = [_np(v) for v in sd.log_probs(S, labels, temperature=1000.0, entropy=True, stats=True)]
    ref.check(_np(S), _np(labels), 1000.0, *res)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [2.0 ** -126, 1e-37, 1e-36, 1e-30])
@pytest.mark.parametrize("n,m", [(12, 40), (12, 900), (12, 3000), (12, 30_000), (12, 70_000), (260, 70_000)])
def test_gradient_of_weights_beyond_the_temperature(cuda, n, m, T, kind):
    """g / T and h / T pass the largest float: labels without weight, and with
    all of it, still have no gradient."""
    import torch
    import libsdca_amd as sd
    print(n, m, kind, T, flush=True)
    S = torch.randint(-30, 30, (n, m), generator=_gen(cuda, m), device=cuda).to(getattr(torch, kind))
    labels = torch.randint(0, m, (n,), generator=_gen(cuda, 1), device=cuda)
    S[torch.arange(n, device=cuda), labels] = 40
    labels[3] = -1
    S[4] *= 1e-38   # (an ordinary column of the smallest numbers, or zeros)
    g = torch.full((n,), 9.0, device=cuda)
    h = torch.full((n,), -3.0, device=cuda)
    g[4] = h[4] = T
    if kind != "float16":   # another label than the largest: a gradient of its size
        labels[5] = (labels[5] + 1) % m
        g[5] = 0.25
    few = slice(0, 12)
    hS, hl = _np(S[few]), _np(labels[few])
    stats = sd.log_probs(S, labels, temperature=T, stats=True)[1]
    for hh, st in ((None, None), (h, None), (None, stats), (h, stats)):
        D, lp = sd.log_probs_grad(S, labels, g, g_entropy=hh, stats=st, temperature=T, logp=True)
        ref.check_grad(_np(D[few]), hS, hl, _np(g[few]).astype(np.float64), None if hh is None else _np(hh[few]), T,
                       *HALF_STEP[kind])
        ref.check(hS, hl, T, _np(lp[few]))
    # a gradient that has no 32-bit value is infinite, the others stay
    g[6], labels[6] = 1e38, (labels[6] + 1) % m
    for st in (None, stats):
        D = sd.log_probs_grad(S, labels, g, stats=st, temperature=T).float()
        top = int(S[6].float().argmax())
        assert D[6, labels[6]] == float("inf") and D[6, top] == -float("inf")
        D[6, labels[6]] = D[6, top] = 0
        assert not bool(D[6].any())
