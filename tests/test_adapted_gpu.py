"""sdca_scores_adapted and sdca_scores_adapted_grad against their plain forms
in 64 bits (tests/adapted_oracle.py)."""
import numpy as np
import pytest

from tests import adapted_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": (2.0 ** -24, 2.0 ** -149), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}
# n, d, m, rank, adapters: the kernels for one and two examples, for few
# classes, tiles of 64, 128 and 256; ranks around 4, 16, 32, 64 and the most
SHAPES = [(1, 1, 1, 1, 1), (1, 4096, 1000, 8, 4), (2, 513, 70, 5, 3), (2, 1024, 9000, 16, 2), (3, 100, 300, 3, 2),
          (5, 17, 137, 128, 2), (31, 513, 137, 10, 3), (33, 64, 256, 16, 40), (48, 600, 513, 17, 5),
          (64, 128, 1024, 33, 3), (65, 4100, 65, 64, 2), (130, 1030, 1001, 65, 4), (200, 256, 700, 31, 1),
          (257, 300, 515, 100, 7), (700, 2048, 600, 16, 3), (1111, 130, 2050, 8, 20), (3000, 72, 1030, 4, 2),
          # terms of many examples together: each number of ranks, in parts and not, 16 and 32 to a workgroup
          (600, 301, 270, 100, 7), (1111, 130, 300, 32, 20), (700, 521, 300, 61, 3), (2200, 300, 280, 16, 5),
          (4100, 200, 300, 32, 4), (4300, 77, 270, 64, 2), (4099, 64, 260, 128, 3)]


def _gen(cuda, seed):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _np(t):
    import torch
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _spaced(t, pitch):
    import torch
    n, d = t.shape
    buf = torch.zeros((n, pitch), dtype=t.dtype, device=t.device)
    buf.fill_(77 if t.dtype == torch.int8 else float("nan"))
    buf[:, :d] = t
    return buf[:, :d]


def _index(cuda, n, count, how, g):
    import torch
    if how == "one":
        return torch.full((n,), count - 1, device=cuda)
    if how == "none":
        return torch.full((n,), -1, device=cuda)
    if how == "mixed":
        return torch.randint(-1, count, (n,), generator=g, device=cuda)
    return torch.sort(torch.randint(-1, count, (n,), generator=g, device=cuda)).values


def _operands(cuda, n, d, m, r, count, kind, how, seed):
    import torch
    import libsdca_amd as sd
    g = _gen(cuda, seed)
    dt = getattr(torch, kind)
    X = torch.randn((n, d), generator=g, device=cuda).to(dt)
    W, sw = sd.quantize_i8(torch.randn((m, d), generator=g, device=cuda) / d ** 0.5)
    A = (torch.randn((count, r, d), generator=g, device=cuda) / d ** 0.5).to(dt)
    B = (torch.randn((count, m, r), generator=g, device=cuda) / r ** 0.5).to(dt)
    scale = 0.25 + torch.rand(count, generator=g, device=cuda)
    return X, W, sw, A, B, _index(cuda, n, count, how, g), scale


def _check(S, X, W, sw, A, B, index, scale, kind):
    ref.check_scores(_np(S), _np(X), _np(W), _np(sw), _np(A), _np(B), _np(index),
                     scale if isinstance(scale, float) else _np(scale), *HALF_STEP[kind])


@pytest.mark.parametrize("n,d,m,r,count", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
def test_scores(cuda, n, d, m, r, count, kind):
    import torch
    import libsdca_amd as sd
    print(n, d, m, r, count, kind, flush=True)
    for how in ("mixed", "one", "runs"):
        X, W, sw, A, B, index, scale = a = _operands(cuda, n, d, m, r, count, kind, how, n + d + m)
        for out in {"float32", kind, "bfloat16"}:
            S = sd.scores_adapted(X, W, sw, A, B, index, scale=scale, dtype=getattr(torch, out))
            assert tuple(S.shape) == (n, m) and S.dtype == getattr(torch, out)
            _check(S, *a, out)
            # rows apart, at odd addresses, W not in place, into a given matrix
            buf = torch.full((n, m + 3), -7, dtype=S.dtype, device=cuda)
            got = sd.scores_adapted(_spaced(X, d + 3), _spaced(W, d + 1), sw, A, B, index, scale=scale, out=buf[:, :m])
            assert torch.equal(got, S) and bool((buf[:, m:] == -7).all())
        S = sd.scores_adapted(X, W, sw, A, B, index, scale=0.5)
        _check(S, X, W, sw, A, B, index, 0.5, "float32")


@pytest.mark.parametrize("n,d,m", [(1, 2048, 500), (2, 600, 300), (40, 77, 100), (40, 700, 900), (300, 300, 500)])
@pytest.mark.parametrize("kind", KINDS)
def test_no_adapter_is_scores_i8(cuda, n, d, m, kind):
    import torch
    import libsdca_amd as sd
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, 8, 3, kind, "none", n)
    assert torch.equal(sd.scores_adapted(X, W, sw, A, B, index), sd.scores_i8(X, W, sw))


@pytest.mark.parametrize("n,d,m", [(2, 600, 300), (40, 77, 100), (80, 700, 900), (1200, 300, 500)])
@pytest.mark.parametrize("kind", KINDS)
def test_adapters_do_not_meet(cuda, n, d, m, kind):
    """An adapter of infinities and NaN, and an index outside, reach their own
    examples alone; the others are as they are without them, bit for bit."""
    import torch
    import libsdca_amd as sd
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, 6, 4, kind, "mixed", n)
    index[0], index[n - 1] = 1, 2
    want = sd.scores_adapted(X, W, sw, A, B, index, scale=scale)
    A2, B2 = A.clone(), B.clone()
    A2[1] = float("inf")
    B2[1] = float("nan")
    got = sd.scores_adapted(X, W, sw, A2, B2, index, scale=scale)
    own = index == 1
    assert torch.equal(got[~own], want[~own]) and bool(torch.isnan(got[own]).all())
    G = torch.randn((n, m), generator=_gen(cuda, 1), device=cuda).to(X.dtype)
    dA, dB = sd.scores_adapted_grad(G, X, A, B, index, scale=scale)
    dA2, dB2 = sd.scores_adapted_grad(G, X, A2, B2, index, scale=scale)
    for a in (0, 2, 3):
        assert torch.equal(dA[a], dA2[a]) and torch.equal(dB[a], dB2[a])
    bad = index.clone()
    bad[0], bad[1] = 4, -2
    got = sd.scores_adapted(X, W, sw, A, B, bad, scale=scale)
    assert bool(torch.isnan(got[:2]).all())
    if n > 2:
        assert torch.equal(got[2:], want[2:])
    bad[0] = bad[1] = 2 ** 40
    got = sd.scores_adapted(X, W, sw, A, B, bad, scale=scale)
    assert bool(torch.isnan(got[:2]).all())
    none = index.clone()
    none[:2] = -1
    for x, y in zip(sd.scores_adapted_grad(G, X, A, B, bad, scale=scale), sd.scores_adapted_grad(G, X, A, B, none, scale=scale)):
        assert torch.equal(x, y)
    # an example with a NaN spoils its own scores, and its adapter's gradients
    X2 = X.clone()
    X2[0, d - 1] = float("nan")
    got = sd.scores_adapted(X2, W, sw, A, B, index, scale=scale)
    assert bool(torch.isnan(got[0]).all()) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("n,d,m,r,count", SHAPES + [(5000, 100, 90, 16, 3), (4000, 33, 600, 70, 1), (900, 50, 60, 8, 300)])
@pytest.mark.parametrize("kind", KINDS)
def test_gradients(cuda, n, d, m, r, count, kind):
    import torch
    import libsdca_amd as sd
    print(n, d, m, r, count, kind, flush=True)
    for how in ("mixed", "one", "runs", "none"):
        X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, r, count, kind, how, n + d + m)
        G = torch.randn((n, m), generator=_gen(cuda, n), device=cuda)
        for g in {"float32", kind, "float16"}:
            Gk = G.to(getattr(torch, g))
            got = sd.scores_adapted_grad(Gk, X, A, B, index, scale=scale)
            assert all(v.dtype == torch.float32 for v in got)
            ref.check_grads([_np(v) for v in got], _np(Gk), _np(X), _np(A), _np(B), _np(index), _np(scale))
            far = sd.scores_adapted_grad(_spaced(Gk, m + 3), _spaced(X, d + 5), A, B, index, scale=scale)
            assert all(torch.equal(x, y) for x, y in zip(got, far))


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("n", [5, 200])
def test_small_values(cuda, kind, n):
    """Gradients, examples and adapters among the type's subnormal numbers,
    as probabilities far from the label's are, and terms far apart."""
    import torch
    import libsdca_amd as sd
    d, m, r = 300, 200, 20
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, r, 3, kind, "mixed", n)
    dt = X.dtype
    small = 2.0 ** (-20 if kind == "float16" else -126)
    G = (torch.randn((n, m), generator=_gen(cuda, 1), device=cuda) * small).to(dt)
    assert bool((G != 0).any())
    got = sd.scores_adapted_grad(G, X, A, B, index, scale=scale)
    if kind == "float16":  # (the sums of the others are no ordinary floats themselves)
        ref.check_grads([_np(v) for v in got], _np(G), _np(X), _np(A), _np(B), _np(index), _np(scale))
    A2 = (A.float() * torch.logspace(-6, 2, r, device=cuda)[None, :, None]).to(dt)
    for X2, B2 in ((X, B), ((X.float() * 2.0 ** -14).to(dt), B), (X, (B.float() * 2.0 ** -18).to(dt))):
        S = sd.scores_adapted(X2, W, sw, A2, B2, index, scale=scale)
        _check(S, X2, W, sw, A2, B2, index, scale, "float32")
        ref.check_grads([_np(v) for v in sd.scores_adapted_grad(G.float(), X2, A2, B2, index, scale=scale)],
                        _np(G.float()), _np(X2), _np(A2), _np(B2), _np(index), _np(scale))


def test_offsets_beyond_32_bits(cuda):
    import torch
    import libsdca_amd as sd
    if torch.cuda.mem_get_info(cuda)[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GiB of device memory")
    n, d, m, r = 70_000, 64, 33_000, 4
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, r, 2, "bfloat16", "mixed", 1)
    S = sd.scores_adapted(X, W, sw, A, B, index, scale=scale, dtype=torch.bfloat16)
    last = slice(n - 40, n)
    _check(S[last], X[last], W, sw, A, B, index[last], scale, "bfloat16")
    G = torch.zeros((n, m), dtype=torch.bfloat16, device=cuda)
    G[last] = S[last]
    dA, dB = sd.scores_adapted_grad(G, X, A, B, index, scale=scale)
    args = [_np(v) for v in (G[last], X[last], A, B, index[last], scale)]
    ref.check_grads([_np(dA), _np(dB)], *args)
    del S, G
    # adapters whose matrices lie beyond 2^32 bytes
    count, m = 40, 1_000_000
    A = torch.zeros((count, 128, d), dtype=torch.float16, device=cuda)
    B = torch.zeros((count, m, 128), dtype=torch.float16, device=cuda)
    A[-1].normal_(generator=_gen(cuda, 2))
    B[-1, -100:].normal_(generator=_gen(cuda, 3))
    W = torch.zeros((m, d), dtype=torch.int8, device=cuda)
    sw = torch.ones(m, device=cuda)
    index = torch.full((3,), count - 1, device=cuda)
    X = X[:3].half()
    S = sd.scores_adapted(X, W, sw, A, B, index)
    _check(S[:, -100:], X, W[-100:], sw[-100:], A, B[:, -100:], index, 1.0, "float32")
    assert not bool(S[:, :-100].any())


def test_more_examples_than_a_grid_row(cuda):
    """More examples than 65535 tiles and workgroups in a row."""
    import torch
    import libsdca_amd as sd
    n, d, m, r = 2 ** 21 + 3, 8, 5, 2
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, r, 3, "float16", "mixed", 6)
    S = sd.scores_adapted(X, W, sw, A, B, index, scale=scale)
    for part in (slice(0, 100), slice(n - 100, n)):
        _check(S[part], X[part], W, sw, A, B, index[part], scale, "float32")
    want = sd.scores_i8(X, W, sw).double()
    for a in range(3):
        T = (X.double() @ A[a].double().T) * scale[a].double()
        want += torch.where((index == a)[:, None], T @ B[a].double().T, 0.0)
    assert float((S.double() - want).abs().max()) < 1e-5
    G = torch.ones((n, m), device=cuda)
    dA, dB = sd.scores_adapted_grad(G, X, A, B, index, scale=scale)
    for a in range(3):
        rows = (index == a).double()[:, None]
        U = scale[a].double() * B[a].double().sum(dim=0)
        want = U[:, None] * (X.double() * rows).sum(dim=0)
        # sums of 7e5 terms of size 1
        assert float((dA[a].double() - want).abs().max()) < 0.2
        T = ((X.double() @ A[a].double().T) * scale[a].double() * rows).sum(dim=0)
        assert float((dB[a].double() - T).abs().max()) < 0.2


def test_another_stream_and_captured(cuda):
    import torch
    import libsdca_amd as sd
    data, want = [], []
    for i, (n, d, m) in enumerate(((1, 3000, 513), (40, 513, 3000), (300, 256, 9000), (30, 100, 200))):
        a = _operands(cuda, n, d, m, 9, 3, "bfloat16", "mixed", i)
        data.append(a + (torch.randn((n, m), generator=_gen(cuda, i), device=cuda),))

    def step(X, W, sw, A, B, index, scale, G):
        return (sd.scores_adapted(X, W, sw, A, B, index, scale=scale),) + sd.scores_adapted_grad(G, X, A, B, index, scale=scale)

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
        again = step(*data[rep])
        assert all(torch.equal(x, y) for x, y in zip(again, want[rep]))


def test_host_arrays(cuda):
    import torch
    import libsdca_amd as sd
    for n, d, m, r in ((20, 77, 50, 5), (1, 600, 90, 4)):
        X, W, sw, A, B, index, scale = a = _operands(cuda, n, d, m, r, 3, "float16", "mixed", n)
        G = torch.randn((n, m), generator=_gen(cuda, n), device=cuda)
        want = (sd.scores_adapted(X, W, sw, A, B, index, scale=scale),) + sd.scores_adapted_grad(G, X, A, B, index, scale=scale)
        hX, hW, hsw, hA, hB, hi, hs = (_np(v) for v in a)
        out = np.full((n, m + 4), 3, np.float32)
        got = (sd.scores_adapted(hX, hW, hsw, hA, hB, hi, scale=hs, out=out[:, :m]),) + \
            sd.scores_adapted_grad(_np(G), hX, hA, hB, hi, scale=list(hs))
        assert all(np.array_equal(x, _np(y)) for x, y in zip(got, want)) and (out[:, m:] == 3).all()


def test_nothing_to_do(cuda):
    import torch
    import libsdca_amd as sd
    X, W, sw, A, B, index, scale = _operands(cuda, 4, 33, 7, 3, 2, "float32", "mixed", 1)
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert tuple(sd.scores_adapted(X[:0], W, sw, A, B, none).shape) == (0, 7)
    dA, dB = sd.scores_adapted_grad(torch.zeros((0, 7), device=cuda), X[:0], A, B, none)
    assert dA.shape == A.shape and dB.shape == B.shape and not bool(dA.any()) and not bool(dB.any())


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_a_training_step_and_an_answer(cuda, kind):
    """The calls as they are used together: adapted scores, the labels' log-
    probabilities, their gradient, the adapters', a step, and drawn labels."""
    import torch
    import libsdca_amd as sd
    n, d, m, r, count = 150, 200, 300, 8, 3
    X, W, sw, A, B, index, scale = _operands(cuda, n, d, m, r, count, kind, "mixed", 5)
    g = _gen(cuda, 6)
    labels = torch.randint(0, m, (n,), generator=g, device=cuda)
    A, B = A.float(), torch.zeros_like(B).float()
    weight = torch.full((n,), 1.0 / n, device=cuda)
    dt = X.dtype
    for step in range(2):
        S = sd.scores_adapted(X, W, sw, A.to(dt), B.to(dt), index, scale=scale)
        D, logp = sd.log_probs_grad(S, labels, weight, logp=True)
        dA, dB = sd.scores_adapted_grad(D, X, A.to(dt), B.to(dt), index, scale=scale)
        # against autograd of the same step in 64 bits
        a, b = (v.to(dt).double().requires_grad_() for v in (A, B))
        q, sx = sd.quantize_i8(X)
        base = (q.double() @ W.double().T) * sx.double()[:, None] * sw.double()
        some = index >= 0
        at = index.clamp(min=0)
        T = torch.matmul(a[at], X.double()[:, :, None])[:, :, 0] * scale.double()[at, None]
        more = torch.matmul(b[at], T[:, :, None])[:, :, 0]
        full = base + torch.where(some[:, None], more, 0.0)
        want = torch.log_softmax(full, dim=1).gather(1, labels[:, None])[:, 0]
        (want * weight.double()).sum().backward()
        assert float((logp.double() - want.detach()).abs().max()) < 1e-4
        for got, w in ((dA, a.grad), (dB, b.grad)):
            assert float((got.double() - w).norm()) <= 1e-5 * float(w.norm()) + 1e-12
        A += 50 * dA
        B += 50 * dB
    S = sd.scores_adapted(X, W, sw, A.to(dt), B.to(dt), index, scale=scale, dtype=torch.bfloat16)
    label = sd.sample(S, torch.rand(n, generator=g, device=cuda), temperature=0.7, top_k=20)
    assert bool(((label >= 0) & (label < m)).all())
    assert bool(torch.isfinite(sd.log_probs(S, label)).all())
