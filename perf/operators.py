"""The operators that answer from a trained model, as cases that can be timed.

  scores   the scores of n examples for m classes by a product in 8-bit
           integers with a scale for each example and each class; float
           examples are quantised on the way
  sample   a label drawn for each example from its scores: temperature,
           top-k, top-p, min-p, with the random numbers given

`run` computes them in their plain form, or where `own` is true by the
library's entry points.  `exact` restates them in 64 bits, apart from both.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def listed():
    return [
        # The smallest call: one example scored against a thousand classes.
        {"name": "scores_one_f32", "op": "scores", "n": 1, "d": 4096, "m": 1000, "x": "f32", "out": "f32"},
        # One token against a large vocabulary: the weights' bytes count.
        {"name": "scores_token_bf16", "op": "scores", "n": 1, "d": 4096, "m": 128_000, "x": "bf16", "out": "f32"},
        # A decoding step of 32 sequences over the same kind of vocabulary.
        {"name": "scores_step_bf16", "op": "scores", "n": 32, "d": 4096, "m": 65_536, "x": "bf16", "out": "bf16"},
        # A prompt's tokens through a wide projection.
        {"name": "scores_prompt_f16", "op": "scores", "n": 1024, "d": 4096, "m": 14_336, "x": "f16", "out": "f16"},
        # A data set's examples for a thousand classes, as the evaluation has them.
        {"name": "scores_eval_f32", "op": "scores", "n": 20_000, "d": 4096, "m": 1000, "x": "f32", "out": "f32"},
        # Sizes that fit no tile.
        {"name": "scores_odd_f16", "op": "scores", "n": 20_011, "d": 513, "m": 137, "x": "f16", "out": "f16"},
        # The largest: examples quantised by the program beforehand.
        {"name": "scores_large_i8", "op": "scores", "n": 16_384, "d": 8192, "m": 8192, "x": "i8", "out": "bf16"},
        # One token drawn, the smallest call.
        {"name": "sample_one_f32", "op": "sample", "n": 1, "m": 32_000, "x": "f32", "how": "both"},
        # A batch whose requests each bring their own settings; some rows are
        # held to a few allowed tokens by a mask, one has none.
        {"name": "sample_batch_bf16", "op": "sample", "n": 64, "m": 128_000, "x": "bf16", "how": "mixed"},
        # Labels for a data set of a thousand classes, among the best five.
        {"name": "sample_classes_f32", "op": "sample", "n": 20_000, "m": 1000, "x": "f32", "how": "top_k"},
        # The nucleus of an odd vocabulary.
        {"name": "sample_nucleus_f16", "op": "sample", "n": 256, "m": 100_003, "x": "f16", "how": "top_p"},
        # The whole distribution, nothing cut.
        {"name": "sample_all_f32", "op": "sample", "n": 500, "m": 65_537, "x": "f32", "how": "none"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        n, d, m = _log_uniform(rng, 1, 20_011), _log_uniform(rng, 100, 8192), _log_uniform(rng, 100, 128_000)
        if rng.random() < 0.5:  # widths of models are round, those of data sets are not
            d = max(128, d // 64 * 64)
        m = max(100, min(m, 500_000_000 // d, 150_000_000 // n, 1_000_000_000_000 // (n * d)))
        return {"op": "scores", "n": n, "d": d, "m": m, "x": rng.choice(["f32", "f16", "bf16", "i8"]),
                "out": rng.choice(["f32", "f16", "bf16"])}
    m = _log_uniform(rng, 100, 256_000)
    return {"op": "sample", "n": _log_uniform(rng, 1, min(20_000, 32_000_000 // m)), "m": m,
            "x": rng.choice(["f32", "f32", "f16", "bf16"]),
            "how": rng.choice(["top_k", "top_p", "min_p", "both", "mixed", "none"])}


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _quantized(a):
    """(q, s) of the rows of a, the rows of q padded to whole 16 bytes."""
    n, d = a.shape
    s = a.abs().amax(dim=1) / 127
    q = torch.zeros((n, -(-d // 16) * 16), dtype=torch.int8, device=a.device)[:, :d]
    q.copy_(torch.round(a / s[:, None]))
    return q, s


def _scores_input(case, seed):
    """Weights as training leaves them, quantised once; activations with a
    few wide channels."""
    g, n, d, m = _generator(seed), case["n"], case["d"], case["m"]
    Wq = torch.zeros((m, -(-d // 16) * 16), dtype=torch.int8, device=DEV)[:, :d]
    sw = torch.empty(m, dtype=torch.float32, device=DEV)
    step = max(1, (1 << 28) // d)
    for i in range(0, m, step):
        w = torch.randn((min(step, m - i), d), generator=g, device=DEV)
        w *= 0.02 + 0.04 * torch.rand((len(w), 1), generator=g, device=DEV)
        Wq[i:i + step], sw[i:i + step] = _quantized(w)
    X = torch.randn((n, d), generator=g, device=DEV)
    X *= 1 + 9 * (torch.rand(d, generator=g, device=DEV) < 0.01)
    X, sx = _quantized(X) if case["x"] == "i8" else (X.to(TYPES[case["x"]]), None)
    return {"op": "scores", "X": X, "sx": sx, "W": Wq, "sw": sw,
            "out": torch.empty((n, m), dtype=TYPES[case["out"]], device=DEV)}


def _logits(case, g):
    """Most labels in a bulk far below, and a head whose probabilities fall
    off as a power of the rank."""
    n, m = case["n"], case["m"]
    S = torch.randn((n, m), generator=g, device=DEV) * 1.5
    head = min(256, m // 2)
    peak = 14 + 4 * torch.rand((n, 1), generator=g, device=DEV)
    fall = 0.8 + 1.2 * torch.rand((n, 1), generator=g, device=DEV)
    rank = torch.arange(1, head + 1, device=DEV, dtype=torch.float32)
    at = torch.randint(0, m, (n, head), generator=g, device=DEV)
    up = torch.zeros_like(S).scatter_reduce_(1, at, peak - fall * rank.log(), "amax", include_self=False)
    S += up
    return S


def _sample_input(case, seed):
    g, n, m, how = _generator(seed), case["n"], case["m"], case["how"]
    S = _logits(case, g)
    s = {"op": "sample", "u": torch.rand(n, generator=g, device=DEV),
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if how == "top_k":
        s["top_k"] = 5
    elif how == "top_p":
        s["top_p"] = 0.95
    elif how == "min_p":
        s["min_p"] = 0.05
    elif how == "both":
        s.update(temperature=0.8, top_k=50, top_p=0.9)
    elif how == "mixed":
        def some(a):
            a = torch.tensor(a, device=DEV)
            return a[torch.randint(0, len(a), (n,), generator=g, device=DEV)]

        s.update(temperature=some([0.0, 0.5, 0.7, 0.8, 1.0, 1.0, 1.1]), top_k=some([0, 0, 20, 50, 100]),
                 top_p=some([0.8, 0.9, 0.95, 1.0]), min_p=some([0.0, 0.0, 0.02, 0.1]))
    S = S.to(TYPES[case["x"]])
    if how == "mixed":
        # An eighth of the rows may only answer with some labels: the others
        # at -inf or at the type's lowest value; the last row has none.
        kind = torch.randint(0, 16, (n, 1), generator=g, device=DEV)
        shut = torch.rand((n, m), generator=g, device=DEV) > min(1.0, 100 / m)
        S.masked_fill_(shut & (kind == 0), -math.inf)
        S.masked_fill_(shut & (kind == 1), torch.finfo(S.dtype).min)
        if n > 1:
            S[n - 1] = -math.inf
    return dict(s, S=S)


def prepare(case, seed):
    return _scores_input(case, seed) if case["op"] == "scores" else _sample_input(case, seed)


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _plain_scores(s):
    X, sx = s["X"].float(), s["sx"]
    if sx is None:
        sx = X.abs().amax(dim=1) / 127
        X = torch.where(sx[:, None] > 0, torch.round(X / sx[:, None]), torch.zeros_like(X))
    S = X @ s["W"].float().T
    S *= sx[:, None]
    S *= s["sw"]
    return S.to(s["out"].dtype)


def _column(v, S, dtype=torch.float32):
    return torch.as_tensor(v, dtype=dtype, device=S.device).reshape(-1, 1)


def _plain_sample(s):
    """Weights in 32 bits; their sums in 64, so that the drawn label does not
    hang on the order in which a long row is added up."""
    S = s["S"].float()
    n, m = S.shape
    T, k = _column(s["temperature"], S), _column(s["top_k"], S, torch.int64)
    p, q = _column(s["top_p"], S), _column(s["min_p"], S)
    top, at = torch.sort(S, dim=1, descending=True, stable=True)
    M = top[:, :1]
    rank = torch.arange(m, device=S.device)
    w = torch.where(top == M, torch.ones_like(top), torch.exp((top - M) * (1 / T)))
    w = torch.where(T > 0, w, (rank == 0).float())
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    c = torch.cumsum(w, 1, dtype=torch.float64)
    keep = (p >= 1) | (c - w < p * c[:, -1:])
    keep &= w >= q
    w = torch.where(keep & (M > -math.inf), w, torch.zeros_like(w))
    kept = (w > 0).sum(dim=1)
    w = torch.zeros_like(w).scatter_(1, at, w)
    c = torch.cumsum(w, 1, dtype=torch.float64)
    total = c[:, -1:]
    label = (c <= s["u"].double()[:, None] * total).sum(dim=1, keepdim=True)
    prob = torch.where(kept > 0, (w.gather(1, label.clamp(max=m - 1)) / total).squeeze(1), 0.0)
    return torch.where(kept > 0, label.squeeze(1), -1), prob.float(), kept


def run(state):
    s = state
    if own:
        import libsdca_amd as sd
        if s["op"] == "scores":
            return sd.scores_i8(s["X"], s["W"], s["sw"], x_scales=s["sx"], out=s["out"])
        return sd.sample(s["S"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                         top_p=s["top_p"], min_p=s["min_p"], prob=True, kept=True)
    return _plain_scores(s) if s["op"] == "scores" else _plain_sample(s)


def work(case):
    n, m = case["n"], case["m"]
    if case["op"] == "scores":
        d = case["d"]
        return {"bytes": n * d * SIZE[case["x"]] + m * d + n * m * SIZE[case["out"]] + 4 * m,
                "flops": 2 * n * m * d}
    # a difference, a product, an exponential and a sum for each score
    return {"bytes": n * m * SIZE[case["x"]] + 24 * n, "flops": 4 * n * m}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------
def _scores_exact(s):
    X = s["X"].double()
    if s["sx"] is None:
        # The scale and the quotient are held in 32 bits by definition: which
        # way a quotient near a half is rounded is no error of the product.
        sx = (X.abs().max(dim=1).values.float() / 127).double()
        X = (X / sx[:, None]).float().double().round()
    else:
        sx = s["sx"].double()
    out = []
    step = max(1, (1 << 27) // s["W"].shape[0])
    W = s["W"].double().mul_(s["sw"].double()[:, None])
    for i in range(0, X.shape[0], step):
        out.append((X[i:i + step] * sx[i:i + step, None]) @ W.T)
    return torch.cat(out)


def _sample_exact(s):
    S = s["S"].double().cpu().numpy()
    n = S.shape[0]
    u = s["u"].double().cpu().numpy()

    def per_row(v):
        return v.double().cpu().numpy() if torch.is_tensor(v) else np.full(n, np.float32(v), np.float64)

    T, K, P, Q = (per_row(s[v]) for v in ("temperature", "top_k", "top_p", "min_p"))
    label, prob, kept = np.full(n, -1), np.zeros(n), np.zeros(n, np.int64)
    for r in range(n):
        row = S[r]
        best = int(np.argmax(row))
        if row[best] == -np.inf:
            continue
        if T[r] == 0:
            label[r], prob[r], kept[r] = best, 1.0, 1
            continue
        w = np.exp((row - row[best]) / T[r])
        order = np.argsort(-row, kind="stable")
        if K[r] > 0:
            order = order[:int(K[r])]
        mass = np.cumsum(w[order])
        if P[r] < 1:
            order = order[:1 + int(np.searchsorted(mass, P[r] * mass[-1]))]
        ids = np.sort(order[w[order] >= Q[r]])
        c = np.cumsum(w[ids])
        label[r] = ids[min(len(ids) - 1, int(np.searchsorted(c, u[r] * c[-1], side="right")))]
        prob[r] = w[label[r]] / c[-1]
        kept[r] = np.count_nonzero(w[ids] > 2.0 ** -150)  # what 32 bits can hold
    return torch.from_numpy(label), torch.from_numpy(prob), torch.from_numpy(kept)


def exact(case, seed):
    s = prepare(case, seed)
    return _scores_exact(s) if case["op"] == "scores" else _sample_exact(s)
