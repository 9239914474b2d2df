"""The adapter tests' 64-bit gradients against differences."""
import numpy as np

from tests import adapted_oracle as ref


def test_gradients_against_differences():
    rng = np.random.default_rng(3)
    n, d, m, r, count = 7, 6, 5, 3, 3
    X, G = rng.standard_normal((n, d)), rng.standard_normal((n, m))
    A, B = rng.standard_normal((count, r, d)), rng.standard_normal((count, m, r))
    index, scale = np.array([0, 2, -1, 0, 2, 2, 0]), np.array([0.5, 2.0, 1.25])

    def value(A, B):
        return (G * ref.by_rows(ref.terms(X, A, index, scale)[0], B, index)).sum()

    (dA, _), (dB, _) = ref.grads(G, X, A, B, index, scale)
    # The value is linear in A and in B: differences have no error but their
    # rounding, some 1e-15 over the step.
    for which, grad in ((0, dA), (1, dB)):
        at = (A, B)[which]
        for i in np.ndindex(at.shape):
            up = at.copy()
            up[i] += 0.5
            args = (up, B) if which == 0 else (A, up)
            assert abs((value(*args) - value(A, B)) / 0.5 - grad[i]) < 1e-11
    assert not dA[1].any() and not dB[1].any()
