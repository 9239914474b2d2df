"""The log-probability tests' 64-bit gradient against differences."""
import numpy as np
import pytest

from tests import log_probs_oracle as ref


@pytest.mark.parametrize("T", [1.0, 0.5, 2.0])
def test_gradient_against_differences(T):
    rng = np.random.default_rng(5)
    n, m = 6, 9
    S = rng.standard_normal((n, m)) * 2
    S[2, 4] = -np.inf
    labels = np.array([0, 8, 3, -1, 5, 1])
    g, h = rng.standard_normal(n), rng.standard_normal(n)

    def value(S):
        _, _, logp, H, *_ = ref.rows(S, T)
        own = np.where(labels >= 0, logp[np.arange(n), labels.clip(0)], 0.0)
        return g * own + h * H

    D = ref.grad(S, labels, g, h, T)
    step = 1e-5
    for j in range(m):
        up, down = S.copy(), S.copy()
        up[:, j] += step
        down[:, j] -= step
        # central differences are off by step^2 / 6 of the third derivative
        # (some units here) and by the values' rounding over the step
        want = (value(up) - value(down)) / (2 * step)
        assert np.abs(D[:, j] - want).max() < 1e-8, j
