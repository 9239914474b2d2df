"""The scratch of the adapters' gradients beside the gradient that they read."""
import pytest

F32, F16, BF16 = 0, 3, 4


@pytest.mark.parametrize("data,grad", [(F32, F32), (BF16, BF16), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("rank", [1, 16, 17, 64, 65, 128])
def test_its_share_of_a_large_gradient(data, grad, rank):
    import libsdca_amd as sd
    n, d, m = 8192, 4096, 128_000
    work = sd.library().sdca_scores_adapted_grad_work(data, grad, d, m, n, 1, rank)
    pitch = (rank + 15) // 16 * 16
    turned = m * rank * 4
    # sums in parts, two places for each segment: dA's of 64 segments at most, dB's of two
    partial = rank * 4 * max(129 * d, 5 * m)
    rows = 2 * n * pitch * 4 + 64 * n
    assert work <= n * m * (4 if grad == F32 else 2) * pitch // 256 + turned + partial + rows
