"""log_probs and log_probs_grad refuse what they cannot take, before any
device work."""
import ctypes

import numpy as np
import pytest


def _refused(status, fn, *args, **kw):
    import libsdca_amd as sd
    with pytest.raises(sd.SdcaError) as e:
        fn(*args, **kw)
    assert e.value.status == status, str(e.value)
    assert str(e.value)


def test_log_probs_refusals():
    import libsdca_amd as sd
    S, labels = np.zeros((3, 8), np.float32), np.zeros(3, np.int64)
    _refused(3, sd.log_probs, S.astype(np.float64), labels)
    _refused(3, sd.log_probs, S.astype(np.int8), labels)
    _refused(2, sd.log_probs, S[0], labels)
    _refused(2, sd.log_probs, S[:, ::2], labels)
    _refused(2, sd.log_probs, S, labels[:2])
    _refused(3, sd.log_probs, S, labels.astype(np.int32))
    _refused(2, sd.log_probs, np.ones((3, 0), np.float32), labels)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-39, 1e39):
        _refused(2, sd.log_probs, S, labels, temperature=t)
    for top in (-1, 65):
        _refused(2, sd.log_probs, S, labels, top=top)
    for bad in (8, -2):
        _refused(8, sd.log_probs, S, np.array([0, bad, 0]))
    torch = pytest.importorskip("torch")
    _refused(2, sd.log_probs, torch.zeros((3, 8)), torch.zeros(3, dtype=torch.int64))
    _refused(2, sd.log_probs, S, torch.zeros(3, dtype=torch.int64))


def test_log_probs_grad_refusals():
    import libsdca_amd as sd
    S, labels, g = np.zeros((3, 8), np.float32), np.zeros(3, np.int64), np.ones(3, np.float32)
    _refused(3, sd.log_probs_grad, S.astype(np.float64), labels, g)
    _refused(2, sd.log_probs_grad, S, labels, g[:2])
    _refused(3, sd.log_probs_grad, S, labels, g.astype(np.float64))
    _refused(3, sd.log_probs_grad, S, labels, g, g_entropy=g.astype(np.float16))
    _refused(2, sd.log_probs_grad, S, labels, g, stats=np.zeros((3, 2), np.float32))
    _refused(2, sd.log_probs_grad, S, labels, g, stats=np.zeros(9, np.float32))
    _refused(2, sd.log_probs_grad, S, labels, g, stats=np.zeros((3, 4), np.float32)[:, :3])
    _refused(3, sd.log_probs_grad, S, labels, g, out=np.zeros((3, 8), np.float16))
    _refused(2, sd.log_probs_grad, S, labels, g, out=np.zeros((3, 7), np.float32))
    _refused(2, sd.log_probs_grad, S, labels, g, temperature=0.0)
    _refused(8, sd.log_probs_grad, S, np.array([0, 9, 0]), g)
    frozen = np.zeros((3, 8), np.float32)
    frozen.flags.writeable = False
    _refused(2, sd.log_probs_grad, S, labels, g, out=frozen)


def test_c_entries_refuse():
    import libsdca_amd as sd
    lib = sd.library()
    a = np.zeros(64, np.float32)
    l = np.zeros(8, np.int64)
    at, lab = a.ctypes.data, l.ctypes.data
    assert lib.sdca_log_probs(0, 4, 2, None, 4, lab, 1.0, 0, at, None, None, None, None, None, 1, None) == 1
    assert lib.sdca_log_probs(0, 4, 2, at, 4, None, 1.0, 0, at, None, None, None, None, None, 1, None) == 1
    assert lib.sdca_log_probs(0, 4, 2, at, 3, lab, 1.0, 0, at, None, None, None, None, None, 1, None) == 2
    assert lib.sdca_log_probs(1, 4, 2, at, 4, lab, 1.0, 0, at, None, None, None, None, None, 1, None) == 3
    assert lib.sdca_log_probs(0, 0, 2, at, 4, lab, 1.0, 0, at, None, None, None, None, None, 1, None) == 2
    assert lib.sdca_log_probs(0, 4, 0, None, 4, None, 1.0, 0, None, None, None, None, None, None, 1, None) == 0
    assert lib.sdca_log_probs_grad(0, 4, 2, at, 4, lab, None, None, None, 1.0, at, 4, None, None, 1, None) == 1
    assert lib.sdca_log_probs_grad(0, 4, 2, at, 4, lab, at, None, None, 1.0, None, 4, None, None, 1, None) == 1
    assert lib.sdca_log_probs_grad(0, 4, 2, at, 5, lab, at, None, None, 1.0, at, 4, None, None, 1, None) == 2
    assert lib.sdca_log_probs_grad(0, 4, 2, at, 4, lab, at, None, None, 1.0, at, 3, None, None, 1, None) == 2
    assert lib.sdca_log_probs_work(0, 1000, 5, 3) == 0
    assert lib.sdca_log_probs_work(0, 200_000, 1, 3) > lib.sdca_log_probs_work(0, 200_000, 1, 0) > 0
    assert lib.sdca_log_probs_grad_work(0, 200_000, 2, None) > 0
    assert lib.sdca_log_probs_grad_work(0, 200_000, 2, ctypes.c_void_p(at)) == 0
