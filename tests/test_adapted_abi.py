"""scores_adapted and scores_adapted_grad refuse what they cannot take, before
any device work; the C++ calls compile."""
import ctypes

import numpy as np
import pytest


def _refused(status, fn, *args, **kw):
    import libsdca_amd as sd
    with pytest.raises(sd.SdcaError) as e:
        fn(*args, **kw)
    assert e.value.status == status, str(e.value)
    assert str(e.value)


def _some():
    X, W, sw = np.ones((3, 8), np.float32), np.ones((5, 8), np.int8), np.ones(5, np.float32)
    return X, W, sw, np.ones((2, 4, 8), np.float32), np.ones((2, 5, 4), np.float32), np.zeros(3, np.int64)


def test_scores_adapted_refusals():
    import libsdca_amd as sd
    f = sd.scores_adapted
    X, W, sw, A, B, index = _some()
    _refused(3, f, X.astype(np.float64), W, sw, A, B, index)
    _refused(3, f, X.astype(np.int8), W, sw, A, B, index)
    _refused(3, f, X, W.astype(np.uint8), sw, A, B, index)
    _refused(2, f, X, W[:, :7], sw, A, B, index)
    _refused(2, f, X, W, sw[:4], A, B, index)
    _refused(3, f, X, W, sw, A.astype(np.float16), B, index)
    _refused(3, f, X, W, sw, A, B.astype(np.float16), index)
    _refused(2, f, X, W, sw, A[0], B, index)
    _refused(2, f, X, W, sw, A[:, :, :7], B, index)
    _refused(2, f, X, W, sw, A, B[:1], index)
    _refused(2, f, X, W, sw, A, B[:, :, :3], index)
    _refused(2, f, X, W, sw, A[:, ::-1], B, index)
    _refused(2, f, X, W, sw, A, B, index[:2])
    _refused(3, f, X, W, sw, A, B, index.astype(np.int32))
    _refused(2, f, X, W, sw, A, B, index, scale=[1.0, 2.0, 3.0])
    _refused(2, f, X, W, sw, A, B, index, scale=float("nan"))
    _refused(2, f, X, W, sw, A, B, index, scale=float("inf"))
    _refused(3, f, X, W, sw, A, B, index, dtype=np.float64)
    _refused(2, f, X, W, sw, A, B, index, out=np.zeros((3, 4), np.float32))
    for bad in (2, -2):
        _refused(2, f, X, W, sw, A, B, np.array([0, bad, 0]))
    _refused(2, f, X, W, sw, np.ones((2, 0, 8), np.float32), np.ones((2, 5, 0), np.float32), index)
    _refused(2, f, X, W, sw, np.ones((2, 129, 8), np.float32), np.ones((2, 5, 129), np.float32), index)
    _refused(2, f, X, W, sw, np.ones((0, 4, 8), np.float32), np.ones((0, 5, 4), np.float32), index)
    torch = pytest.importorskip("torch")
    _refused(2, f, X, W, sw, torch.ones((2, 4, 8)), B, index)
    _refused(2, f, *(torch.from_numpy(v) for v in _some()))


def test_scores_adapted_grad_refusals():
    import libsdca_amd as sd
    f = sd.scores_adapted_grad
    X, W, sw, A, B, index = _some()
    G = np.ones((3, 5), np.float32)
    _refused(3, f, G.astype(np.float64), X, A, B, index)
    _refused(3, f, G, X.astype(np.float64), A, B, index)
    _refused(2, f, G[:2], X, A, B, index)
    _refused(2, f, G[:, :4], X, A, B, index)
    _refused(2, f, G[0], X, A, B, index)
    _refused(3, f, G, X, A.astype(np.float16), B, index)
    _refused(2, f, G, X, A, B, np.array([0, 2, 0]))
    _refused(2, f, G, X, A, B, index, scale=float("nan"))


def test_c_entries_refuse():
    import libsdca_amd as sd
    lib = sd.library()
    a = np.zeros(256, np.float32)
    i = np.zeros(8, np.int64)
    at = a.ctypes.data
    ad = sd.Adapters(2, 4, at, at, i.ctypes.data, None, 1.0)
    assert lib.sdca_scores_adapted(0, 0, 8, 5, 3, at, 8, at, 8, at, None, at, 5, None, 1, None) == 1
    assert lib.sdca_scores_adapted(0, 0, 8, 5, 3, None, 8, at, 8, at, ad, at, 5, None, 1, None) == 1
    assert lib.sdca_scores_adapted(0, 0, 8, 5, 3, at, 7, at, 8, at, ad, at, 5, None, 1, None) == 2
    assert lib.sdca_scores_adapted(5, 0, 8, 5, 3, at, 8, at, 8, at, ad, at, 5, None, 1, None) == 3
    assert lib.sdca_scores_adapted(0, 1, 8, 5, 3, at, 8, at, 8, at, ad, at, 5, None, 1, None) == 3
    assert lib.sdca_scores_adapted(0, 0, 131_072, 5, 3, at, 131_072, at, 131_072, at, ad, at, 5, None, 1, None) == 2
    assert lib.sdca_scores_adapted(0, 0, 8, 5, 0, None, 8, None, 8, None, ad, None, 5, None, 1, None) == 0
    for bad in (sd.Adapters(2, 4, None, at, i.ctypes.data, None, 1.0), sd.Adapters(2, 4, at, at, None, None, 1.0)):
        assert lib.sdca_scores_adapted(0, 0, 8, 5, 3, at, 8, at, 8, at, bad, at, 5, None, 1, None) == 1
        assert lib.sdca_scores_adapted_grad(0, 0, 8, 5, 3, at, 5, at, 8, bad, at, at, None, 1, None) == 1
    for bad in (sd.Adapters(0, 4, at, at, i.ctypes.data, None, 1.0), sd.Adapters(65_536, 4, at, at, i.ctypes.data, None, 1.0),
                sd.Adapters(2, 0, at, at, i.ctypes.data, None, 1.0), sd.Adapters(2, 129, at, at, i.ctypes.data, None, 1.0)):
        assert lib.sdca_scores_adapted(0, 0, 8, 5, 3, at, 8, at, 8, at, bad, at, 5, None, 1, None) == 2
    assert lib.sdca_scores_adapted_grad(0, 0, 8, 5, 3, at, 5, at, 8, ad, None, at, None, 1, None) == 1
    assert lib.sdca_scores_adapted_grad(0, 0, 8, 5, 3, at, 4, at, 8, ad, at, at, None, 1, None) == 2
    assert lib.sdca_scores_adapted_work(0, 8, 5, 3, ctypes.c_void_p(at), 8, 2, 4) > 0
    assert lib.sdca_scores_adapted_grad_work(0, 0, 8, 5, 3, 2, 4) > 0


HPP_PROGRAM = r"""
#include "sdca_hip.hpp"
#include <cstdio>
int main() {
  const int d = 19, m = 7, n = 4, r = 2;
  std::vector<float> W(d * m), X(d * n), A(3 * r * d), B(3 * r * m), g(n, 0.5f), stats(3 * n), H(n);
  for (int i = 0; i < d * m; ++i) W[i] = static_cast<float>((i * 37) % 23 - 11) / 16;
  for (int i = 0; i < d * n; ++i) X[i] = static_cast<float>((i * 29) % 17 - 8) / 16;
  for (int i = 0; i < 3 * r * d; ++i) A[i] = static_cast<float>((i * 31) % 19 - 9) / 32;
  for (int i = 0; i < 3 * r * m; ++i) B[i] = static_cast<float>((i * 41) % 13 - 6) / 32;
  const std::int64_t index[n] = {2, -1, 0, 2}, labels[n] = {6, 0, 3, -1};
  const sdca_adapters ad = {3, r, A.data(), B.data(), index, nullptr, 0.5};
  const sdca::hip::quantized q = sdca::hip::quantize_i8(d, m, W.data());
  const std::vector<float> S = sdca::hip::scores_adapted(n, X.data(), q, ad);
  const std::vector<float> lp = sdca::hip::log_probs(m, n, S.data(), labels, 0.5, H.data(), stats.data());
  const std::vector<float> D = sdca::hip::log_probs_grad(m, n, S.data(), labels, g.data(), g.data(), 0.5);
  const std::pair<std::vector<float>, std::vector<float>> dAB =
      sdca::hip::scores_adapted_grad(d, m, n, D.data(), X.data(), ad);
  const std::vector<float>* all[] = {&S, &lp, &H, &stats, &D, &dAB.first, &dAB.second};
  for (const std::vector<float>* v : all)
    for (float x : *v) std::printf("%.9g\n", x);
  try {
    sdca::hip::log_probs(m, n, S.data(), labels, 0.0);
  } catch (const sdca::hip::error& e) {
    std::printf("refused %d\n", e.status());
  }
  return 0;
}
"""


def build_program(tmp_path):
    import os
    import shutil
    import subprocess
    import libsdca_amd as sd
    if shutil.which("g++") is None:
        pytest.skip("g++ not found")
    src, exe = tmp_path / "adapted.cpp", tmp_path / "adapted"
    src.write_text(HPP_PROGRAM)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    libdir = os.path.dirname(sd.LIB_PATH)
    out = subprocess.run(
        ["g++", "-std=c++11", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(exe),
         "-L", libdir, "-l:" + os.path.basename(sd.LIB_PATH), "-Wl,-rpath," + libdir, "-Wl,-rpath,/opt/rocm/lib",
         "-Wl,--allow-shlib-undefined"], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    return str(exe)


def test_cpp_calls_compile(tmp_path):
    build_program(tmp_path)


@pytest.mark.gpu
def test_cpp_calls_give_what_python_gives(cuda, tmp_path):
    import subprocess
    import libsdca_amd as sd
    run = subprocess.run([build_program(tmp_path)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stderr
    lines = run.stdout.split("\n")
    d, m, n, r = 19, 7, 4, 2

    def made(count, by, mod, off, over, *shape):
        return (((np.arange(count) * by) % mod - off).astype(np.float32) / np.float32(over)).reshape(shape)

    W, X = made(d * m, 37, 23, 11, 16, m, d), made(d * n, 29, 17, 8, 16, n, d)
    A, B = made(3 * r * d, 31, 19, 9, 32, 3, r, d), made(3 * r * m, 41, 13, 6, 32, 3, m, r)
    index, labels, g = np.array([2, -1, 0, 2]), np.array([6, 0, 3, -1]), np.full(n, 0.5, np.float32)
    S = sd.scores_adapted(X, *sd.quantize_i8(W), A, B, index, scale=0.5)
    lp, H, stats = sd.log_probs(S, labels, temperature=0.5, entropy=True, stats=True)
    D = sd.log_probs_grad(S, labels, g, g_entropy=g, temperature=0.5)
    dA, dB = sd.scores_adapted_grad(D, X, A, B, index, scale=0.5)
    want = np.concatenate([v.ravel() for v in (S, lp, H, stats, D, dA, dB)])
    assert np.array_equal(np.array(lines[:len(want)], np.float32), want)
    assert lines[len(want)] == "refused 2"
