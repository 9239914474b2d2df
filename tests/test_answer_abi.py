"""The answering calls refuse what they cannot take, before any device work."""
import ctypes

import numpy as np
import pytest


def _refused(status, fn, *args, **kw):
    import libsdca_amd as sd
    with pytest.raises(sd.SdcaError) as e:
        fn(*args, **kw)
    assert e.value.status == status, str(e.value)
    assert str(e.value)


def test_quantize_refusals():
    import libsdca_amd as sd
    a = np.ones((3, 8), np.float32)
    _refused(3, sd.quantize_i8, a.astype(np.int32))
    _refused(3, sd.quantize_i8, a.astype(np.int8))
    _refused(2, sd.quantize_i8, a[0])
    _refused(2, sd.quantize_i8, a[:, ::2])
    _refused(2, sd.quantize_i8, np.broadcast_to(a[:1], (3, 8)))
    _refused(2, sd.quantize_i8, a, out=np.zeros((3, 7), np.int8))
    _refused(3, sd.quantize_i8, a, out=np.zeros((3, 8), np.uint8))
    _refused(3, sd.quantize_i8, a, scales=np.zeros(3, np.float64))
    _refused(2, sd.quantize_i8, a, scales=np.zeros(4, np.float32))
    _refused(2, sd.quantize_i8, np.ones((3, 0), np.float32))


def test_scores_refusals():
    import libsdca_amd as sd
    X, W = np.ones((3, 8), np.float32), np.ones((5, 8), np.int8)
    sw, sx = np.ones(5, np.float32), np.ones(3, np.float32)
    _refused(3, sd.scores_i8, X.astype(np.int16), W, sw)
    _refused(3, sd.scores_i8, X, W.astype(np.uint8), sw)
    _refused(2, sd.scores_i8, X, W[:, :7], sw)
    _refused(2, sd.scores_i8, X, W, sw[:4])
    _refused(3, sd.scores_i8, X, W, sw.astype(np.float64))
    _refused(1, sd.scores_i8, X, W, sw, x_scales=sx)
    _refused(1, sd.scores_i8, X.astype(np.int8), W, sw)
    _refused(3, sd.scores_i8, X, W, sw, dtype=np.float64)
    _refused(2, sd.scores_i8, X, W, sw, out=np.zeros((3, 4), np.float32))
    _refused(2, sd.scores_i8, X, W, sw, out=np.zeros((5, 3), np.float32).T)
    _refused(2, sd.scores_i8, X, np.ones((0, 8), np.int8), np.ones(0, np.float32))
    torch = pytest.importorskip("torch")
    _refused(2, sd.scores_i8, X, torch.ones((5, 8), dtype=torch.int8), sw)
    _refused(2, sd.scores_i8, torch.ones((3, 8)), torch.ones((5, 8), dtype=torch.int8), torch.ones(5))


def test_sample_refusals():
    import libsdca_amd as sd
    S, u = np.zeros((3, 8), np.float32), np.full(3, 0.5, np.float32)
    _refused(3, sd.sample, S.astype(np.int64), u)
    _refused(2, sd.sample, S[0], u)
    _refused(2, sd.sample, S, u[:2])
    _refused(3, sd.sample, S, u.astype(np.float64))
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
               dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.1),
               dict(top_k=-1), dict(temperature=[1.0, 1.0, -1.0]), dict(top_k=[1, 2]), dict(top_p=[1.0, 0.0, 1.0])):
        _refused(2, sd.sample, S, u, **kw)
    _refused(2, sd.sample, S, np.array([0.0, 1.0, 0.5], np.float32))


def test_c_entries_refuse():
    """The C ABI's own checks, without the wrapper's."""
    import libsdca_amd as sd
    lib = sd.library()
    a = np.zeros(64, np.float32)
    at = a.ctypes.data
    assert lib.sdca_quantize_i8(0, 4, 2, at, 3, at, 4, at, 1, None) == 2
    assert lib.sdca_quantize_i8(0, 4, 2, at, 4, None, 4, at, 1, None) == 1
    assert lib.sdca_quantize_i8(5, 4, 2, at, 4, at, 4, at, 1, None) == 3
    assert lib.sdca_quantize_i8(2, 4, 2, at, 4, at, 4, at, 1, None) == 3
    assert lib.sdca_quantize_i8(0, 4, -1, at, 4, at, 4, at, 1, None) == 2
    assert lib.sdca_scores_i8(5, 0, 4, 2, 2, at, 4, None, at, 4, at, at, 2, 1, None) == 1
    assert lib.sdca_scores_i8(0, 0, 4, 2, 2, at, 4, at, at, 4, at, at, 2, 1, None) == 1
    assert lib.sdca_scores_i8(0, 1, 4, 2, 2, at, 4, None, at, 4, at, at, 2, 1, None) == 3
    assert lib.sdca_scores_i8(0, 0, 4, 2, 2, at, 4, None, at, 4, at, at, 1, 1, None) == 2
    assert lib.sdca_scores_i8(0, 0, 131_072, 2, 2, at, 131_072, None, at, 131_072, at, at, 2, 1, None) == 2
    assert b"131071" in lib.sdca_last_error()
    p = sd.SampleParams()
    lib.sdca_sample_params_default(ctypes.byref(p))
    assert (p.temperature, p.top_p, p.min_p, p.top_k) == (1, 1, 0, 0)
    lib.sdca_sample_params_default(None)
    assert lib.sdca_sample(0, 0, 2, at, 4, at, None, None, at, None, None, 1, None) == 2
    assert lib.sdca_sample(0, 4, 2, at, 4, None, None, None, at, None, None, 1, None) == 1
    assert lib.sdca_sample(5, 4, 2, at, 4, at, None, None, at, None, None, 1, None) == 3
    assert lib.sdca_sample(0, 4, 0, None, 4, None, None, None, None, None, None, 1, None) == 0


HPP_PROGRAM = r"""
#include "sdca_hip.hpp"
#include <cstdio>
int main() {
  const int d = 19, m = 7, n = 3;
  std::vector<float> W(d * m), X(d * n), u(n, 0.5f), prob(n);
  for (int i = 0; i < d * m; ++i) W[i] = static_cast<float>((i * 37) % 23 - 11);
  for (int i = 0; i < d * n; ++i) X[i] = static_cast<float>((i * 29) % 17 - 8);
  const sdca::hip::quantized q = sdca::hip::quantize_i8(d, m, W.data());
  const std::vector<float> S = sdca::hip::scores_i8(n, X.data(), q);
  sdca_sample_params p = sdca::hip::sample_params();
  p.temperature = 100;
  p.top_k = 3;
  const std::vector<std::int64_t> label = sdca::hip::sample(m, n, S.data(), u.data(), p, prob.data());
  for (int i = 0; i < n; ++i) std::printf("%d %.9g\n", static_cast<int>(label[i]), prob[i]);
  for (float s : S) std::printf("%.9g\n", s);
  p.top_p = 2;
  try {
    sdca::hip::sample(m, n, S.data(), u.data(), p);
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
    src, exe = tmp_path / "answer.cpp", tmp_path / "answer"
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
    d, m, n = 19, 7, 3
    W = ((np.arange(d * m) * 37) % 23 - 11).astype(np.float32).reshape(m, d)
    X = ((np.arange(d * n) * 29) % 17 - 8).astype(np.float32).reshape(n, d)
    S = sd.scores_i8(X, *sd.quantize_i8(W))
    label, prob = sd.sample(S, np.full(n, 0.5, np.float32), temperature=100.0, top_k=3, prob=True)
    got = [line.split() for line in lines[:n]]
    assert [int(a) for a, _ in got] == label.tolist()
    assert np.array_equal(np.array([b for _, b in got], np.float32), prob)
    assert np.array_equal(np.array(lines[n:n + m * n], np.float32).reshape(n, m), S)
    assert lines[n + m * n] == "refused 2"
