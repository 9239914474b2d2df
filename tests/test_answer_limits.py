"""The answering calls at the limits of a dispatch and of their own: columns
beyond one grid's threads, offsets at the ends of a buffer."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "libsdca_amd", "csrc")


def _run_host(tmp_path, body, *flags):
    """Compiles and runs a program on the host-only header of the limits."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not found")
    src, exe = tmp_path / "limits.cpp", tmp_path / "limits"
    src.write_text(f'#include "answer_limits.hpp"\n#include <cstdio>\n#include <initializer_list>\nusing namespace sdca_gpu;\nint main() {{\n{body}\n}}\n')
    out = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", *flags, "-I", CSRC, str(src), "-o", str(exe)],
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
    return run.stdout


def test_slices_cover_and_fit_a_dispatch(tmp_path):
    """Slices follow one another to the end, and each is a grid of fewer than
    2^32 threads."""
    out = _run_host(tmp_path, r"""
  const int64_t many[] = {0, 1, 5, 1 << 21, (1 << 22) + 3, (1 << 24) + 3, (int64_t(1) << 30) - 1, INT32_MAX};
  for (int64_t n : many)
    for (int threads : {64, 256, 512, 1024})
      for (int64_t per : {1, 4, 16, 64, 256}) {
        int64_t next = 0;
        each_slice(n, per, threads, [&](int64_t first, int64_t count) {
          const int64_t blocks = (count + per - 1) / per;
          if (first != next || count < 1 || blocks * threads >= int64_t(1) << 32 || first % per) std::printf("bad\n");
          next = first + count;
        });
        if (next != n) std::printf("left out\n");
      }
""")
    assert out == ""


def _room(cuda, gib):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(cuda)[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GiB of device memory")


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", [(2 ** 28 + 5, 2), (2 ** 24 + 3, 1025)])
def test_quantize_more_columns_than_a_dispatch(cuda, n, d):
    """Sixteen threads to a column and a workgroup to a column, beyond 2^32
    threads.  Every column is of ones but the ones around the places where a
    grid could end, which are compared with the same columns alone."""
    import torch
    import libsdca_amd as sd
    _room(cuda, 70)
    print(n, d, flush=True)
    A = torch.ones((n, d), dtype=torch.float16, device=cuda)
    edge = torch.tensor(sorted({r for e in range(20, 29) for r in range(2 ** e - 2, 2 ** e + 2) if r < n} | {0, n - 2, n - 1}),
                        device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(d)
    some = torch.randn((len(edge), d), generator=g, device=cuda).half()
    A[edge] = some
    Q = torch.zeros((n, d), dtype=torch.int8, device=cuda)
    s = torch.full((n,), -1.0, device=cuda)
    sd.quantize_i8(A, out=Q, scales=s)
    want_q, want_s = sd.quantize_i8(some)
    assert torch.equal(Q[edge], want_q) and torch.equal(s[edge], want_s)
    rest = torch.ones(n, dtype=torch.bool, device=cuda)
    rest[edge] = False
    one = sd.quantize_i8(A[3:4])[1]
    assert bool(((s == one) | ~rest).all())
    for i in range(0, n, 1 << 22):
        assert bool(((Q[i:i + (1 << 22)] == 127).all(dim=1) | ~rest[i:i + (1 << 22)]).all()), i


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(2 ** 26 + 5, 10), (2 ** 24 + 3, 2049), (2 ** 22 + 3, 4097)])
def test_sample_more_columns_than_a_dispatch(cuda, n, m):
    """A wave, four waves and sixteen waves to a column, beyond 2^32 threads.
    Every column has one label that can be drawn but the ones around the
    places where a grid could end, which are compared with the same columns
    alone, settings of their own included."""
    import torch
    import libsdca_amd as sd
    _room(cuda, 80)
    print(n, m, flush=True)
    g = torch.Generator(device=cuda)
    g.manual_seed(m)
    S = torch.full((n, m), -30000.0, dtype=torch.float16, device=cuda)
    at = torch.randint(0, m, (n,), generator=g, device=cuda)
    S.scatter_(1, at[:, None], 1.0)
    edge = torch.tensor(sorted({r for e in range(20, 27) for r in range(2 ** e - 5, 2 ** e + 5) if r < n} | {0, n - 2, n - 1}),
                        device=cuda)
    S[edge] = torch.randn((len(edge), m), generator=g, device=cuda).half()
    u = torch.rand(n, generator=g, device=cuda)
    kw = dict(temperature=0.5 + torch.rand(n, generator=g, device=cuda), top_p=0.5 + 0.5 * torch.rand(n, generator=g, device=cuda),
              min_p=0.1 * torch.rand(n, generator=g, device=cuda), top_k=torch.randint(0, 9, (n,), generator=g, device=cuda))
    label, prob, kept = sd.sample(S, u, prob=True, kept=True, **kw)
    want = sd.sample(S[edge], u[edge], prob=True, kept=True, **{name: v[edge] for name, v in kw.items()})
    for a, b in zip((label, prob, kept), want):
        assert torch.equal(a[edge], b)
    rest = torch.ones(n, dtype=torch.bool, device=cuda)
    rest[edge] = False
    assert bool(((label == at) | ~rest).all())
    assert bool((((prob == 1) & (kept == 1)) | ~rest).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,d", [(3, 2 ** 30 - 1, 16), (2 ** 29 + 70, 3, 128)])
def test_scores_more_tiles_than_a_dispatch(cuda, n, m, d):
    """Tiles of one side beyond a dispatch's threads: each score equal to the
    integers' sum times its scales."""
    import torch
    import libsdca_amd as sd
    _room(cuda, 100)
    print(n, m, d, flush=True)
    g = torch.Generator(device=cuda)
    g.manual_seed(d)
    long = torch.empty((max(n, m), d), dtype=torch.int8, device=cuda)
    for part in long.split(1 << 26):
        part.random_(-127, 128, generator=g)
    short = torch.randint(-127, 128, (min(n, m), d), generator=g, device=cuda, dtype=torch.int8)
    scale = 0.01 + torch.rand(max(n, m), generator=g, device=cuda)
    own = 0.01 + torch.rand(min(n, m), generator=g, device=cuda)
    X, sx, W, sw = (short, own, long, scale) if n < m else (long, scale, short, own)
    S = torch.full((n, m), float("nan"), dtype=torch.bfloat16, device=cuda)
    sd.scores_i8(X, W, sw, x_scales=sx, out=S)
    step = 1 << 24
    for i in range(0, max(n, m), step):
        x, s = (X, sx) if n < m else (X[i:i + step], sx[i:i + step])
        w, t = (W[i:i + step], sw[i:i + step]) if n < m else (W, sw)
        sums = x.float() @ w.float().T  # whole numbers below 2^24
        want = (sums * s[:, None] * t).to(torch.bfloat16)
        assert torch.equal(S[:, i:i + step] if n < m else S[i:i + step], want), i


def test_offsets_outside_stay_outside(tmp_path):
    """The product's loads of tiles that are not there: whatever row's offset
    the one outside is added to, the sum is defined and beyond any buffer."""
    out = _run_host(tmp_path, r"""
  for (int64_t pitch : {int64_t(16), int64_t(4096), int64_t(1) << 20, kI8MaxPitch})
    for (int row = 0; row < 256; ++row) {
      const auto from = i8_offset(static_cast<uint32_t>(row * pitch), 7 * 16);
      const auto at = i8_offset(from, kOutside);
      if (int64_t(at) != row * pitch + 7 * 16 + int64_t(kOutside) || from > kI8MostOffset) std::printf("%d %lld\n", row, (long long)pitch);
    }
""", "-fsanitize=undefined", "-fno-sanitize-recover=all")
    assert out == ""


def test_sample_refuses_columns_beyond_its_sums():
    """Beyond 2^23 labels the sums' units would be too coarse."""
    import ctypes
    import libsdca_amd as sd
    lib = sd.library()
    at = ctypes.c_void_p(16)  # never read
    for m in (2 ** 23 + 1, 2 ** 28, 2 ** 30 - 1):
        assert lib.sdca_sample(0, m, 0, at, m, at, None, None, at, None, None, 0, None) == 2
        assert b"8388608" in lib.sdca_last_error()
    assert lib.sdca_sample(0, 2 ** 23, 0, at, 2 ** 23, at, None, None, at, None, None, 0, None) == 0


@pytest.mark.gpu
def test_sample_longest_columns(cuda):
    """2^23 labels, the tail's weights just below and just above half a unit
    of the sums (2^-40): all of it is lost or counted twice, 2^-17 of the
    largest weight, within what the weights' own rounding allows."""
    import numpy as np
    import torch
    import libsdca_amd as sd
    from tests import answer_oracle as ref
    m = 2 ** 23
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    S = torch.empty((4, m), device=cuda)
    S[0] = float(np.log(0.97 * 2.0 ** -40))
    S[1] = float(np.log(1.03 * 2.0 ** -40))
    S[2:] = torch.randn((2, m), generator=g, device=cuda)
    S[:2, m // 3] = 0
    for u, kw in (([0.5, 0.5, 0.5, 0.9], dict()), ([0.999999, 0.999999, 0.1, 0.3], dict(top_p=0.9)),
                  ([0.2, 0.99999, 0.7, 0.999], dict(temperature=1.5, top_k=500, min_p=1e-3))):
        print(kw, flush=True)
        u = torch.tensor(u, device=cuda)
        label, prob, kept = sd.sample(S, u, prob=True, kept=True, **kw)
        full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw)
        ref.check_sample(S.cpu().numpy(), u.cpu().numpy(), *(np.float32(v) for v in full.values()),
                         label.cpu().numpy(), prob.cpu().numpy(), kept.cpu().numpy())


def test_read_only_results_are_refused():
    import numpy as np
    import libsdca_amd as sd
    A = np.ones((3, 8), np.float32)
    W, w = np.ones((5, 8), np.int8), np.ones(5, np.float32)
    held = lambda shape, dtype: np.frombuffer(bytes(int(np.prod(shape)) * np.dtype(dtype).itemsize), dtype).reshape(shape)  # noqa: E731
    for fn, args, kw in ((sd.quantize_i8, (A,), dict(out=held((3, 8), np.int8))),
                         (sd.quantize_i8, (A,), dict(scales=held((3,), np.float32))),
                         (sd.scores_i8, (A, W, w), dict(out=held((3, 5), np.float32)))):
        with pytest.raises(sd.SdcaError) as e:
            fn(*args, **kw)
        assert e.value.status == 2 and "read-only" in str(e.value)
