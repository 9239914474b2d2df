// What low-rank adapters need besides the score product: the examples' terms
// T_i = scale_a X_i A_a', and the adapters' gradients.  With G the scores'
// gradient and U_i = scale_a G_i B_a (a product of the same form as T),
//   dB_a = sum over the rows i of a of G_i (x) T_i,
//   dA_a = sum over the rows i of a of U_i (x) X_i,
// in 32 bits throughout.  The rows are brought into the order of their
// adapters first (positions, not data), and each adapter's into segments;
// sums over several segments are joined in the segments' order, so that
// results do not change from run to run.
#include <algorithm>
#include <type_traits>

#include "answer_launch.hpp"
#include "answer_limits.hpp"
#include "answer_types.hpp"
#include "common.hpp"

namespace sdca_gpu {
namespace {

// ---------------------------------------------------------------------------
// Terms, and with them the rows in 8 bits where Q is given.
// ---------------------------------------------------------------------------
struct TermsArgs {
  int64_t ldx, lda;  // lda: from one adapter's A to the next one's
  int wide, rank, pitch, count;
  const int64_t* index;
  const int* order;  // or NULL
  PerColumn<float> scale;
  float* terms;
  int parts;      // of the wide axis, and from one's terms to the next one's
  int64_t apart;
  int8_t* Q;
  int pad;
  float* scales;
};

// Eight neighbouring values of a row from `at` on, zeros from `len` on.
template <class T>
__device__ inline void load_raw(const T* row, int64_t at, int64_t len, T (&v)[8]) {
  if (at + 8 <= len) {
    __builtin_memcpy(v, row + at, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < len ? row[at + e] : from_float<T>(0.f);
  }
}

// `lanes` lanes take the column x of d values to 8 bits with that scale, and
// zeros up to pad.
template <class T>
__device__ inline void write_column(const T* x, int d, const ColumnScale& s, int8_t* q, int pad, int lane,
                                    int lanes) {
  constexpr int kOnce = sizeof(T) == 4 ? 2 : 4;
  const auto write = [&](const T (&raw)[8], int at, bool whole) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_float(raw[e]);
    unsigned w[2];
    quantize8(v, s, w);
    if (!whole) end_column(at, d, w);
    __builtin_memcpy(q + at, w, 8);  // (pad is whole tiles)
  };
  int first = 0;
  for (; first + lanes * 8 * kOnce <= d; first += lanes * 8 * kOnce) {
    T raw[kOnce][8];
#pragma unroll
    for (int i = 0; i < kOnce; ++i) __builtin_memcpy(raw[i], x + first + (i * lanes + lane) * 8, sizeof(raw[i]));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kOnce; ++i) write(raw[i], first + (i * lanes + lane) * 8, true);
  }
  for (int at = first + lane * 8; at < pad; at += lanes * 8) {
    T raw[8];
    load_column(x, at, d, raw);
    write(raw, at, false);
  }
}

// A workgroup takes eight of the adapter's rows for one example; the last of
// an example's workgroups its 8-bit form.  With parts the terms are there
// already, and only that last one runs, which adds them up.
template <class TX, class TA>
__global__ __launch_bounds__(256) void terms_row_kernel(const TX* __restrict__ X,
                                                        const TA* __restrict__ A, TermsArgs a) {
  __shared__ float part[4][8];
  __shared__ unsigned most_of[4];
  const int64_t p = blockIdx.x, row = a.order ? a.order[p] : p;
  const TX* x = X + row * a.ldx;
  if (a.parts > 1 || static_cast<int>(blockIdx.y) * 8 >= a.pitch) {
    if (a.parts > 1 && static_cast<int>(threadIdx.x) < a.pitch) {
      float* t = a.terms + p * a.pitch + threadIdx.x;
      float sum = t[0];
#pragma unroll 4
      for (int i = 1; i < a.parts; ++i) sum += t[i * a.apart];
      t[0] = sum;
    }
    unsigned most = 0;
    for (int at = threadIdx.x * 8; at < a.wide; at += 256 * 8) {
      TX raw[8];
      load_column(x, at, a.wide, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, magnitude(to_float(raw[e])));
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) most = max(most, static_cast<unsigned>(__shfl_xor(most, off)));
    if ((threadIdx.x & 63) == 0) most_of[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) most = max(most, most_of[w]);
    const ColumnScale s(most);
    if (threadIdx.x == 0) a.scales[p] = s.scale;
    write_column(x, a.wide, s, a.Q + p * a.pad, a.pad, threadIdx.x, 256);
    return;
  }
  const int64_t id = a.index[row];
  if (id < 0 || id >= a.count) return;
  const int k0 = blockIdx.y * 8;
  if (k0 >= a.rank) {
    if (threadIdx.x < 8) a.terms[p * a.pitch + k0 + threadIdx.x] = 0.f;
    return;
  }
  const TA* w = A + id * a.lda + static_cast<int64_t>(k0) * a.wide;
  float acc[8] = {};
  const auto add = [&](int at, auto load) {
    TX v[8];
    TA u[8][8];
    load(x, v);
#pragma unroll
    for (int k = 0; k < 8; ++k)  // (rows behind the rank: the last one again)
      load(w + static_cast<int64_t>(min(k, a.rank - 1 - k0)) * a.wide, u[k]);
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[k] = fmaf(to_float(v[e]), to_float(u[k][e]), acc[k]);
  };
  for (int at0 = 0; at0 < a.wide; at0 += 256 * 8) {
    const int at = at0 + threadIdx.x * 8;
    if (at0 + 256 * 8 <= a.wide) {
      add(at, [&](const auto* from, auto& v) { __builtin_memcpy(v, from + at, sizeof(v)); });
    } else {
      add(at, [&](const auto* from, auto& v) { load_raw(from, at, a.wide, v); });
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = wave_total(acc[k]);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) part[threadIdx.x >> 6][k] = acc[k];
  }
  __syncthreads();
  if (threadIdx.x < 8) {
    const int k = threadIdx.x;
    const float sum = part[0][k] + part[1][k] + part[2][k] + part[3][k];
    const float scale = a.scale.each ? a.scale.each[id] : a.scale.value;
    a.terms[p * a.pitch + k0 + k] = k0 + k < a.rank ? sum * scale : 0.f;
  }
}

// sum += a product of 16 rows by 16 columns over 32 values: a lane has eight
// of row and of column lane % 16.  Two halves or two bfloat16 multiply as
// they are, others in 32 bits; the sums are 32-bit either way.
template <class TA, class TB>
__device__ inline v4f multiply(const TA (&a)[8], const TB (&b)[8], v4f sum) {
  if constexpr (std::is_same<TA, TB>::value && sizeof(TA) == 2) {
    return multiply_16<TA>(a, b, sum);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sum = __builtin_amdgcn_mfma_f32_16x16x4f32(to_float(a[e]), to_float(b[e]), sum, 0, 0, 0);
    return sum;
  }
}

// A workgroup takes 16 NE examples with all ranks (16 RF); its waves share the
// wide axis and add up through LDS.  Examples of different adapters take
// turns; in the adapters' order that is rare.  With QUANT the largest
// magnitudes come with the first reading, and the rows are read again for
// their 8-bit form, by then mostly from the last-level cache (20000 rows of
// 4096 floats, rank 16: 147 us, in two kernels 97 and 76).  A compute unit
// takes some 60 GB/s here, half of it A's rows from the L2.
constexpr int steps_ahead(int registers) {  // 72 registers of loads at most
  return registers <= 9 ? 8 : registers <= 18 ? 4 : registers <= 36 ? 2 : 1;
}
template <class TX, class TA, int NE, int RF, int kTermWaves, bool QUANT>
__global__ __launch_bounds__(64 * kTermWaves) void terms_tile_kernel(
    const TX* __restrict__ X, const TA* __restrict__ A, TermsArgs a, int64_t n,
    const int2* __restrict__ spans, int64_t first) {
  constexpr bool kOneType = std::is_same<TX, TA>::value;
  constexpr int kAhead = steps_ahead(kOneType ? (NE + RF) * 2 * static_cast<int>(sizeof(TX)) : (NE + RF) * 8);
  constexpr int kFrags = NE * RF;
  constexpr int kOnce = kFrags < 4 ? kFrags : 4;
  __shared__ v4f part[kOnce][kTermWaves][64];
  __shared__ unsigned most_of[kTermWaves][NE * 16];
  const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t total = a.order && !QUANT ? spans[a.count].x : n;
  const int64_t p0 = (first + blockIdx.x) * (16 * NE);
  if (p0 >= total) return;
  const auto row_of = [&](int64_t p) { return a.order ? static_cast<int64_t>(a.order[p]) : p; };
  int64_t row[NE];
  int id[NE];
  unsigned long long left[NE];
  unsigned most[NE] = {};
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const int64_t p = p0 + j * 16 + low;
    row[j] = p < total ? row_of(p) : -1;
    const int64_t given = row[j] >= 0 ? a.index[row[j]] : -1;
    id[j] = given >= 0 && given < a.count ? static_cast<int>(given) : -1;
    left[j] = __ballot(id[j] >= 0);
  }
  // A wave's part of the wide axis.  Rows of a width like 4096 begin on one
  // channel of the L2, all sixteen, so waves work far from one another and
  // workgroups begin at different places.
  const int waves = kTermWaves * gridDim.y, share = (a.wide + 32 * waves - 1) / (32 * waves) * 32;
  const int begin = min((static_cast<int>(blockIdx.y) * kTermWaves + wave) * share, a.wide);
  const int behind = min(begin + share, a.wide);
  bool seen = !QUANT;
  while (true) {
    int me = -1;
#pragma unroll
    for (int j = NE - 1; j >= 0; --j)
      if (left[j]) me = __builtin_amdgcn_readlane(id[j], __builtin_ctzll(left[j]));
    if (me < 0 && seen) break;
    // (Rows behind the rank are the last one again, and examples of other
    // adapters multiply like the rest: neither's sums are used.)
    const TA* w[RF];
    const TX* x[NE];
#pragma unroll
    for (int f = 0; f < RF; ++f)
      w[f] = A + max(me, 0) * a.lda + static_cast<int64_t>(min(f * 16 + low, a.rank - 1)) * a.wide;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      left[j] &= ~__ballot(id[j] == me);
      x[j] = X + max(row[j], int64_t(0)) * a.ldx;
    }
    v4f acc[NE][RF] = {};
    TX u[kAhead][NE][8];
    TA v[kAhead][RF][8];
    const auto products = [&] {
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
#pragma unroll
        for (int j = 0; j < NE; ++j) {
#pragma unroll
          for (int f = 0; f < RF; ++f) acc[j][f] = multiply(v[s][f], u[s][j], acc[j][f]);
          if constexpr (QUANT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) most[j] = max(most[j], magnitude(to_float(u[s][j][e])));
          }
        }
    };
    const int turns = (behind - begin + 32 * kAhead - 1) / (32 * kAhead);
    for (int i = 0; i < turns; ++i) {
      int turn = i + static_cast<int>(blockIdx.x % turns);  // (turns is 0 for a wave without a part)
      turn -= turn >= turns ? turns : 0;
      const int at0 = begin + turn * 32 * kAhead + high * 8;
      if (begin + (turn + 1) * 32 * kAhead <= behind) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
#pragma unroll
          for (int j = 0; j < NE; ++j) __builtin_memcpy(u[s][j], x[j] + at0 + s * 32, sizeof(u[s][j]));
#pragma unroll
          for (int f = 0; f < RF; ++f) __builtin_memcpy(v[s][f], w[f] + at0 + s * 32, sizeof(v[s][f]));
        }
      } else {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
#pragma unroll
          for (int j = 0; j < NE; ++j) load_raw(x[j], at0 + s * 32, behind, u[s][j]);
#pragma unroll
          for (int f = 0; f < RF; ++f) load_raw(w[f], at0 + s * 32, behind, v[s][f]);
        }
      }
      // (All loads first: in an order of its own choice the compiler has few on
      // their way at a time.)
      __builtin_amdgcn_sched_barrier(0);
      products();
      __builtin_amdgcn_sched_barrier(0);
    }
    seen = true;
    if (me < 0) break;
    const float scale = a.scale.each ? a.scale.each[me] : a.scale.value;
#pragma unroll
    for (int g = 0; g < kFrags; g += kOnce) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kOnce; ++i) part[i][wave][lane] = acc[(g + i) / RF][(g + i) % RF];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kOnce; ++i) {
        const int j = (g + i) / RF, k = (g + i) % RF * 16 + high * 4;
        if (wave != i || id[j] != me) continue;
        v4f sum = part[i][0][lane];
#pragma unroll
        for (int q = 1; q < kTermWaves; ++q) sum += part[i][q][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = k + e < a.rank ? sum[e] * scale : 0.f;
        if (k < a.pitch)
          *reinterpret_cast<v4f*>(a.terms + blockIdx.y * a.apart + (p0 + j * 16 + low) * a.pitch + k) = sum;
      }
    }
  }
  if constexpr (QUANT) {
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      most[j] = max(most[j], static_cast<unsigned>(__shfl_xor(most[j], 16)));
      most[j] = max(most[j], static_cast<unsigned>(__shfl_xor(most[j], 32)));
      if (lane < 16) most_of[wave][j * 16 + lane] = most[j];
    }
    __syncthreads();
    for (int r = wave; r < 16 * NE; r += kTermWaves) {
      const int64_t p = p0 + r;
      if (p >= total) break;
      unsigned all = 0;
#pragma unroll
      for (int w = 0; w < kTermWaves; ++w) all = max(all, most_of[w][r]);
      const ColumnScale s(all);
      if (lane == 0) a.scales[p] = s.scale;
      write_column(X + row_of(p) * a.ldx, a.wide, s, a.Q + p * a.pad, a.pad, lane, 64);
    }
  }
}

template <class TX, class TA, int NE, int RF, int WAVES, bool QUANT>
void start_terms(const TermsLaunch& l, const TermsArgs& a) {
  each_slice((l.n + 16 * NE - 1) / (16 * NE), 1, 64 * WAVES * l.parts, [&](int64_t first, int64_t count) {
    terms_tile_kernel<TX, TA, NE, RF, WAVES, QUANT>
        <<<dim3(static_cast<unsigned>(count), l.parts), 64 * WAVES, 0, l.stream>>>(
        static_cast<const TX*>(l.X), static_cast<const TA*>(l.A), a, l.n, l.spans, first);
  });
}
template <class TX, class TA, int NE, int RF, int WAVES>
void start_terms(const TermsLaunch& l, const TermsArgs& a) {
  if constexpr (std::is_same<TX, TA>::value) {
    if (l.Q && l.parts == 1) return start_terms<TX, TA, NE, RF, WAVES, true>(l, a);
  }
  start_terms<TX, TA, NE, RF, WAVES, false>(l, a);
}
// Of A there is as much to read as of 16 examples, or more for a rank above
// 16: 32 share it.  (8192 rows of 14336 bfloat16, rank 16: 49 us, 16 at a time
// 59; 20000 rows of 4096 floats take 88 either way, with twice the registers
// for the same loads.)  Few workgroups have sixteen waves each.
template <class TX, class TA>
void start_terms(const TermsLaunch& l, const TermsArgs& a) {
  const bool many = l.n >= 4096;
  if (a.rank <= 16) {
    if (!many) start_terms<TX, TA, 1, 1, 16>(l, a);
    else if (sizeof(TX) == 2) start_terms<TX, TA, 2, 1, 8>(l, a);
    else start_terms<TX, TA, 1, 1, 8>(l, a);
  } else if (a.rank <= 32) {
    many ? start_terms<TX, TA, 2, 2, 8>(l, a) : start_terms<TX, TA, 1, 2, 16>(l, a);
  } else if (a.rank <= 64) {
    many ? start_terms<TX, TA, 2, 4, 8>(l, a) : start_terms<TX, TA, 1, 4, 16>(l, a);
  } else {
    start_terms<TX, TA, 1, 8, 8>(l, a);
  }
}

template <class TX, class TA>
hipError_t terms(const TermsLaunch& l) {
  const Adapters& ad = *l.adapters;
  TermsArgs a;
  a.ldx = l.ldx;
  a.lda = ad.rank * l.wide;
  a.wide = static_cast<int>(l.wide);
  a.rank = static_cast<int>(ad.rank);
  a.pitch = static_cast<int>(terms_pitch(ad.rank));
  a.count = static_cast<int>(ad.count);
  a.scale = ad.scale;
  a.index = ad.index;
  a.order = l.order;
  a.terms = l.terms;
  a.Q = l.Q;
  a.pad = static_cast<int>(l.pad);
  a.scales = l.scales;
  a.parts = l.parts;
  a.apart = l.n * a.pitch;
  if (l.n == 0) return hipSuccess;
  if (!terms_by_rows(l.n, ad.rank)) {
    start_terms<TX, TA>(l, a);
    if (l.parts > 1) {
      terms_row_kernel<TX, TA><<<static_cast<unsigned>(l.n), 256, 0, l.stream>>>(
          static_cast<const TX*>(l.X), static_cast<const TA*>(l.A), a);
    }
    return hipGetLastError();
  }
  const unsigned groups = static_cast<unsigned>(a.pitch / 8 + (l.Q ? 1 : 0));
  terms_row_kernel<TX, TA><<<dim3(static_cast<unsigned>(l.n), groups), 256, 0, l.stream>>>(
      static_cast<const TX*>(l.X), static_cast<const TA*>(l.A), a);
  return hipGetLastError();
}
template <class TX>
hipError_t terms(const TermsLaunch& l) {
  switch (l.adapters->data) {
    case SDCA_F32: return terms<TX, float>(l);
    case SDCA_F16: return terms<TX, __half>(l);
    default: return terms<TX, __hip_bfloat16>(l);
  }
}

// ---------------------------------------------------------------------------
// The rows by adapter, and segments of at most `length` of them.
// ---------------------------------------------------------------------------
struct Segment {
  int adapter, first, rows, slot;  // slot: where the partial sums go; -1: the result itself
};
// Segment numbers need no sum over the adapters before: with `before` rows of
// those, adapter a's begin at before / length + a, and there are
// ceil(rows / length) <= (before + rows) / length - before / length + 1.  In
// the same way the slots of adapters of several segments begin at
// 2 before / length.  Numbers that are not taken have no rows.
struct Segments {
  int length;
  Segment* table;
  __host__ __device__ int64_t first(int64_t before, int64_t a) const { return before / length + a; }
  __host__ __device__ int64_t slot(int64_t before) const { return 2 * before / length; }
};

struct GroupArgs {
  const int64_t* index;
  int n, count;
  int* order;    // rows by adapter, rising within each, those without one last
  int2* spans;   // an adapter's first place in `order`, and its number of rows; the others' last
  int* ids;      // or NULL: the rows' adapters in their order, -1, or -2 for no adapter's number
  Segments by[2];
};

// A workgroup finds the places of one adapter's rows, or the last one those
// of the rows without: its waves each count their part of the index, then
// write.
__device__ void group(const GroupArgs& a, int me) {
  constexpr int kWaves = 16, kBatch = 8;
  __shared__ int less_of[kWaves], equal_of[kWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t share = ((static_cast<int64_t>(a.n) + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int64_t begin = min(static_cast<int64_t>(a.n), wave * share);
  const int64_t end = min(static_cast<int64_t>(a.n), begin + share);
  // kBatch rows' adapters, the rows without as `count`, none behind the end.
  // (All loaded, and held to be used, so that the loads are on their way
  // together: left to itself the compiler makes each wait for the one before,
  // and 20000 rows took 18 us.  The adapters' gradients of 16 x 8 examples, of
  // which this is a good part, with 4, 8 and 16 at once, us: 3000 rows 51.6, 51.8,
  // 54.9; 20000 62.9, 63.7, 67; 10^6 1530, 1494, 1506.)
  int64_t raw[kBatch];
  const auto adapters = [&](int64_t i0, int (&id)[kBatch]) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) raw[b] = a.index[min(i0 + b * 64 + lane, end - 1)];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) asm volatile("" : "+v"(raw[b]));
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      id[b] = i0 + b * 64 + lane >= end ? 0x7fffffff : raw[b] >= 0 && raw[b] < a.count ? static_cast<int>(raw[b]) : a.count;
  };
  int less = 0, equal = 0;
  for (int64_t i0 = begin; i0 < end; i0 += 64 * kBatch) {
    int id[kBatch];
    adapters(i0, id);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      less += id[b] < me;
      equal += id[b] == me;
    }
  }
  less = wave_total(less);
  equal = wave_total(equal);
  if (lane == 0) less_of[wave] = less, equal_of[wave] = equal;
  __syncthreads();
  int before = 0, rows = 0, place = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += less_of[w];
    if (w < wave) place += equal_of[w];
    rows += equal_of[w];
  }
  place += before;
  if (equal) {
    for (int64_t i0 = begin; i0 < end; i0 += 64 * kBatch) {
      int id[kBatch];
      adapters(i0, id);
      const int64_t i = i0 + lane;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const bool mine = id[b] == me;
        const unsigned long long mask = __ballot(mine);
        if (mine) {
          const int to = place + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                                           __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0));
          a.order[to] = static_cast<int>(i + b * 64);
          if (a.ids) a.ids[to] = me < a.count ? me : raw[b] == -1 ? -1 : -2;
        }
        place += __popcll(mask);
      }
    }
  }
  if (threadIdx.x == 0) a.spans[me] = make_int2(before, rows);
  if (me == a.count) return;
  const bool last = me == a.count - 1;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const Segments& s = a.by[t];
    if (!s.table) continue;
    const int64_t first = s.first(before, me);
    const int64_t behind = last ? s.first(a.n, a.count) : s.first(before + rows, me + 1);
    for (int64_t i = first + threadIdx.x; i < behind; i += 1024) {
      const int64_t done = (i - first) * s.length;
      Segment g;
      g.adapter = static_cast<int>(me);
      g.first = before + static_cast<int>(min(done, static_cast<int64_t>(rows)));
      g.rows = static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(s.length), rows - done)));
      g.slot = rows > s.length ? static_cast<int>(s.slot(before) + i - first) : -1;
      s.table[i] = g;
    }
  }
}

// ---------------------------------------------------------------------------
// B (m x rank for each adapter) with its classes in a row.
// ---------------------------------------------------------------------------
struct TurnArgs {
  const void* B;
  int64_t m;
  int rank;
  void* to;
};
template <class T, class TO>
__device__ void turn(const TurnArgs& a, int64_t id) {
  constexpr int kClasses = 64;
  __shared__ T tile[kClasses * (kMostRank + 1)];
  const int64_t blocks = (a.m + kClasses - 1) / kClasses;
  const int64_t which = id / blocks, c0 = id % blocks * kClasses;
  const int classes = static_cast<int>(min(static_cast<int64_t>(kClasses), a.m - c0)), rank = a.rank;
  const T* b = static_cast<const T*>(a.B) + (which * a.m + c0) * rank;
  for (int i = threadIdx.x; i < classes * rank; i += 1024) tile[i / rank * (rank + 1) + i % rank] = b[i];
  __syncthreads();
  const int c = threadIdx.x % kClasses;
  if (c >= classes) return;
  for (int k = threadIdx.x / kClasses; k < rank; k += 1024 / kClasses) {
    const T x = tile[c * (rank + 1) + k];
    TO* to = static_cast<TO*>(a.to) + (which * rank + k) * a.m + c0 + c;
    if constexpr (std::is_same<T, TO>::value) *to = x;
    else *to = to_float(x);
  }
}

__global__ __launch_bounds__(1024) void group_kernel(GroupArgs a) { group(a, blockIdx.x); }

// Both in one launch: the first workgroups group, the others turn.
template <class T, class TO>
__global__ __launch_bounds__(1024) void group_turn_kernel(GroupArgs g, TurnArgs t, int64_t first) {
  const int64_t id = first + blockIdx.x;
  if (id <= g.count) group(g, static_cast<int>(id));
  else turn<T, TO>(t, id - g.count - 1);
}

// 16 bytes of a row from `at` on as words, zeros from `len` on.
template <class T>
__device__ inline void load_some(const T* row, int64_t at, int64_t len, unsigned (&w)[4]) {
  constexpr int kIn = 4 / static_cast<int>(sizeof(T));
  if (at + 4 * kIn <= len) {
    __builtin_memcpy(w, row + at, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < kIn; ++e) {
        const int64_t k = at + i * kIn + e;
        unsigned b = 0;
        if (k < len) __builtin_memcpy(&b, row + k, sizeof(T));
        w[i] |= b << (16 * e);
      }
    }
  }
}

// Sums over rows: out[c][k] or out[k][c] = sum_i Z_ic V_ik for the rows of a
// segment, by 16 x 16 x 4 products in 32 bits.  A lane loads 16 bytes of a
// row, V neighbouring values, four rows at a time; value e of all lanes makes
// an operand, 16 columns V apart by four rows, without a turn through LDS.
// A wave has 16 V columns and 16 RF ranks.
//
// With TERMS the rows' own terms with Z, sum_c Z_ic Bt_kc, come from the same
// reading: 16 rows go through LDS to lanes by row, the wave's part of Bt stays
// in registers, the four waves' sums are added up in LDS, and the columns'
// workgroups' by a kernel behind this one.
// ---------------------------------------------------------------------------
struct SumArgs {
  int64_t ldz;
  int wide, rank, pitch;
  const float* terms;
  const int* order;
  const Segment* segments;
  int64_t blocks, first;  // of columns; the launch's first workgroup
  float *out, *partial;
  // With TERMS: Bt of Z's type, rank rows of `wide` for each adapter; the
  // columns' workgroups' terms, `rows` of them each.
  const void* turned;
  PerColumn<float> scale;
  float* parts;
  int64_t rows;
};

template <class T, int RF, bool RANKS_FIRST, bool TERMS>
__global__ __launch_bounds__(256) void sum_kernel(const T* __restrict__ Z, SumArgs a) {
  // (kSteps loads of a lane ahead of its products: with eight 8192 x 14336
  // bfloat16 with terms take the same 78 us.)
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kSteps = 4;
  constexpr int kPitch = 16 * V + V;             // other banks for each row
  constexpr int kChunks = TERMS ? 16 * V / 32 : 1;  // of 32 columns
  static_assert(!(TERMS && RANKS_FIRST), "terms go with the columns' order");
  __shared__ __align__(16) T turn[TERMS ? 4 : 1][TERMS ? 16 * kPitch : 1];
  __shared__ v4f sums[TERMS ? 2 : 1][TERMS ? 4 : 1][TERMS ? RF : 1][TERMS ? 64 : 1];
  const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = a.first + blockIdx.x;
  const Segment seg = a.segments[id / a.blocks];
  const int64_t c0 = (id % a.blocks * 4 + wave) * (16 * V);
  if (!seg.rows || (!TERMS && c0 >= a.wide)) return;
  const int rank0 = blockIdx.y * 16 * RF;
  T b[kChunks][TERMS ? RF : 1][8];
  float scale = 0.f;
  if constexpr (TERMS) {
    scale = a.scale.each ? a.scale.each[seg.adapter] : a.scale.value;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      // (Ranks behind the last are the last one again: their terms are not used.)
      const int k = min(rank0 + f * 16 + low, a.rank - 1);
      const T* from = static_cast<const T*>(a.turned) + (static_cast<int64_t>(seg.adapter) * a.rank + k) * a.wide;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) load_raw(from, c0 + i * 32 + high * 8, a.wide, b[i][f]);
    }
  }
  const int64_t c = c0 + low * V;
  const int* order = a.order + seg.first;
  const float* terms = a.terms + static_cast<int64_t>(seg.first) * a.pitch;
  v4f acc[V][RF] = {};
  // The next rows' places, then the next rows, come while these multiply.
  unsigned z[kSteps][4];
  float t[kSteps][RF];
  int64_t row[kSteps];
  const auto places = [&](int p0) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) row[s] = order[min(p0 + 4 * s + high, seg.rows - 1)];
  };
  const bool across = c0 + 16 * V <= a.wide && rank0 + 16 * RF <= a.pitch;
  const auto fetch = [&](int p0) {
    if (across && p0 + 4 * kSteps <= seg.rows) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        __builtin_memcpy(z[s], Z + row[s] * a.ldz + c, 16);
#pragma unroll
        for (int f = 0; f < RF; ++f) t[s][f] = terms[static_cast<int64_t>(p0 + 4 * s + high) * a.pitch + rank0 + f * 16 + low];
      }
      return;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bool in = p0 + 4 * s + high < seg.rows;
      load_some(Z + row[s] * a.ldz, c, in ? a.wide : 0, z[s]);
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        const int k = rank0 + f * 16 + low;
        t[s][f] = in && k < a.pitch ? terms[static_cast<int64_t>(p0 + 4 * s + high) * a.pitch + k] : 0.f;
      }
    }
  };
  places(0);
  fetch(0);
  places(4 * kSteps);
  for (int p0 = 0; p0 < seg.rows; p0 += 4 * kSteps) {
    unsigned zn[kSteps][4];
    float tn[kSteps][RF];
    __builtin_memcpy(zn, z, sizeof(z));
    __builtin_memcpy(tn, t, sizeof(t));
    __builtin_amdgcn_sched_barrier(0);
    if (p0 + 4 * kSteps < seg.rows) {
      fetch(p0 + 4 * kSteps);
      places(p0 + 8 * kSteps);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (TERMS) {
#pragma unroll
      for (int h = 0; h < kSteps / 4; ++h) {  // sixteen rows
#pragma unroll
        for (int s = 0; s < 4; ++s)
          __builtin_memcpy(__builtin_assume_aligned(&turn[wave][(4 * s + high) * kPitch + low * V], 16), zn[4 * h + s], 16);
        wave_lds_sync();
        v4f own[RF] = {};
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          T u[8];
          __builtin_memcpy(u, __builtin_assume_aligned(&turn[wave][low * kPitch + i * 32 + high * 8], 16), sizeof(u));
#pragma unroll
          for (int f = 0; f < RF; ++f) own[f] = multiply(b[i][f], u, own[f]);
        }
        wave_lds_sync();
        const int p = p0 + 16 * h, turns = p / 16, which = turns & 1;
#pragma unroll
        for (int f = 0; f < RF; ++f) sums[which][wave][f][lane] = own[f];
        // (The next turn's sums go to the other half, and those after them come
        // behind the next barrier, when these have been read.)
        __syncthreads();
        if (wave == (turns & 3) && p + low < seg.rows) {
          float* to = a.parts + (id % a.blocks * a.rows + seg.first + p + low) * a.pitch + rank0 + high * 4;
#pragma unroll
          for (int f = 0; f < RF; ++f) {
            if (rank0 + f * 16 >= a.pitch) break;
            const v4f all = ((sums[which][0][f][lane] + sums[which][1][f][lane]) + sums[which][2][f][lane]) + sums[which][3][f][lane];
            *reinterpret_cast<v4f*>(to + f * 16) = all * scale;
          }
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[V];
      unpack<T>(zn[s], x);
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int f = 0; f < RF; ++f)
          acc[e][f] = RANKS_FIRST ? __builtin_amdgcn_mfma_f32_16x16x4f32(tn[s][f], x[e], acc[e][f], 0, 0, 0)
                                  : __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], tn[s][f], acc[e][f], 0, 0, 0);
    }
  }
  const int64_t size = static_cast<int64_t>(a.rank) * a.wide;
  float* out = seg.slot < 0 ? a.out + seg.adapter * size : a.partial + seg.slot * size;
#pragma unroll
  for (int f = 0; f < RF; ++f)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (RANKS_FIRST) {
        const int k = rank0 + f * 16 + high * 4 + x;
        if (k >= a.rank) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = acc[e][f][x];
        float* to = out + static_cast<int64_t>(k) * a.wide;
        if (c + V <= a.wide) {
          __builtin_memcpy(to + c, v, sizeof(v));
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < a.wide) to[c + e] = v[e];
        }
      } else {
        const int k = rank0 + f * 16 + low;
        const int64_t at = c0 + V * (high * 4 + x);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (k < a.rank && at + e < a.wide) out[(at + e) * a.rank + k] = acc[e][f][x];
      }
    }
}

// What is left of sums in parts: the rows' terms from those of the columns'
// workgroups (by the first `terms_blocks` workgroups), and the adapters of
// several segments from their partial sums, zeros for those without rows (by
// `each` for each adapter).
struct JoinArgs {
  const int2* spans;
  int count, pitch;
  int64_t terms_blocks, rows, parts;
  const float* part_terms;
  float* terms;
  Segments segments;
  int64_t each, size;
  const float* partial;
  float* out;
};
// The sum of `parts` values `apart` from one another, in their order, 64 bytes
// on their way together: of many narrow rows there are hundreds of parts (20000
// x 100 and 512 floats, rank 8: 313 and 209 for few results; the gradients took
// 99 us with four loads at a time that the compiler kept apart, 73 so).
template <class V>
__device__ inline V in_order(const V* from, int64_t parts, int64_t apart) {
  constexpr int kBatch = 64 / static_cast<int>(sizeof(V));
  V sum = {};
  int64_t p = 0;
  for (; p + kBatch <= parts; p += kBatch) {
    V v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = from[(p + i) * apart];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) sum += v[i];
  }
#pragma unroll 4
  for (; p < parts; ++p) sum += from[p * apart];
  return sum;
}
__global__ __launch_bounds__(256) void join_kernel(JoinArgs j, int64_t first) {
  const int64_t id = first + blockIdx.x;
  if (id < j.terms_blocks) {
    const int64_t size = static_cast<int64_t>(j.spans[j.count].x) * j.pitch / 4, apart = j.rows * j.pitch / 4;
    const v4f* from = reinterpret_cast<const v4f*>(j.part_terms);
    for (int64_t i = id * 256 + threadIdx.x; i < size; i += j.terms_blocks * 256) {
      reinterpret_cast<v4f*>(j.terms)[i] = in_order(from + i, j.parts, apart);
    }
    return;
  }
  const int64_t a = (id - j.terms_blocks) / j.each, block = (id - j.terms_blocks) % j.each;
  const int2 span = j.spans[a];
  if (span.y && span.y <= j.segments.length) return;
  const int parts = (span.y + j.segments.length - 1) / j.segments.length;
  const float* from = j.partial + j.segments.slot(span.x) * j.size;
  for (int64_t i = block * 256 + threadIdx.x; i < j.size; i += j.each * 256) {
    j.out[a * j.size + i] = in_order(from + i, parts, j.size);
  }
}

// Rows of a segment, so that the columns' workgroups times the segments come
// to about 512, two waves to a SIMD (8192 x 14336 bfloat16 with terms: 78 us;
// 256 of them 112; 1024 83, and 6 more for the joining of their sums).
int segment_length(int es, int64_t wide, int64_t n) {
  const int64_t columns = 4 * 16 * (16 / es), blocks = (wide + columns - 1) / columns;
  const int64_t parts = std::max<int64_t>(1, 512 / blocks);
  const int64_t length = ((n + parts - 1) / parts + 31) / 32 * 32;
  return static_cast<int>(std::max<int64_t>(length, 64));
}

template <class T>
int64_t column_blocks(int64_t wide) {
  constexpr int64_t kColumns = 4 * 16 * (16 / sizeof(T));
  return (wide + kColumns - 1) / kColumns;
}

template <class T, int RF, bool RANKS_FIRST, bool TERMS>
void start_sums(const T* Z, SumArgs a, int64_t segments, hipStream_t stream) {
  a.blocks = column_blocks<T>(a.wide);
  const unsigned ranks = (a.rank + 16 * RF - 1) / (16 * RF);
  each_slice(segments * a.blocks, 1, 256 * static_cast<int64_t>(ranks), [&](int64_t first, int64_t count) {
    a.first = first;
    sum_kernel<T, RF, RANKS_FIRST, TERMS><<<dim3(static_cast<unsigned>(count), ranks), 256, 0, stream>>>(Z, a);
  });
}
template <class T, bool RANKS_FIRST, bool TERMS>
void start_sums(const T* Z, const SumArgs& a, int64_t segments, hipStream_t stream) {
  if (a.rank <= 16) start_sums<T, 1, RANKS_FIRST, TERMS>(Z, a, segments, stream);
  else if (a.rank <= 32) start_sums<T, 2, RANKS_FIRST, TERMS>(Z, a, segments, stream);
  else start_sums<T, 4, RANKS_FIRST, TERMS>(Z, a, segments, stream);
}

// Whether G's terms come with dB's sums: Bt is then of G's type.  They are kept
// for each workgroup's columns first, 1024 bytes of a row of G, which takes as
// much as G itself times rank (in whole 16) over 256.  In a launch of their own
// they take G's reading once more: 8192 x 14336 bfloat16, rank 128, 755 us for
// 707 and 283 MB of scratch for 400; floats 1217 for 1105 and 152 MB for 387;
// 512 x 30000 floats with adapters in halves 840 for 250.
bool terms_with_sums(int grad, int data) { return grad == data || grad == SDCA_F32; }

struct GradPlan {
  int length[2];  // of segments: dB's, dA's
  int64_t segments[2];
  size_t order, spans, table[2], turned, terms[2], parts, partial, end;
};
GradPlan plan_grad(int grad, int data, int64_t d, int64_t m, int64_t n, int64_t count, int64_t rank) {
  GradPlan p;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const auto es = [](int type) { return type == SDCA_F32 ? 4 : 2; };
  p.length[0] = segment_length(es(grad), m, n);
  p.length[1] = segment_length(es(data), d, n);
  p.order = take(n * sizeof(int));
  p.spans = take((count + 1) * sizeof(int2));
  size_t partial = 0;
  for (int t = 0; t < 2; ++t) {
    const Segments s = {p.length[t], nullptr};
    p.segments[t] = s.first(n, count);
    p.table[t] = take(p.segments[t] * sizeof(Segment));
    if (n > p.length[t])
      partial = std::max(partial, static_cast<size_t>(s.slot(n) + 1) * rank * (t ? d : m) * sizeof(float));
    p.terms[t] = take(static_cast<size_t>(n) * terms_pitch(rank) * sizeof(float));
  }
  const bool with = terms_with_sums(grad, data);
  p.turned = take(static_cast<size_t>(count) * m * rank * es(with ? grad : data));
  const int64_t blocks = grad == SDCA_F32 ? column_blocks<float>(m) : column_blocks<__half>(m);
  p.parts = take(with ? static_cast<size_t>(blocks) * n * terms_pitch(rank) * sizeof(float) : 0);
  p.partial = take(partial);
  p.end = at;
  return p;
}

template <class T, bool RANKS_FIRST, bool TERMS>
void sums(const void* Z, int64_t ldz, int64_t wide, const GradPlan& p, const float* terms, float* out,
          const AdaptedGradLaunch& l) {
  constexpr int t = RANKS_FIRST ? 1 : 0;
  char* work = static_cast<char*>(l.work);
  SumArgs a = {};
  a.ldz = ldz;
  a.wide = static_cast<int>(wide);
  a.rank = static_cast<int>(l.adapters.rank);
  a.pitch = static_cast<int>(terms_pitch(a.rank));
  a.terms = terms;
  a.order = reinterpret_cast<const int*>(work + p.order);
  a.segments = reinterpret_cast<const Segment*>(work + p.table[t]);
  a.out = out;
  a.partial = reinterpret_cast<float*>(work + p.partial);
  a.turned = work + p.turned;
  a.scale = l.adapters.scale;
  a.parts = reinterpret_cast<float*>(work + p.parts);
  a.rows = l.n;
  start_sums<T, RANKS_FIRST, TERMS>(static_cast<const T*>(Z), a, p.segments[t], l.stream);
  JoinArgs j = {};
  j.spans = reinterpret_cast<const int2*>(work + p.spans);
  j.count = static_cast<int>(l.adapters.count);
  j.pitch = a.pitch;
  j.terms_blocks = TERMS ? std::min<int64_t>((l.n * a.pitch / 4 + 255) / 256, 8192) : 0;
  j.rows = l.n;
  j.parts = column_blocks<T>(wide);
  j.part_terms = a.parts;
  j.terms = reinterpret_cast<float*>(work + p.terms[1]);
  j.segments = Segments{p.length[t], nullptr};
  j.size = wide * a.rank;
  j.each = std::min<int64_t>((j.size + 255) / 256, std::max<int64_t>(1, 16384 / j.count));
  j.partial = a.partial;
  j.out = out;
  each_slice(j.terms_blocks + j.each * j.count, 1, 256, [&](int64_t first, int64_t count) {
    join_kernel<<<static_cast<unsigned>(count), 256, 0, l.stream>>>(j, first);
  });
}

template <class T, class TO>
void group_turn(const GroupArgs& g, const TurnArgs& t, hipStream_t stream) {
  each_slice((t.m + 63) / 64 * g.count + g.count + 1, 1, 1024, [&](int64_t first, int64_t count) {
    group_turn_kernel<T, TO><<<static_cast<unsigned>(count), 1024, 0, stream>>>(g, t, first);
  });
}
template <class T>
void group_turn(const GroupArgs& g, const TurnArgs& t, int grad, hipStream_t stream) {
  if constexpr (!std::is_same<T, float>::value) {
    if (grad == SDCA_F32) return group_turn<T, float>(g, t, stream);
  }
  group_turn<T, T>(g, t, stream);
}

}  // namespace

// A few workgroups of 16 examples read at some 60 GB/s each: the wide axis is
// shared by more of them until they come to one for each compute unit (1024
// rows of 4096 halves, rank 32, and their 8-bit form, all in tiles: 31 us in one
// part, 20 in four with the sums and the 8-bit form in a launch behind).
int terms_parts(int64_t n, int64_t rank) {
  const int64_t tiles = (n + 15) / 16;
  return terms_by_rows(n, rank) || tiles > 128 ? 1 : static_cast<int>(std::min<int64_t>(8, 256 / tiles));
}

hipError_t launch_terms(const TermsLaunch& l) {
  switch (l.data) {
    case SDCA_F32: return terms<float>(l);
    case SDCA_F16: return terms<__half>(l);
    default: return terms<__hip_bfloat16>(l);
  }
}

hipError_t launch_group(const Adapters& ad, int64_t n, int* order, int2* spans, int* ids,
                        hipStream_t stream) {
  GroupArgs g = {};
  g.index = ad.index;
  g.n = static_cast<int>(n);
  g.count = static_cast<int>(ad.count);
  g.order = order;
  g.spans = spans;
  g.ids = ids;
  group_kernel<<<static_cast<unsigned>(ad.count + 1), 1024, 0, stream>>>(g);
  return hipGetLastError();
}

size_t adapted_grad_work_bytes(int grad, int data, int64_t d, int64_t m, int64_t n, int64_t count,
                               int64_t rank) {
  return plan_grad(grad, data, d, m, n, count, rank).end;
}

hipError_t launch_adapted_grad(const AdaptedGradLaunch& l) {
  const Adapters& ad = l.adapters;
  const GradPlan p = plan_grad(l.grad, ad.data, l.d, l.m, l.n, ad.count, ad.rank);
  char* work = static_cast<char*>(l.work);
  GroupArgs g = {};
  g.index = ad.index;
  g.n = static_cast<int>(l.n);
  g.count = static_cast<int>(ad.count);
  g.order = reinterpret_cast<int*>(work + p.order);
  g.spans = reinterpret_cast<int2*>(work + p.spans);
  for (int t = 0; t < 2; ++t) g.by[t] = Segments{p.length[t], reinterpret_cast<Segment*>(work + p.table[t])};
  void* Bt = work + p.turned;
  const TurnArgs turned = {ad.B, l.m, static_cast<int>(ad.rank), Bt};
  switch (ad.data) {
    case SDCA_F32: group_turn<float>(g, turned, l.grad, l.stream); break;
    case SDCA_F16: group_turn<__half>(g, turned, l.grad, l.stream); break;
    default: group_turn<__hip_bfloat16>(g, turned, l.grad, l.stream);
  }
  float *T = reinterpret_cast<float*>(work + p.terms[0]), *U = reinterpret_cast<float*>(work + p.terms[1]);
  TermsLaunch t;
  t.adapters = &ad;
  t.n = l.n;
  t.order = g.order;
  t.spans = g.spans;
  t.parts = 1;
  t.Q = nullptr;
  t.pad = 0;
  t.scales = nullptr;
  t.stream = l.stream;
  t.data = ad.data;
  t.wide = l.d;
  t.X = l.X;
  t.ldx = l.ldx;
  t.A = ad.A;
  t.terms = T;
  hipError_t e = launch_terms(t);
  if (e != hipSuccess) return e;
  const bool with = terms_with_sums(l.grad, ad.data);
  if (!with) {
    t.data = l.grad;
    t.wide = l.m;
    t.X = l.G;
    t.ldx = l.ldg;
    t.A = Bt;
    t.terms = U;
    if ((e = launch_terms(t)) != hipSuccess) return e;
  }
  switch (l.grad) {
    case SDCA_F32: sums<float, false, true>(l.G, l.ldg, l.m, p, T, l.dB, l); break;
    case SDCA_F16:
      with ? sums<__half, false, true>(l.G, l.ldg, l.m, p, T, l.dB, l)
           : sums<__half, false, false>(l.G, l.ldg, l.m, p, T, l.dB, l);
      break;
    default:
      with ? sums<__hip_bfloat16, false, true>(l.G, l.ldg, l.m, p, T, l.dB, l)
           : sums<__hip_bfloat16, false, false>(l.G, l.ldg, l.m, p, T, l.dB, l);
  }
  switch (ad.data) {
    case SDCA_F32: sums<float, true, false>(l.X, l.ldx, l.d, p, U, l.dA, l); break;
    case SDCA_F16: sums<__half, true, false>(l.X, l.ldx, l.d, p, U, l.dA, l); break;
    default: sums<__hip_bfloat16, true, false>(l.X, l.ldx, l.d, p, U, l.dA, l);
  }
  return hipGetLastError();
}

}  // namespace sdca_gpu
