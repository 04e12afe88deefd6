// The best continuations of groups of beams (include/sophia_pages.h): score +
// log-softmax over the vocabulary, and of all beams' candidates the greatest.
//
// Two passes, the first over the logits, read once: a work-group takes a part of a row and
// leaves its maximum, the sum of e^(x - maximum) and its `keep` greatest logits (of one row
// the order of the logits is that of the candidates).  The second, a work-group per group,
// joins the sums of each row, in double precision, and takes the greatest of what the parts left.
//
// The greatest of many values without sorting them: the values are divided into K >= keep sets
// of equal size; the least of the sets' maxima is not above the keep-th greatest, as
// K values are not below it, and only about K log K values are: those are collected, and each
// finds its place by counting the greater ones.  Equal values are ordered by their index.
// More than fit (many equal values, or few values above -inf) are found one after the other.
#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_pages.h"

namespace sophia {
namespace {

constexpr int kMost = SOPHIA_BEAMS;   // of keep
constexpr int kRoom = 1024;           // collected values

struct BeamArgs {
  const void *x;
  int64_t x_stride;
  int64_t rows;
  int vocab;
  const float *scores;
  const uint8_t *ended;     // NULL: none
  int64_t pad;
  int beams, keep, sets, parts;
  // Of each (row, part): maximum and sum, and its greatest logits with their tokens.
  double *sum;              // [rows][parts]
  float *top;               // [rows][parts]
  float *value;             // [rows][parts][keep]
  int32_t *token;
  float *out_score;
  int32_t *out_parent;
  int64_t *out_token;
};

// A work-group's maximum and sum, in every thread.  `s` holds a value per wavefront.
template <typename T, typename F>
__device__ __forceinline__ T across(T v, T *s, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if (lane == 0) s[wave] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < waves; ++i) v = f(v, s[i]);
  return v;
}

// The least of the maxima of `sets` sets of threads, a power of two up to the threads of the
// work-group and at least one per wavefront; `v` is this thread's maximum.
template <typename T>
__device__ __forceinline__ T least_of_sets(T v, int sets, T *s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int size = blockDim.x / sets;   // threads of a set
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_xor(v, off, 64);
    v = (off < size) == (o > v) ? o : v;
  }
  __syncthreads();
  if (lane == 0) s[wave] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < waves; ++i) v = s[i] < v ? s[i] : v;
  return v;
}

// The greatest `keep` of the work-group's values in order; each(f) calls f(value, index) for those
// of this thread that are candidates, in ascending order of their indexes.  write(place, value,
// index) is called once per place, by any thread; returns how many there are.
template <typename T>
struct Collected {
  T value[kRoom];
  int index[kRoom];
  int n;
  T wave[16];
  int wave_index[16];
};
template <typename T, typename E, typename W>
__device__ __forceinline__ int greatest(Collected<T> &c, T mine, int sets, int keep, E each, W write) {
  const T floor = least_of_sets(mine, sets, c.wave);
  if (threadIdx.x == 0) c.n = 0;
  __syncthreads();
  each([&](T v, int i) {
    if (v >= floor) {
      const int at = atomicAdd(&c.n, 1);
      if (at < kRoom) {
        c.value[at] = v;
        c.index[at] = i;
      }
    }
  });
  __syncthreads();
  const int n = c.n;
  if (n <= kRoom) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const T v = c.value[i];
      const int at = c.index[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += c.value[j] > v || (c.value[j] == v && c.index[j] < at);
      if (place < keep) write(place, v, at);
    }
    return min(n, keep);
  }
  // One after the other: the greatest of those behind the last one.
  T last = 0;
  int last_at = -1;
  for (int place = 0; place < keep; ++place) {
    T best = -INFINITY;
    int best_at = 0x7fffffff;
    each([&](T v, int i) {
      if (place > 0 && !(v < last || (v == last && i > last_at))) return;
      if (v > best || (v == best && i < best_at)) best = v, best_at = i;
    });
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const T v = __shfl_xor(best, off, 64);
      const int at = __shfl_xor(best_at, off, 64);
      if (v > best || (v == best && at < best_at)) best = v, best_at = at;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      c.wave[threadIdx.x >> 6] = best;
      c.wave_index[threadIdx.x >> 6] = best_at;
    }
    __syncthreads();
    best = c.wave[0];
    best_at = c.wave_index[0];
    for (int i = 1; i < static_cast<int>(blockDim.x >> 6); ++i)
      if (c.wave[i] > best || (c.wave[i] == best && c.wave_index[i] < best_at)) best = c.wave[i], best_at = c.wave_index[i];
    if (threadIdx.x == 0) write(place, best, best_at);   // (there are more than kRoom >= keep)
    last = best;
    last_at = best_at;
  }
  return keep;
}

// Values of a thread in the first pass: EPT of them, eight consecutive ones of 2,048 at a time
// (VEC), or every 256th.
template <int DT, bool VEC, int EPT>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a) {
  __shared__ Collected<float> s;
  __shared__ double s_sum[4];
  const int64_t row = blockIdx.y;
  const int part = blockIdx.x, t = threadIdx.x;
  // (a beam that has ended, or cannot be continued, has no use for its logits)
  if (!(fabsf(a.scores[row]) < INFINITY) || (a.ended && a.ended[row])) return;
  const int v0 = part * 256 * EPT, width = min(256 * EPT, a.vocab - v0);
  const int64_t at = row * a.x_stride + v0;
  float x[EPT];
#pragma unroll
  for (int e = 0; e < EPT; e += 8) {
    if constexpr (VEC) {
      const int i = 256 * e + 8 * t;
      if (i + 8 <= width) {
        const f4 lo = load4(a.x, at + i, DT), hi = load4(a.x, at + i + 4, DT);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[e + k] = lo[k], x[e + 4 + k] = hi[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[e + k] = i + k < width ? load_elem(a.x, at + i + k, DT) : -INFINITY;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = 256 * (e + k) + t;
        x[e + k] = i < width ? load_elem(a.x, at + i, DT) : -INFINITY;
      }
    }
  }
  const auto index = [&](int e) { return VEC ? 256 * (e & ~7) + 8 * t + (e & 7) : 256 * e + t; };
  float mine = -INFINITY;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    if (!(x[e] > -INFINITY)) x[e] = -INFINITY;   // NaN: no candidate
    mine = fmaxf(mine, x[e]);
  }
  const float top = across(mine, s.wave, [](float p, float q) { return fmaxf(p, q); });
  const int64_t slot = row * a.parts + part;
  double sum = 0.0;
  if (top > -INFINITY && top < INFINITY) {
    float p = 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) p += __expf(x[e] - top);
    sum = across(static_cast<double>(p), s_sum, [](double q, double r) { return q + r; });
  }
  if (t == 0) {
    a.top[slot] = top;
    a.sum[slot] = sum;
  }
  float *value = a.value + slot * a.keep;
  int32_t *token = a.token + slot * a.keep;
  const int n = top > -INFINITY
                    ? greatest<float>(
                          s, mine, a.sets, a.keep,
                          [&](auto f) {
#pragma unroll
                            for (int e = 0; e < EPT; ++e)
                              if (x[e] > -INFINITY) f(x[e], index(e));
                          },
                          [&](int place, float v, int i) {
                            value[place] = v;
                            token[place] = v0 + i;
                          })
                    : 0;
  for (int i = n + t; i < a.keep; i += 256) token[i] = -1;
}

// A group's candidates: of beam b, part p and place j the index ((b parts) + p) keep + j; equal
// values of one beam are in the order of their tokens, as parts and places are.
__global__ __launch_bounds__(256) void beam_join_kernel(BeamArgs a) {
  __shared__ Collected<double> s;
  __shared__ double s_lse[kMost];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.beams;
  const int t = threadIdx.x;
  for (int b = t; b < a.beams; b += 256) {
    const int64_t row = row0 + b;
    double lse = INFINITY;   // (no candidates)
    if (fabsf(a.scores[row]) < INFINITY && !(a.ended && a.ended[row])) {
      float top = -INFINITY;
      for (int p = 0; p < a.parts; ++p) top = fmaxf(top, a.top[row * a.parts + p]);
      if (top > -INFINITY && top < INFINITY) {
        double sum = 0.0;
        for (int p = 0; p < a.parts; ++p) {
          const float m = a.top[row * a.parts + p];
          if (m > -INFINITY) sum += a.sum[row * a.parts + p] * exp(static_cast<double>(m) - static_cast<double>(top));
        }
        lse = static_cast<double>(top) + log(sum);
      }
    }
    s_lse[b] = lse;
  }
  __syncthreads();
  const int each_beam = a.parts * a.keep, all = a.beams * each_beam;
  const auto candidate = [&](int i) {
    const int b = i / each_beam;
    const int64_t row = row0 + b;
    const float score = a.scores[row];
    if (!(fabsf(score) < INFINITY)) return -static_cast<double>(INFINITY);
    if (a.ended && a.ended[row]) return i == b * each_beam ? static_cast<double>(score) : -static_cast<double>(INFINITY);
    const int64_t at = row0 * each_beam + i;
    if (!(s_lse[b] < INFINITY) || a.token[at] < 0) return -static_cast<double>(INFINITY);
    return static_cast<double>(score) + (static_cast<double>(a.value[at]) - s_lse[b]);
  };
  double mine = -INFINITY;
  for (int i = t; i < all; i += 256) {
    const double v = candidate(i);
    mine = v > mine ? v : mine;
  }
  float *out_score = a.out_score + static_cast<int64_t>(blockIdx.x) * a.keep;
  int32_t *out_parent = a.out_parent + static_cast<int64_t>(blockIdx.x) * a.keep;
  int64_t *out_token = a.out_token + static_cast<int64_t>(blockIdx.x) * a.keep;
  const int n = greatest<double>(
      s, mine, a.sets, a.keep,
      [&](auto f) {
        for (int i = t; i < all; i += 256) {
          const double v = candidate(i);
          if (v > -INFINITY) f(v, i);
        }
      },
      [&](int place, double v, int i) {
        const int b = i / each_beam;
        out_score[place] = static_cast<float>(v);
        out_parent[place] = b;
        out_token[place] = a.ended && a.ended[row0 + b] ? a.pad : a.token[row0 * each_beam + i];
      });
  for (int i = n + t; i < a.keep; i += 256) {
    out_score[i] = -INFINITY;
    out_parent[i] = -1;
    out_token[i] = -1;
  }
}

// Values of a thread: many where there are rows enough to fill the chip.
int part_values(int64_t rows, int vocab) {
  return rows * ((vocab + 8191) / 8192) >= 1024 ? 32 : 8;
}

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" size_t sophia_beam_select_workspace_size(int64_t rows, int vocab, int keep) {
  if (rows < 1 || vocab < 1 || keep < 1) return 0;
  const int64_t each = 256 * part_values(rows, vocab), parts = (vocab + each - 1) / each;
  return static_cast<size_t>(rows * parts) * (8 + 4 + 8 * static_cast<size_t>(keep));
}

extern "C" int sophia_beam_select(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                                  const float *scores, const uint8_t *ended, int64_t pad_token, int beams, int keep,
                                  float *out_scores, int32_t *out_parent, int64_t *out_token, void *workspace,
                                  size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "beam_select: dtype not supported");
  SOPHIA_REQUIRE(vocab >= 1 && vocab <= 1 << 28, "beam_select: vocab must be in [1, 2^28]");
  SOPHIA_REQUIRE(beams >= 1 && beams <= SOPHIA_BEAMS && keep >= 1 && keep <= SOPHIA_BEAMS,
                 "beam_select: beams and keep must be in [1, %d]", SOPHIA_BEAMS);
  SOPHIA_REQUIRE(rows >= 0 && rows % beams == 0 && rows <= 65535, "beam_select: rows must be a multiple of beams, at most 65535");
  SOPHIA_REQUIRE(logits_stride >= vocab, "beam_select: row stride smaller than a row");
  if (rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(logits && scores && out_scores && out_parent && out_token, "beam_select: NULL pointer");
  const int values = part_values(rows, vocab), each = 256 * values, parts = (vocab + each - 1) / each;
  SOPHIA_REQUIRE(static_cast<int64_t>(beams) * parts * keep <= 1 << 30, "beam_select: too many candidates");
  SOPHIA_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                     workspace_bytes >= sophia_beam_select_workspace_size(rows, vocab, keep),
                 "beam_select: workspace too small");
  int sets = 4;
  while (sets < keep) sets *= 2;
  BeamArgs a{logits, logits_stride, rows, vocab, scores, ended, pad_token, beams, keep, sets, parts,
             nullptr, nullptr, nullptr, nullptr, out_scores, out_parent, out_token};
  const int64_t n = rows * parts;
  a.sum = static_cast<double *>(workspace);
  a.top = reinterpret_cast<float *>(a.sum + n);
  a.value = a.top + n;
  a.token = reinterpret_cast<int32_t *>(a.value + n * keep);
  const int esz = dtype == SOPHIA_DTYPE_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && logits_stride * esz % 16 == 0;
  const dim3 grid(parts, static_cast<unsigned>(rows));
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SOPHIA_BEAM(dt, v, n) hipLaunchKernelGGL((beam_part_kernel<dt, v, n>), grid, dim3(256), 0, st, a)
#define SOPHIA_BEAM_DT(dt)                                                           \
  do {                                                                               \
    if (values == 32) {                                                              \
      if (vec) SOPHIA_BEAM(dt, true, 32); else SOPHIA_BEAM(dt, false, 32);           \
    } else {                                                                         \
      if (vec) SOPHIA_BEAM(dt, true, 8); else SOPHIA_BEAM(dt, false, 8);             \
    }                                                                                \
  } while (0)
  if (dtype == SOPHIA_DTYPE_F32) SOPHIA_BEAM_DT(SOPHIA_DTYPE_F32);
  else SOPHIA_BEAM_DT(SOPHIA_DTYPE_BF16);
#undef SOPHIA_BEAM_DT
#undef SOPHIA_BEAM
  hipLaunchKernelGGL(beam_join_kernel, dim3(static_cast<unsigned>(rows / beams)), dim3(256), 0, st, a);
  return check_launch("beam_select");
}
