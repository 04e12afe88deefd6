// The best continuations of groups of beams (include/sophia_pages.h): score +
// log-softmax over the vocabulary, and of all beams' candidates the greatest.
//
// Two passes, the first over the logits, read once: a work-group takes a part of a row and
// leaves its maximum, the sum of e^(x - maximum) and its `keep` greatest logits (of one row
// the order of the logits is that of the candidates).  The second, a work-group per group,
// joins the sums of each row, in double precision, and takes the greatest of what the parts left.
//
// The greatest of many values without sorting them: of 64 sets of them (256 where more than 32 are kept) the keep-th
// greatest of the sets' maxima is not above the keep-th greatest of all, and few values are not below it: those
// are collected, and each finds its place by counting the greater ones.  Equal values are ordered by
// their keys: the token's index, and in the join the beam, then the logit, then the token, so that the order of a
// beam's candidates is that of its logits also where their sums are equal in 64 bits.  More than there is room for (many equal values, or few sets with a value above -inf)
// are found one after the other.
//
// 512 rows of 65,536 logits in bf16 (67 MB): 19.2 us, 10.6 of them until the maxima are known, 2.4 for the sums and
// 6 for what is collected, which the loads of other work-groups hide in part; then 9.8 to join them.  Four rows in
// fp32: 5.1 and 5.4, latency; 64 rows of 32 beams, of which 64 are kept, 12 and 40.
#include <limits>

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
  int beams, keep, parts;
  // Of each (row, part): maximum and sum, and its greatest logits with their tokens.
  double *sum;              // [rows][parts]
  float *top;               // [rows][parts]
  float *value;             // [rows][parts][keep]
  int32_t *token;
  float *out_score;
  int32_t *out_parent;
  int64_t *out_token;
};

// What the lanes hold l ^ 1, ^ 2, ^ 4 and ^ 8 away, without the LDS crossbar, of values that
// are equal within 1, 2, 4 and 8 lanes; then the row swaps.
template <int OFF>
__device__ __forceinline__ float lane_other(float v) {
  if constexpr (OFF == 1) return dpp_rotate<0xb1>(v);    // quad_perm 1, 0, 3, 2
  if constexpr (OFF == 2) return dpp_rotate<0x4e>(v);    // quad_perm 2, 3, 0, 1
  if constexpr (OFF == 4) return dpp_rotate<0x141>(v);   // row_half_mirror
  if constexpr (OFF == 8) return dpp_rotate<0x140>(v);   // row_mirror
  if constexpr (OFF == 16) return lane_xor16(v);
  return lane_xor32(v);
}

// Of a wavefront's values, which are equal within sets of 4 lanes, the greatest.
__device__ __forceinline__ float top_of_quads(float v) {
  v = fmaxf(v, lane_other<4>(v));
  v = fmaxf(v, lane_other<8>(v));
  v = fmaxf(v, lane_other<16>(v));
  return fmaxf(v, lane_other<32>(v));
}
__device__ __forceinline__ float top_of_lanes(float v) {
  v = fmaxf(v, lane_other<1>(v));
  return top_of_quads(fmaxf(v, lane_other<2>(v)));
}

__device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Of 256 sets' maxima, a set per thread of four wavefronts: the least of those of a wavefront that fewer than `keep`
// are above (inf: none); of all wavefronts the keep-th greatest.
__device__ __forceinline__ float kth_of_sets(const float *sets, float mine, int keep) {
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < 256; i += 4) {
    const f4 o = *reinterpret_cast<const f4 *>(sets + i);
    above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
  }
  return -top_of_lanes(above < keep ? -mine : -INFINITY);
}
constexpr int kFewKept = 32;   // to which 64 sets are enough: of 8,192 values 44 are collected of 32, 300 of 64 (of 256 sets 75)

// Collected values with their keys, the lower before the higher where values are equal.
template <typename T, typename K>
struct Room {
  T value[kRoom];
  K key[kRoom];
  __device__ __forceinline__ void set(int at, T v, K k) { value[at] = v, key[at] = k; }
  // How many of those from j0 to j1 come before entry i.
  __device__ __forceinline__ int before(int i, int j0, int j1) const {
    const T v = value[i];
    const K at = key[i];
    int n = 0;
#pragma unroll 4
    for (int j = j0; j < j1; ++j) n += (value[j] > v) | ((value[j] == v) & (key[j] < at));
    return n;
  }
};
template <typename T, typename K, int WAVES>
struct Collected {
  Room<T, K> room;
  int n;
  float top[WAVES], floor[WAVES];
  double sum[WAVES];
  T best[WAVES];
  K best_key[WAVES];
};

template <typename T, typename K, int WAVES>
__device__ __forceinline__ void collect(Collected<T, K, WAVES> &c, T v, K k) {
  const int at = atomicAdd(&c.n, 1);
  if (at < kRoom) c.room.set(at, v, k);
}

// The greatest `keep` of what was collected (after a barrier), in order:
// write(place, value, key) once per place, by any thread.  Returns how many there are.  each(f) calls
// f(value, key) for this thread's candidates: where more were collected than there is room for, they
// are found one after the other, each the greatest of those behind the last one.
template <typename T, typename K, int WAVES, typename E, typename W>
__device__ __forceinline__ int greatest(Collected<T, K, WAVES> &c, int keep, E each, W write) {
  const int n = c.n, t = threadIdx.x;
  constexpr int kThreads = 64 * WAVES;
  if (n <= kRoom) {
    for (int i = t; i < n; i += kThreads) {
      const int place = c.room.before(i, 0, n);
      if (place < keep) write(place, c.room.value[i], c.room.key[i]);
    }
    return min(n, keep);
  }
  T last = 0;
  K last_key = 0;
  for (int place = 0; place < keep; ++place) {
    T best = -INFINITY;
    K best_key = std::numeric_limits<K>::max();
    each([&](T v, K k) {
      if (place > 0 && !(v < last || (v == last && k > last_key))) return;
      if (v > best || (v == best && k < best_key)) best = v, best_key = k;
    });
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const T v = __shfl_xor(best, off, 64);
      const K k = __shfl_xor(best_key, off, 64);
      if (v > best || (v == best && k < best_key)) best = v, best_key = k;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      c.best[threadIdx.x >> 6] = best;
      c.best_key[threadIdx.x >> 6] = best_key;
    }
    __syncthreads();
    best = c.best[0];
    best_key = c.best_key[0];
    for (int i = 1; i < WAVES; ++i)
      if (c.best[i] > best || (c.best[i] == best && c.best_key[i] < best_key)) best = c.best[i], best_key = c.best_key[i];
    if (threadIdx.x == 0) write(place, best, best_key);   // (there are more than kRoom >= keep)
    last = best;
    last_key = best_key;
  }
  return keep;
}

// Values of a thread in the first pass, and of a part: eight consecutive ones of 2,048 at a time (VEC), or every
// 256th.  (With 8 in place of 32 four times as many parts are joined: 64 rows of 65,536 logits in bf16, eight beams of which 16 are
// kept, 20.3 us in place of 15.1, 8 rows 16.7 and 12.8, one row 8.6 and 8.7.)
constexpr int kValues = 32, kPartSize = 256 * kValues;
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a) {
  __shared__ Collected<float, int, 4> s;
  __shared__ __attribute__((aligned(16))) float s_quad[64], s_set[256];   // the maxima of four threads each, and of each
  const int64_t row = blockIdx.y;
  const int part = blockIdx.x, t = threadIdx.x;
  // (a beam that has ended, or cannot be continued, has no use for its logits)
  if (!(fabsf(a.scores[row]) < INFINITY) || (a.ended && a.ended[row])) return;
  constexpr int EPT = kValues;
  const int v0 = part * kPartSize, width = min(kPartSize, a.vocab - v0);
  const int64_t at = row * a.x_stride + v0;
  float x[EPT];
  if (VEC && width % 8 == 0) {   // (no branch between the loads: all are under way together)
    constexpr int kRaw = DT == SOPHIA_DTYPE_BF16 ? 1 : 2;
    u4 raw[EPT / 8][kRaw];
#pragma unroll
    for (int e = 0; e < EPT; e += 8)
#pragma unroll
      for (int k = 0; k < kRaw; ++k)
        raw[e / 8][k] = reinterpret_cast<const u4 *>(static_cast<const char *>(a.x) + (at + min(256 * e + 8 * t, width - 8)) * (2 * kRaw))[k];
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const u4 &r = raw[e / 8][DT == SOPHIA_DTYPE_BF16 ? 0 : (e & 7) / 4];
      if constexpr (DT == SOPHIA_DTYPE_BF16)
        x[e] = __uint_as_float(e & 1 ? r[(e & 7) / 2] & 0xffff0000u : r[(e & 7) / 2] << 16);
      else
        x[e] = __uint_as_float(r[e & 3]);
    }
    if (width < kPartSize) {
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = 256 * (e & ~7) + 8 * t < width ? x[e] : -INFINITY;
    }
  } else {
    uint32_t raw[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const int i = VEC ? 256 * (e & ~7) + 8 * t + (e & 7) : 256 * e + t;
      raw[e] = load_raw(a.x, at + min(i, width - 1), DT);
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const int i = VEC ? 256 * (e & ~7) + 8 * t + (e & 7) : 256 * e + t;
      x[e] = i < width ? raw_to_f32(raw[e], DT) : -INFINITY;
    }
  }
  const auto index = [&](int e) { return VEC ? 256 * (e & ~7) + 8 * t + (e & 7) : 256 * e + t; };
  // (a maximum passes over NaN, and NaN is not above anything)
  float top4[EPT / 4], quad = -INFINITY;
#pragma unroll
  for (int e = 0; e < EPT; e += 4) {
    top4[e / 4] = fmaxf(fmaxf(x[e], x[e + 1]), fmaxf(x[e + 2], x[e + 3]));
    quad = fmaxf(quad, top4[e / 4]);
  }
  const float mine = quad;
  quad = fmaxf(quad, lane_other<1>(quad));
  quad = fmaxf(quad, lane_other<2>(quad));
  const int lane = t & 63, wave = t >> 6;
  if ((lane & 3) == 0) s_quad[t >> 2] = quad;
  if (a.keep > kFewKept) s_set[t] = mine;
  float top = top_of_quads(quad);
  if (lane == 0) s.top[wave] = top;
  if (t == 0) s.n = 0;
  __syncthreads();
  top = fmaxf(fmaxf(s.top[0], s.top[1]), fmaxf(s.top[2], s.top[3]));
  const int64_t slot = row * a.parts + part;
  float *value = a.value + slot * a.keep;
  int32_t *token = a.token + slot * a.keep;
  if (!(top > -INFINITY)) {
    if (t == 0) a.top[slot] = -INFINITY;
    for (int i = t; i < a.keep; i += 256) token[i] = -1;
    return;
  }
  if (a.keep > kFewKept) {
    const float kth = kth_of_sets(s_set, mine, a.keep);
    if (lane == 0) s.floor[wave] = kth;
  } else {
    // How many of the 64 maxima are above this one, a quarter of them compared by each lane of the four.
    int above = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 o = *reinterpret_cast<const f4 *>(s_quad + 16 * (lane & 3) + 4 * i);
      above += (o.x > quad) + (o.y > quad) + (o.z > quad) + (o.w > quad);
    }
    above += __builtin_amdgcn_update_dpp(0, above, 0xb1, 0xf, 0xf, true);
    above += __builtin_amdgcn_update_dpp(0, above, 0x4e, 0xf, 0xf, true);
    const float kth = -top_of_quads(above < a.keep ? -quad : -INFINITY);
    if (lane == 0) s.floor[wave] = kth;
  }
  if (top < INFINITY) {
    // The maximum subtracted first: exact near it whatever its size, and at most -inf for the lowest values.  (A rounded product
    // top log2 e as reference would be off by a factor of its own in each part, 3e-4 of a sum at 10,000, and infinite from 2.4e38 on.)
    const auto add = [&](float v) { return __builtin_amdgcn_exp2f((v - top) * 1.44269504088896341f); };
    float p[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < EPT; ++e) p[e & 3] += add(x[e]);
    float sum = (p[0] + p[1]) + (p[2] + p[3]);
    if (__any(sum != sum)) {   // NaN among them
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < EPT; ++e) sum += x[e] == x[e] ? add(x[e]) : 0.f;
    }
    sum = wave_sum_dpp(sum);
    if ((t & 63) == 0) s.sum[t >> 6] = static_cast<double>(sum);
  }
  __syncthreads();
  const float least = fmaxf(fminf(fminf(s.floor[0], s.floor[1]), fminf(s.floor[2], s.floor[3])), -3.402823466e38f);
  if (mine >= least) {
#pragma unroll
    for (int e = 0; e < EPT; e += 4)
      if (top4[e / 4] >= least) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (x[e + k] >= least) collect(s, x[e + k], index(e + k));
      }
  }
  __syncthreads();
  if (t == 0) {
    a.top[slot] = top;
    a.sum[slot] = (s.sum[0] + s.sum[1]) + (s.sum[2] + s.sum[3]);
  }
  const int n = greatest(
      s, a.keep,
      [&](auto f) {
#pragma unroll
        for (int e = 0; e < EPT; ++e)
          if (x[e] > -INFINITY) f(x[e], index(e));
      },
      [&](int place, float v, int i) {
        value[place] = v;
        token[place] = v0 + i;
      });
  for (int i = n + t; i < a.keep; i += 256) token[i] = -1;
}

// A group's candidates: of beam b, part p and place j the index ((b parts) + p) keep + j, which among equal logits
// of a beam is in the order of their tokens, as parts and places are.  A wavefront
// joins the sums of a beam, a part per lane; meanwhile the candidates are under way, the first of
// all lists first.  The parts' lists are sorted: the keep-th of any of them is not above the
// keep-th greatest of all, and neither is the keep-th of the threads' sets.
constexpr int kJoin = 1024, kHeld = 2;   // threads, and candidates of each that stay in registers
// A candidate's key: its beam, its logit, the greater first, and its index within the beam: of 2^15 parts of 2^28 logits, 64 of each.
constexpr int kIndexBits = 21;
static_assert((1 << 28) / kPartSize * kMost <= 1 << kIndexBits && kMost <= 1 << (63 - 32 - kIndexBits), "a key has 63 bits");
__device__ __forceinline__ int64_t candidate_key(int beam, float x, int in) {
  const uint32_t bits = __float_as_uint(x + 0.f);   // (+0, not -0)
  const uint32_t descending = bits & 0x80000000u ? bits : ~bits & 0x7fffffffu;
  return static_cast<int64_t>(beam) << (32 + kIndexBits) | static_cast<int64_t>(descending) << kIndexBits | in;
}
__global__ __launch_bounds__(kJoin) void beam_join_kernel(BeamArgs a) {
  constexpr int kWaves = kJoin / 64;
  __shared__ Collected<double, int64_t, kWaves> s;
  // Of a beam its greatest logit and the logarithm of its sum relative to it; apart, as next to a large one the other would be lost.
  __shared__ double s_top[kMost], s_log[kMost];
  __shared__ int s_kind[kMost];     // of a beam: 0 no candidates, 1 its logits', 2 itself
  __shared__ __attribute__((aligned(16))) float s_first[kWaves][64], s_set[256];
  __shared__ float s_floor;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.beams;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int lists = a.beams * a.parts, all = lists * a.keep;
  const int64_t base = row0 * a.parts * a.keep;
  // Candidate c is place c / lists of list c % lists.
  const auto index = [&](int c) {
    const int place = c / lists;
    return (c - place * lists) * a.keep + place;
  };
  float held[kHeld];
  int held_token[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int64_t at = base + index(min(t + k * kJoin, all - 1));
    held[k] = a.value[at];
    held_token[k] = a.token[at];
  }
  for (int b = wave; b < a.beams; b += kWaves) {
    const int64_t row = row0 + b;
    const float score = a.scores[row];
    const bool done = a.ended && a.ended[row];
    float top = -INFINITY;
    double log_sum = 0.0;
    int kind = fabsf(score) < INFINITY ? 2 : 0;
    if (kind && !done) {
      for (int p = lane; p < a.parts; p += 64) top = fmaxf(top, a.top[row * a.parts + p]);
      top = top_of_lanes(top);
      kind = top > -INFINITY && top < INFINITY;
      if (kind) {
        double sum = 0.0;
        for (int p = lane; p < a.parts; p += 64) {
          const float m = a.top[row * a.parts + p];
          if (m > -INFINITY) sum += a.sum[row * a.parts + p] * exp(static_cast<double>(m) - static_cast<double>(top));
        }
        log_sum = log(sum_lanes(sum));
      }
    }
    if (lane == 0) {
      s_top[b] = top;
      s_log[b] = log_sum;
      s_kind[b] = kind;
    }
  }
  if (t == 0) s.n = 0;
  __syncthreads();
  const int each_beam = a.parts * a.keep;
  const auto candidate = [&](int i, float x, int token) {
    const int b = i / each_beam;
    const double score = a.scores[row0 + b];
    if (s_kind[b] == 1 && token >= 0) return score + ((static_cast<double>(x) - s_top[b]) - s_log[b]);
    return s_kind[b] == 2 && i == b * each_beam ? score : -static_cast<double>(INFINITY);
  };
  double v[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    v[k] = t + k * kJoin < all ? candidate(index(t + k * kJoin), held[k], held_token[k]) : -INFINITY;
  const auto each = [&](auto f) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (v[k] > -INFINITY) f(v[k], index(t + k * kJoin), held[k]);
    for (int c = t + kHeld * kJoin; c < all; c += kJoin) {
      const int i = index(c);
      const float x = a.value[base + i];
      const double w = candidate(i, x, a.token[base + i]);
      if (w > -INFINITY) f(w, i, x);
    }
  };
  const auto key = [&](int i, float x) {
    const int b = i / each_beam;
    return candidate_key(b, x, i - b * each_beam);
  };
  // (rounding to fp32 keeps the order, but for equal ones)
  float last = -INFINITY;   // the keep-th of a list
  each([&](double w, int i, float) {
    if (i % a.keep == a.keep - 1) last = fmaxf(last, static_cast<float>(w));
  });
  double best = v[0];
#pragma unroll
  for (int k = 1; k < kHeld; ++k) best = fmax(best, v[k]);
  s_first[wave][lane] = static_cast<float>(best);
  last = top_of_lanes(last);
  if (lane == 0) s.top[wave] = last;
  __syncthreads();
  if (a.keep > kFewKept) {   // (as in the first pass, four threads to a set)
    float first = -INFINITY;
    if (wave < 4) {
      for (int i = wave; i < kWaves; i += 4) first = fmaxf(first, s_first[i][lane]);
      s_set[t] = first;
    }
    __syncthreads();
    if (wave < 4) {
      const float kth = kth_of_sets(s_set, first, a.keep);
      if (lane == 0) s.floor[wave] = kth;
    }
    __syncthreads();
    if (wave == 0) {
      const float floor = top_of_lanes(s.top[lane & (kWaves - 1)]);
      if (lane == 0) s_floor = fmaxf(floor, fminf(fminf(s.floor[0], s.floor[1]), fminf(s.floor[2], s.floor[3])));
    }
  } else if (wave == 0) {
    float first = s_first[0][lane], floor = s.top[lane & (kWaves - 1)];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) first = fmaxf(first, s_first[i][lane]);
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < 64; ++i)
      above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(first), i)) > first;
    floor = top_of_lanes(floor);
    // the least of those that fewer than keep are above: the keep-th (-inf: there are not so many)
    const float kth = -top_of_lanes(above < a.keep ? -first : -INFINITY);
    if (lane == 0) s_floor = fmaxf(floor, kth);
  }
  __syncthreads();
  const float floor = s_floor;
  each([&](double w, int i, float x) {
    if (static_cast<float>(w) >= floor) collect(s, w, key(i, x));
  });
  __syncthreads();
  float *out_score = a.out_score + static_cast<int64_t>(blockIdx.x) * a.keep;
  int32_t *out_parent = a.out_parent + static_cast<int64_t>(blockIdx.x) * a.keep;
  int64_t *out_token = a.out_token + static_cast<int64_t>(blockIdx.x) * a.keep;
  const auto each_key = [&](auto f) { each([&](double w, int i, float x) { f(w, key(i, x)); }); };
  const int n = greatest(s, a.keep, each_key, [&](int place, double w, int64_t k) {
    const int b = static_cast<int>(k >> (32 + kIndexBits)), in = static_cast<int>(k & ((1 << kIndexBits) - 1));
    out_score[place] = static_cast<float>(w);
    out_parent[place] = b;
    out_token[place] = s_kind[b] == 2 ? a.pad : a.token[base + b * each_beam + in];
  });
  for (int i = n + t; i < a.keep; i += kJoin) {
    out_score[i] = -INFINITY;
    out_parent[i] = -1;
    out_token[i] = -1;
  }
}

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" size_t sophia_beam_select_workspace_size(int64_t rows, int vocab, int keep) {
  if (rows < 1 || vocab < 1 || keep < 1) return 0;
  const int64_t parts = (vocab + kPartSize - 1) / kPartSize;
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
  const int parts = (vocab + kPartSize - 1) / kPartSize;
  SOPHIA_REQUIRE(static_cast<int64_t>(beams) * parts * keep <= 1 << 30, "beam_select: too many candidates");
  SOPHIA_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                     workspace_bytes >= sophia_beam_select_workspace_size(rows, vocab, keep),
                 "beam_select: workspace too small");
  BeamArgs a{logits, logits_stride, rows, vocab, scores, ended, pad_token, beams, keep, parts,
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
#define SOPHIA_BEAM(dt, v) hipLaunchKernelGGL((beam_part_kernel<dt, v>), grid, dim3(256), 0, st, a)
  if (dtype == SOPHIA_DTYPE_F32) {
    if (vec) SOPHIA_BEAM(SOPHIA_DTYPE_F32, true); else SOPHIA_BEAM(SOPHIA_DTYPE_F32, false);
  } else {
    if (vec) SOPHIA_BEAM(SOPHIA_DTYPE_BF16, true); else SOPHIA_BEAM(SOPHIA_DTYPE_BF16, false);
  }
#undef SOPHIA_BEAM
  hipLaunchKernelGGL(beam_join_kernel, dim3(static_cast<unsigned>(rows / beams)), dim3(kJoin), 0, st, a);
  return check_launch("beam_select");
}
