// MLA attention in latent space over paged latents, and the latent norms that write
// them (include/sophia_pages.h).
//
// Keys and values are the same rows, so a tile of them is staged in LDS once and read
// twice, as K rows and, transposed, as V, under a running maximum and sum.  The columns of
// the products are the (token, head) pairs of a sequence, packed: with 16 heads 32 columns
// are two tokens.  Two forms of one kernel:
//   wide   : a work-group takes 4 x 32 columns (fp32: 4 x 16) and a range of their keys; its
//            wavefronts share tiles of 64 keys and differ in their columns.
//   narrow : a sequence of at most 16 columns, so a token of 16 heads: a work-group
//            takes a range of its keys, and the wavefronts differ in their keys, each with tiles
//            of its own and no barrier until they join through LDS at the end.
// A sequence of several ranges leaves partials, which a second kernel joins.
//
// What bounds them (rank 128, 16 heads, bf16): the wide form the matrix pipes and the vector unit in turn, as a
// wavefront's tile is 48 products (1,536 cycles) and 300 vector instructions (1,700) that wait for one another, of
// 3,700 in all: 8 sequences of 300 to 777 new tokens after up to 2,221 in 81 us and 9 to join them (411 TFLOP/s with both), 16 new
// ones of 1,024 161 (426).  Eight wavefronts that take turns at products and softmax, with tiles in threes, were slower
// (100, 180), and so was a work-group that goes on to its next item by itself (95).  The narrow form is latency: one
// token after 700 9.2 us, 96 tokens after 221 to 3,090 each 12.8 and 4.  Between the forms, two tokens of each of 96 sequences
// after 208 to 3,982 are the wide form's, three of whose four wavefronts have no columns: 47 us, four tokens 51, one 16.5.
#include "common.hpp"
#include "pages.hpp"
#include "tree.hpp"

#include "../../include/sophia_pages.h"

namespace sophia {
namespace {

constexpr float kSlack = 8.f;    // (powers of 2)
constexpr int kWideKeys = 64;    // keys of a tile of the wide form

struct PagedArgs {
  Pages p;
  const void *qa;
  int64_t qa_stride;
  void *out;
  int64_t out_stride;
  float scale_log2;
  int heads, max_new;
  // Narrow: key ranges of a sequence at most, keys of one, and the partials [sequence][range] if there are several.
  int narrow_blocks, narrow_splits, narrow_keys;
  float *narrow_part;
  // Wide: ranges of a sequence at most (a division of it into `wide_splits` > 0), and the partials, of four wavefronts each.
  int wide_blocks, wide_used, wide_splits, part_cap;
  float *wide_part;
};
constexpr int kLeast = 2;     // tiles of a wide range at least
// Tiles of a range in shares of the whole work: with fewer more partials, with more the chip waits for the last
// ones (8 sequences of 300 to 777 new tokens after up to 2,221: 1.0 96.1 us, 1.3 96.2, 1.6 92.1, 2.0 96.7, with the merge;
// four of 700 after 2,000 118.9, 118.5, 111.9, 118.6).
constexpr float kStretch = 1.6f;
// Work-groups that run at a time.
template <int R>
constexpr int kSlots = R <= 128 ? 512 : 256;

template <int R, bool F32, bool NARROW>
struct Form {
  static constexpr bool k16 = F32 || NARROW;                      // 16 columns to a wavefront, in 16x16 products
  static constexpr int kCols = k16 ? 16 : 32;
  static constexpr int kGroup = NARROW ? kCols : 4 * kCols;       // of a work-group
  static constexpr int kKeys = !NARROW ? kWideKeys : F32 && R == 256 ? 16 : 32;   // of a tile
  static constexpr int kBytes = R * (F32 ? 4 : 2);                // of a row
  static constexpr int kChunks = kBytes / 16;
  static constexpr int kTile = kKeys * kBytes;
  static constexpr int kQuads = k16 ? R / 16 : R / 8;             // four ranks each, of a lane's column
  static constexpr int kPart = 64 * (4 * kQuads + 2);             // floats of a wavefront's partial: [kQuads][64 lanes] times four,
                                                                  // then maximum and sum [64 lanes]
  static __device__ __forceinline__ int rank(int j) {             // the first of quad j's
    const int lane = threadIdx.x & 63;
    return k16 ? 16 * j + 4 * (lane >> 4) : 8 * j + 4 * (lane >> 5);
  }
  static constexpr int kOwn = NARROW ? kKeys : kKeys / 4;         // rows that a wavefront stages
  static constexpr int kLoads = kOwn * kChunks / 64;
};

typedef float f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ bf8 bits_to_bf8(const u4 &v) { return __builtin_bit_cast(bf8, v); }
__device__ __forceinline__ f16v mfma32x32(const bf8 &a, const bf8 &b, const f16v &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ const u4 zero_rows[2048] = {};   // what keys that are not there are read from: 32 rows of 1 KiB at most

// Chunk c (16 bytes) of an LDS row lies at place c ^ turn(row): in bf16 eight rows of one chunk
// (K) and four rows of two chunks (V, transposing reads), in fp32 sixteen rows of one chunk and
// four rows of four, touch all banks.
template <bool F32>
__device__ __forceinline__ int turn(int row) {
  return F32 ? row & 15 : ((row & 7) << 1) | ((row >> 3) & 1);
}
template <int R, bool F32>
__device__ __forceinline__ int place(int row, int chunk) {   // in bytes
  constexpr int kChunks = R * (F32 ? 4 : 2) / 16;
  return 16 * (row * kChunks + (chunk ^ (turn<F32>(row) & (kChunks - 1))));
}

// What a work-group does.
struct Work {
  Sequence q;
  int col0, cols;           // its first column, and the sequence's
  int first, last;          // tokens of its first and its last column
  int k0, k1;               // its keys
  int used;                 // ranges of these columns
  int64_t part;             // its partial; that of the next range is `step` on
  int step;
};

// Whether a sequence is the narrow form's: by the rows that are computed, max_new of them at most.
__device__ __forceinline__ bool narrow_cols(const PagedArgs &a, int n, int cols) {
  return a.narrow_blocks && min(n, a.max_new) <= cols / a.heads;
}

// The columns from w.col0 on of sequence w.q (which is that of all of its rows; those past max_new
// have no columns); returns the keys that their last token sees.
__device__ __forceinline__ int columns(const PagedArgs &a, Work &w, int group) {
  w.q.n = min(w.q.n, a.max_new);
  w.cols = w.q.n * a.heads;
  w.first = w.col0 / a.heads;
  w.last = (min(w.col0 + group, w.cols) - 1) / a.heads;
  return max(0, min(w.q.pos0 + w.last + 1, w.q.keys));
}

// Narrow: range `split` of sequence s.
template <int R, bool F32>
__device__ __forceinline__ bool find_narrow(const PagedArgs &a, Work &w, int s, int split) {
  using F = Form<R, F32, true>;
  w.q = sequence(a.p, s);
  if (w.q.n == 0 || !narrow_cols(a, w.q.n, F::kCols)) return false;
  w.col0 = 0;
  const int keys = columns(a, w, F::kGroup);
  // (the last range has what max_len did not tell of)
  w.used = max(1, min((keys + a.narrow_keys - 1) / a.narrow_keys, a.narrow_splits));
  w.k0 = split * a.narrow_keys;
  w.k1 = split == a.narrow_splits - 1 ? keys : min(keys, w.k0 + a.narrow_keys);
  w.part = static_cast<int64_t>(s) * a.narrow_splits + split;
  w.step = 1;
  return split < w.used;
}

// Wide: a sequence per lane, 64 at a time.  The host does not know the lengths, so every work-group
// finds its share in the list of all (sequence, range, group), which it counts itself.  Ranges are about
// equally long, which follows from the whole work.
template <int R, bool F32>
struct Lanes {
  using F = Form<R, F32, false>;
  const PagedArgs &a;
  Sequence q;
  int groups = 0, tiles = 0, fewest = 0;         // of this lane's sequence; tiles of its last group and of its first
  int used = 0, items = 0, parts = 0;            // ranges, (range, group) items, those of them that are partials
  __device__ __forceinline__ explicit Lanes(const PagedArgs &args) : a(args) {}
  __device__ __forceinline__ void look(int s) {
    const int in = min(s, a.p.n_seqs - 1);
    q = sequence(a.p, in);
    const int n = s == in && !narrow_cols(a, q.n, Form<R, F32, true>::kCols) ? min(q.n, a.max_new) : 0;
    groups = (n * a.heads + F::kGroup - 1) / F::kGroup;
    const auto tiles_to = [&](int token) { return (max(0, min(q.pos0 + token + 1, q.keys)) + kWideKeys - 1) / kWideKeys; };
    tiles = tiles_to(n - 1);
    fewest = tiles_to(0);
  }
  __device__ __forceinline__ void divide(int length) {
    const int least = a.wide_splits ? (tiles + a.wide_splits - 1) / a.wide_splits : max(length, (tiles + a.wide_used - 1) / a.wide_used);
    used = tiles ? (tiles + least - 1) / least : 1;
    items = used * groups;
    parts = used > 1 ? items : 0;
  }
  // Tiles of a range at most.  With W = sum of groups x tiles, kSlots work-groups at a time have W / kSlots
  // tiles each.  A sequence's last group has at most twice the tiles of its groups on average, so there are at most
  // 2 W / length items and one more per group; those of sequences of two ranges or more, the partials, are
  // at most 4 W / length.
  __device__ __forceinline__ int range_tiles(int lane) {
    float work = 0.f;
    for (int s0 = (a.p.n_seqs - 1) & ~63; s0 >= 0; s0 -= 64) {
      look(s0 + lane);
      work += 0.5f * static_cast<float>(groups) * static_cast<float>(tiles + fewest);
    }
    work = row_sum16(work);
    work += lane_xor16(work);
    work = (work + lane_xor32(work)) * 1.0001f + 1.f;   // (not less than it is, by rounding)
    return max(kLeast, static_cast<int>(fminf(ceilf(work * kStretch / static_cast<float>(kSlots<R>)), 1 << 29)));
  }
};

// Up to 64 sequences' shares of the list, the longest ranges first, so that the last items are short ones: of place i
// in this order the sequence, its groups, ranges and tiles, and items and partials up to and including it.
struct Shares {
  int groups[64], used[64], tiles[64], items[64], parts[64];
  Sequence q[64];
  int n, length;
};

// By one wavefront; the lanes have looked at the sequences from s0 on.
template <int R, bool F32>
__device__ __forceinline__ void share(Lanes<R, F32> &l, Shares &t, int s0, int length) {
  const int lane = threadIdx.x & 63;
  l.divide(length);
  const bool real = l.groups > 0;
  const int key = real ? (l.tiles + l.used - 1) / l.used << 6 | (63 - lane) : -1;
  int place = 0;
  for (uint64_t m = __ballot(real); m; m &= m - 1)
    place += __builtin_amdgcn_readlane(key, __ffsll(static_cast<unsigned long long>(m)) - 1) > key;
  t.groups[lane] = t.items[lane] = t.parts[lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  if (real) {
    t.q[place] = l.q;
    t.groups[place] = l.groups;
    t.used[place] = l.used;
    t.tiles[place] = l.tiles;
    t.items[place] = l.items;
    t.parts[place] = l.parts;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  const int items = wave_scan(t.items[lane]), parts = wave_scan(t.parts[lane]);
  t.items[lane] = items;
  t.parts[lane] = parts;
  if (lane == 0) t.n = __popcll(__ballot(real));
}

// Group g of place i, its range `split`; `parts` partials come before those of these 64 sequences.
template <int R, bool F32>
__device__ __forceinline__ bool take(const PagedArgs &a, const Shares &t, Work &w, int i, int g, int split, int parts) {
  using F = Form<R, F32, false>;
  const int groups = t.groups[i], used = t.used[i];
  w.q = t.q[i];
  w.col0 = (groups - 1 - g) * F::kGroup;     // (late groups, which see most keys, first)
  const int keys = columns(a, w, F::kGroup), tiles = (keys + kWideKeys - 1) / kWideKeys;
  const int least = max(1, (t.tiles[i] + used - 1) / used);
  w.used = max(1, (tiles + least - 1) / least);
  const int mine = tiles / w.used, more = tiles - mine * w.used;   // the first `more` ranges have one more
  w.k0 = kWideKeys * (mine * split + min(split, more));
  w.k1 = min(keys, w.k0 + kWideKeys * (mine + (split < more ? 1 : 0)));
  w.part = parts + (i ? t.parts[i - 1] : 0) + split * groups + g;
  w.step = groups;
  return split < w.used && (w.used == 1 || w.part + static_cast<int64_t>(w.used - 1 - split) * groups < a.part_cap);   // (always, see range_tiles)
}

// The place of the first 64 whose sum is above `item`, by a wavefront.
__device__ __forceinline__ int place_of(const int *sums, int item) {
  return __ffsll(static_cast<unsigned long long>(__ballot(item < sums[threadIdx.x & 63]))) - 1;
}

// The lane's column `col` of a range: the result, or a partial at p.
template <int R, bool F32, typename V>
__device__ __forceinline__ void put(const PagedArgs &a, const Work &w, float *p, int col, float m, float l, V value) {
  using F = Form<R, F32, false>;
  constexpr int kQuads = F::kQuads;
  const int lane = threadIdx.x & 63;
  if (w.used > 1) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) reinterpret_cast<f4 *>(p)[64 * j + lane] = value(j);
    reinterpret_cast<f2 *>(p + 256 * kQuads)[lane] = f2{m, l};
  } else if (col < w.cols) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;   // (no key: zeros)
    const int token = col / a.heads, head = col - token * a.heads;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
      store4(a.out, (w.q.base + token) * a.out_stride + static_cast<int64_t>(head) * R + F::rank(j),
             F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, value(j) * inv);
  }
}

// A tile on its way into LDS: the ids of its pages, a key per lane, and the copies.
template <int R, bool F32, bool NARROW>
struct Stage {
  using F = Form<R, F32, NARROW>;
  const PagedArgs &a;
  const Work &w;
  int lane, row0;                 // this wavefront's first row
  uint32_t offset[F::kLoads];     // of this lane's chunks from that row on, in bytes
  __device__ __forceinline__ Stage(const PagedArgs &args, const Work &work)
      : a(args), w(work), lane(threadIdx.x & 63), row0(NARROW ? 0 : F::kOwn * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
#pragma unroll
    for (int t = 0; t < F::kLoads; ++t) {
      const int row = 64 / F::kChunks * t + lane / F::kChunks;
      offset[t] = row * F::kBytes + 16 * ((lane % F::kChunks) ^ (turn<F32>(row0 + row) & (F::kChunks - 1)));
    }
  }
  // The page of key k0 + lane, as the table has it (k0 < k1; of the tile's keys, lanes past them repeat;
  // past the last key its page), and whether it is one and the key is there: apart, so that nothing waits for the load.
  __device__ __forceinline__ int load_id(int k0) const {
    const int j = min(k0 + (lane & (F::kKeys - 1)), w.k1 - 1);
    return a.p.table[w.q.slot * a.p.table_stride + (j >> a.p.shift)];
  }
  __device__ __forceinline__ int id_of(int k0, int id) const {
    return k0 + (lane & (F::kKeys - 1)) < w.k1 && id >= 0 && id < a.p.n_pages ? id : -1;
  }
  // Where this wavefront's rows of a tile lie in one page there is one address, a scalar, and offsets per lane
  // that do not change; else (small pages, the last keys) each lane has its own addresses.
  __device__ __forceinline__ void copy(char *tile, int k0, int id) const {
    char *to = tile + 16 * row0 * F::kChunks;
    const int of = lane / F::kChunks;
    if ((1 << a.p.shift) >= F::kOwn && k0 + F::kKeys <= w.k1) {
      const int page = __builtin_amdgcn_readlane(id, row0), at = (k0 + row0) & ((1 << a.p.shift) - 1);
      const int64_t skip = page * (a.p.page_stride * (F32 ? 4 : 2)) + at * F::kBytes;
      const char *from = page >= 0 ? static_cast<const char *>(a.p.pages) + skip : reinterpret_cast<const char *>(zero_rows);
#pragma unroll
      for (int t = 0; t < F::kLoads; ++t)
        __builtin_amdgcn_global_load_lds(from + offset[t], to + 1024 * t, 16, 0, 0);
    } else {
#pragma unroll
      for (int t = 0; t < F::kLoads; ++t) {
        const int row = row0 + 64 / F::kChunks * t + of, c = (lane % F::kChunks) ^ (turn<F32>(row) & (F::kChunks - 1));
        const int page = __shfl(id, row, 64);
        const int at = (k0 + row) & ((1 << a.p.shift) - 1);
        const char *from = static_cast<const char *>(a.p.pages) +
                           (page * a.p.page_stride * (F32 ? 4 : 2) + static_cast<int64_t>(at) * F::kBytes + 16 * c);
        __builtin_amdgcn_global_load_lds(page >= 0 ? from : reinterpret_cast<const char *>(zero_rows), to + 1024 * t, 16, 0, 0);
      }
    }
  }
  // Chunks that hold a value that is not finite become zeros; returns the rows that had one, of
  // those that this wavefront copied.
  __device__ __forceinline__ uint64_t clean(char *tile) const {
    uint64_t rows = 0;
#pragma unroll
    for (int t = 0; t < F::kLoads; ++t) {
      u4 *at = reinterpret_cast<u4 *>(tile + 16 * (row0 * F::kChunks + 64 * t) + 16 * lane);
      const u4 v = *at;
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (F32)
          any |= (v[i] & 0x7f800000u) == 0x7f800000u;
        else
          any |= (v[i] & 0x7f800000u) == 0x7f800000u || (v[i] & 0x7f80u) == 0x7f80u;
      }
      if (any) *at = u4{0u, 0u, 0u, 0u};
      const uint64_t hit = __ballot(any);
#pragma unroll
      for (int r = 0; r < 64 / F::kChunks; ++r)
        if ((hit >> (r * F::kChunks)) & (~0ull >> (64 - F::kChunks))) rows |= 1ull << (row0 + 64 / F::kChunks * t + r);
    }
    return rows;
  }
};

// The softmax and value product of a wavefront's columns: bf16 in 32x32x16 MFMAs (wide).  A
// probability enters the value product as two bf16 numbers, the second what the first has
// lost (2^-16 of it remains lost), so that outputs are as close as their own rounding;
// scores, maxima and sums are fp32.
template <int R>
struct Bf16Columns {
  using F = Form<R, false, false>;
  static constexpr int KS = R / 16, DT = R / 32, KT = F::kKeys / 32;
  const PagedArgs &a;
  bf8 qf[KS];
  f16v ot[DT];
  float m, l;          // l over this lane's keys alone
  int lane, half;
  int ko[KS], vo[DT];  // places of this lane's reads in a tile
  __device__ __forceinline__ explicit Bf16Columns(const PagedArgs &args) : a(args), m(-INFINITY), l(0.f) {
    lane = threadIdx.x & 63;
    half = lane >> 5;
    const int l16 = lane & 15;
    // K row lane % 32 (32 kt rows on: a constant); V rows 4 half + l16 / 4 (16 kp rows on: a
    // constant; 8 rows on: the chunk's lowest bit turns).
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ko[ks] = place<R, false>(lane & 31, 2 * ks + half);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      vo[dt] = place<R, false>(4 * half + (l16 >> 2), 4 * dt + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1)) + 8 * (l16 & 1);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) ot[dt][i] = 0.f;
  }
  __device__ __forceinline__ int column() const { return lane & 31; }
  __device__ __forceinline__ void queries(int64_t row, int head) {
    const uint16_t *qp = static_cast<const uint16_t *>(a.qa) + row * a.qa_stride + static_cast<int64_t>(head) * R + 8 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = bits_to_bf8(*reinterpret_cast<const u4 *>(qp + 16 * ks));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));   // (waited for here, not in the loop)
  }
  // One tile, of which this lane's column sees the keys `seen` (`all`: every key).
  __device__ __forceinline__ void tile(const char *lds, bool all, uint64_t seen) {
    // st[kt][i] = score(key 32 kt + 8 (i / 4) + 4 half + i % 4 of the tile, this column)
    f16v st[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
    // K rows two steps ahead of their products, by hand: left to itself the compiler waits for each read.
    constexpr int kAhead = 3;
    bf8 k[kAhead][KT];
    const auto read_k = [&](int ks) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        k[ks % kAhead][kt] = bits_to_bf8(*reinterpret_cast<const u4 *>(lds + ko[ks] + 32 * kt * F::kBytes));
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int ks = 0; ks < kAhead - 1 && ks < KS; ++ks) read_k(ks);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + kAhead - 1 < KS) read_k(ks + kAhead - 1);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) st[kt] = mfma32x32(k[ks % kAhead][kt], qf[ks], st[kt]);
    }
    if (!all) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t bits = static_cast<uint32_t>(seen >> (32 * kt)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) st[kt][i] = bits & (1u << (8 * (i >> 2) + (i & 3))) ? st[kt][i] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      float top[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = st[kt][8 * i];
#pragma unroll
        for (int j = 1; j < 8; ++j) top[i] = fmaxf(top[i], st[kt][8 * i + j]);
      }
      mx = fmaxf(mx, fmaxf(top[0], top[1]));
    }
    mx = fmaxf(mx, lane_xor32(mx)) * a.scale_log2;
    // The reference follows the maximum where that has risen by more than kSlack: until
    // then probabilities are up to 2^kSlack, as exact as below 1.
    if (__any(mx > m + kSlack)) {
      const float m_new = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) ot[dt] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;   // (a column without a key so far)
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = __builtin_amdgcn_exp2f(fmaf(st[kt][i], a.scale_log2, -ref));
      float s2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s2[i] = st[kt][8 * i];
#pragma unroll
        for (int j = 1; j < 8; ++j) s2[i] += st[kt][8 * i + j];
      }
      ps += s2[0] + s2[1];
    }
    l += ps;
#pragma unroll
    for (int kp = 0; kp < 2 * KT; ++kp) {   // 16 keys from 16 kp on
      const f16v &sv = st[kp >> 1];
      u4 pw, pr;   // rounded, and the rest
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = sv[8 * (kp & 1) + 2 * i], p1 = sv[8 * (kp & 1) + 2 * i + 1];
        pw[i] = pack_bf16x2(p0, p1);
        pr[i] = pack_bf16x2(p0 - __uint_as_float(pw[i] << 16), p1 - __uint_as_float(pw[i] & 0xffff0000u));
      }
      bf8 vf[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u2 lo = lds_read_tr(reinterpret_cast<const uint16_t *>(lds + vo[dt] + 16 * kp * F::kBytes));
        const u2 hi = lds_read_tr(reinterpret_cast<const uint16_t *>(lds + (vo[dt] ^ 16) + (16 * kp + 8) * F::kBytes));
        vf[dt] = bits_to_bf8(u4{lo.x, lo.y, hi.x, hi.y});
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) ot[dt] = mfma32x32(vf[dt], bits_to_bf8(pw), ot[dt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) ot[dt] = mfma32x32(vf[dt], bits_to_bf8(pr), ot[dt]);
    }
  }
  __device__ __forceinline__ void finish(bool poison) {
    l += lane_xor32(l);
    if (poison) l = NAN;
  }
  // ot[dt][i] = O[this column][rank 32 dt + 8 (i / 4) + 4 half + i % 4] before the 1 / l
  __device__ __forceinline__ f4 quad(int j) const {
    const f16v &v = ot[j >> 2];
    const int i = 4 * (j & 3);
    return f4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  }
};

// The same for the 16 columns of the narrow form, 16x16x32 MFMAs over 32 keys: one token of 16 heads would leave
// half of 32 columns empty (4,000 keys by one work-group 47 us in place of 52, as copies were then; now 31).
template <int R>
struct Bf16Narrow {
  using F = Form<R, false, true>;
  static constexpr int KS = R / 32, DT = R / 16;
  static_assert(F::kKeys == 32, "two products of 16 keys");
  const PagedArgs &a;
  bf8 qf[KS];
  f4 ot[DT];
  float m, l;          // l over this lane's keys alone
  int lane, grp, l16;
  int ko[KS], vo[DT];
  __device__ __forceinline__ explicit Bf16Narrow(const PagedArgs &args) : a(args), m(-INFINITY), l(0.f) {
    lane = threadIdx.x & 63;
    grp = lane >> 4;
    l16 = lane & 15;
    // K row l16 (16 rows on: a constant), chunk 4 ks + grp; V rows 4 grp + l16 / 4 (16 rows on: a constant).
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ko[ks] = place<R, false>(l16, 4 * ks + grp);
#pragma unroll
    for (int b = 0; b < DT; ++b) vo[b] = place<R, false>(4 * grp + (l16 >> 2), 2 * b + ((l16 & 3) >> 1)) + 8 * (l16 & 1);
#pragma unroll
    for (int b = 0; b < DT; ++b) ot[b] = f4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ int column() const { return l16; }
  __device__ __forceinline__ void queries(int64_t row, int head) {
    const uint16_t *qp = static_cast<const uint16_t *>(a.qa) + row * a.qa_stride + static_cast<int64_t>(head) * R + 8 * grp;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = bits_to_bf8(*reinterpret_cast<const u4 *>(qp + 32 * ks));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  }
  __device__ __forceinline__ void tile(const char *lds, bool all, uint64_t seen) {
    f4 st[2];   // score(key 16 kt + 4 grp + i, this column)
    st[0] = st[1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        st[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            bits_to_bf8(*reinterpret_cast<const u4 *>(lds + ko[ks] + 16 * kt * F::kBytes)), qf[ks], st[kt], 0, 0, 0);
    if (!all) {
      const uint32_t bits = static_cast<uint32_t>(seen) >> (4 * grp);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[kt][i] = bits & (1u << (16 * kt + i)) ? st[kt][i] : -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                     fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
    mx = fmaxf(mx, lane_xor16(mx));
    mx = fmaxf(mx, lane_xor32(mx)) * a.scale_log2;
    if (__any(mx > m + kSlack)) {   // (as in the wide form)
      const float m_new = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < DT; ++b) ot[b] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    u4 pw, pr;   // the probabilities rounded, and the rest
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(st[kt][2 * i], a.scale_log2, -ref));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(st[kt][2 * i + 1], a.scale_log2, -ref));
        ps += p0 + p1;
        const uint32_t w = pack_bf16x2(p0, p1);
        pw[2 * kt + i] = w;
        pr[2 * kt + i] = pack_bf16x2(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
      }
    l += ps;
    // (the k index of lane group grp runs over keys 4 grp .. + 3 and 16 + 4 grp .. + 3, as the scores lie)
    bf8 vf[DT];
#pragma unroll
    for (int b = 0; b < DT; ++b) {
      const u2 lo = lds_read_tr(reinterpret_cast<const uint16_t *>(lds + vo[b]));
      const u2 hi = lds_read_tr(reinterpret_cast<const uint16_t *>(lds + vo[b] + 16 * F::kBytes));
      vf[b] = bits_to_bf8(u4{lo.x, lo.y, hi.x, hi.y});
    }
#pragma unroll
    for (int b = 0; b < DT; ++b) ot[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[b], bits_to_bf8(pw), ot[b], 0, 0, 0);
#pragma unroll
    for (int b = 0; b < DT; ++b) ot[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[b], bits_to_bf8(pr), ot[b], 0, 0, 0);
  }
  __device__ __forceinline__ void finish(bool poison) {
    l += lane_xor16(l);
    l += lane_xor32(l);
    if (poison) l = NAN;
  }
  // ot[b][i] = O[this column][rank 16 b + 4 grp + i] before the 1 / l
  __device__ __forceinline__ f4 quad(int j) const { return ot[j]; }
};

// The same in fp32, 16x16x4 MFMAs: a lane's four consecutive ranks of a key are the A
// operands of four steps (the k index runs 4 (lane / 16) + step), and the scores'
// accumulator, keys 4 (lane / 16) + i, is the B operand of the value product in the same order.
template <int R, bool NARROW>
struct F32Columns {
  using F = Form<R, true, NARROW>;
  static constexpr int KB = R / 16, KT = F::kKeys / 16;
  const PagedArgs &a;
  f4 qf[KB], ot[KB];
  float m, l;
  int lane, grp, l16;
  __device__ __forceinline__ explicit F32Columns(const PagedArgs &args) : a(args), m(-INFINITY), l(0.f) {
    lane = threadIdx.x & 63;
    grp = lane >> 4;
    l16 = lane & 15;
#pragma unroll
    for (int b = 0; b < KB; ++b) ot[b] = f4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ int column() const { return l16; }
  __device__ __forceinline__ void queries(int64_t row, int head) {
    const float *qp = static_cast<const float *>(a.qa) + row * a.qa_stride + static_cast<int64_t>(head) * R + 4 * grp;
#pragma unroll
    for (int b = 0; b < KB; ++b) qf[b] = *reinterpret_cast<const f4 *>(qp + 16 * b);
#pragma unroll
    for (int b = 0; b < KB; ++b) asm volatile("" : "+v"(qf[b]));
  }
  __device__ __forceinline__ void tile(const char *lds, bool, uint64_t seen) {
    f4 st[KT];   // score(key 16 kt + 4 grp + i, this column)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) st[kt] = f4{0.f, 0.f, 0.f, 0.f};
    // LDS reads a step ahead of their products, here and below: by hand, as scheduling groups
    // over that many products take the compiler a minute.
    f4 k[2][KT];
    const auto read_k = [&](int b) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        k[b & 1][kt] = *reinterpret_cast<const f4 *>(lds + place<R, true>(l16, 4 * b + grp) + 16 * kt * F::kBytes);
      __builtin_amdgcn_sched_barrier(0);
    };
    read_k(0);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      if (b + 1 < KB) read_k(b + 1);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) st[kt] = mfma_f32(k[b & 1][kt][s], qf[b][s], st[kt]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st[kt][i] = (seen >> (16 * kt + 4 * grp + i)) & 1 ? st[kt][i] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, st[kt][i]);
      }
    mx = fmaxf(mx, lane_xor16(mx));
    mx = fmaxf(mx, lane_xor32(mx));
    const float m_new = fmaxf(m, mx);
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    const float ref = m == -INFINITY ? 0.f : m;
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st[kt][i] = __builtin_amdgcn_exp2f(st[kt][i] - ref);
        ps += st[kt][i];
      }
    l = l * alpha + ps;
#pragma unroll
    for (int b = 0; b < KB; ++b) ot[b] *= alpha;
    float v[2][KB];
    const auto read_v = [&](int i) {   // of key 16 (i / 4) + 4 grp + i % 4
#pragma unroll
      for (int b = 0; b < KB; ++b)
        v[i & 1][b] = *reinterpret_cast<const float *>(lds + place<R, true>(4 * grp + (i & 3), 4 * b + (l16 >> 2)) +
                                                       16 * (i >> 2) * F::kBytes + 4 * (l16 & 3));
      __builtin_amdgcn_sched_barrier(0);
    };
    read_v(0);
#pragma unroll
    for (int i = 0; i < 4 * KT; ++i) {
      if (i + 1 < 4 * KT) read_v(i + 1);
#pragma unroll
      for (int b = 0; b < KB; ++b) ot[b] = mfma_f32(v[i & 1][b], st[i >> 2][i & 3], ot[b]);
    }
  }
  __device__ __forceinline__ void finish(bool poison) {
    l += lane_xor16(l);
    l += lane_xor32(l);
    if (poison) l = NAN;
  }
  // ot[b][i] = O[this column][rank 16 b + 4 grp + i] before the 1 / l
  __device__ __forceinline__ f4 quad(int j) const { return ot[j]; }
};

template <int R, bool F32, bool NARROW>
struct ColumnsOf {
  using type = Bf16Columns<R>;
};
template <int R>
struct ColumnsOf<R, false, true> {
  using type = Bf16Narrow<R>;
};
template <int R, bool NARROW>
struct ColumnsOf<R, true, NARROW> {
  using type = F32Columns<R, NARROW>;
};

// Keys of the tile from k0 on that a column at position pos sees, of those there are.
__device__ __forceinline__ uint64_t seen_keys(uint64_t there, int pos, int k0) {
  const int n = pos + 1 - k0;
  return n >= 64 ? there : n <= 0 ? 0 : there & ((1ull << n) - 1);
}

// The tiles of the kernel: two of each kind, in objects of their own, so that the compiler knows that reads of the
// one do not wait for copies into the other.
template <int R, bool F32>
constexpr int kTileBytes = 4 * Form<R, F32, true>::kTile > Form<R, F32, false>::kTile ? 4 * Form<R, F32, true>::kTile
                                                                                       : Form<R, F32, false>::kTile;

template <int R, bool F32>
__device__ __forceinline__ void wide(const PagedArgs &a, const Work &w, char *tile0, char *tile1, uint64_t *s_bad) {
  using F = Form<R, F32, false>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Stage<R, F32, false> stage(a, w);
  typename ColumnsOf<R, F32, false>::type c(a);
  const int col = w.col0 + F::kCols * wave + c.column(), in = min(col, w.cols - 1);
  const int token = in / a.heads, pos = w.q.pos0 + token;
  const int wave_col = w.col0 + F::kCols * wave;
  const bool idle = wave_col >= w.cols;   // (of the whole wavefront)
  const int wave_last = w.q.pos0 + (min(wave_col + F::kCols, w.cols) - 1) / a.heads, wave_first = w.q.pos0 + wave_col / a.heads;
  uint64_t there = 0;
  int id = 0;
  if (w.k0 < w.k1) {
    id = stage.id_of(w.k0, stage.load_id(w.k0));
    there = __ballot(id >= 0);
    stage.copy(tile0, w.k0, id);
    id = stage.load_id(w.k0 + F::kKeys);
  }
  c.queries(w.q.base + token, in - token * a.heads);
  uint64_t poison = 0;
  const auto step = [&](int k0, char *tile, char *next) {
    // This wavefront's copies, then the others'.  The next tile's go out only after that, into
    // the buffer that all have left.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : "+v"(id)::"memory");
    __syncthreads();
    const uint64_t now = there;
    if (k0 + F::kKeys < w.k1) {
      id = stage.id_of(k0 + F::kKeys, id);
      there = __ballot(id >= 0);
      stage.copy(next, k0 + F::kKeys, id);
    }
    id = stage.load_id(k0 + 2 * F::kKeys);   // (of the last key's page past the end: no branch, which would wait for it)
    // A key that not every column sees would reach all of them through the products (0 times
    // infinity): it enters them as zeros where it is not finite, and the columns that do see it
    // end as NaN.
    uint64_t bad = 0;
    if (k0 + F::kKeys - 1 > w.q.pos0 + w.first && w.first != w.last) {
      const uint64_t mine = stage.clean(tile);
      if (lane == 0) s_bad[wave] = mine;
      lds_barrier();
      bad = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    }
    if (!idle && wave_last >= k0) {
      const uint64_t seen = seen_keys(now, pos, k0);
      poison |= bad & seen;
      c.tile(tile, now == ~0ull && wave_first >= k0 + F::kKeys - 1, seen);
    }
  };
  for (int k0 = w.k0; k0 < w.k1; k0 += 2 * F::kKeys) {
    step(k0, tile0, tile1);
    if (k0 + F::kKeys < w.k1) step(k0 + F::kKeys, tile1, tile0);
  }
  if (idle) return;
  c.finish(poison != 0);
  put<R, F32>(a, w, a.wide_part + (4 * w.part + wave) * F::kPart, col, c.m, c.l, [&](int j) { return c.quad(j); });
}

template <int R, bool F32>
__device__ __forceinline__ void narrow(const PagedArgs &a, const Work &w, char *tiles0, char *tiles1, f2 (*s_ml)[64]) {
  using F = Form<R, F32, true>;
  constexpr int kQuads = F::kQuads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Stage<R, F32, true> stage(a, w);
  typename ColumnsOf<R, F32, true>::type c(a);
  const int col = c.column(), in = min(col, w.cols - 1);
  const int token = in / a.heads, pos = w.q.pos0 + token;
  constexpr uint64_t kAll = ~0ull >> (64 - F::kKeys);
  constexpr int kStep = 4 * F::kKeys;
  char *const tile0 = tiles0 + wave * F::kTile, *const tile1 = tiles1 + wave * F::kTile;   // this wavefront's
  const int first = w.k0 + F::kKeys * wave;
  uint64_t there = 0;
  int id = 0;
  if (first < w.k1) {
    id = stage.id_of(first, stage.load_id(first));
    there = __ballot(id >= 0) & kAll;
    stage.copy(tile0, first, id);
    id = stage.load_id(first + kStep);
  }
  c.queries(w.q.base + token, in - token * a.heads);
  uint64_t poison = 0;
  const auto step = [&](int k0, char *tile, char *next) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : "+v"(id)::"memory");   // (its own copies; nobody else reads them)
    const uint64_t now = there;
    if (k0 + kStep < w.k1) {
      id = stage.id_of(k0 + kStep, id);
      there = __ballot(id >= 0) & kAll;
      stage.copy(next, k0 + kStep, id);
    }
    id = stage.load_id(k0 + 2 * kStep);
    const uint64_t seen = seen_keys(now, pos, k0);
    if (k0 + F::kKeys - 1 > w.q.pos0 && w.last != 0) {   // (as in the wide form)
      poison |= stage.clean(tile) & seen;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
    }
    c.tile(tile, now == kAll && w.q.pos0 >= k0 + F::kKeys - 1, seen);
  };
  for (int k0 = first; k0 < w.k1; k0 += 2 * kStep) {
    step(k0, tile0, tile1);
    if (k0 + kStep < w.k1) step(k0 + kStep, tile1, tile0);
  }
  c.finish(poison != 0);
  // The wavefronts' columns joined: each scaled to the common maximum, then summed four ranks a thread.
  s_ml[wave][lane] = f2{c.m, c.l};
  __syncthreads();
  float m = s_ml[0][lane].x;
#pragma unroll
  for (int i = 1; i < 4; ++i) m = fmaxf(m, s_ml[i][lane].x);
  const auto weight = [&](int i) {
    const float mi = s_ml[i][lane].x;
    return mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - m);
  };
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) l = fmaf(s_ml[i][lane].y, weight(i), l);
  // Quad j of wavefront i: the even ones where tile 0 was, the odd ones where tile 1 was.
  static_assert(4 * (kQuads / 2) * 64 * sizeof(f4) <= 4 * F::kTile, "the sums fit the tiles");
  const auto sums = [&](int i, int j) {
    return reinterpret_cast<f4 *>(j & 1 ? tiles1 : tiles0) + (i * (kQuads / 2) + (j >> 1)) * 64 + lane;
  };
  const float own = weight(wave);
#pragma unroll
  for (int j = 0; j < kQuads; ++j) *sums(wave, j) = c.quad(j) * own;
  __syncthreads();
  constexpr int kMine = (kQuads + 3) / 4;
  f4 v[kMine];
#pragma unroll
  for (int t = 0; t < kMine; ++t) {
    const int j = wave + 4 * t;
    v[t] = f4{0.f, 0.f, 0.f, 0.f};
    if (j < kQuads)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[t] += *sums(i, j);
  }
  if (w.used > 1) {
    float *p = a.narrow_part + w.part * F::kPart;
#pragma unroll
    for (int t = 0; t < kMine; ++t)
      if (wave + 4 * t < kQuads) reinterpret_cast<f4 *>(p)[64 * (wave + 4 * t) + lane] = v[t];
    if (wave == 0) reinterpret_cast<f2 *>(p + 256 * kQuads)[lane] = f2{m, l};
  } else if (col < w.cols) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int t = 0; t < kMine; ++t)
      if (wave + 4 * t < kQuads)
        store4(a.out, (w.q.base + token) * a.out_stride + static_cast<int64_t>(in - token * a.heads) * R + F::rank(wave + 4 * t),
               F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, v[t] * inv);
  }
}

// The narrow work-groups first, as one of them may have a long chain of tiles.  Of the wide ones there are as many as the
// host's bound on the items, so each has one at most; it would take more in turn if offsets that descend made more
// of them.  WIDE, NARROW: which there are.
template <int R, bool F32, bool WIDE, bool NARROW>
__global__ __launch_bounds__(256, R <= 128 ? 2 : 1) void mla_paged_kernel(PagedArgs a) {
  constexpr int kBytes = NARROW ? kTileBytes<R, F32> : Form<R, F32, false>::kTile;
  __shared__ __attribute__((aligned(1024))) char s_tile0[kBytes], s_tile1[kBytes];
  Work w;
  if (NARROW && static_cast<int>(blockIdx.x) < a.narrow_blocks) {
    __shared__ f2 s_ml[4][64];
    // (an odd number of work-groups per sequence: with 8 or 16 the first ranges, which all sequences have, would be on
    // one XCD: 96 sequences 26 us in place of 18)
    const int each = a.narrow_splits | 1;
    if (find_narrow<R, F32>(a, w, blockIdx.x / each, blockIdx.x % each))
      narrow<R, F32>(a, w, s_tile0, s_tile1, s_ml);
  } else if constexpr (WIDE) {
    __shared__ uint64_t s_bad[4];
    __shared__ Shares s_shares;
    const int grid = gridDim.x - a.narrow_blocks;
    int block = blockIdx.x - a.narrow_blocks, parts = 0;
    for (int s0 = 0; s0 < a.p.n_seqs; s0 += 64) {
      if (threadIdx.x < 64) {
        Lanes<R, F32> l(a);
        const int length = s0 == 0 ? l.range_tiles(threadIdx.x) : s_shares.length;
        if (s0 > 0) l.look(s0 + threadIdx.x);
        share(l, s_shares, s0, length);
        if (threadIdx.x == 0) s_shares.length = length;
      }
      __syncthreads();
      const int all = s_shares.items[63];
      for (; block < all; block += grid) {
        const int i = __builtin_amdgcn_readfirstlane(place_of(s_shares.items, block));
        const int item = block - (i ? s_shares.items[i - 1] : 0), groups = s_shares.groups[i];
        const int split = __builtin_amdgcn_readfirstlane(item / groups), g = __builtin_amdgcn_readfirstlane(item - split * groups);
        if (take<R, F32>(a, s_shares, w, i, g, split, parts)) wide<R, F32>(a, w, s_tile0, s_tile1, s_bad);
        __syncthreads();   // (the tiles are free)
      }
      block -= all;
      parts += s_shares.parts[63];
      __syncthreads();
    }
  }
}

// Joins the ranges of a wavefront's columns, the partials one after the other, several loaded before the first is
// used.  Work-groups of narrow sequences first (if they have partials): a wavefront four ranks of each column;
// then those of wide groups: a wavefront EACH times four ranks of its own columns.
template <int R, bool F32, bool NARROW, int QUADS>
__device__ __forceinline__ void join(const PagedArgs &a, const Work &w, const float *p, int64_t step, int col, int j0) {
  using F = Form<R, F32, NARROW>;
  constexpr int kQuads = F::kQuads, kAhead = 8 / QUADS;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f;
  f4 acc[QUADS];
#pragma unroll
  for (int q = 0; q < QUADS; ++q) acc[q] = f4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < w.used; s0 += kAhead) {
    f2 ml[kAhead];
    f4 v[kAhead][QUADS];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const float *ps = p + min(s0 + s, w.used - 1) * step;   // the last one again, unused
      ml[s] = reinterpret_cast<const f2 *>(ps + 256 * kQuads)[lane];
#pragma unroll
      for (int q = 0; q < QUADS; ++q) v[s][q] = reinterpret_cast<const f4 *>(ps)[64 * (j0 + q) + lane];
    }
    float top = m;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) top = fmaxf(top, ml[s].x);
    const float ref = top == -INFINITY ? 0.f : top;
    const float e0 = __builtin_amdgcn_exp2f(m - ref);
    l *= e0;
#pragma unroll
    for (int q = 0; q < QUADS; ++q) acc[q] *= e0;
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
      if (s0 + s < w.used) {
        const float e = __builtin_amdgcn_exp2f(ml[s].x - ref);
        l = fmaf(ml[s].y, e, l);
#pragma unroll
        for (int q = 0; q < QUADS; ++q) acc[q] += v[s][q] * e;
      }
    m = top;
  }
  if (col >= w.cols) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int token = col / a.heads, head = col - token * a.heads;
#pragma unroll
  for (int q = 0; q < QUADS; ++q)
    store4(a.out, (w.q.base + token) * a.out_stride + static_cast<int64_t>(head) * R + F::rank(j0 + q),
           F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, acc[q] * inv);
}

template <int R, bool F32, int EACH>
__global__ __launch_bounds__(256) void mla_paged_merge_kernel(PagedArgs a, int narrow_units) {
  using F = Form<R, F32, false>;
  constexpr int kEach = F::kQuads < EACH ? F::kQuads : EACH;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Work w;
  if (static_cast<int>(blockIdx.x) < narrow_units) {
    using N = Form<R, F32, true>;
    const int j = 4 * blockIdx.y + wave;
    if (j >= N::kQuads || !find_narrow<R, F32>(a, w, blockIdx.x, 0) || w.used == 1) return;
    join<R, F32, true, 1>(a, w, a.narrow_part + w.part * N::kPart, N::kPart, lane & (N::kCols - 1), j);
  } else {
    // (many groups: all quads in one work-group)
    const int j0 = EACH > 1 ? 0 : blockIdx.y, j1 = EACH > 1 ? F::kQuads : j0 + 1;
    if (EACH > 1 ? blockIdx.y > 0 : j0 >= F::kQuads) return;
    __shared__ Shares s_all[4];
    Shares &t = s_all[wave];     // (each wavefront its own: no barrier)
    Lanes<R, F32> l(a);
    const int length = l.range_tiles(lane);
    int group = blockIdx.x - narrow_units, parts = 0;
    for (int s0 = 0; s0 < a.p.n_seqs; s0 += 64) {
      if (s0 > 0) l.look(s0 + lane);
      share(l, t, s0, length);
      const int sum = wave_scan(t.groups[lane]), all = __builtin_amdgcn_readlane(sum, 63);
      if (group < all) {
        const int i = __ffsll(static_cast<unsigned long long>(__ballot(group < sum))) - 1;
        const int g = group - (__builtin_amdgcn_readlane(sum, i) - t.groups[i]);
        if (!take<R, F32>(a, t, w, i, g, 0, parts) || w.used == 1 || w.col0 + F::kCols * wave >= w.cols) return;
        const float *p = a.wide_part + (4 * w.part + wave) * F::kPart;
        for (int j = j0; j < j1; j += kEach)
          join<R, F32, false, kEach>(a, w, p, 4ll * w.step * F::kPart, (lane & (F::kCols - 1)) + w.col0 + F::kCols * wave, j);
        return;
      }
      group -= all;
      parts += t.parts[63];
    }
  }
}

// ---- norms ---------------------------------------------------------------------
// The normalisations that follow MLA's down projections, in place, and the latents into
// their pages: a wavefront has two rows, whose places its halves look up while the rows are under way;
// lanes [0, q_rank / 8) hold 8 elements of q each, the next kv_rank / 8 lanes 8 of the latent.  16,624 rows of
// 384 + 128 in bf16: 38 MB read and written in 10.4 us (3.7 TB/s; a copy has 5.1); 96 rows 4.2, a launch and two waits.
struct PagedNormArgs {
  Pages p;
  void *q;
  int64_t q_stride;
  void *kv;
  int64_t kv_stride;
  int q_rank, kv_rank;
  const float *q_w, *kv_w;
  float q_eps, kv_eps;
};

// Of n ascending offsets, how many are <= row, which may differ between the halves of a wavefront: by 32nds,
// a step per factor of 32.
__device__ __forceinline__ int count_not_above(const int32_t *cu, int n, int64_t row) {
  const int lane = threadIdx.x & 63, in = lane & 31, half = lane >> 5;
  int lo = 0, hi = n;   // the count lies within [lo, hi]
  while (__any(hi > lo)) {
    const int step = max(1, (hi - lo + 31) >> 5);
    const int at = lo + (in + 1) * step - 1;
    const uint64_t both = __ballot(at < hi && cu[min(at, n - 1)] <= row);
    const uint32_t not_above = static_cast<uint32_t>(both >> (32 * half));
    const int first = not_above == ~0u ? 32 : __ffs(~not_above) - 1;   // lanes from 0 on
    const int from = lo + first * step;
    hi = min(hi, from + step - 1);
    lo = min(from, hi);
  }
  return lo;
}

template <int DT>
__device__ __forceinline__ void load8(const void *base, float (&v)[8]) {
  if constexpr (DT == SOPHIA_DTYPE_BF16) {
    const u4 w = *static_cast<const u4 *>(base);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
    const f4 a = static_cast<const f4 *>(base)[0], b = static_cast<const f4 *>(base)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  }
}
template <int DT>
__device__ __forceinline__ void store8(void *base, const float (&v)[8]) {
  if constexpr (DT == SOPHIA_DTYPE_BF16) {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *static_cast<u4 *>(base) = w;
  } else {
    static_cast<f4 *>(base)[0] = f4{v[0], v[1], v[2], v[3]};
    static_cast<f4 *>(base)[1] = f4{v[4], v[5], v[6], v[7]};
  }
}

template <int DT>
__global__ __launch_bounds__(256) void mla_paged_norm_kernel(PagedNormArgs a) {
  constexpr int kEsz = DT == SOPHIA_DTYPE_BF16 ? 2 : 4;
  const int64_t row0 = 2 * (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6));
  if (row0 >= a.p.rows) return;  // uniform over the wavefront
  const int l = threadIdx.x & 63;
  const int qc = a.q_rank / 8, kc = a.kv_rank / 8;
  const bool isq = l < qc, iskv = l >= qc && l < qc + kc;
  const int c = isq ? l : l - qc;  // 8-element chunk within its part
  const int64_t stride = isq ? a.q_stride : a.kv_stride;
  uint8_t *base = static_cast<uint8_t *>(isq ? a.q : a.kv) + (row0 * stride + 8 * c) * kEsz;
  const bool two = row0 + 1 < a.p.rows;
  float v[2][8] = {};
  if (isq || iskv) {
    load8<DT>(base, v[0]);
    if (two) load8<DT>(base + stride * kEsz, v[1]);
  }
  // Where a half's row goes (the first half of the lanes has the first row): its place in the pages, or -1.
  const int64_t row = row0 + (l >> 5);
  int64_t place = -1;
  const int s = count_not_above(a.p.cu + 1, a.p.n_seqs, row);
  if (s < a.p.n_seqs) {
    const Sequence q = sequence(a.p, s);
    const int64_t pos = q.pos0 + (row - q.base);
    if (row >= q.base && row < q.base + q.n && pos >= 0 && pos < q.keys) {
      const int page = page_of(a.p, q.slot, static_cast<int>(pos));
      if (page >= 0) place = page * a.p.page_stride + (pos & ((1 << a.p.shift) - 1)) * a.kv_rank;
    }
  }
  const float *w = (isq ? a.q_w : a.kv_w) + 8 * c;
  float weight[8] = {};
  if (isq || iskv) {
#pragma unroll
    for (int i = 0; i < 8; ++i) weight[i] = as_dtype(w[i], DT);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r == 1 && !two) return;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[r][i], v[r][i], ss);
    const float sq = wave_sum_dpp(isq ? ss : 0.f), sk = wave_sum_dpp(iskv ? ss : 0.f);
    const float scale = isq ? rsqrtf(sq / static_cast<float>(a.q_rank) + a.q_eps)
                            : rsqrtf(sk / static_cast<float>(a.kv_rank) + a.kv_eps);
    const int64_t to = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(
                                                static_cast<int>(place >> 32), 32 * r)))
                                                << 32 |
                                            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place), 32 * r)));
    if (isq || iskv) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[r][i] = v[r][i] * scale * weight[i];
      store8<DT>(base + r * stride * kEsz, v[r]);
      if (iskv && to >= 0) store8<DT>(static_cast<uint8_t *>(const_cast<void *>(a.p.pages)) + (to + 8 * c) * kEsz, v[r]);
    }
  }
}

// ---- the host's side -------------------------------------------------------------
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// How the work is divided: which of the two forms there are, their groups and key ranges.
struct Plan {
  bool narrow, wide;
  int64_t wide_groups, wide_items, wide_parts;      // at most
  int narrow_splits, narrow_keys, wide_used;
  size_t narrow_bytes, wide_bytes;                  // of their partials
};

Plan plan(int n_seqs, int64_t rows, int max_new, int64_t max_len, int heads, int rank, int dtype, int splits) {
  const bool f32 = dtype == SOPHIA_DTYPE_F32;
  if (max_new > rows) max_new = static_cast<int>(rows);
  const int cols = 16, group = f32 ? 64 : 128;
  const int64_t part = 64ll * (4 * (f32 ? rank / 16 : rank / 8) + 2) * 4, narrow_part = 64ll * (4 * (rank / 16) + 2) * 4;
  const int64_t slots = rank <= 128 ? kSlots<128> : kSlots<256>;
  Plan p = {};
  p.wide = static_cast<int64_t>(max_new) * heads > cols;
  // (as many rows as sequences of max_new tokens have: there is no shorter one)
  p.narrow = !p.wide || (heads <= cols && rows != static_cast<int64_t>(n_seqs) * max_new);
  const int64_t keys = max_len < 1 ? 1 : max_len < 1 << 29 ? max_len : 1 << 29;
  if (p.wide) {
    const int64_t a = rows * heads / group + n_seqs, b = n_seqs * ((static_cast<int64_t>(max_new) * heads + group - 1) / group);
    p.wide_groups = a < b ? a : b;
    if (p.wide_groups < 1) p.wide_groups = 1;
    const int64_t tiles = (keys + kWideKeys - 1) / kWideKeys;
    p.wide_used = static_cast<int>(splits > 0 ? imin64(splits, tiles) : imin64(1024, (tiles + kLeast - 1) / kLeast));
    const int64_t most = p.wide_groups * p.wide_used;
    p.wide_items = splits > 0 ? p.wide_groups * splits : imin64(most, p.wide_groups + 2 * slots);
    p.wide_parts = splits > 0 ? p.wide_groups * splits : imin64(most, 4 * slots);
    p.wide_bytes = (splits > 0 ? splits : p.wide_used) > 1 ? static_cast<size_t>(4 * p.wide_parts) * part : 0;
    if (p.wide_bytes == 0) p.wide_parts = 0;
  }
  if (p.narrow) {
    const int64_t tiles = (keys + 127) / 128;
    // Beside wide groups that fill the chip a chain of tiles has time.  Else ranges to about 768 work-groups, were all
    // sequences as long as the longest, and 16 at most: more cost the merge what they save.  us in 1, 4, 8 and 16
    // ranges: one sequence of 4,000 keys 30.9, 14.2, 10.8, 10.2; 32 of 200 to 4,000 30.1, 14.5, 12.8, 12.3; 96 of them
    // 31.5, 18.4, 15.4, 19.8; 200 of up to 3,400 27.3, 20.4, 22.2, 25.7.  Of six tiles one range, a launch
    // less for the host: 9.4, and 8.4 in six on the device.
    int64_t want = splits > 0 ? splits : (p.wide && p.wide_groups >= slots) || tiles <= 6 ? 1 : imin64(16, (768 + n_seqs - 1) / n_seqs);
    want = iclamp64(want, 1, tiles);
    const int64_t each = (tiles + want - 1) / want;
    p.narrow_splits = static_cast<int>((tiles + each - 1) / each);
    p.narrow_keys = static_cast<int>(128 * each);
    p.narrow_bytes = p.narrow_splits > 1 ? static_cast<size_t>(n_seqs) * p.narrow_splits * narrow_part : 0;
  }
  return p;
}

template <int R, bool F32>
int launch(PagedArgs a, const Plan &p, int splits, char *workspace, hipStream_t st) {
  if (p.narrow) {
    a.narrow_blocks = a.p.n_seqs * (p.narrow_splits | 1);
    a.narrow_splits = p.narrow_splits;
    a.narrow_keys = p.narrow_keys;
    a.narrow_part = reinterpret_cast<float *>(workspace);
  }
  if (p.wide) {
    a.wide_blocks = static_cast<int>(p.wide_items);
    a.wide_used = p.wide_bytes ? p.wide_used : 1;
    a.wide_splits = splits;
    a.part_cap = static_cast<int>(p.wide_parts);
    a.wide_part = reinterpret_cast<float *>(workspace + p.narrow_bytes);
  }
  const dim3 grid(static_cast<unsigned>(a.narrow_blocks + a.wide_blocks));
  if (p.narrow && p.wide) hipLaunchKernelGGL((mla_paged_kernel<R, F32, true, true>), grid, dim3(256), 0, st, a);
  else if (p.wide) hipLaunchKernelGGL((mla_paged_kernel<R, F32, true, false>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mla_paged_kernel<R, F32, false, true>), grid, dim3(256), 0, st, a);
  const int narrow_units = p.narrow_bytes ? a.p.n_seqs : 0;
  const int64_t units = narrow_units + (p.wide_bytes ? p.wide_groups : 0);
  // Few groups: a work-group per quad, whose chain of ranges is short; many: four quads, as finding a group costs as
  // much as joining it (520 groups: 19 us with one, 10 with four; 16 groups in fp32: 7 and 12).
  constexpr int kQuads = Form<R, F32, false>::kQuads;
  const unsigned x = static_cast<unsigned>(units);
  if (p.wide_bytes && p.wide_groups < 256)
    hipLaunchKernelGGL((mla_paged_merge_kernel<R, F32, 1>), dim3(x, kQuads), dim3(256), 0, st, a, narrow_units);
  else if (units > 0)
    hipLaunchKernelGGL((mla_paged_merge_kernel<R, F32, 4>), dim3(x, (kQuads + 3) / 4), dim3(256), 0, st, a, narrow_units);
  return check_launch("mla_paged_attn");
}

// What both entry points ask of the pages.
int check_pages(const char *what, const void *pages, int64_t page_stride, int64_t n_pages, int page_size,
                const int32_t *table, int64_t table_stride, int table_rows, int max_pages, const int32_t *cu,
                const int64_t *kv_len, int n_seqs, int64_t rows, int rank) {
  SOPHIA_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && rows >= 0 && rows <= 0x1fffffff,
                 "%s: n_seqs must be 0..65535 and rows 0..2^29 - 1", what);
  SOPHIA_REQUIRE(page_size >= 1 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
                 "%s: page_size must be a power of two, at most 65536", what);
  SOPHIA_REQUIRE(n_pages >= 0 && n_pages <= 0x7fffffff && page_stride >= static_cast<int64_t>(page_size) * rank &&
                     page_stride % 8 == 0,
                 "%s: n_pages must be 0..2^31 - 1, page_stride hold a page and be a multiple of 8", what);
  SOPHIA_REQUIRE(table_rows >= 0 && max_pages >= 0 && table_stride >= max_pages &&
                     static_cast<int64_t>(max_pages) * page_size <= 1 << 29,
                 "%s: the table's rows must hold max_pages entries, of at most 2^29 tokens", what);
  if (n_seqs == 0 || rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(cu && kv_len && (table || max_pages == 0 || table_rows == 0) && (pages || n_pages == 0), "%s: NULL pointer", what);
  SOPHIA_REQUIRE(aligned16(pages), "%s: pages must be 16-byte aligned", what);
  return SOPHIA_OK;
}

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" size_t sophia_mla_paged_workspace_size(int n_seqs, int64_t rows, int max_new, int64_t max_len, int heads, int rank,
                                                  int dtype, int splits) {
  if (n_seqs < 1 || rows < 1 || max_new < 1 || heads < 1 || rank < 1 || splits < 0) return 0;
  const Plan p = plan(n_seqs, rows, max_new, max_len, heads, rank, dtype, splits);
  return p.narrow_bytes + p.wide_bytes;
}

extern "C" int sophia_mla_paged_attn(const void *qa, int64_t qa_stride, int dtype, const void *pages, int64_t page_stride,
                                     int64_t n_pages, int page_size, const int32_t *table, int64_t table_stride,
                                     int table_rows, int max_pages, const int32_t *slots, const int32_t *cu_seqlens,
                                     const int64_t *kv_len, int n_seqs, int64_t rows, int max_new, int64_t max_len,
                                     float scale, void *out, int64_t out_stride, int heads, int rank, int splits,
                                     void *workspace, size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "mla_paged_attn: dtype not supported");
  SOPHIA_REQUIRE(rank == 32 || rank == 64 || rank == 128 || rank == 256,
                 "mla_paged_attn: rank %d not supported (32, 64, 128 or 256)", rank);
  SOPHIA_REQUIRE(heads >= 1 && heads <= 128, "mla_paged_attn: heads must be in [1, 128]");
  SOPHIA_REQUIRE(scale > 0.f && scale < 1e38f, "mla_paged_attn: scale must be > 0 and finite");
  SOPHIA_REQUIRE(max_new >= 1 && splits >= 0 && splits <= 1024, "mla_paged_attn: max_new must be >= 1 and splits 0..1024");
  if (int rc = check_pages("mla_paged_attn", pages, page_stride, n_pages, page_size, table, table_stride, table_rows, max_pages,
                           cu_seqlens, kv_len, n_seqs, rows, rank))
    return rc;
  SOPHIA_REQUIRE(qa_stride >= static_cast<int64_t>(heads) * rank && out_stride >= static_cast<int64_t>(heads) * rank &&
                     qa_stride % 8 == 0 && out_stride % 8 == 0,
                 "mla_paged_attn: row strides must hold a row and be multiples of 8");
  SOPHIA_REQUIRE(rows * heads <= 1 << 30, "mla_paged_attn: rows * heads must be at most 2^30");
  if (n_seqs == 0 || rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(qa && out, "mla_paged_attn: NULL pointer");
  SOPHIA_REQUIRE(aligned16(qa) && aligned16(out), "mla_paged_attn: qa and out must be 16-byte aligned");
  const Plan p = plan(n_seqs, rows, max_new, max_len, heads, rank, dtype, splits);
  SOPHIA_REQUIRE(p.narrow_bytes + p.wide_bytes == 0 ||
                     (workspace && aligned16(workspace) && workspace_bytes >= p.narrow_bytes + p.wide_bytes),
                 "mla_paged_attn: workspace too small");
  SOPHIA_REQUIRE(p.wide_items <= 1 << 28 && 4 * p.wide_groups <= 1 << 28, "mla_paged_attn: too much work for one call");
  const PagedArgs a{{pages, page_stride, n_pages, log2_of(page_size), table, table_stride, table_rows, max_pages, slots,
                     cu_seqlens, kv_len, n_seqs, rows},
                    qa, qa_stride, out, out_stride, scale * 1.44269504088896341f, heads, max_new, 0, 1, 1, nullptr, 0, 1, 0, 0, nullptr};
  char *ws = static_cast<char *>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (rank) {
#define SOPHIA_MLA_PAGED(r) \
  case r:                   \
    return dtype == SOPHIA_DTYPE_F32 ? launch<r, true>(a, p, splits, ws, st) : launch<r, false>(a, p, splits, ws, st);
    SOPHIA_MLA_PAGED(32) SOPHIA_MLA_PAGED(64) SOPHIA_MLA_PAGED(128) SOPHIA_MLA_PAGED(256)
#undef SOPHIA_MLA_PAGED
  }
  return SOPHIA_OK;
}

extern "C" int sophia_mla_latent_norms_paged(void *q_lat, int64_t q_stride, void *kv_lat, int64_t kv_stride, int64_t rows,
                                             int q_rank, int kv_rank, int dtype, const float *q_norm_weight, float q_eps,
                                             const float *kv_norm_weight, float kv_eps, void *pages, int64_t page_stride,
                                             int64_t n_pages, int page_size, const int32_t *table, int64_t table_stride,
                                             int table_rows, int max_pages, const int32_t *slots, const int32_t *cu_seqlens,
                                             const int64_t *kv_len, int n_seqs, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "mla_latent_norms_paged: dtype not supported");
  SOPHIA_REQUIRE(q_rank > 0 && kv_rank > 0 && q_rank % 8 == 0 && kv_rank % 8 == 0 && q_rank + kv_rank <= 512,
                 "mla_latent_norms_paged: ranks must be positive multiples of 8 with q_rank + kv_rank <= 512");
  SOPHIA_REQUIRE(q_stride % 8 == 0 && kv_stride % 8 == 0 && q_stride >= q_rank && kv_stride >= kv_rank,
                 "mla_latent_norms_paged: strides must be multiples of 8 elements and cover a row");
  if (int rc = check_pages("mla_latent_norms_paged", pages, page_stride, n_pages, page_size, table, table_stride, table_rows,
                           max_pages, cu_seqlens, kv_len, n_seqs, rows, kv_rank))
    return rc;
  if (rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(q_lat && kv_lat && q_norm_weight && kv_norm_weight, "mla_latent_norms_paged: NULL pointer");
  SOPHIA_REQUIRE(aligned16(q_lat) && aligned16(kv_lat) && aligned16(q_norm_weight) && aligned16(kv_norm_weight),
                 "mla_latent_norms_paged: pointers must be 16-byte aligned");
  const PagedNormArgs a{{pages, page_stride, n_pages, log2_of(page_size), table, table_stride, table_rows, max_pages, slots,
                         cu_seqlens, kv_len, n_seqs, rows},
                        q_lat, q_stride, kv_lat, kv_stride, q_rank, kv_rank, q_norm_weight, kv_norm_weight, q_eps, kv_eps};
  const dim3 grid(static_cast<unsigned>((rows + 7) / 8));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SOPHIA_DTYPE_BF16)
    hipLaunchKernelGGL(mla_paged_norm_kernel<SOPHIA_DTYPE_BF16>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(mla_paged_norm_kernel<SOPHIA_DTYPE_F32>, grid, dim3(256), 0, st, a);
  return check_launch("mla_latent_norms_paged");
}
