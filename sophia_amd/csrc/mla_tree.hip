// MLA attention in latent space for a tree of drafted tokens: every node attends
// to the cached latents of its sequence and to the drafted latents of itself and
// its ancestors (include/sophia_draft.h), in one pass with a running maximum and
// sum.  Keys and values are the same rows, so a tile of 64 of them is staged in
// LDS once and read twice, as K rows and, transposed, as V.
//
// A work-group (4 wavefronts) takes some nodes of one tree and a range of its keys:
// the 16 heads of a node are 16 columns of the matrix products, so a wavefront
// holds 2 nodes in bf16, 1 in fp32.  Contexts and trees of a batch differ by far, and
// the host does not know them: every work-group finds its share in the list of all
// (tree, range, nodes), which it counts itself, a tree per lane.  A tree's ranges are
// equally long, and all have about the same length, which follows from the whole work.  Neighbours in the list, which
// read the same keys, run on one XCD, whose L2 serves all but the first of them.  A
// tree of one range writes its result at once, the others partials that a second
// kernel joins, both in the order in which the lanes hold them.
//
// The drafted latents are one more tile of the last range, taken first, the only one
// with a mask per column.  A drafted latent that is not finite would reach every
// node through the products (0 times infinity): it enters them as zeros, and the
// nodes that do see it end as NaN.
//
// What bounds it: 32 trees of 24 to 64 nodes after 60 to 4,000 keys (11.7 GFLOP, 11 us at
// the rate of a large product) take 32 us and 10 for the merge.  A tile of 8 nodes is 48
// MFMAs per wavefront, 1,536 cycles (a third of them for what the probabilities lose when
// rounded once); 128 KB of LDS reads for its four wavefronts, 1,024 cycles of the CU; and
// about 300 vector instructions, mostly the softmax, with 32 exponentials.  Two wavefronts
// per SIMD (226 registers) share these; over the whole kernel the matrix pipes are busy 35 %
// of the time, the vector unit 42 and LDS 21, as a work-group spends 8,000 cycles before its
// first tile and after its last, and some have a tile more than others.  One tree of 7 nodes
// after 523 keys takes 10 us and 4, all of it latency.  The same 32 trees at other ranks, with
// the merge: 32 27 us, 64 32, 128 42, 256 150 (76 bytes of a lane's state in scratch).
// On the way, for the 32 trees: ranges by number instead of length 79; three copies of the
// tile's code for masked and whole tiles, whose spilled registers were waited for together
// with the next tile 50 + 8; one copy 42 + 8; shares from a list of what there is, instead of
// a grid over the bounds, which left CUs without work beside others with two shares, and
// partials stored as the lanes hold them 29 + 9; rows read ahead of their products and a
// reference that seldom moves 27 + 10; probabilities in two parts 32 + 10.  Not kept, as no
// faster: two tiles in LDS and one barrier a tile, lines of the tiles ahead loaded early.
#include <type_traits>

#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_draft.h"

namespace sophia {
namespace {

template <bool F32>
constexpr int kGroup = F32 ? 4 : 8;   // nodes per work-group
constexpr int kTile = 64;        // keys per tile (a whole tree)
constexpr float kSlack = 8.f;    // (powers of 2)
static_assert(kTile == kTreeNodes, "the drafted latents are one tile");

struct MlaTreeArgs {
  Trees trees;
  const void *qa;
  int64_t qa_stride;
  const void *latent;      // drafted [rows, R], of qa's type
  int64_t latent_stride;
  const float *cache;
  int64_t slot_stride;
  int max_seq, n_slots;
  const int32_t *slots;
  const int64_t *cached;
  float scale_log2;
  void *out;
  int64_t out_stride;
  float *part;             // when splits > 1: `part_cap` partials of kPart<R, F32> floats
  int part_cap;
  int heads, splits, split_tiles, n_trees;
};

// Work-groups that run at a time.
template <int R>
constexpr int kSlots = R <= 128 ? 512 : 256;

typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ bf8 bits_to_bf8(const u4 &v) { return __builtin_bit_cast(bf8, v); }
__device__ __forceinline__ f16v mfma32x32(const bf8 &a, const bf8 &b, const f16v &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Cached keys of a tree: -1 when its slot is out of range (its rows are then zeros).
// No branch: both loads are then under way together.
__device__ __forceinline__ int cached_keys(const MlaTreeArgs &a, int tree, int64_t &slot) {
  const int64_t keys = iclamp64(a.cached[tree], 0, a.max_seq);
  slot = a.slots ? a.slots[tree] : tree;
  return slot >= 0 && slot < a.n_slots ? static_cast<int>(keys) : -1;
}

// What a work-group does.
struct Work {
  int tree, node0, split, n, keys, t0, t1;   // tiles [t0, t1) of the cached keys
  int part;                                  // its partial
  bool drafted, whole;                       // the range has the drafted tile too; is the tree's only one
  int64_t base, slot;
};

// A tree per lane, 64 at a time.
template <int R, bool F32>
struct Lanes {
  const MlaTreeArgs &a;
  int64_t base = 0, slot = 0;
  int n = 0, keys = 0, groups = 0, tiles = 0;   // of this lane's tree; groups 0 behind the last one
  int used = 0, items = 0, parts = 0;           // its ranges, (range, group) items, those of them that are partials
  __device__ __forceinline__ explicit Lanes(const MlaTreeArgs &args) : a(args) {}
  __device__ __forceinline__ void look(int tree) {
    const int in = min(tree, a.n_trees - 1);
    keys = cached_keys(a, in, slot);
    n = tree_nodes(a.trees, in, base);
    groups = tree == in ? (n + kGroup<F32> - 1) / kGroup<F32> : 0;
    tiles = keys < 0 ? 1 : (keys + kTile - 1) / kTile + 1;
  }
  __device__ __forceinline__ void divide(int length) {
    used = min(a.splits, (tiles + length - 1) / length);
    items = used * groups;
    parts = used > 1 ? items : 0;
  }
  // Tiles of a range at most.  With W = sum of groups x tiles and G = sum of groups there
  // are about W / length + G / 2 items, as many as run at a time if that can be: one more
  // takes as long as all of them.  At least split_tiles.  A tree of two ranges or more has
  // fewer than 2 tiles / length of them, so there are at most 2 kSlots partials.  Looks at
  // the first 64 trees last.
  __device__ __forceinline__ int range_tiles(int lane) {
    float work = 0.f;
    int all = 0;
    for (int t0 = (a.n_trees - 1) & ~63; t0 >= 0; t0 -= 64) {
      look(t0 + lane);
      work += static_cast<float>(groups) * static_cast<float>(tiles);
      all += groups;
    }
    all = __builtin_amdgcn_readlane(wave_scan(all), 63);
    work = row_sum16(work);
    work += lane_xor16(work);
    work = (work + lane_xor32(work)) * 1.0001f + 1.f;   // (not less than it is, by rounding)
    const int fill = max(kSlots<R> - all / 2, kSlots<R> / 2);
    work = fminf(ceilf(work / static_cast<float>(fill)), 1 << 29);
    return max(a.split_tiles, static_cast<int>(work));
  }
};

// Work-group b's share: item (b % 8) ceil(items / 8) + b / 8 of the list, in which
// the nodes of a (tree, range) are next to each other.  False behind its end.
template <int R, bool F32>
__device__ __forceinline__ bool find_work(const MlaTreeArgs &a, Work &w) {
  const int lane = threadIdx.x & 63;
  Lanes<R, F32> l(a);
  const int length = l.range_tiles(lane);
  l.divide(length);
  int sum = wave_scan(l.items), all = __builtin_amdgcn_readlane(sum, 63), items = all;
  if (a.n_trees > 64) {
    for (int t0 = 64; t0 < a.n_trees; t0 += 64) {
      l.look(t0 + lane);
      l.divide(length);
      items += __builtin_amdgcn_readlane(wave_scan(l.items), 63);
    }
    l.look(lane);
    l.divide(length);
  }
  const int share = (items + 7) >> 3, b = blockIdx.x;
  int item = (b & 7) * share + (b >> 3);
  if ((b >> 3) >= share || item >= items) return false;
  int t0 = 0, parts = 0;
  while (item >= all) {
    item -= all;
    parts += __builtin_amdgcn_readlane(wave_scan(l.parts), 63);
    t0 += 64;
    if (t0 >= a.n_trees) return false;
    l.look(t0 + lane);
    l.divide(length);
    sum = wave_scan(l.items);
    all = __builtin_amdgcn_readlane(sum, 63);
  }
  const int at = __ffsll(static_cast<unsigned long long>(__ballot(item < sum))) - 1;
  const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
  const auto of64 = [&](int64_t v) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(of(static_cast<int>(v >> 32)))) << 32 |
                                static_cast<uint32_t>(of(static_cast<int>(v))));
  };
  item -= of(sum - l.items);
  w.part = parts + of(wave_scan(l.parts) - l.parts) + item;
  w.tree = t0 + at;
  w.keys = of(l.keys);
  w.n = of(l.n);
  w.base = of64(l.base);
  w.slot = of64(l.slot);
  const int used = of(l.used), groups = of(l.groups), tiles = of(l.tiles);
  w.split = item / groups;
  w.node0 = (item - w.split * groups) * kGroup<F32>;
  const int each = tiles / used, more = tiles - each * used;   // the first `more` ranges have one more
  w.t0 = each * w.split + min(w.split, more);
  w.t1 = w.t0 + each + (w.split < more ? 1 : 0);
  w.drafted = w.split + 1 == used;
  if (w.drafted) --w.t1;
  w.whole = used == 1;
  return w.whole || w.part < a.part_cap;   // (there is always room, see range_tiles)
}

// Partials: of each item and wavefront, four ranks of a lane's column at a time,
// [R / 8 or R / 16 of them][64 lanes], then maximum and sum [64 lanes].  They lie in the
// order of the list, those of a group `groups` apart.
template <int R, bool F32>
constexpr int kQuads = F32 ? R / 16 : R / 8;
template <int R, bool F32>
constexpr int kPart = 4 * 64 * (4 * kQuads<R, F32> + 2);
template <int R, bool F32>
__device__ __forceinline__ float *partial(const MlaTreeArgs &a, int64_t part, int wave) {
  return a.part + part * kPart<R, F32> + wave * (kPart<R, F32> / 4);
}

template <bool F32>
__device__ __forceinline__ void zero_rows(const MlaTreeArgs &a, const Work &w, int rank) {
  const int rows = min(kGroup<F32>, w.n - w.node0), width = a.heads * rank;
  for (int i = threadIdx.x; i < rows * width; i += 256) {
    const int64_t at = (w.base + w.node0 + i / width) * a.out_stride + i % width;
    if constexpr (F32)
      static_cast<float *>(a.out)[at] = 0.f;
    else
      static_cast<uint16_t *>(a.out)[at] = 0;
  }
}

// The lane's column (head `head` of row `row`, `real`) of a range, quad j being four
// ranks from rank(j) on: the result, or a partial.
template <int R, bool F32, typename V, typename K>
__device__ __forceinline__ void put(const MlaTreeArgs &a, const Work &w, int64_t row, int head, bool real, float m, float l,
                                    V value, K rank) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (!w.whole) {
    float *p = partial<R, F32>(a, w.part, wave);
#pragma unroll
    for (int j = 0; j < kQuads<R, F32>; ++j) reinterpret_cast<f4 *>(p)[64 * j + lane] = value(j);
    reinterpret_cast<f2 *>(p + 256 * kQuads<R, F32>)[lane] = f2{m, l};
  } else if (real) {
    const float inv = 1.0f / l;
#pragma unroll
    for (int j = 0; j < kQuads<R, F32>; ++j)
      store4(a.out, row * a.out_stride + static_cast<int64_t>(head) * R + rank(j),
             F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, value(j) * inv);
  }
}

// Rows of tile t, four ranks per thread and step (whole 128-byte lines per
// wavefront).  Rows past the last key repeat it: their probability is 0, and what
// lies behind the keys in the cache never enters a product.
template <int R, bool F32>
struct Stage {
  static constexpr int kQuads = R / 4, kRows = 256 / kQuads, kSteps = kTile / kRows;
  f4 v[kSteps];
  // A tile of cached keys: a scalar base and 32-bit offsets.
  __device__ __forceinline__ void load(const MlaTreeArgs &a, const Work &w, int t) {
    const int q = threadIdx.x % kQuads, r0 = threadIdx.x / kQuads;
    const char *p = reinterpret_cast<const char *>(a.cache + (w.slot * a.slot_stride + static_cast<int64_t>(kTile * t) * R));
    const int last = w.keys - 1 - kTile * t;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      v[i] = *reinterpret_cast<const f4 *>(p + static_cast<uint32_t>(min(r0 + kRows * i, last) * (4 * R) + 16 * q));
  }
  // The drafted tile: zeros for what is not finite, and which rows held it.
  __device__ __forceinline__ void load_drafted(const MlaTreeArgs &a, const Work &w, int (&bad)[kTile]) {
    const int q = threadIdx.x % kQuads, r0 = threadIdx.x / kQuads, lane0 = (threadIdx.x & 63) - q;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      v[i] = load4(a.latent, (w.base + min(r0 + kRows * i, w.n - 1)) * a.latent_stride + 4 * q,
                   F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      bool any = false;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool ok = is_finite(v[i][c]);
        any |= !ok;
        v[i][c] = ok ? v[i][c] : 0.f;
      }
      const uint64_t row = (__ballot(any) >> lane0) & (~0ull >> (64 - kQuads));
      if (q == 0) bad[r0 + kRows * i] = row != 0;
    }
  }
};

// The path of a node, which may differ from lane to lane (0 behind the tree's nodes);
// `parent` is that of node `lane`.
__device__ __forceinline__ uint64_t path_of(const Work &w, int parent, int node) {
  const int lane = threadIdx.x & 63, from = min(node, kTreeNodes - 1);
  const uint64_t paths = tree_paths(parent, w.n, lane, [](int, int) {});
  const uint32_t lo = __shfl(static_cast<uint32_t>(paths), from, 64);
  const uint32_t hi = __shfl(static_cast<uint32_t>(paths >> 32), from, 64);
  return node < w.n ? static_cast<uint64_t>(hi) << 32 | lo : 0;
}

// ---- bf16: 32x32x16 MFMAs, as the causal attention uses them ---------------------
// The cached latents are rounded to bf16 on their way into LDS: a bf16 model wrote
// them from bf16 values, so nothing is lost.  A probability enters the value product
// as two bf16 numbers, the second what the first has lost (2^-16 of it remains lost):
// as one, the outputs of 32 trees were 0.0020 off a float64 form, of which their own
// rounding is 0.0017; as two 0.0017, for 38.6 us in place of 34.3 (with the merge).
// Scores, maxima and sums are fp32.
//
// An LDS row is R / 8 chunks of 16 bytes, chunk c of row r at place c ^ f(r), f =
// r % 16 rotated left by one bit: eight rows of one chunk (K) and four rows of two
// chunks (V, transposing reads) both touch all banks.
template <int R>
__device__ __forceinline__ int place(int row, int chunk) {
  const int f = ((row & 7) << 1) | ((row >> 3) & 1);
  return row * R + 8 * (chunk ^ (f & (R / 8 - 1)));
}

template <int R>
__global__ __launch_bounds__(256, R <= 128 ? 2 : 1) void mla_tree_kernel(MlaTreeArgs a) {
  constexpr int KS = R / 16, DT = R / 32;
  __shared__ __attribute__((aligned(1024))) uint16_t s_lat[kTile * R];
  __shared__ int s_bad[kTile];
  Work w;
  if (!find_work<R, false>(a, w)) return;
  if (w.keys < 0) return zero_rows<false>(a, w, R);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ln = lane & 31, half = lane >> 5, l16 = lane & 15;
  const int parent = w.drafted ? tree_parent(a.trees, w.base, w.n, lane) : -1;
  Stage<R, false> next;
  if (w.drafted)
    next.load_drafted(a, w, s_bad);
  else
    next.load(a, w, w.t0);
  const int node = w.node0 + 2 * wave + (ln >> 4);   // this lane's column: (node, head)
  const int64_t row = w.base + min(node, w.n - 1);
  bf8 qf[KS];
  {
    const uint16_t *qp = static_cast<const uint16_t *>(a.qa) + row * a.qa_stride +
                         static_cast<int64_t>(min(l16, a.heads - 1)) * R + 8 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = bits_to_bf8(*reinterpret_cast<const u4 *>(qp + 16 * ks));
  }
  const uint64_t path = w.drafted ? path_of(w, parent, node) : 0;
  const bool idle = w.node0 + 2 * wave >= w.n;   // (of the whole wavefront)

  // Q is waited for here: a wait for it inside the loop would be one for the next
  // tile's loads too, every time.
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  // This lane's places within a tile: K row ln (32 kt rows on: a constant), V rows
  // 4 half + l16 / 4 (16 kp rows on: a constant; 8 rows on: the chunk's lowest bit turns).
  int ko[KS], vo[DT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) ko[ks] = place<R>(ln, 2 * ks + half);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    vo[dt] = place<R>(4 * half + (l16 >> 2), 4 * dt + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1)) + 4 * (l16 & 1);
  f16v ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) ot[dt][i] = 0.f;
  float l_run = 0.f;   // over this lane's keys alone
  float m_run = -INFINITY;
  const auto stage = [&]() {
    using St = Stage<R, false>;
    const int q = tid % St::kQuads, r0 = tid / St::kQuads;
#pragma unroll
    for (int i = 0; i < St::kSteps; ++i)
      *reinterpret_cast<u2 *>(s_lat + place<R>(r0 + St::kRows * i, q >> 1) + 4 * (q & 1)) =
          u2{pack_bf16x2(next.v[i].x, next.v[i].y), pack_bf16x2(next.v[i].z, next.v[i].w)};
    lds_barrier();
  };
  // One tile from LDS, of which this lane's column sees the keys `seen` (`all`: every
  // key; one copy of this code, as three held more than the registers there are).
  const auto block = [&](bool all, uint64_t seen) {
    // st[kt][i] = score(key 32 kt + 8 (i / 4) + 4 half + i % 4 of the tile, column ln)
    f16v st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        st[kt] = mfma32x32(bits_to_bf8(*reinterpret_cast<const u4 *>(s_lat + ko[ks] + 32 * kt * R)), qf[ks], st[kt]);
    // (K rows two steps ahead of their products)
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      if (ks + 3 < KS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    if (!all) {
      const uint32_t bits[2] = {static_cast<uint32_t>(seen) >> (4 * half), static_cast<uint32_t>(seen >> 32) >> (4 * half)};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[kt][i] = bits[kt] & (1u << (8 * (i >> 2) + (i & 3))) ? st[kt][i] : -INFINITY;
    }
    float top[4];   // (four chains: one of 32 waits for every step of it)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[i] = st[i >> 1][8 * (i & 1)];
#pragma unroll
      for (int j = 1; j < 8; ++j) top[i] = fmaxf(top[i], st[i >> 1][8 * (i & 1) + j]);
    }
    float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    mx = fmaxf(mx, lane_xor32(mx)) * a.scale_log2;
    // The reference follows the maximum where that has risen by more than kSlack: until
    // then probabilities are up to 2^kSlack, as exact as below 1.
    if (__any(mx > m_run + kSlack)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) ot[dt] *= alpha;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = __builtin_amdgcn_exp2f(fmaf(st[kt][i], a.scale_log2, -m_run));
    float ps[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ps[i] = st[i >> 1][8 * (i & 1)];
#pragma unroll
      for (int j = 1; j < 8; ++j) ps[i] += st[i >> 1][8 * (i & 1) + j];
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
    for (int kp = 0; kp < 4; ++kp) {   // 16 keys from 16 kp on
      const f16v &sv = st[kp >> 1];
      u4 pw, pr;   // rounded, and the rest
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = sv[8 * (kp & 1) + 2 * i], p1 = sv[8 * (kp & 1) + 2 * i + 1];
        pw[i] = pack_bf16x2(p0, p1);
        pr[i] = pack_bf16x2(p0 - __uint_as_float(pw[i] << 16), p1 - __uint_as_float(pw[i] & 0xffff0000u));
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u2 lo = lds_read_tr(s_lat + vo[dt] + 16 * kp * R);
        const u2 hi = lds_read_tr(s_lat + (vo[dt] ^ 8) + (16 * kp + 8) * R);
        const bf8 vf = bits_to_bf8(u4{lo.x, lo.y, hi.x, hi.y});
        ot[dt] = mfma32x32(vf, bits_to_bf8(pw), ot[dt]);
        ot[dt] = mfma32x32(vf, bits_to_bf8(pr), ot[dt]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
#pragma unroll
    for (int i = 0; i < 4 * DT; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 1);
      if (i + 3 < 4 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
  };
  for (int t = w.t0 - (w.drafted ? 1 : 0); t < w.t1; ++t) {
    stage();
    if (t + 1 < w.t1) next.load(a, w, t + 1);
    if (!idle) {
      const int left = t < w.t0 ? 0 : w.keys - kTile * t;
      block(left >= kTile, t < w.t0 ? path : (1ull << (left & 63)) - 1);
    }
    lds_barrier();
  }
  if (w.drafted && (__ballot(s_bad[lane] != 0) & path)) l_run = NAN;
  l_run += lane_xor32(l_run);
  // ot[dt][i] = O[column ln][rank 32 dt + 8 (i / 4) + 4 half + i % 4] before the 1 / l
  put<R, false>(
      a, w, row, l16, node < w.n && l16 < a.heads, m_run, l_run,
      [&](int j) {
        const f16v &v = ot[j >> 2];
        const int i = 4 * (j & 3);
        return f4{v[i], v[i + 1], v[i + 2], v[i + 3]};
      },
      [&](int j) { return 8 * j + 4 * half; });
}

// ---- fp32 ----------------------------------------------------------------------
// 16x16x4 MFMAs in fp32 throughout: an fp32 model's latents have more bits than
// bf16 holds.  5 trees of 1 to 32 nodes after up to 3,001 keys: 16 us and 7 for the
// merge; a tile takes a wavefront 256 MFMAs of 32 cycles (9,700 in all; 12,100 while the
// compiler read V right before each product), and only the keys divide it further.  A
// lane's four consecutive ranks of a key are the A operands of four steps (the k index runs 4 (lane / 16) + step), and the scores' accumulator, keys
// 4 (lane / 16) + i, is the B operand of the value product in the same order.
template <int R>
__global__ __launch_bounds__(256, R <= 128 ? 2 : 1) void mla_tree_f32_kernel(MlaTreeArgs a) {
  constexpr int KB = R / 16, LD = R + 4;
  __shared__ __attribute__((aligned(16))) float s_lat[kTile][LD];
  __shared__ int s_bad[kTile];
  Work w;
  if (!find_work<R, true>(a, w)) return;
  if (w.keys < 0) return zero_rows<true>(a, w, R);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, grp = lane >> 4;
  const int parent = w.drafted ? tree_parent(a.trees, w.base, w.n, lane) : -1;
  Stage<R, true> next;
  if (w.drafted)
    next.load_drafted(a, w, s_bad);
  else
    next.load(a, w, w.t0);
  const int node = w.node0 + wave;   // (the same for the whole wavefront)
  const int64_t row = w.base + min(node, w.n - 1);
  f4 qf[KB], ot[KB];
  const float *qp = static_cast<const float *>(a.qa) + row * a.qa_stride +
                    static_cast<int64_t>(min(l16, a.heads - 1)) * R + 4 * grp;
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    qf[b] = *reinterpret_cast<const f4 *>(qp + 16 * b);
    ot[b] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const uint64_t path = w.drafted ? path_of(w, parent, node) : 0;
#pragma unroll
  for (int b = 0; b < KB; ++b) asm volatile("" : "+v"(qf[b]));   // (waited for here, not in the loop)
  float m_run = -INFINITY, l_run = 0.f;   // l_run over this lane's keys alone
  const auto stage = [&]() {
    using St = Stage<R, true>;
#pragma unroll
    for (int i = 0; i < St::kSteps; ++i)
      *reinterpret_cast<f4 *>(&s_lat[tid / St::kQuads + St::kRows * i][4 * (tid % St::kQuads)]) = next.v[i];
    lds_barrier();
  };
  const auto block = [&](uint64_t seen) {
    f4 st[4];   // score(key 16 kt + 4 grp + i, head l16)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) st[kt] = f4{0.f, 0.f, 0.f, 0.f};
    // LDS reads a step ahead of their products, here and below: by hand, as scheduling groups
    // over that many products take the compiler a minute.
    f4 k[2][4];
    const auto read_k = [&](int b) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) k[b & 1][kt] = *reinterpret_cast<const f4 *>(&s_lat[16 * kt + l16][16 * b + 4 * grp]);
      __builtin_amdgcn_sched_barrier(0);
    };
    read_k(0);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      if (b + 1 < KB) read_k(b + 1);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) st[kt] = mfma_f32(k[b & 1][kt][s], qf[b][s], st[kt]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st[kt][i] = (seen >> (16 * kt + 4 * grp + i)) & 1 ? st[kt][i] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, st[kt][i]);
      }
    mx = fmaxf(mx, lane_xor16(mx));
    mx = fmaxf(mx, lane_xor32(mx));
    const float m_new = fmaxf(m_run, mx);
    const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st[kt][i] = __builtin_amdgcn_exp2f(st[kt][i] - m_new);
        ps += st[kt][i];
      }
    l_run = l_run * alpha + ps;
#pragma unroll
    for (int b = 0; b < KB; ++b) ot[b] *= alpha;
    float v[2][KB];
    const auto read_v = [&](int i) {   // of key 16 (i / 4) + 4 grp + i % 4
#pragma unroll
      for (int b = 0; b < KB; ++b) v[i & 1][b] = s_lat[16 * (i >> 2) + 4 * grp + (i & 3)][16 * b + l16];
      __builtin_amdgcn_sched_barrier(0);
    };
    read_v(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i + 1 < 16) read_v(i + 1);
#pragma unroll
      for (int b = 0; b < KB; ++b) ot[b] = mfma_f32(v[i & 1][b], st[i >> 2][i & 3], ot[b]);
    }
  };
  for (int t = w.t0 - (w.drafted ? 1 : 0); t < w.t1; ++t) {
    stage();
    if (t + 1 < w.t1) next.load(a, w, t + 1);
    if (node < w.n) {
      const int left = t < w.t0 ? 0 : w.keys - kTile * t;
      block(t < w.t0 ? path : left >= kTile ? ~0ull : (1ull << left) - 1);
    }
    lds_barrier();
  }
  if (w.drafted && (__ballot(s_bad[lane] != 0) & path)) l_run = NAN;
  // ot[b][i] = O[head l16][rank 16 b + 4 grp + i] before the 1 / l
  l_run += lane_xor16(l_run);
  l_run += lane_xor32(l_run);
  put<R, true>(
      a, w, row, l16, node < w.n && l16 < a.heads, m_run, l_run, [&](int j) { return ot[j]; },
      [&](int j) { return 16 * j + 4 * grp; });
}

// Joins the ranges of a tree: work-groups (group of nodes and an eighth of the
// quads, tree), a wavefront as in the attention, a thread four ranks at a time.  Eight
// partials are loaded before the first is used.
constexpr int kMergeParts = 8;
template <int R, bool F32>
__global__ __launch_bounds__(256) void mla_tree_merge_kernel(MlaTreeArgs a) {
  constexpr int kParts = kQuads<R, F32> < 8 ? kQuads<R, F32> : 8, QW = kQuads<R, F32> / kParts;   // quads per work-group
  const int tree = blockIdx.y, node0 = static_cast<int>(blockIdx.x / kMergeParts) * kGroup<F32>;
  if (blockIdx.x % kMergeParts >= kParts) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15;
  Lanes<R, F32> trees(a);
  const int length = trees.range_tiles(lane);
  trees.divide(length);
  int64_t part = 0;     // the tree's first
  for (int t0 = 64; t0 <= tree; t0 += 64) {
    part += __builtin_amdgcn_readlane(wave_scan(trees.parts), 63);
    trees.look(t0 + lane);
    trees.divide(length);
  }
  const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, tree & 63); };
  part += of(wave_scan(trees.parts) - trees.parts);
  const int used = of(trees.used), n = of(trees.n), groups = of(trees.groups);
  const int64_t base = iclamp64(a.trees.cu[tree], 0, a.trees.rows);
  const int node = node0 + (F32 ? wave : 2 * wave + ((lane >> 4) & 1));
  // (one range: written already; and there is always room, see range_tiles)
  if (node >= n || l16 >= a.heads || used == 1 || part + used * groups > a.part_cap) return;
  const float *p = partial<R, F32>(a, part + node0 / kGroup<F32>, wave);
  const int64_t step = static_cast<int64_t>(groups) * kPart<R, F32>;
  const int j0 = static_cast<int>(blockIdx.x % kMergeParts) * QW;
  float m = -INFINITY, l = 0.f;
  f4 acc[QW];
#pragma unroll
  for (int j = 0; j < QW; ++j) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 8;
  for (int s0 = 0; s0 < used; s0 += kAhead) {
    f2 ml[kAhead];
    f4 v[kAhead][QW];
    float top = m;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const float *ps = p + min(s0 + s, used - 1) * step;   // the last one again, unused
      ml[s] = reinterpret_cast<const f2 *>(ps + 256 * kQuads<R, F32>)[lane];
#pragma unroll
      for (int j = 0; j < QW; ++j) v[s][j] = reinterpret_cast<const f4 *>(ps)[64 * (j0 + j) + lane];
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) top = fmaxf(top, ml[s].x);
    const float e0 = __builtin_amdgcn_exp2f(m - top);
    l *= e0;
#pragma unroll
    for (int j = 0; j < QW; ++j) acc[j] *= e0;
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
      if (s0 + s < used) {
        const float e = __builtin_amdgcn_exp2f(ml[s].x - top);
        l = fmaf(ml[s].y, e, l);
#pragma unroll
        for (int j = 0; j < QW; ++j) acc[j] += v[s][j] * e;
      }
    m = top;
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int j = 0; j < QW; ++j)
    store4(a.out, (base + node) * a.out_stride + static_cast<int64_t>(l16) * R + (F32 ? 16 * (j0 + j) + 4 * (lane >> 4)
                                                                                      : 8 * (j0 + j) + 4 * (lane >> 5)),
           F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, acc[j] * inv);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace sophia

using namespace sophia;

namespace {
// Items of a list at most, were every range one of its own; how many partials there can
// be (Lanes::range_tiles), and the floats of one.
int64_t tree_items(int n_trees, int max_nodes, bool f32, int splits) {
  const int group = f32 ? kGroup<true> : kGroup<false>;
  return static_cast<int64_t>(n_trees) * ((max_nodes + group - 1) / group) * splits;
}
constexpr int64_t kMostParts = 2 * 512;
int64_t part_floats(int rank, bool f32) { return 4 * 64 * (4 * (rank / (f32 ? 16 : 8)) + 2); }
}  // namespace

extern "C" size_t sophia_mla_tree_workspace_size(int n_trees, int max_nodes, int rank, int dtype, int splits) {
  if (n_trees < 0 || max_nodes < 1 || rank <= 0 || splits < 2) return 0;
  const bool f32 = dtype == SOPHIA_DTYPE_F32;
  return static_cast<size_t>(imin64(kMostParts, tree_items(n_trees, max_nodes, f32, splits)) * part_floats(rank, f32)) *
         sizeof(float);
}

extern "C" int sophia_mla_tree_attn(const void *qa, int64_t qa_stride, const void *latent, int64_t latent_stride,
                                    int dtype, const float *cache, int64_t slot_stride, int n_slots, int max_seq,
                                    const int32_t *slots, const int64_t *cached, const int32_t *cu_nodes,
                                    const int32_t *parents, int n_trees, int64_t rows, int max_nodes, float scale,
                                    void *out, int64_t out_stride, int heads, int rank, int splits, int split_keys,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "mla_tree_attn: dtype not supported");
  SOPHIA_REQUIRE(rank == 32 || rank == 64 || rank == 128 || rank == 256,
                 "mla_tree_attn: rank %d not supported (32, 64, 128 or 256)", rank);
  SOPHIA_REQUIRE(heads >= 1 && heads <= 16, "mla_tree_attn: heads must be in [1, 16]");
  SOPHIA_REQUIRE(n_trees >= 0 && n_trees <= 65535 && rows >= 0 && splits >= 1 && splits <= 1024,
                 "mla_tree_attn: n_trees must be 0..65535, rows >= 0 and splits 1..1024");
  SOPHIA_REQUIRE(split_keys > 0 && split_keys % kTile == 0, "mla_tree_attn: split_keys must be a multiple of %d", kTile);
  SOPHIA_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeNodes, "mla_tree_attn: max_nodes must be in [1, %d]", kTreeNodes);
  SOPHIA_REQUIRE(scale > 0.f, "mla_tree_attn: scale must be > 0");
  SOPHIA_REQUIRE(n_slots >= 0 && max_seq >= 0 && slot_stride >= static_cast<int64_t>(max_seq) * rank,
                 "mla_tree_attn: slot stride smaller than a slot");
  SOPHIA_REQUIRE(qa_stride >= static_cast<int64_t>(heads) * rank && out_stride >= static_cast<int64_t>(heads) * rank &&
                     latent_stride >= rank && qa_stride % 8 == 0 && out_stride % 8 == 0 && latent_stride % 8 == 0 &&
                     slot_stride % 8 == 0,
                 "mla_tree_attn: row strides must hold a row and be multiples of 8");
  if (n_trees == 0 || rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(qa && latent && cache && cached && cu_nodes && parents && out, "mla_tree_attn: NULL pointer");
  SOPHIA_REQUIRE(aligned16(qa) && aligned16(latent) && aligned16(cache) && aligned16(out),
                 "mla_tree_attn: qa, latent, cache and out must be 16-byte aligned");
  SOPHIA_REQUIRE(splits == 1 || (workspace && aligned16(workspace) &&
                                 workspace_bytes >= sophia_mla_tree_workspace_size(n_trees, max_nodes, rank, dtype, splits)),
                 "mla_tree_attn: workspace too small");
  const bool f32 = dtype == SOPHIA_DTYPE_F32;
  const int64_t items = tree_items(n_trees, max_nodes, f32, splits), groups = tree_items(1, max_nodes, f32, 1);
  const int64_t most = imin64(items, groups * n_trees + 512);   // of the list: no more than run at a time, or a group each
  const int part_cap = splits > 1 ? static_cast<int>(imin64(kMostParts, items)) : 0;
  const MlaTreeArgs a{{cu_nodes, parents, rows, max_nodes}, qa, qa_stride, latent, latent_stride, cache, slot_stride,
                      max_seq, n_slots, slots, cached, scale * 1.44269504088896341f, out, out_stride,
                      static_cast<float *>(workspace), part_cap, heads, splits, split_keys / kTile, n_trees};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>((most + 7) / 8 * 8)), merge(static_cast<unsigned>(kMergeParts * groups), n_trees);
  switch (rank) {
#define SOPHIA_MLA_TREE(r)                                                                      \
  case r:                                                                                       \
    if (dtype == SOPHIA_DTYPE_BF16) {                                                           \
      hipLaunchKernelGGL(mla_tree_kernel<r>, grid, dim3(256), 0, st, a);                        \
      if (splits > 1) hipLaunchKernelGGL((mla_tree_merge_kernel<r, false>), merge, dim3(256), 0, st, a); \
    } else {                                                                                    \
      hipLaunchKernelGGL(mla_tree_f32_kernel<r>, grid, dim3(256), 0, st, a);                    \
      if (splits > 1) hipLaunchKernelGGL((mla_tree_merge_kernel<r, true>), merge, dim3(256), 0, st, a);  \
    }                                                                                           \
    break;
    SOPHIA_MLA_TREE(32) SOPHIA_MLA_TREE(64) SOPHIA_MLA_TREE(128) SOPHIA_MLA_TREE(256)
#undef SOPHIA_MLA_TREE
  }
  return check_launch("mla_tree_attn");
}
