// MLA attention in latent space for a tree of drafted tokens: every node attends
// to the cached latents of its sequence and to the drafted latents of itself and
// its ancestors (include/sophia_draft.h), in one pass with a running maximum and
// sum.  Keys and values are the same rows, so a tile of 64 of them is staged in
// LDS once and read twice, as K rows and, transposed, as V.
//
// A work-group (4 wavefronts) takes 8 nodes of one tree and a range of its keys:
// the 16 heads of a node are 16 columns of the matrix products, so a wavefront
// holds 2 nodes.  The drafted latents are the last tile of the last range, the
// only one with a mask per column.  A drafted latent that is not finite would
// reach every node through the products (0 times infinity): it enters them as
// zeros, and the nodes that do see it end as NaN.  Work-groups of one (tree, range) run on one
// XCD, whose L2 serves all but the first of them.
#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_draft.h"

namespace sophia {
namespace {

constexpr int kGroup = 8;        // nodes per work-group
constexpr int kTile = 64;        // keys per tile (a whole tree)
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
  float *part;             // [rows, splits, 16, R + 4] when splits > 1
  int heads, splits, groups, n_trees;
};

typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ bf8 bits_to_bf8(const u4 &v) { return __builtin_bit_cast(bf8, v); }
__device__ __forceinline__ f16v mfma32x32(const bf8 &a, const bf8 &b, const f16v &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Cached keys of a tree: -1 when its slot is out of range (its rows are then zeros).
__device__ __forceinline__ int cached_keys(const MlaTreeArgs &a, int tree, int64_t &slot) {
  slot = a.slots ? a.slots[tree] : tree;
  if (slot < 0 || slot >= a.n_slots) return -1;
  return static_cast<int>(iclamp64(a.cached[tree], 0, a.max_seq));
}

// Tiles of a range: an even division.
__device__ __forceinline__ int tiles_per_split(int tiles, int splits) { return (tiles + splits - 1) / splits; }

// What a work-group does: tree, first node, range; false when there is nothing.
struct Work {
  int tree, node0, split, n, keys, t0, t1;   // tiles [t0, t1); tile keys / 64 rounded up is the drafted one
  int64_t base, slot;
};
__device__ __forceinline__ bool find_work(const MlaTreeArgs &a, Work &w) {
  // unit (tree, range) u: work-groups 8 (groups (u / 8) + group) + u % 8
  const int b = blockIdx.x, r = b >> 3;
  const int unit = (r / a.groups) * 8 + (b & 7);
  if (unit >= a.n_trees * a.splits) return false;
  w.tree = unit / a.splits;
  w.split = unit % a.splits;
  w.node0 = (r % a.groups) * kGroup;
  w.n = tree_nodes(a.trees, w.tree, w.base);
  if (w.node0 >= w.n) return false;
  w.keys = cached_keys(a, w.tree, w.slot);
  const int tiles = (w.keys + kTile - 1) / kTile + 1;
  const int per = tiles_per_split(tiles, a.splits);
  w.t0 = w.split * per;
  w.t1 = min(tiles, w.t0 + per);
  return w.keys < 0 ? w.split == 0 : w.t0 < tiles;
}

template <bool F32>
__device__ __forceinline__ void zero_rows(const MlaTreeArgs &a, const Work &w, int rank) {
  const int rows = min(kGroup, w.n - w.node0), width = a.heads * rank;
  for (int i = threadIdx.x; i < rows * width; i += 256) {
    const int64_t at = (w.base + w.node0 + i / width) * a.out_stride + i % width;
    if constexpr (F32)
      static_cast<float *>(a.out)[at] = 0.f;
    else
      static_cast<uint16_t *>(a.out)[at] = 0;
  }
}

// Four ranks from `rank` on of (row, head): the result, or a partial with its
// running maximum and sum behind it.
template <int R, bool F32>
__device__ __forceinline__ void put4(const MlaTreeArgs &a, const Work &w, int64_t row, int head, int rank, f4 v, float m,
                                     float l) {
  if (a.splits > 1) {
    float *p = a.part + ((row * a.splits + w.split) * 16 + head) * (R + 4);
    *reinterpret_cast<f4 *>(p + rank) = v;
    if (rank == 0) *reinterpret_cast<f2 *>(p + R) = f2{m, l};
  } else {
    store4(a.out, row * a.out_stride + static_cast<int64_t>(head) * R + rank,
           F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16, v * (1.0f / l));
  }
}

// Rows of tile t, four ranks per thread and step (whole 128-byte lines per
// wavefront).  Rows past the last key repeat it: their probability is 0, and what
// lies behind the keys in the cache never enters a product.
template <int R, bool F32>
struct Stage {
  static constexpr int kQuads = R / 4, kRows = 256 / kQuads, kSteps = kTile / kRows;
  f4 v[kSteps];
  __device__ __forceinline__ void load(const MlaTreeArgs &a, const Work &w, int t) {
    const int q = threadIdx.x % kQuads, r0 = threadIdx.x / kQuads;
    if (kTile * t < w.keys) {
      const float *p = a.cache + w.slot * a.slot_stride + 4 * q;
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        v[i] = *reinterpret_cast<const f4 *>(p + static_cast<int64_t>(min(kTile * t + r0 + kRows * i, w.keys - 1)) * R);
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        v[i] = load4(a.latent, (w.base + min(r0 + kRows * i, w.n - 1)) * a.latent_stride + 4 * q,
                     F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16);
    }
  }
  // Of the drafted tile: zeros for what is not finite, and which rows held it.
  __device__ __forceinline__ void clean(int (&bad)[kTile]) {
    const int q = threadIdx.x % kQuads, r0 = threadIdx.x / kQuads, lane0 = (threadIdx.x & 63) - q;
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

// ---- bf16: 32x32x16 MFMAs, as the causal attention uses them ---------------------
// The cached latents are rounded to bf16 on their way into LDS (a bf16 model wrote
// them from bf16 values, so nothing is lost), probabilities to bf16 for the value
// product; scores, maxima and sums are fp32.
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
  __shared__ __attribute__((aligned(1024))) uint16_t s_lat[2][kTile * R];
  __shared__ int s_bad[kTile];
  Work w;
  if (!find_work(a, w)) return;
  if (w.keys < 0) return zero_rows<false>(a, w, R);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ln = lane & 31, half = lane >> 5, l16 = lane & 15;
  Stage<R, false> next;
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
  const uint64_t paths = tree_paths(tree_parent(a.trees, w.base, w.n, lane), w.n, lane, [](int, int) {});
  const uint64_t path = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(paths >> 32), min(node, 63), 64)) << 32 |
                        __shfl(static_cast<uint32_t>(paths), min(node, 63), 64);
  const bool idle = w.node0 + 2 * wave >= w.n;   // (of the whole wavefront)

  f16v ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) ot[dt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;   // l_run over this lane's keys alone
  for (int t = w.t0; t < w.t1; ++t) {
    uint16_t *lat = s_lat[(t - w.t0) & 1];
    const bool drafted = kTile * t >= w.keys;
    if (drafted) next.clean(s_bad);
    {
      using St = Stage<R, false>;
      const int q = tid % St::kQuads, r0 = tid / St::kQuads;
#pragma unroll
      for (int i = 0; i < St::kSteps; ++i)
        *reinterpret_cast<u2 *>(lat + place<R>(r0 + St::kRows * i, q >> 1) + 4 * (q & 1)) =
            u2{pack_bf16x2(next.v[i].x, next.v[i].y), pack_bf16x2(next.v[i].z, next.v[i].w)};
    }
    lds_barrier();   // (the other buffer's reads ended before each wavefront's last barrier)
    if (t + 1 < w.t1) next.load(a, w, t + 1);
    if (idle) continue;
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
        st[kt] = mfma32x32(
            bits_to_bf8(*reinterpret_cast<const u4 *>(lat + place<R>(32 * kt + ln, 2 * ks + half))), qf[ks], st[kt]);
    if (kTile * (t + 1) > w.keys) {
      const uint64_t seen = drafted ? path : (1ull << (w.keys - kTile * t)) - 1;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          st[kt][i] = (seen >> (32 * kt + 8 * (i >> 2) + 4 * half + (i & 3))) & 1 ? st[kt][i] : -INFINITY;
    }
    float mx = st[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) mx = fmaxf(mx, st[i >> 4][i & 15]);
    mx = fmaxf(mx, lane_xor32(mx)) * a.scale_log2;
    if (__any(mx > m_run)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) ot[dt] *= alpha;
    }
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[kt][i] = __builtin_amdgcn_exp2f(fmaf(st[kt][i], a.scale_log2, -m_run));
        ps += st[kt][i];
      }
    l_run += ps;
    if (drafted && (__ballot(s_bad[lane] != 0) & path)) l_run = NAN;
#pragma unroll
    for (int kp = 0; kp < 4; ++kp) {   // 16 keys from 16 kp on
      const f16v &sv = st[kp >> 1];
      u4 pw;
#pragma unroll
      for (int i = 0; i < 4; ++i) pw[i] = pack_bf16x2(sv[8 * (kp & 1) + 2 * i], sv[8 * (kp & 1) + 2 * i + 1]);
      const bf8 pf = bits_to_bf8(pw);
      const int vr = 16 * kp + 4 * half + (l16 >> 2);
      const int vc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u2 lo = lds_read_tr(lat + place<R>(vr, 4 * dt + vc) + 4 * (l16 & 1));
        const u2 hi = lds_read_tr(lat + place<R>(vr + 8, 4 * dt + vc) + 4 * (l16 & 1));
        ot[dt] = mfma32x32(bits_to_bf8(u4{lo.x, lo.y, hi.x, hi.y}), pf, ot[dt]);
      }
    }
  }
  // ot[dt][i] = O[column ln][rank 32 dt + 8 (i / 4) + 4 half + i % 4] before the 1 / l
  l_run += lane_xor32(l_run);
  if (node >= w.n || l16 >= a.heads) return;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      put4<R, false>(a, w, row, l16, 32 * dt + 8 * i + 4 * half,
                     f4{ot[dt][4 * i], ot[dt][4 * i + 1], ot[dt][4 * i + 2], ot[dt][4 * i + 3]}, m_run, l_run);
}

// ---- fp32 ----------------------------------------------------------------------
// 16x16x4 MFMAs in fp32 throughout: an fp32 model's latents have more bits than
// bf16 holds.  A lane's four consecutive ranks of a key are the A operands of four
// steps (the k index runs 4 (lane / 16) + step), and the scores' accumulator, keys
// 4 (lane / 16) + i, is the B operand of the value product in the same order.
template <int R>
__global__ __launch_bounds__(256, 1) void mla_tree_f32_kernel(MlaTreeArgs a) {
  constexpr int KB = R / 16, LD = R + 4;
  __shared__ __attribute__((aligned(16))) float s_lat[kTile][LD];
  __shared__ int s_bad[kTile];
  Work w;
  if (!find_work(a, w)) return;
  if (w.keys < 0) return zero_rows<true>(a, w, R);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, grp = lane >> 4;
  Stage<R, true> next;
  next.load(a, w, w.t0);
  const uint64_t paths = tree_paths(tree_parent(a.trees, w.base, w.n, lane), w.n, lane, [](int, int) {});
  f4 qf[2][KB], ot[2][KB];
  uint64_t path[2];
  float m_run[2], l_run[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int node = min(w.node0 + 2 * wave + e, w.n - 1);
    const float *qp = static_cast<const float *>(a.qa) + (w.base + node) * a.qa_stride +
                      static_cast<int64_t>(min(l16, a.heads - 1)) * R + 4 * grp;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      qf[e][b] = *reinterpret_cast<const f4 *>(qp + 16 * b);
      ot[e][b] = f4{0.f, 0.f, 0.f, 0.f};
    }
    path[e] = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(paths >> 32), node, 64)) << 32 |
              __shfl(static_cast<uint32_t>(paths), node, 64);
    m_run[e] = -INFINITY;
    l_run[e] = 0.f;
  }
  const bool idle = w.node0 + 2 * wave >= w.n;
  for (int t = w.t0; t < w.t1; ++t) {
    using St = Stage<R, true>;
    if (t > w.t0) lds_barrier();
    const bool drafted = kTile * t >= w.keys;
    if (drafted) next.clean(s_bad);
#pragma unroll
    for (int i = 0; i < St::kSteps; ++i)
      *reinterpret_cast<f4 *>(&s_lat[tid / St::kQuads + St::kRows * i][4 * (tid % St::kQuads)]) = next.v[i];
    lds_barrier();
    if (t + 1 < w.t1) next.load(a, w, t + 1);
    if (idle) continue;
    f4 st[2][4];   // score(key 16 kt + 4 grp + i, head l16 of node e)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      st[0][kt] = st[1][kt] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const f4 k = *reinterpret_cast<const f4 *>(&s_lat[16 * kt + l16][16 * b + 4 * grp]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) st[e][kt] = mfma_f32(k[s], qf[e][b][s], st[e][kt]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint64_t seen = ~0ull;
      if (drafted)
        seen = path[e];
      else if (kTile * (t + 1) > w.keys)
        seen = (1ull << (w.keys - kTile * t)) - 1;
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st[e][kt][i] = (seen >> (16 * kt + 4 * grp + i)) & 1 ? st[e][kt][i] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, st[e][kt][i]);
        }
      mx = fmaxf(mx, lane_xor16(mx));
      mx = fmaxf(mx, lane_xor32(mx));
      const float m_new = fmaxf(m_run[e], mx);
      const float alpha = m_run[e] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[e] - m_new);
      m_run[e] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st[e][kt][i] = __builtin_amdgcn_exp2f(st[e][kt][i] - m_new);
          ps += st[e][kt][i];
        }
      l_run[e] = l_run[e] * alpha + ps;
      if (drafted && (__ballot(s_bad[lane] != 0) & path[e])) l_run[e] = NAN;
#pragma unroll
      for (int b = 0; b < KB; ++b) ot[e][b] *= alpha;
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float v = s_lat[16 * kt + 4 * grp + s][16 * b + l16];
#pragma unroll
          for (int e = 0; e < 2; ++e) ot[e][b] = mfma_f32(v, st[e][kt][s], ot[e][b]);
        }
  }
  // ot[e][b][i] = O[head l16 of node e][rank 16 b + 4 grp + i] before the 1 / l
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float l = l_run[e];
    l += lane_xor16(l);
    l += lane_xor32(l);
    const int node = w.node0 + 2 * wave + e;
    if (node >= w.n || l16 >= a.heads) continue;
#pragma unroll
    for (int b = 0; b < KB; ++b)
      put4<R, true>(a, w, w.base + node, l16, 16 * b + 4 * grp, ot[e][b], m_run[e], l);
  }
}

// Joins the ranges of a tree's rows: work-group per (node, tree), a thread four
// ranks of a head.
template <int R, bool F32>
__global__ __launch_bounds__(256) void mla_tree_merge_kernel(MlaTreeArgs a) {
  int64_t base, slot;
  const int n = tree_nodes(a.trees, blockIdx.y, base);
  if (static_cast<int>(blockIdx.x) >= n) return;
  const int keys = cached_keys(a, blockIdx.y, slot);
  if (keys < 0) return;   // (zeros already)
  const int tiles = (keys + kTile - 1) / kTile + 1;
  const int per = tiles_per_split(tiles, a.splits);
  const int used = (tiles + per - 1) / per;
  const int64_t row = base + blockIdx.x;
  for (int i = threadIdx.x; i < a.heads * (R / 4); i += 256) {
    const int h = i / (R / 4), r = 4 * (i % (R / 4));
    const float *p = a.part + (row * a.splits * 16 + h) * (R + 4);
    float m = -INFINITY, l = 0.f;
    f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < used; ++s, p += 16 * (R + 4)) {
      const f2 ml = *reinterpret_cast<const f2 *>(p + R);
      const f4 v = *reinterpret_cast<const f4 *>(p + r);
      const float m_new = fmaxf(m, ml.x);
      const float e0 = __builtin_amdgcn_exp2f(m - m_new), e1 = __builtin_amdgcn_exp2f(ml.x - m_new);
      acc = acc * e0 + v * e1;
      l = l * e0 + ml.y * e1;
      m = m_new;
    }
    store4(a.out, row * a.out_stride + static_cast<int64_t>(h) * R + r, F32 ? SOPHIA_DTYPE_F32 : SOPHIA_DTYPE_BF16,
           acc * (1.0f / l));
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" size_t sophia_mla_tree_workspace_size(int64_t rows, int rank, int splits) {
  if (rows < 0 || rank <= 0 || splits < 1) return 0;
  return splits > 1 ? static_cast<size_t>(rows) * splits * 16 * (rank + 4) * sizeof(float) : 0;
}

extern "C" int sophia_mla_tree_attn(const void *qa, int64_t qa_stride, const void *latent, int64_t latent_stride,
                                    int dtype, const float *cache, int64_t slot_stride, int n_slots, int max_seq,
                                    const int32_t *slots, const int64_t *cached, const int32_t *cu_nodes,
                                    const int32_t *parents, int n_trees, int64_t rows, int max_nodes, float scale,
                                    void *out, int64_t out_stride, int heads, int rank, int splits, void *workspace,
                                    size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "mla_tree_attn: dtype not supported");
  SOPHIA_REQUIRE(rank == 32 || rank == 64 || rank == 128 || rank == 256,
                 "mla_tree_attn: rank %d not supported (32, 64, 128 or 256)", rank);
  SOPHIA_REQUIRE(heads >= 1 && heads <= 16, "mla_tree_attn: heads must be in [1, 16]");
  SOPHIA_REQUIRE(n_trees >= 0 && n_trees <= 65535 && rows >= 0 && splits >= 1 && splits <= 1024,
                 "mla_tree_attn: n_trees must be 0..65535, rows >= 0 and splits 1..1024");
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
                                 workspace_bytes >= sophia_mla_tree_workspace_size(rows, rank, splits)),
                 "mla_tree_attn: workspace too small");
  const int groups = (max_nodes + kGroup - 1) / kGroup;
  const int64_t blocks = (static_cast<int64_t>(n_trees) * splits + 7) / 8 * 8 * groups;
  SOPHIA_REQUIRE(blocks <= 0x7fffffff, "mla_tree_attn: too many trees and splits");
  const MlaTreeArgs a{{cu_nodes, parents, rows, max_nodes}, qa, qa_stride, latent, latent_stride, cache, slot_stride,
                      max_seq, n_slots, slots, cached, scale * 1.44269504088896341f, out, out_stride,
                      static_cast<float *>(workspace), heads, splits, groups, n_trees};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), merge(max_nodes, n_trees);
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
