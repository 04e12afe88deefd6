// The KDA recurrence along the paths of a tree of drafted tokens, and the
// accepted path's write-back into the caches of all layers.
//
// Step.  The chunk form of the delta rule with the ancestor mask in the place of
// the lower triangle (include/sophia_draft.h has the formulas): with A_ij =
// beta_i k_i . k_j e^(G_i - G_j) over strict ancestors and B_ij = q_i . k_j
// e^(G_i - G_j) over ancestors and the node itself,
//   (I + A) U = beta (V - (K e^G) S),   O = (Q e^G) S + B U.
// The state is read once and not written; a node's own state is never formed.
//
// One 256-thread work-group per (tree, head).  Each wavefront owns 32 value
// columns, of which its lanes hold S as B operands of v_mfma_f32_16x16x4_f32
// from the start (issued before anything else); q, k, G, A and B are formed
// together in LDS, and from the products with S on no wavefront waits for
// another: an accumulator holds rows 4 (lane / 16) + i of a 16-row tile, which
// is a B operand whose k index runs 4 (lane / 16) + step, so U goes from one
// product to the next in registers.
//
// Everything is fp32 (the matrix products too): u enters the cached state with
// the accepted path, and the decode step that the state otherwise comes from
// is fp32 as well.  The exponents e^(G_i - G_j) are formed per pair, on the
// vector unit, for ancestors alone: their arguments are never positive, however
// long the path and strong the decay, where a factored form e^(G_i) e^(-G_j)
// overflows past 17 steps of the lower bound -5.
//
// A node with an input that is not finite would reach its siblings through the
// products (0 times infinity): its rows enter them as zeros, and what lies on a
// path with it ends as NaN.
#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_draft.h"

namespace sophia {
namespace {

constexpr int kD = 128;
constexpr int kLd = kD + 4;     // row stride of the LDS matrices: 16 rows 4 banks apart
constexpr int kTape = 3 * kD;   // floats of a node's tape per head

struct TreeStepArgs {
  Trees trees;
  const void *x[3];          // q, k, v before the conv
  int64_t x_stride;
  const float *conv_w;       // [3 * heads * 128, taps]
  const float *conv_state;   // [n_slots, 3 * heads * 128, taps - 1]
  int taps;
  const void *g;
  int64_t g_stride;
  int g_dtype;
  const void *beta;
  int64_t beta_stride;
  int beta_dtype;
  const float *A_log, *dt_bias;
  float scale, lower_bound;
  unsigned flags;
  const float *state;
  int n_slots;
  const int32_t *slots;
  int heads;
  void *o;
  int64_t o_stride;
  float *tape;
};

template <int N>
struct alignas(4 * N) Floats {
  float v[N];
};

// N consecutive elements (N * size bytes aligned) as floats.
template <int DT, int N>
__device__ __forceinline__ void load_n(const void *base, int64_t idx, float (&r)[N]) {
  if constexpr (N == 2 && DT == SOPHIA_DTYPE_BF16) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(base) + idx);
    r[0] = __uint_as_float(w << 16);
    r[1] = __uint_as_float(w & 0xffff0000u);
  } else if constexpr (N == 2) {
    const f2 w = *reinterpret_cast<const f2 *>(static_cast<const float *>(base) + idx);
    r[0] = w.x;
    r[1] = w.y;
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const f4 w = load4(base, idx + c, DT);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[c + i] = w[i];
    }
  }
}

// silu(conv) of N consecutive channels (the first is `ch` of the fused q | k | v
// channels, `col` of its own part `x`) at a node.  Predecessors are counted from
// the oldest history sample: 0, 1, 2, then node i as 3 + i.
template <int DT, int N>
__device__ __forceinline__ void conv_node(const TreeStepArgs &a, const void *x, int64_t base, int64_t col, int64_t ch,
                                          const float *hist, const int *par, int node, float (&y)[N]) {
  float acc[N];
#pragma unroll
  for (int c = 0; c < N; ++c) acc[c] = 0.f;
  int e = node + 3;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if (d >= a.taps) break;
    float s[N];
    if (e >= 3) {
      load_n<DT>(x, (base + e - 3) * a.x_stride + col, s);
      const int p = par[e - 3];
      e = p < 0 ? 2 : p + 3;
    } else {
      const int hist_len = a.taps - 1;   // (e + hist_len - 3 >= 0: the taps reach that far)
#pragma unroll
      for (int c = 0; c < N; ++c) s[c] = hist[(ch + c) * hist_len + e + hist_len - 3];
      --e;
    }
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] = fmaf(a.conv_w[(ch + c) * a.taps + a.taps - 1 - d], s[c], acc[c]);
  }
#pragma unroll
  for (int c = 0; c < N; ++c) y[c] = acc[c] * sigmoid_f(acc[c]);
}

// MT: tiles of 16 nodes.
template <int MT, int DT>
__global__ __launch_bounds__(256, MT == 1 ? 2 : 1) void kda_tree_step_kernel(TreeStepArgs a) {
  constexpr int T = 16 * MT, LA = T + 4;
  __shared__ __align__(16) float s_q[T][kLd], s_k[T][kLd], s_g[T][kLd];
  __shared__ __align__(16) float s_a[T][LA];   // -A, its diagonal blocks later (I + A)^-1
  __shared__ __align__(16) float s_b[T][LA];
  __shared__ float s_beta[T];
  __shared__ int s_bad[kTreeNodes];
  __shared__ uint64_t s_path[kTreeNodes];
  __shared__ int s_up[6][kTreeNodes];          // s_up[0]: parents

  const int h = blockIdx.x, tree = blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int c16 = lane & 15, grp = lane >> 4;
  int64_t base;
  const int n = tree_nodes(a.trees, tree, base);
  if (n == 0) return;
  const int slot = a.slots ? a.slots[tree] : tree;
  const int col2 = 32 * wave + 2 * c16;   // this lane's two value columns
  if (slot < 0 || slot >= a.n_slots) {
    for (int i = t; i < n * kD; i += 256) {
      const int64_t row = base + i / kD;
      store_elem(a.o, row * a.o_stride + static_cast<int64_t>(h) * kD + i % kD, DT, 0.f);
      float *tp = a.tape + (row * a.heads + h) * kTape + i % kD;
      tp[0] = tp[kD] = tp[2 * kD] = 0.f;
    }
    return;
  }
  // S rows 16 blk + 4 grp + s of the lane's columns: 4 rows of 128 bytes per load.
  f2 st[kD / 4];
  const float *S = a.state + (static_cast<int64_t>(slot) * a.heads + h) * kD * kD;
#pragma unroll
  for (int i = 0; i < kD / 4; ++i)
    st[i] = __builtin_nontemporal_load(
        reinterpret_cast<const f2 *>(S + (16 * (i >> 2) + 4 * grp + (i & 3)) * kD + col2));

  const int parent = tree_parent(a.trees, base, n, lane);
  const uint64_t path = tree_paths(parent, n, lane, [&](int r, int up) {
    if (wave == 0) s_up[r][lane] = up;
  });
  if (wave == 0) s_path[lane] = path;
  int depth = __popcll(path);
#pragma unroll
  for (int m = 1; m < 64; m *= 2) depth = max(depth, __shfl_xor(depth, m, 64));
  for (int i = t; i < T * LA; i += 256) (&s_a[0][0])[i] = (&s_b[0][0])[i] = 0.f;
  if (t < T) {
    float b = t < n ? load_elem(a.beta, (base + t) * a.beta_stride + h, a.beta_dtype) : 0.f;
    if (a.flags & SOPHIA_KDA_BETA_SIGMOID) b = sigmoid_f(b);
    s_beta[t] = t < n && is_finite(b) ? b : 0.f;
    s_bad[t] = !is_finite(b);
  }
  __syncthreads();

  // q, k and the log-decay: 16 nodes at a time, 8 channels per thread.
  const int64_t inner = static_cast<int64_t>(a.heads) * kD;
  const float *hist = a.conv_state + static_cast<int64_t>(slot) * 3 * inner * (a.taps - 1);
  const int seg = 8 * (t & 15);
  const int64_t hc = static_cast<int64_t>(h) * kD + seg;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int node = 16 * m + (t >> 4);
    float q[8], k[8], g[8];
    if (node < n) {
      conv_node<DT>(a, a.x[0], base, hc, hc, hist, s_up[0], node, q);
      conv_node<DT>(a, a.x[1], base, hc, inner + hc, hist, s_up[0], node, k);
      if (a.g_dtype == SOPHIA_DTYPE_BF16)
        load_n<SOPHIA_DTYPE_BF16>(a.g, (base + node) * a.g_stride + hc, g);
      else
        load_n<SOPHIA_DTYPE_F32>(a.g, (base + node) * a.g_stride + hc, g);
      if (a.flags & SOPHIA_KDA_GATE_IN_KERNEL) {
        const float head_scale = __expf(a.A_log[h]);
#pragma unroll
        for (int c = 0; c < 8; ++c) g[c] = kda_log_decay(g[c], head_scale, a.dt_bias[hc + c], a.lower_bound);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) q[c] = k[c] = g[c] = 0.f;
    }
    float qs = a.scale, ks = 1.f;
    if (a.flags & SOPHIA_KDA_QK_L2NORM) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        sq = fmaf(q[c], q[c], sq);
        sk = fmaf(k[c], k[c], sk);
      }
      qs = a.scale / fmaxf(sqrtf(row_sum16(sq)), 1e-12f);
      ks = 1.f / fmaxf(sqrtf(row_sum16(sk)), 1e-12f);
    }
    bool ok = true;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      q[c] *= qs;
      k[c] *= ks;
      ok &= is_finite(q[c]) && is_finite(k[c]) && is_finite(g[c]);
    }
    if (((__ballot(!ok) >> (lane & 48)) & 0xffff) != 0) {   // (of the node's 16 threads alike)
#pragma unroll
      for (int c = 0; c < 8; ++c) q[c] = k[c] = g[c] = 0.f;
      s_bad[node] = 1;
    }
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      *reinterpret_cast<f4 *>(&s_q[node][seg + c]) = f4{q[c], q[c + 1], q[c + 2], q[c + 3]};
      *reinterpret_cast<f4 *>(&s_k[node][seg + c]) = f4{k[c], k[c + 1], k[c + 2], k[c + 3]};
      *reinterpret_cast<f4 *>(&s_g[node][seg + c]) = f4{g[c], g[c + 1], g[c + 2], g[c + 3]};
    }
  }
  __syncthreads();

  uint64_t bad = __ballot(lane < T && s_bad[lane < T ? lane : 0] != 0);

  // G: sums of the log-decay along the paths, by doubling (as many rounds as the
  // deepest path needs).
  for (int r = 0; (1 << r) < depth; ++r) {
    f4 add[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int up = s_up[r][16 * m + (t >> 4)];
      add[m][0] = up < 0 ? f4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f4 *>(&s_g[up][seg]);
      add[m][1] = up < 0 ? f4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f4 *>(&s_g[up][seg + 4]);
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      *reinterpret_cast<f4 *>(&s_g[16 * m + (t >> 4)][seg]) += add[m][0];
      *reinterpret_cast<f4 *>(&s_g[16 * m + (t >> 4)][seg + 4]) += add[m][1];
    }
    __syncthreads();
  }

  // A and B: a wavefront takes every fourth node, 16 lanes one of its ancestors.
  for (int i = wave; i < n; i += 4) {
    uint64_t left = s_path[i];
    float qi[8], ki[8], gi[8];
    load_n<SOPHIA_DTYPE_F32>(&s_q[i][0], 8 * c16, qi);
    load_n<SOPHIA_DTYPE_F32>(&s_k[i][0], 8 * c16, ki);
    load_n<SOPHIA_DTYPE_F32>(&s_g[i][0], 8 * c16, gi);
    while (left) {
      int j = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int low = left ? __ffsll(static_cast<unsigned long long>(left)) - 1 : -1;
        if (grp == e) j = low;
        left &= left - 1;   // (0 stays 0)
      }
      float kk = 0.f, qk = 0.f;
      if (j >= 0) {
        float kj[8], gj[8];
        load_n<SOPHIA_DTYPE_F32>(&s_k[j][0], 8 * c16, kj);
        load_n<SOPHIA_DTYPE_F32>(&s_g[j][0], 8 * c16, gj);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float w = kj[c] * __expf(gi[c] - gj[c]);
          kk = fmaf(ki[c], w, kk);
          qk = fmaf(qi[c], w, qk);
        }
      }
      kk = row_sum16(kk);
      qk = row_sum16(qk);
      if (j >= 0 && c16 == 0) {
        s_b[i][j] = qk;
        if (j != i) s_a[i][j] = -s_beta[i] * kk;
      }
    }
  }
  __syncthreads();

  // The tape's k and G, and in their place K e^G and Q e^G.  One wavefront also
  // inverts the unit lower triangular diagonal blocks of I + A, a column per lane.
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int node = 16 * m + (t >> 4);
    float *tp = a.tape + ((base + node) * a.heads + h) * kTape + seg;
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      f4 *pq = reinterpret_cast<f4 *>(&s_q[node][seg + c]), *pk = reinterpret_cast<f4 *>(&s_k[node][seg + c]);
      const f4 gv = *reinterpret_cast<const f4 *>(&s_g[node][seg + c]), kv = *pk;
      if (node < n) {
        const float nan = s_path[node] & bad ? NAN : 0.f;
        *reinterpret_cast<f4 *>(tp + kD + c) = kv + nan;
        *reinterpret_cast<f4 *>(tp + 2 * kD + c) = gv + nan;
      }
      f4 e;
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = __expf(gv[i]);
      *pq *= e;
      *pk = kv * e;
    }
  }
  if (wave == 3 && grp < MT) {
    float inv[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = i == c16 ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) x = fmaf(s_a[16 * grp + i][16 * grp + j], inv[j], x);
      inv[i] = x;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_a[16 * grp + i][16 * grp + c16] = inv[i];
  }
  __syncthreads();

  // (K e^G) S and (Q e^G) S for this wavefront's columns.
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 u[MT][2], o[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) u[m][0] = u[m][1] = o[m][0] = o[m][1] = zero;
#pragma unroll
  for (int blk = 0; blk < kD / 16; ++blk)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const f4 ak = *reinterpret_cast<const f4 *>(&s_k[16 * m + c16][16 * blk + 4 * grp]);
      const f4 aq = *reinterpret_cast<const f4 *>(&s_q[16 * m + c16][16 * blk + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u[m][e] = mfma_f32(ak[s], st[4 * blk + s][e], u[m][e]);
          o[m][e] = mfma_f32(aq[s], st[4 * blk + s][e], o[m][e]);
        }
    }

  // Block forward substitution, and the outputs.
  const int64_t vc = static_cast<int64_t>(h) * kD + col2;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    f4 rhs[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int node = 16 * m + 4 * grp + i;
      float v[2] = {0.f, 0.f};
      if (node < n) conv_node<DT>(a, a.x[2], base, vc, 2 * inner + vc, hist, s_up[0], node, v);
      const bool ok = is_finite(v[0]) && is_finite(v[1]);
      const uint64_t rows = __ballot(!ok);
      if (rows) {   // (of this wavefront's columns)
        if (!ok) v[0] = v[1] = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((rows >> (16 * r)) & 0xffff) bad |= 1ull << (16 * m + 4 * r + i);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) rhs[e][i] = s_beta[node] * (v[e] - u[m][e][i]);
    }
#pragma unroll
    for (int p = 0; p < m; ++p) {
      const f4 l = *reinterpret_cast<const f4 *>(&s_a[16 * m + c16][16 * p + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) rhs[e] = mfma_f32(l[s], u[p][e][s], rhs[e]);
    }
    const f4 inv = *reinterpret_cast<const f4 *>(&s_a[16 * m + c16][16 * m + 4 * grp]);
    u[m][0] = u[m][1] = zero;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) u[m][e] = mfma_f32(inv[s], rhs[e][s], u[m][e]);
#pragma unroll
    for (int p = 0; p <= m; ++p) {
      const f4 b = *reinterpret_cast<const f4 *>(&s_b[16 * m + c16][16 * p + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[m][e] = mfma_f32(b[s], u[p][e][s], o[m][e]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int node = 16 * m + 4 * grp + i;
      if (node >= n) continue;
      const int64_t row = base + node;
      const float nan = s_path[node] & bad ? NAN : 0.f;
      const float o0 = o[m][0][i] + nan, o1 = o[m][1][i] + nan;
      if constexpr (DT == SOPHIA_DTYPE_BF16)
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.o) + row * a.o_stride + vc) = pack_bf16x2(o0, o1);
      else
        *reinterpret_cast<f2 *>(static_cast<float *>(a.o) + row * a.o_stride + vc) = f2{o0, o1};
      *reinterpret_cast<f2 *>(a.tape + (row * a.heads + h) * kTape + col2) = f2{u[m][0][i] + nan, u[m][1][i] + nan};
    }
  }
}

// ---------------------------------------------------------------------------
// Commit: work-group (layer, head, half of the value columns) x tree for the KDA
// layers, (layer) x tree for the MLA layers, all layers in one launch: the few
// trees of a small batch then still fill the chip, and 28 launches become one.
// Bound by the state: 64 KiB read and written per (layer, tree, head), in place,
// as the decode step moves it (thread: 4 columns of every 16th row).
struct CommitArgs {
  Trees trees;
  const int32_t *path;
  int64_t path_stride;
  const int32_t *n_path;
  int max_path;
  const int32_t *slots;
  int n_slots, heads, taps, x_dtype;
  const int64_t *cached;
  int max_seq, rank, latent_dtype;
  int n_kda;
  sophia_commit_kda kda[SOPHIA_COMMIT_KDA];
  sophia_commit_mla mla[SOPHIA_COMMIT_MLA];
};

constexpr int kCommitCols = 64;

__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
  __shared__ int s_path[kTreeNodes];
  __shared__ int s_n;
  __shared__ __align__(16) float s_w[kTreeNodes][kD];
  __shared__ __align__(16) float s_u[kTreeNodes][kCommitCols];
  __shared__ float s_end[kD];
  const int tree = blockIdx.y, t = threadIdx.x;
  int64_t base;
  const int nodes = tree_nodes(a.trees, tree, base);
  const int slot = a.slots ? a.slots[tree] : tree;
  if (slot < 0 || slot >= a.n_slots) return;
  if (t < 64) {
    const int want = min(a.n_path[tree], a.max_path);
    const int p = t < want ? a.path[tree * a.path_stride + t] : -1;
    const uint64_t bad = __ballot(p < 0 || p >= nodes);
    s_path[t] = p;
    if (t == 0) s_n = bad ? __ffsll(static_cast<unsigned long long>(bad)) - 1 : 64;
  }
  __syncthreads();
  const int n = s_n;
  if (n == 0) return;

  const int per_layer = a.heads * (kD / kCommitCols);
  const int kda_blocks = a.n_kda * per_layer;
  if (static_cast<int>(blockIdx.x) >= kda_blocks) {
    const sophia_commit_mla &l = a.mla[blockIdx.x - kda_blocks];
    const int64_t pos = a.cached[tree];
    const int quads = a.rank / 4;
    for (int i = t; i < n * quads; i += 256) {
      const int at = i / quads, c = 4 * (i % quads);
      if (pos + at < 0 || pos + at >= a.max_seq) continue;
      *reinterpret_cast<f4 *>(l.cache + slot * l.slot_stride + (pos + at) * a.rank + c) =
          load4(l.latent, (base + s_path[at]) * l.latent_stride + c, a.latent_dtype);
    }
    return;
  }
  const sophia_commit_kda &l = a.kda[blockIdx.x / per_layer];
  const int part = blockIdx.x % per_layer;
  const int h = part / (kD / kCommitCols), col0 = (part % (kD / kCommitCols)) * kCommitCols;
  const int cg = t & 15, rg = t >> 4;
  float *S = l.state + (static_cast<int64_t>(slot) * a.heads + h) * kD * kD;
  f4 st[kD / 16];
#pragma unroll
  for (int r = 0; r < kD / 16; ++r)
    st[r] = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(S + (rg + 16 * r) * kD + col0 + 4 * cg));
  const auto tape = [&](int at) { return l.tape + ((base + s_path[at]) * a.heads + h) * kTape; };
  const int c = t & (kD - 1);
  const float end = tape(n - 1)[2 * kD + c];
  if (t < kD) s_end[c] = __expf(end);
  for (int at = t >> 7; at < n; at += 2) s_w[at][c] = tape(at)[kD + c] * __expf(end - tape(at)[2 * kD + c]);
  for (int at = t >> 6; at < n; at += 4) s_u[at][t & 63] = tape(at)[col0 + (t & 63)];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kD / 16; ++r) st[r] *= s_end[rg + 16 * r];
  for (int at = 0; at < n; ++at) {
    const f4 u = *reinterpret_cast<const f4 *>(&s_u[at][4 * cg]);
#pragma unroll
    for (int r = 0; r < kD / 16; ++r) st[r] += s_w[at][rg + 16 * r] * u;
  }
#pragma unroll
  for (int r = 0; r < kD / 16; ++r)
    __builtin_nontemporal_store(st[r], reinterpret_cast<f4 *>(S + (rg + 16 * r) * kD + col0 + 4 * cg));

  // The head's q, k and v histories, a channel per thread: the samples kept move
  // down, the path's last ones follow.
  const int hist = a.taps - 1;
  if (col0 != 0 || hist == 0) return;
  const int64_t inner = static_cast<int64_t>(a.heads) * kD;
  for (int i = t; i < 3 * kD; i += 256) {
    const int64_t ch = (i / kD) * inner + static_cast<int64_t>(h) * kD + i % kD;
    float *p = l.conv_state + (static_cast<int64_t>(slot) * 3 * inner + ch) * hist;
    float keep[3];
    for (int j = 0; j < hist; ++j) {
      const int at = n + j;   // of (history, path): hist + n samples
      keep[j] = at < hist ? p[at] : load_elem(l.x, (base + s_path[at - hist]) * l.x_stride + ch, a.x_dtype);
    }
    for (int j = 0; j < hist; ++j) p[j] = keep[j];
  }
}

bool dtype_ok(int dtype) { return dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16; }
bool aligned(const void *p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" int sophia_kda_tree_step(const void *x_q, const void *x_k, const void *x_v, int64_t x_row_stride, int x_dtype,
                                    const float *conv_weight, const float *conv_state, int kernel_size, const void *g,
                                    int64_t g_row_stride, int g_dtype, const void *beta, int64_t beta_row_stride,
                                    int beta_dtype, const float *A_log, const float *dt_bias, float scale,
                                    float lower_bound, unsigned flags, const float *state, int n_slots,
                                    const int32_t *slots, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                                    int64_t rows, int max_nodes, int num_heads, int head_dim, void *o,
                                    int64_t o_row_stride, float *tape, void *stream) {
  SOPHIA_REQUIRE(head_dim == kD, "kda_tree_step: head_dim must be 128 (got %d)", head_dim);
  SOPHIA_REQUIRE(kernel_size >= 1 && kernel_size <= 4, "kda_tree_step: kernel_size must be in [1, 4]");
  SOPHIA_REQUIRE(n_trees >= 0 && n_trees <= 65535 && num_heads > 0 && rows >= 0,
                 "kda_tree_step: n_trees must be 0..65535, num_heads > 0 and rows >= 0");
  SOPHIA_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeNodes, "kda_tree_step: max_nodes must be in [1, %d]", kTreeNodes);
  SOPHIA_REQUIRE(dtype_ok(x_dtype) && dtype_ok(g_dtype) && dtype_ok(beta_dtype), "kda_tree_step: dtype not supported");
  SOPHIA_REQUIRE(n_slots >= 0, "kda_tree_step: n_slots must be >= 0");
  const int64_t inner = static_cast<int64_t>(num_heads) * kD;
  SOPHIA_REQUIRE(x_row_stride >= inner && g_row_stride >= inner && beta_row_stride >= num_heads && o_row_stride >= inner,
                 "kda_tree_step: row stride smaller than a row");
  SOPHIA_REQUIRE(x_row_stride % 8 == 0 && g_row_stride % 8 == 0 && o_row_stride % 8 == 0,
                 "kda_tree_step: row strides of x, g and o must be multiples of 8");
  if (n_trees == 0 || rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(x_q && x_k && x_v && conv_weight && g && beta && state && cu_nodes && parents && o && tape &&
                     (conv_state || kernel_size == 1),
                 "kda_tree_step: NULL pointer");
  SOPHIA_REQUIRE(!(flags & SOPHIA_KDA_GATE_IN_KERNEL) || (A_log && dt_bias),
                 "kda_tree_step: gate in kernel needs A_log and dt_bias");
  SOPHIA_REQUIRE(aligned(x_q, 16) && aligned(x_k, 16) && aligned(x_v, 16) && aligned(g, 16) && aligned(o, 16) &&
                     aligned(state, 16) && aligned(tape, 16),
                 "kda_tree_step: x, g, o, state and tape must be 16-byte aligned");
  const TreeStepArgs a{{cu_nodes, parents, rows, max_nodes}, {x_q, x_k, x_v}, x_row_stride, conv_weight, conv_state,
                       kernel_size, g, g_row_stride, g_dtype, beta, beta_row_stride, beta_dtype, A_log, dt_bias, scale,
                       lower_bound, flags, state, n_slots, slots, num_heads, o, o_row_stride, tape};
  const dim3 grid(num_heads, n_trees);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SOPHIA_TREE_STEP(MT)                                                                              \
  if (x_dtype == SOPHIA_DTYPE_BF16)                                                                       \
    hipLaunchKernelGGL((kda_tree_step_kernel<MT, SOPHIA_DTYPE_BF16>), grid, dim3(256), 0, st, a);         \
  else                                                                                                    \
    hipLaunchKernelGGL((kda_tree_step_kernel<MT, SOPHIA_DTYPE_F32>), grid, dim3(256), 0, st, a);
  if (max_nodes <= 16) {
    SOPHIA_TREE_STEP(1)
  } else if (max_nodes <= 32) {
    SOPHIA_TREE_STEP(2)
  } else {
    SOPHIA_TREE_STEP(4)
  }
#undef SOPHIA_TREE_STEP
  return check_launch("kda_tree_step");
}

extern "C" int sophia_tree_commit(const int32_t *path, int64_t path_stride, const int32_t *n_path, int max_path,
                                  const int32_t *cu_nodes, int n_trees, int64_t rows, const int32_t *slots, int n_slots,
                                  const sophia_commit_kda *kda, int n_kda, int num_heads, int head_dim, int kernel_size,
                                  int x_dtype, const sophia_commit_mla *mla, int n_mla, const int64_t *cached,
                                  int max_seq, int rank, int latent_dtype, void *stream) {
  SOPHIA_REQUIRE(n_trees >= 0 && n_trees <= 65535 && rows >= 0 && n_slots >= 0 && n_kda >= 0 && n_mla >= 0,
                 "tree_commit: n_trees must be 0..65535, rows, n_slots and layer counts >= 0");
  SOPHIA_REQUIRE(max_path >= 1 && max_path <= kTreeNodes && path_stride >= max_path,
                 "tree_commit: max_path must be in [1, %d] and path rows at least as long", kTreeNodes);
  SOPHIA_REQUIRE((n_kda == 0 || kda) && (n_mla == 0 || mla), "tree_commit: NULL layer list");
  if (n_kda > 0) {
    SOPHIA_REQUIRE(head_dim == kD, "tree_commit: head_dim must be 128 (got %d)", head_dim);
    SOPHIA_REQUIRE(num_heads > 0 && num_heads <= 4096 && kernel_size >= 1 && kernel_size <= 4 && dtype_ok(x_dtype),
                   "tree_commit: num_heads must be 1..4096, kernel_size 1..4, x fp32 or bf16");
  }
  if (n_mla > 0)
    SOPHIA_REQUIRE(rank > 0 && rank % 4 == 0 && max_seq >= 0 && dtype_ok(latent_dtype),
                   "tree_commit: rank must be a multiple of 4, max_seq >= 0, latents fp32 or bf16");
  if (n_trees == 0 || rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(path && n_path && cu_nodes && (n_mla == 0 || cached), "tree_commit: NULL pointer");
  const int64_t inner = static_cast<int64_t>(num_heads) * kD;
  for (int l = 0; l < n_kda; ++l) {
    SOPHIA_REQUIRE(kda[l].tape && kda[l].x && kda[l].state && (kda[l].conv_state || kernel_size == 1),
                   "tree_commit: NULL pointer in KDA layer %d", l);
    SOPHIA_REQUIRE(kda[l].x_stride >= 3 * inner, "tree_commit: x row stride smaller than a row in KDA layer %d", l);
    SOPHIA_REQUIRE(aligned(kda[l].state, 16), "tree_commit: state must be 16-byte aligned in KDA layer %d", l);
  }
  for (int l = 0; l < n_mla; ++l) {
    SOPHIA_REQUIRE(mla[l].latent && mla[l].cache, "tree_commit: NULL pointer in MLA layer %d", l);
    SOPHIA_REQUIRE(mla[l].latent_stride >= rank && mla[l].latent_stride % 4 == 0 &&
                       mla[l].slot_stride >= static_cast<int64_t>(max_seq) * rank && mla[l].slot_stride % 4 == 0,
                   "tree_commit: bad strides in MLA layer %d", l);
    SOPHIA_REQUIRE(aligned(mla[l].cache, 16) && aligned(mla[l].latent, latent_dtype == SOPHIA_DTYPE_BF16 ? 8 : 16),
                   "tree_commit: rows not aligned in MLA layer %d", l);
  }
  for (int k0 = 0, m0 = 0; k0 < n_kda || m0 < n_mla;) {
    const int nk = n_kda - k0 < SOPHIA_COMMIT_KDA ? n_kda - k0 : SOPHIA_COMMIT_KDA;
    const int nm = n_mla - m0 < SOPHIA_COMMIT_MLA ? n_mla - m0 : SOPHIA_COMMIT_MLA;
    CommitArgs a{{cu_nodes, nullptr, rows, kTreeNodes}, path, path_stride, n_path, max_path, slots, n_slots, num_heads,
                 kernel_size, x_dtype, cached, max_seq, rank, latent_dtype, nk, {}, {}};
    for (int l = 0; l < nk; ++l) a.kda[l] = kda[k0 + l];
    for (int l = 0; l < nm; ++l) a.mla[l] = mla[m0 + l];
    const unsigned blocks = static_cast<unsigned>(nk) * num_heads * (kD / kCommitCols) + nm;
    hipLaunchKernelGGL(tree_commit_kernel, dim3(blocks, n_trees), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    k0 += nk;
    m0 += nm;
  }
  return check_launch("tree_commit");
}
