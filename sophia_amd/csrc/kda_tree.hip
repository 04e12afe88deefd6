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
// One work-group of 8 wavefronts per (tree, head).  A wavefront owns 16 value columns,
// of which its lanes hold S as B operands of v_mfma_f32_16x16x4_f32; loads are asked
// for long before they are used, the state behind the rest, a quarter at a time.  q,
// k, v and the log-decay of a node are then 8 channels in each of 16 threads, in
// registers; the conv's samples, G along the paths, and the operands of the matrix
// products go through LDS.  From the products with S on no wavefront waits for another
// but once: an accumulator holds rows 4 (lane / 16) + i of a 16-row tile, which is a B
// operand whose k index runs 4 (lane / 16) + step, so U goes from one product to the
// next in registers.
//
// Everything is fp32 (the matrix products too): u enters the cached state with
// the accepted path, and the decode step that the state otherwise comes from
// is fp32 as well.  A and B are (K e^G) (K e^-G)^T and (Q e^G) (K e^-G)^T on MFMAs
// where |G| stays below kFactored.  Beyond it e^-G would leave the range of fp32: then
// tile by tile of 16 nodes with a reference near both (K e^(G - R)) (K e^(R - G))^T, and
// tiles whose nodes have lost too different parts for any one reference per pair of a node
// and an ancestor on the vector unit, from e^(G_i - G_j), whose argument is never positive.
//
// What bounds it: the steps' latency.  One tree of 7 nodes takes 13 us (16 heads on
// as many CUs, 25,000 cycles from the first load to the last store), 64 trees of 8 to
// 24 nodes 55 us, two work-groups per CU in two rounds, where their 114 MB take 22 us
// at the rate of a copy; there the matrix pipes are busy 27 % of the time, the
// vector unit 31 and LDS 20.  8 fp32 chains of 17 to 64 nodes take 39 us: half
// the CUs, 72,000 cycles for 64 nodes, of which the products with S, at the fp32 MFMA
// rate, are 20,000.  On the way (us, these three cases): samples gathered from memory tap
// by tap 21, 128, 121; samples through LDS, pairs on the vector unit 23, 83, 59; conv taps
// by distance in LDS, where by channel all 16 threads of a node met in one bank, tiles
// without nodes left out 13, 57, 56; strong decays by tiles in place of pairs (62,000 of
// the slowest head's cycles, 23,000 since) 13, 55, 39.  Not kept: 4 wavefronts of 32
// columns (58 for the second), the solve step by step along shallow paths in place of the
// inverse (58), taps in bf16 (57).
//
// A node with an input that is not finite would reach its siblings through the
// products (0 times infinity): its rows enter them as zeros, and what lies on a
// path with it ends as NaN; where that is its q alone, which no other node reads, its
// own output.
#include <type_traits>

#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_draft.h"

namespace sophia {
namespace {

constexpr int kD = 128;
constexpr int kLd = kD + 4;     // row stride of the LDS matrices: 16 rows 4 banks apart
constexpr int kTape = 3 * kD;   // floats of a node's tape per head
constexpr int kStateParts = 4;  // (all of S at once: 57 us in place of 55 for the 64 trees)

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

// |G| up to which A and B are formed from e^G and e^-G: e^-60 times a component of
// k stays a normal fp32 number down to 1.3e-12.  Each exponential is then off by up to
// 2.6e-6, the rounding of its argument, and a pair's weight by up to 5.3e-6.  That counts
// where a weight is near 1 far down, in a channel that lost e^-50 at one node and little
// since (one that lost it evenly has small weights); the roundings of G itself, 1.9e-6 a
// sum at 60, are in e^(G_i - G_j) too.  With the references below up to 1.3e-5: both
// exponents are up to 80 then, and rounded differences.
constexpr float kFactored = 60.f;
// Beyond it the exponents are G_i - R and R - G_j, R the largest G of i's 16 nodes, so the
// first is never positive.  The second may reach kFar, where e^x is in the range of fp32
// still; past kNear the first must stay in that range too, as e^(G_i - G_j) may then be
// large although e^(G_i - R) is lost (below kNear it is under e^-60).
constexpr float kFar = 80.f, kNear = 20.f;

// Log-decays below this one count as it: e^-104 is 0 in fp32 as theirs is, and a G that
// holds them still tells apart what is added to it (-inf and the lowest float do not).
constexpr float kForgotten = -104.f;

// Eight elements of a row as they lie, and as floats: four from p on and the four 64
// places behind them.  Over 16 threads each half is contiguous, which eight in a row
// per thread are not (two of them then meet in every LDS bank).
constexpr int kHalf = kD / 2;
template <int DT>
struct Raw8 {
  typename std::conditional<DT == SOPHIA_DTYPE_BF16, u2, u4>::type w[2];
};
template <int DT, typename E>
__device__ __forceinline__ Raw8<DT> raw8(const E *p) {
  using V = decltype(Raw8<DT>::w[0] + 0);
  return {{*reinterpret_cast<const V *>(p), *reinterpret_cast<const V *>(p + kHalf)}};
}
template <int DT>
__device__ __forceinline__ void to_float(const Raw8<DT> &r, float (&f)[8]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    if constexpr (DT == SOPHIA_DTYPE_BF16) {
      const uint32_t w = r.w[c >> 2][(c & 3) >> 1];
      f[c] = __uint_as_float(c & 1 ? w & 0xffff0000u : w << 16);
    } else {
      f[c] = __uint_as_float(r.w[c >> 2][c & 3]);
    }
  }
}
__device__ __forceinline__ void read8(const float *p, float (&f)[8]) { to_float(raw8<SOPHIA_DTYPE_F32>(p), f); }
__device__ __forceinline__ void write8(float *p, const float (&f)[8]) {
  reinterpret_cast<f4 *>(p)[0] = f4{f[0], f[1], f[2], f[3]};
  reinterpret_cast<f4 *>(p + kHalf)[0] = f4{f[4], f[5], f[6], f[7]};
}

// LDS of the step: first the rows before the conv, then the matrices.
template <int MT, int DT>
struct StepLds {
  static constexpr int T = 16 * MT, LA = T + 4;
  static constexpr int kRow = 3 * kD + 8;   // elements of a raw row: q | k | v
  using Elem = typename std::conditional<DT == SOPHIA_DTYPE_BF16, uint16_t, float>::type;
  struct Conv {
    float w[4][3 * kD];                     // by the distance of the sample
    Elem x[3 + T][kRow];                    // the history, oldest first, then the nodes
  };
  struct Mat {
    float q[T][kLd], k[T][kLd], g[T][kLd];
    float a[T][LA];                         // -A, its diagonal blocks later (I + A)^-1
    float b[T][LA];
  };
  union {
    Conv conv;
    Mat mat;
  };
};

constexpr int kThreads = 512, kWaves = kThreads / 64;
static_assert(kWaves * 16 == kD, "16 value columns per wavefront");

// MT: tiles of 16 nodes.
template <int MT, int DT>
__global__ __launch_bounds__(kThreads, MT == 4 ? 2 : 4) void kda_tree_step_kernel(TreeStepArgs a) {
  using Lds = StepLds<MT, DT>;
  constexpr int T = Lds::T;
  constexpr int RP = kThreads / 16, P = (T + RP - 1) / RP;    // nodes at a time, and how often
  __shared__ __align__(16) Lds lds;
  __shared__ float s_beta[T];
  __shared__ uint64_t s_path[kTreeNodes];
  __shared__ int s_up[6][kTreeNodes];                   // s_up[0]: parents
  __shared__ int s_bad[kTreeNodes], s_bad_q[kTreeNodes], s_far;
  auto &mat = lds.mat;

  const int h = blockIdx.x, tree = blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  int64_t base;
  const int n = tree_nodes(a.trees, tree, base);
  const int slot = a.slots ? a.slots[tree] : tree;
  if (n == 0) return;
  if (slot < 0 || slot >= a.n_slots) {
    for (int i = t; i < n * kD; i += kThreads) {
      const int64_t row = base + i / kD;
      store_elem(a.o, row * a.o_stride + static_cast<int64_t>(h) * kD + i % kD, DT, 0.f);
      float *tp = a.tape + (row * a.heads + h) * kTape + i % kD;
      tp[0] = tp[kD] = tp[2 * kD] = 0.f;
    }
    return;
  }

  // ---- loads
  const int64_t inner = static_cast<int64_t>(a.heads) * kD;
  const int r0 = t >> 4, seg = 4 * (t & 15);            // this thread's nodes r0 + RP p, channels seg .. + 3, seg + 64 ..
  const int64_t hc = static_cast<int64_t>(h) * kD + seg;
  using Elem = typename Lds::Elem;
  const int parent = tree_parent(a.trees, base, n, lane);
  Raw8<DT> raw[P][3];
  u2 raw_g[P][4];
  const bool g16 = a.g_dtype == SOPHIA_DTYPE_BF16;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int64_t row = base + min(r0 + RP * p, n - 1);
#pragma unroll
    for (int part = 0; part < 3; ++part)
      raw[p][part] = raw8<DT>(static_cast<const Elem *>(a.x[part]) + row * a.x_stride + hc);
    // (of bf16 the first half of what is loaded; no branch around a load)
    const int gsz = g16 ? 2 : 4;
    const uint8_t *gp = static_cast<const uint8_t *>(a.g) + (row * a.g_stride + hc) * gsz;
    raw_g[p][0] = *reinterpret_cast<const u2 *>(gp);
    raw_g[p][1] = *reinterpret_cast<const u2 *>(gp + (g16 ? 0 : 8));
    raw_g[p][2] = *reinterpret_cast<const u2 *>(gp + kHalf * gsz);
    raw_g[p][3] = *reinterpret_cast<const u2 *>(gp + kHalf * gsz + (g16 ? 0 : 8));
  }
  // Taps by distance and history samples of channels t, t + kThreads of the head's 384;
  // those that a shorter conv lacks are zeros.
  constexpr int kCh = (3 * kD + kThreads - 1) / kThreads;
  float taps[kCh][4], past[kCh][3];
  const int hist = a.taps - 1;
#pragma unroll
  for (int j = 0; j < kCh; ++j) {
    const int i = min(t + kThreads * j, 3 * kD - 1);
    const int64_t ch = (i / kD) * inner + static_cast<int64_t>(h) * kD + i % kD;
#pragma unroll
    for (int d = 0; d < 4; ++d) taps[j][d] = d <= hist ? a.conv_w[ch * a.taps + hist - d] : 0.f;
#pragma unroll
    for (int e = 0; e < 3; ++e)
      past[j][e] = e + hist >= 3 ? a.conv_state[(static_cast<int64_t>(slot) * 3 * inner + ch) * hist + e + hist - 3] : 0.f;
  }
  const uint32_t raw_beta = load_raw(a.beta, (base + min(t, n - 1)) * a.beta_stride + h, a.beta_dtype);
  const bool gate = (a.flags & SOPHIA_KDA_GATE_IN_KERNEL) != 0;
  Raw8<SOPHIA_DTYPE_F32> raw_bias = {};
  if (gate) raw_bias = raw8<SOPHIA_DTYPE_F32>(a.dt_bias + hc);
  const float a_log = gate ? a.A_log[h] : 0.f;
  // S rows 16 blk + 4 grp + s of the lane's columns: behind the other loads, whose waits
  // do not include them, and a quarter at a time between the steps below, as a
  // wavefront stands still while the memory queue takes no more.
  float st[kD / 4];
  const int col = 16 * wave + c16;
  const auto load_state = [&](auto part) {
    constexpr int kPer = kD / 4 / kStateParts, i0 = decltype(part)::value * kPer;
    const float *S = a.state + (static_cast<int64_t>(slot) * a.heads + h) * kD * kD + col;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = i0; i < i0 + kPer; ++i)
      st[i] = __builtin_nontemporal_load(S + (16 * (i >> 2) + 4 * grp + (i & 3)) * kD);
    __builtin_amdgcn_sched_barrier(0);
  };
  load_state(std::integral_constant<int, 0>{});
  // ---- paths, and the raw rows into LDS
  if (wave == 0) s_up[0][lane] = parent;
  const uint64_t path = tree_paths(parent, n, lane, [&](int r, int up) {
    if (wave == 0) s_up[r][lane] = up;
  });
  int depth = __popcll(path);
#pragma unroll
  for (int m = 1; m < 64; m *= 2) depth = max(depth, __shfl_xor(depth, m, 64));
  depth = __builtin_amdgcn_readfirstlane(depth);
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (r0 + RP * p < T)
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        using V = decltype(raw[p][part].w[0] + 0);
        Elem *d = &lds.conv.x[3 + r0 + RP * p][part * kD + seg];
        *reinterpret_cast<V *>(d) = raw[p][part].w[0];
        *reinterpret_cast<V *>(d + kHalf) = raw[p][part].w[1];
      }
#pragma unroll
  for (int j = 0; j < kCh; ++j) {
    const int i = t + kThreads * j;
    if (i >= 3 * kD) continue;
#pragma unroll
    for (int d = 0; d < 4; ++d) lds.conv.w[d][i] = taps[j][d];
#pragma unroll
    for (int e = 0; e < 3; ++e) store_elem(lds.conv.x[e], i, DT, past[j][e]);
  }
  if (wave == 0) s_path[lane] = path;
  if (t < kTreeNodes) {
    float b = t < n ? raw_to_f32(raw_beta, a.beta_dtype) : 0.f;
    if (a.flags & SOPHIA_KDA_BETA_SIGMOID) b = sigmoid_f(b);
    const bool ok = is_finite(b);
    if (t < T) s_beta[t] = t < n && ok ? b : 0.f;
    s_bad[t] = !ok;
    s_bad_q[t] = 0;
  }
  if (t == 0) s_far = 0;
  load_state(std::integral_constant<int, 1>{});
  lds_barrier();

  // ---- conv, norms, log-decay: in registers
  // Predecessors, counted from the oldest history sample: 0, 1, 2, then node i as 3 + i.
  // Where a shorter conv has none, the node itself: its tap is 0, and 0 times another
  // node's sample need not be.
  float qkv[3][P][8], g[P][8], bias[8];
  to_float(raw_bias, bias);
  const float head_scale = __expf(a_log);
  auto &q = qkv[0], &k = qkv[1], &v = qkv[2];
  int e[P][4];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int node = r0 + RP * p;
    e[p][0] = 3 + (node < n ? node : 0);
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int at = e[p][d - 1], up = s_up[0][max(at - 3, 0)];
      e[p][d] = d > hist ? e[p][0] : at < 3 ? at - 1 : (up < 0 ? 2 : up + 3);
    }
  }
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    float w[4][8];
#pragma unroll
    for (int d = 0; d < 4; ++d) read8(&lds.conv.w[d][part * kD + seg], w[d]);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float (&y)[8] = qkv[part][p];
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] = 0.f;
      if (r0 + RP * p >= n) continue;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        float s[8];
        to_float(raw8<DT>(&lds.conv.x[e[p][d]][part * kD + seg]), s);
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = fmaf(w[d][c], s[c], y[c]);
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] *= sigmoid_f(y[c]);
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int node = r0 + RP * p;
#pragma unroll
    for (int c = 0; c < 8; ++c) g[p][c] = 0.f;
    if (node >= n) continue;
    float qs = a.scale, ks = 1.f;
    if (a.flags & SOPHIA_KDA_QK_L2NORM) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        sq = fmaf(q[p][c], q[p][c], sq);
        sk = fmaf(k[p][c], k[p][c], sk);
      }
      qs = a.scale / fmaxf(sqrtf(row_sum16(sq)), 1e-12f);
      ks = 1.f / fmaxf(sqrtf(row_sum16(sk)), 1e-12f);
    }
    bool ok = true, ok_q = true;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      q[p][c] *= qs;
      k[p][c] *= ks;
      const uint32_t w = raw_g[p][2 * (c >> 2)][(c & 3) >> 1];
      const float z = g16 ? __uint_as_float(c & 1 ? w & 0xffff0000u : w << 16)
                          : __uint_as_float(raw_g[p][2 * (c >> 2) + ((c & 3) >> 1)][c & 1]);
      g[p][c] = gate ? kda_log_decay(z, head_scale, bias[c], a.lower_bound) : z;
      g[p][c] = g[p][c] < kForgotten ? kForgotten : g[p][c];   // (NaN stays)
      ok &= is_finite(k[p][c]) && is_finite(v[p][c]) && is_finite(g[p][c]);
      ok_q &= is_finite(q[p][c]);
    }
    const auto any16 = [&](bool x) { return ((__ballot(x) >> (lane & 48)) & 0xffff) != 0; };   // (of the node's 16 threads)
    if (any16(!ok)) {
#pragma unroll
      for (int c = 0; c < 8; ++c) k[p][c] = v[p][c] = g[p][c] = 0.f;
      s_bad[node] = 1;
    }
    if (any16(!ok_q)) {
#pragma unroll
      for (int c = 0; c < 8; ++c) q[p][c] = 0.f;
      s_bad_q[node] = 1;
    }
  }
  load_state(std::integral_constant<int, 2>{});
  lds_barrier();

  // ---- G: sums of the log-decay along the paths, by doubling (as many rounds as the
  // deepest path needs), between two buffers
  const auto put_g = [&](float (*buf)[kLd]) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (r0 + RP * p < T) {
        write8(&buf[r0 + RP * p][seg], g[p]);
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) top = fmaxf(top, fabsf(g[p][c]));
        if (top > kFactored) s_far = 1;
      }
  };
  put_g(mat.g);
  load_state(std::integral_constant<int, 3>{});
  lds_barrier();
  for (int r = 0; (1 << r) < depth; ++r) {
    float (*from)[kLd] = r & 1 ? mat.q : mat.g, (*to)[kLd] = r & 1 ? mat.g : mat.q;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int up = r0 + RP * p < T ? s_up[r][r0 + RP * p] : -1;
      if (up >= 0) {
        float add[8];
        read8(&from[up][seg], add);
#pragma unroll
        for (int c = 0; c < 8; ++c) g[p][c] += add[c];
      }
    }
    put_g(to);
    lds_barrier();
  }
  const uint64_t bad = __ballot(s_bad[lane] != 0), bad_q = __ballot(s_bad_q[lane] != 0);
  const bool far = s_far != 0;
  const int mt = MT == 1 ? 1 : (n + 15) >> 4;   // tiles that hold nodes

  // ---- the tape's k and G; the operands
  const auto operands = [&]() {   // Q e^G, K e^G
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int node = r0 + RP * p;
      if (node >= T) continue;
      float qe[8], ke[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float e = __expf(g[p][c]);
        qe[c] = q[p][c] * e;
        ke[c] = k[p][c] * e;
      }
      write8(&mat.q[node][seg], qe);
      write8(&mat.k[node][seg], ke);
    }
  };
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int node = r0 + RP * p;
    if (node >= n) continue;
    const float nan = s_path[node] & bad ? NAN : 0.f;
    float *tp = a.tape + ((base + node) * a.heads + h) * kTape + seg;
    float kt[8], gt[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      kt[c] = k[p][c] + nan;
      gt[c] = g[p][c] + nan;
    }
    write8(tp + kD, kt);
    write8(tp + 2 * kD, gt);
  }
  if (!far) {
    operands();
#pragma unroll
    for (int p = 0; p < P; ++p) {   // K e^-G
      if (r0 + RP * p >= T) continue;
      float ki[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) ki[c] = k[p][c] * __expf(-g[p][c]);
      write8(&mat.g[r0 + RP * p][seg], ki);
    }
    lds_barrier();
    // Units (row tile, column tile, A or B), one wavefront each.
    for (int u = wave; u < mt * (mt + 1); u += kWaves) {
      int ti = 0, tj = u >> 1;
      while (tj > ti) tj -= ++ti;
      const float (*left)[kLd] = u & 1 ? mat.q : mat.k;
      f4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int blk = 0; blk < kD / 16; ++blk) {
        const f4 l = *reinterpret_cast<const f4 *>(&left[16 * ti + c16][16 * blk + 4 * grp]);
        const f4 r = *reinterpret_cast<const f4 *>(&mat.g[16 * tj + c16][16 * blk + 4 * grp]);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc[s & 1] = mfma_f32(l[s], r[s], acc[s & 1]);
      }
      const int j = 16 * tj + c16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * ti + 4 * grp + i;
        const bool on = (s_path[row] >> j) & 1;
        const float x = acc[0][i] + acc[1][i];
        if (u & 1)
          mat.b[row][j] = on ? x : 0.f;
        else
          mat.a[row][j] = on && row != j ? -s_beta[row] * x : 0.f;
      }
    }
    lds_barrier();
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (r0 + RP * p < T) {
        write8(&mat.q[r0 + RP * p][seg], q[p]);
        write8(&mat.k[r0 + RP * p][seg], k[p]);
        write8(&mat.g[r0 + RP * p][seg], g[p]);
      }
    lds_barrier();
    // Tiles (ti, tj) of A and of B, one wavefront each.
    for (int u = wave; u < mt * (mt + 1) / 2; u += kWaves) {
      int ti = 0, tj = u;
      while (tj > ti) tj -= ++ti;
      const uint64_t mine = s_path[16 * ti + c16] >> (16 * tj) & 0xffff;
      bool seen = false;        // node c16 of tile tj is on the path of one of tile ti
#pragma unroll
      for (int i = 0; i < 16; ++i) seen |= (s_path[16 * ti + i] >> (16 * tj + c16)) & 1;
      f4 acc_a = {0.f, 0.f, 0.f, 0.f}, acc_b = acc_a;
      float low = 0.f, high = 0.f;   // of the exponents
      if (__any(mine != 0)) {
#pragma unroll
        for (int blk = 0; blk < kD / 16; ++blk) {
          const int at = 16 * blk + 4 * grp, i = 16 * ti + c16, j = 16 * tj + c16;
          const f4 ki = *reinterpret_cast<const f4 *>(&mat.k[i][at]), qi = *reinterpret_cast<const f4 *>(&mat.q[i][at]);
          const f4 gi = *reinterpret_cast<const f4 *>(&mat.g[i][at]);
          const f4 kj = *reinterpret_cast<const f4 *>(&mat.k[j][at]), gj = *reinterpret_cast<const f4 *>(&mat.g[j][at]);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float r = row_max16(i < n ? gi[s] : -INFINITY);
            const float ei = gi[s] - r, ej = r - gj[s];
            if (i < n) low = fminf(low, ei);
            if (seen) high = fmaxf(high, ej);
            const float e = __expf(ei), right = kj[s] * __expf(ej);
            acc_a = mfma_f32(ki[s] * e, right, acc_a);
            acc_b = mfma_f32(qi[s] * e, right, acc_b);
          }
        }
      }
      const bool in_range = !__any(high > kFar) && !(__any(high > kNear) && __any(low < -kFar));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * ti + 4 * grp + i, j = 16 * tj + c16;
        const bool on = in_range && ((s_path[row] >> j) & 1);
        mat.a[row][j] = on && row != j ? -s_beta[row] * acc_a[i] : 0.f;
        mat.b[row][j] = on ? acc_b[i] : 0.f;
      }
      if (in_range) continue;
      // Pair by pair, 16 lanes each.
      for (int i = 16 * ti; i < min(n, 16 * ti + 16); ++i) {
        uint64_t left = s_path[i] & 0xffffull << 16 * tj;
        float qi[8], ki[8], gi[8];
        read8(&mat.q[i][4 * c16], qi);
        read8(&mat.k[i][4 * c16], ki);
        read8(&mat.g[i][4 * c16], gi);
        while (left) {
          int j = -1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int next = left ? __ffsll(static_cast<unsigned long long>(left)) - 1 : -1;
            if (grp == e) j = next;
            left &= left - 1;   // (0 stays 0)
          }
          float kk = 0.f, qk = 0.f;
          if (j >= 0) {
            float kj[8], gj[8];
            read8(&mat.k[j][4 * c16], kj);
            read8(&mat.g[j][4 * c16], gj);
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
            mat.b[i][j] = qk;
            if (j != i) mat.a[i][j] = -s_beta[i] * kk;
          }
        }
      }
    }
    lds_barrier();
    operands();
    lds_barrier();
  }

  // ---- v to where K e^-G was; one wavefront inverts the unit lower triangular
  // diagonal blocks of I + A, a column per lane; (K e^G) S and (Q e^G) S
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (r0 + RP * p < T) write8(&mat.g[r0 + RP * p][seg], v[p]);
  if (wave == kWaves - 1 && grp < MT) {
    float inv[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = i == c16 ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) x = fmaf(mat.a[16 * grp + i][16 * grp + j], inv[j], x);
      inv[i] = x;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) mat.a[16 * grp + i][16 * grp + c16] = inv[i];
  }
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 u[MT], o[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) u[m] = o[m] = zero;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m >= mt) break;
#pragma unroll
    for (int blk = 0; blk < kD / 16; ++blk) {
      const f4 ak = *reinterpret_cast<const f4 *>(&mat.k[16 * m + c16][16 * blk + 4 * grp]);
      const f4 aq = *reinterpret_cast<const f4 *>(&mat.q[16 * m + c16][16 * blk + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        u[m] = mfma_f32(ak[s], st[4 * blk + s], u[m]);
        o[m] = mfma_f32(aq[s], st[4 * blk + s], o[m]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);   // (reads ahead of their products)
#pragma unroll
    for (int blk = 0; blk < kD / 16; ++blk) {
      __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
      if (blk + 2 < kD / 16) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  }
  lds_barrier();

  // ---- block forward substitution, and the outputs
  const int64_t vc = static_cast<int64_t>(h) * kD + col;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m >= mt) break;
    f4 rhs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int node = 16 * m + 4 * grp + i;
      rhs[i] = s_beta[node] * (mat.g[node][col] - u[m][i]);
    }
#pragma unroll
    for (int p = 0; p < m; ++p) {
      const f4 l = *reinterpret_cast<const f4 *>(&mat.a[16 * m + c16][16 * p + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s) rhs = mfma_f32(l[s], u[p][s], rhs);
    }
    const f4 inv = *reinterpret_cast<const f4 *>(&mat.a[16 * m + c16][16 * m + 4 * grp]);
    u[m] = zero;
#pragma unroll
    for (int s = 0; s < 4; ++s) u[m] = mfma_f32(inv[s], rhs[s], u[m]);
#pragma unroll
    for (int p = 0; p <= m; ++p) {
      const f4 b = *reinterpret_cast<const f4 *>(&mat.b[16 * m + c16][16 * p + 4 * grp]);
#pragma unroll
      for (int s = 0; s < 4; ++s) o[m] = mfma_f32(b[s], u[p][s], o[m]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int node = 16 * m + 4 * grp + i;
      if (node >= n) continue;
      const int64_t row = base + node;
      const float nan = s_path[node] & bad ? NAN : 0.f;
      store_elem(a.o, row * a.o_stride + vc, DT, o[m][i] + ((bad_q >> node) & 1 ? NAN : nan));
      a.tape[(row * a.heads + h) * kTape + col] = u[m][i] + nan;
    }
  }
}

// ---------------------------------------------------------------------------
// Commit: work-group (layer, head, half of the value columns) x tree for the KDA
// layers, (layer) x tree for the MLA layers, all layers in one launch: the few
// trees of a small batch then still fill the chip, and 28 launches become one.
// Bound by the state: 64 KiB read and written per (layer, tree, head), in place,
// as the decode step moves it (thread: 4 columns of every 16th row).  28 layers of 48
// trees: 2.3 GB in 410 us, 5.6 TB/s (a copy of 1 GiB: 5.15); of 4 trees: 192 MB in 38 us.
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
                     aligned(state, 16) && aligned(tape, 16) && aligned(dt_bias, 16),
                 "kda_tree_step: x, g, o, state, tape and dt_bias must be 16-byte aligned");
  const TreeStepArgs a{{cu_nodes, parents, rows, max_nodes}, {x_q, x_k, x_v}, x_row_stride, conv_weight, conv_state,
                       kernel_size, g, g_row_stride, g_dtype, beta, beta_row_stride, beta_dtype, A_log, dt_bias, scale,
                       lower_bound, flags, state, n_slots, slots, num_heads, o, o_row_stride, tape};
  const dim3 grid(num_heads, n_trees);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SOPHIA_TREE_STEP(MT)                                                                            \
  if (x_dtype == SOPHIA_DTYPE_BF16)                                                                     \
    hipLaunchKernelGGL((kda_tree_step_kernel<MT, SOPHIA_DTYPE_BF16>), grid, dim3(kThreads), 0, st, a);        \
  else                                                                                                  \
    hipLaunchKernelGGL((kda_tree_step_kernel<MT, SOPHIA_DTYPE_F32>), grid, dim3(kThreads), 0, st, a);
  // By the bound on a tree's nodes: the least that holds it has the least LDS and registers,
  // so more of its work-groups run together.  us, 16 heads, bf16: 64 trees of 32 nodes 62 as
  // 32, 86 as 64; 64 of 8 nodes 38 as 16 or 32, 59 as 64; 8 of 16 nodes 17 as any.
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
  return sophia_tree_commit_within(path, path_stride, n_path, max_path, cu_nodes, n_trees, rows, kTreeNodes, slots, n_slots,
                                   kda, n_kda, num_heads, head_dim, kernel_size, x_dtype, mla, n_mla, cached, max_seq, rank,
                                   latent_dtype, stream);
}

extern "C" int sophia_tree_commit_within(const int32_t *path, int64_t path_stride, const int32_t *n_path, int max_path,
                                         const int32_t *cu_nodes, int n_trees, int64_t rows, int max_nodes,
                                         const int32_t *slots, int n_slots, const sophia_commit_kda *kda, int n_kda,
                                         int num_heads, int head_dim, int kernel_size, int x_dtype,
                                         const sophia_commit_mla *mla, int n_mla, const int64_t *cached, int max_seq,
                                         int rank, int latent_dtype, void *stream) {
  SOPHIA_REQUIRE(n_trees >= 0 && n_trees <= 65535 && rows >= 0 && n_slots >= 0 && n_kda >= 0 && n_mla >= 0,
                 "tree_commit: n_trees must be 0..65535, rows, n_slots and layer counts >= 0");
  SOPHIA_REQUIRE(max_path >= 1 && max_path <= kTreeNodes && path_stride >= max_path,
                 "tree_commit: max_path must be in [1, %d] and path rows at least as long", kTreeNodes);
  SOPHIA_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeNodes, "tree_commit: max_nodes must be in [1, %d]", kTreeNodes);
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
    CommitArgs a{{cu_nodes, nullptr, rows, max_nodes}, path, path_stride, n_path, max_path, slots, n_slots, num_heads,
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
