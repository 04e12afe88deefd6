// Logits of the next tokens: penalties, biases and masks on them, and the greedy
// walk along a tree of drafted tokens (include/sophia_draft.h).
//
// Both read every logit once and are bound by that.
//
// Adjust: a work-group takes a tile of the vocabulary for some rows of one
// sequence.  It counts the sequence's history into LDS (integer atomics, whose
// order does not matter), lays the biases of the tile beside the counts, and then
// streams its rows through both.  Tokens of a tree are few and mostly in other
// tiles, so a row's ancestors are compared one by one.
//
// Accept: the chosen tokens of all rows in parts, then one wavefront per tree,
// whose lanes are the nodes, joins the parts and walks: a step is one ballot.
#include "common.hpp"
#include "tree.hpp"

#include "../../include/sophia_draft.h"

namespace sophia {
namespace {

constexpr int kVec = 8;                 // consecutive logits per thread and step
constexpr int kTileV = 256 * kVec;      // vocabulary per work-group

struct AdjustArgs {
  Trees trees;              // cu NULL: row r is sequence r
  const int64_t *tokens;    // of the trees' nodes
  const void *x;
  int64_t x_stride;
  void *y;
  int64_t y_stride;
  int64_t rows;
  int vocab;
  const int64_t *history;   // NULL: none
  int64_t history_stride;
  const int32_t *history_len, *prompt_len;
  int history_max;
  const float *repetition, *presence, *frequency;
  const int64_t *bias_ids;  // NULL: none
  const float *bias;
  int n_bias;
  const int32_t *allowed;   // NULL: none
  const int32_t *allowed_rows;
  int n_masks, mask_words;
  int rows_per_group;
};

// The generated count of a token, and whether it was seen at all (bit 31).
constexpr uint32_t kSeen = 0x80000000u;

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void adjust_logits_kernel(AdjustArgs a) {
  __shared__ __align__(16) uint32_t s_count[kTileV];
  __shared__ __align__(16) float s_bias[kTileV];
  __shared__ int s_tok[kTreeNodes];
  __shared__ uint64_t s_path[kTreeNodes];
  const int t = threadIdx.x, lane = t & 63;
  const int v0 = blockIdx.x * kTileV, seq = blockIdx.z;
  const int width = min(kTileV, a.vocab - v0);
  int64_t base = seq;
  int n = 1;
  uint64_t in_tile = 0;   // nodes whose token lies in this tile
  if (a.trees.cu) n = tree_nodes(a.trees, seq, base);
  const int first = blockIdx.y * a.rows_per_group, last = min(n, first + a.rows_per_group);
  if (first >= last) return;
  if (a.trees.cu) {
    const uint64_t path = tree_paths(tree_parent(a.trees, base, n, lane), n, lane, [](int, int) {});
    const int64_t tok = lane < n ? a.tokens[base + lane] - v0 : -1;
    in_tile = __ballot(tok >= 0 && tok < width);
    if (t < 64) {
      s_path[lane] = path;
      s_tok[lane] = tok >= 0 && tok < width ? static_cast<int>(tok) : -1;
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; i += 4) {
    *reinterpret_cast<u4 *>(&s_count[kVec * t + i]) = u4{0, 0, 0, 0};
    *reinterpret_cast<f4 *>(&s_bias[kVec * t + i]) = f4{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  if (a.history) {
    const int len = max(0, min(a.history_len[seq], a.history_max));
    const int prompt = a.prompt_len ? a.prompt_len[seq] : 0;
    const int64_t *h = a.history + seq * a.history_stride;
    for (int i = t; i < len; i += 256) {
      const int64_t tok = h[i] - v0;
      if (tok < 0 || tok >= width) continue;
      if (i < prompt)
        atomicOr(&s_count[tok], kSeen);
      else
        atomicAdd(&s_count[tok], 1u);
    }
  }
  if (a.bias_ids) {
    // An id given more than once: its first entry adds all of them, in order.
    const int64_t *ids = a.bias_ids + static_cast<int64_t>(seq) * a.n_bias;
    const float *b = a.bias + static_cast<int64_t>(seq) * a.n_bias;
    for (int i = t; i < a.n_bias; i += 256) {
      const int64_t id = ids[i];
      if (id < v0 || id >= v0 + width) continue;
      bool again = false;
      for (int j = 0; j < i && !again; ++j) again = ids[j] == id;
      if (again) continue;
      float sum = b[i];
      for (int j = i + 1; j < a.n_bias; ++j)
        if (ids[j] == id) sum += b[j];
      s_bias[id - v0] = sum;
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[seq] : 1.f, inv = 1.f / rep;
  const float pres = a.presence ? a.presence[seq] : 0.f;
  const float freq = a.frequency ? a.frequency[seq] : 0.f;
  // y = x (/ or *) rep - freq count - pres (count > 0) + bias, -inf where not allowed
  const auto one = [&](float x, uint32_t c, float b, bool allowed) {
    const uint32_t count = c & ~kSeen;
    float y = x * (x > 0.f ? inv : rep);
    y -= freq * static_cast<float>(count);
    y -= count ? pres : 0.f;
    return allowed ? (c ? y : x) + b : -INFINITY;
  };
  for (int i = first; i < last; ++i) {
    const int64_t row = base + i;
    const int64_t xr = row * a.x_stride + v0, yr = row * a.y_stride + v0;
    uint64_t extra = a.trees.cu ? s_path[i] & in_tile : 0;
    const uint8_t *mask = nullptr;
    if (a.allowed) {
      const int64_t m = a.allowed_rows ? a.allowed_rows[row] : row;
      if (m >= 0 && m < a.n_masks) mask = reinterpret_cast<const uint8_t *>(a.allowed + m * a.mask_words) + v0 / 8;
    }
    const auto count_of = [&](int at) {
      uint32_t c = s_count[at];
      for (uint64_t e = extra; e; e &= e - 1)
        c += s_tok[__ffsll(static_cast<unsigned long long>(e)) - 1] == at;
      return c;
    };
    if (VEC && kVec * t + kVec <= width) {
      const int at = kVec * t;
      f4 x[2] = {load4(a.x, xr + at, DT), load4(a.x, xr + at + 4, DT)};
      const unsigned bits = mask ? mask[t] : 0xffu;
#pragma unroll
      for (int c = 0; c < kVec; ++c) x[c >> 2][c & 3] = one(x[c >> 2][c & 3], count_of(at + c), s_bias[at + c], bits >> c & 1);
      store4(a.y, yr + at, DT, x[0]);
      store4(a.y, yr + at + 4, DT, x[1]);
    } else if (!VEC) {
      for (int at = t; at < width; at += 256)
        store_elem(a.y, yr + at, DT, one(load_elem(a.x, xr + at, DT), count_of(at), s_bias[at],
                                         mask ? mask[at >> 3] >> (at & 7) & 1 : true));
    } else {
      for (int at = kVec * t; at < width; ++at)   // the vocabulary's last logits
        store_elem(a.y, yr + at, DT, one(load_elem(a.x, xr + at, DT), count_of(at), s_bias[at],
                                         mask ? mask[at >> 3] >> (at & 7) & 1 : true));
    }
  }
}

// ---------------------------------------------------------------------------
struct AcceptArgs {
  Trees trees;
  const void *x;
  int64_t x_stride;
  int vocab;
  const int64_t *tokens;
  int parts, per_part;      // logits per part, a multiple of kTileV
  f2 *part;                 // [rows, parts]: greatest logit, its index as bits
  int32_t *path;
  int64_t path_stride;
  int32_t *n_path;
  int64_t *next, *chosen;
};

// The greater logit, of equal ones the lower index.
__device__ __forceinline__ void better(float &v, int &i, float v2, int i2) {
  const bool take = v2 > v || (v2 == v && i2 < i);
  v = take ? v2 : v;
  i = take ? i2 : i;
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void argmax_part_kernel(AcceptArgs a) {
  __shared__ float s_v[4];
  __shared__ int s_i[4];
  const int64_t row = blockIdx.y;
  const int t = threadIdx.x, part = blockIdx.x;
  const int v0 = part * a.per_part, v1 = min(a.vocab, v0 + a.per_part);
  const int64_t xr = row * a.x_stride;
  float best = -INFINITY;
  int at = 0x7fffffff;   // nothing above -inf
  const auto see = [&](float v, int i) {
    if (v > best) {      // (never for NaN; indices rise, so an equal one is not lower)
      best = v;
      at = i;
    }
  };
  if constexpr (VEC) {
    int i = v0 + kVec * t;
    for (; i + kVec <= v1; i += kTileV) {
      const f4 lo = load4(a.x, xr + i, DT), hi = load4(a.x, xr + i + 4, DT);
#pragma unroll
      for (int c = 0; c < 4; ++c) see(lo[c], i + c);
#pragma unroll
      for (int c = 0; c < 4; ++c) see(hi[c], i + 4 + c);
    }
    for (; i < v1; ++i) see(load_elem(a.x, xr + i, DT), i);   // the row's last logits, one thread's
  } else {
    for (int i = v0 + t; i < v1; i += 256) see(load_elem(a.x, xr + i, DT), i);
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) better(best, at, __shfl_xor(best, m, 64), __shfl_xor(at, m, 64));
  if ((t & 63) == 0) {
    s_v[t >> 6] = best;
    s_i[t >> 6] = at;
  }
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < 4; ++w) better(best, at, s_v[w], s_i[w]);
    a.part[row * a.parts + part] = f2{best, __int_as_float(at)};
  }
}

// A row's choice from its parts.
__device__ __forceinline__ int join_parts(const AcceptArgs &a, int64_t row) {
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int p = 0; p < a.parts; ++p) {
    const f2 v = a.part[row * a.parts + p];
    better(best, at, v.x, __float_as_int(v.y));
  }
  return at == 0x7fffffff ? 0 : at;
}

// Work-group per tree (the walk), then one per 64 rows (`chosen`, of all rows).
__global__ __launch_bounds__(64) void tree_walk_kernel(AcceptArgs a, int n_trees) {
  const int tree = blockIdx.x, lane = threadIdx.x;
  if (tree >= n_trees) {
    const int64_t row = static_cast<int64_t>(tree - n_trees) * 64 + lane;
    if (row < a.trees.rows) a.chosen[row] = join_parts(a, row);
    return;
  }
  int64_t base;
  const int n = tree_nodes(a.trees, tree, base);
  const int at = lane < n ? join_parts(a, base + lane) : 0;
  const int parent = tree_parent(a.trees, base, n, lane);
  const int64_t token = lane < n ? a.tokens[base + lane] : -1;
  int cur = 0, len = n > 0 ? 1 : 0, mine = n > 0 && lane == 0 ? 0 : -1;   // mine: path entry `lane`
  while (len > 0) {   // (a child is a later node: at most n steps)
    const int want = __shfl(at, cur, 64);
    const uint64_t next = __ballot(lane < n && parent == cur && token == want);
    if (next == 0) break;
    cur = __ffsll(static_cast<unsigned long long>(next)) - 1;
    if (lane == len) mine = cur;
    ++len;
  }
  if (lane < a.trees.max_nodes) a.path[tree * a.path_stride + lane] = mine;
  const int last = __shfl(at, cur, 64);
  if (lane == 0) {
    a.n_path[tree] = len;
    a.next[tree] = n > 0 ? last : -1;
  }
}

bool dtype_ok(int dtype) { return dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Parts of a row's argmax: enough work-groups to fill the chip several times,
// whole tiles each.
int argmax_parts(int64_t rows, int vocab) {
  const int64_t tiles = (static_cast<int64_t>(vocab) + kTileV - 1) / kTileV;
  const int64_t want = (4096 + rows - 1) / (rows > 0 ? rows : 1);
  return static_cast<int>(iclamp64(want, 1, tiles));
}

}  // namespace
}  // namespace sophia

using namespace sophia;

extern "C" int sophia_adjust_logits(const void *logits, int64_t logits_stride, void *out, int64_t out_stride, int dtype,
                                    int64_t rows, int vocab, const int64_t *history, int64_t history_stride,
                                    const int32_t *history_len, const int32_t *prompt_len, int history_max,
                                    const float *repetition, const float *presence, const float *frequency,
                                    const int64_t *bias_ids, const float *bias, int n_bias, const int32_t *allowed,
                                    int n_masks, const int32_t *allowed_rows, const int32_t *cu_nodes,
                                    const int32_t *parents, const int64_t *tokens, int n_seqs, int max_nodes,
                                    void *stream) {
  SOPHIA_REQUIRE(dtype_ok(dtype), "adjust_logits: dtype not supported");
  SOPHIA_REQUIRE(rows >= 0 && vocab >= 0 && vocab <= 1 << 30 && n_seqs >= 0 && n_seqs <= 65535,
                 "adjust_logits: n_seqs must be 0..65535, rows >= 0 and vocab 0..2^30");
  SOPHIA_REQUIRE(cu_nodes ? (max_nodes >= 1 && max_nodes <= kTreeNodes) : n_seqs == rows,
                 "adjust_logits: trees need max_nodes in [1, %d]; without them a row is a sequence", kTreeNodes);
  SOPHIA_REQUIRE(logits_stride >= vocab && out_stride >= vocab, "adjust_logits: row stride smaller than a row");
  SOPHIA_REQUIRE(history_max >= 0 && history_stride >= history_max && n_bias >= 0 && n_masks >= 0,
                 "adjust_logits: history rows must hold history_max tokens, counts be >= 0");
  if (rows == 0 || vocab == 0 || n_seqs == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(logits && out, "adjust_logits: NULL pointer");
  SOPHIA_REQUIRE(!cu_nodes || (parents && tokens), "adjust_logits: trees need parents and tokens");
  SOPHIA_REQUIRE(!history || history_len, "adjust_logits: history needs history_len");
  SOPHIA_REQUIRE(n_bias == 0 || (bias_ids && bias), "adjust_logits: biases need ids and values");
  SOPHIA_REQUIRE(!allowed || allowed_rows || n_masks == rows, "adjust_logits: a mask per row, or allowed_rows");
  const int tiles = (vocab + kTileV - 1) / kTileV;
  AdjustArgs a{{cu_nodes, parents, rows, cu_nodes ? max_nodes : 1}, tokens, logits, logits_stride, out, out_stride, rows,
               vocab, history, history_stride, history_len, prompt_len, history_max, repetition, presence, frequency,
               n_bias ? bias_ids : nullptr, bias, n_bias, allowed, allowed_rows, n_masks, (vocab + 31) / 32, 0};
  // Rows of a sequence per work-group: all of them once there are 2,048 work-groups.
  const int64_t fill = static_cast<int64_t>(tiles) * n_seqs;
  const int groups = static_cast<int>(iclamp64((2048 + fill - 1) / fill, 1, (a.trees.max_nodes + 3) / 4));
  a.rows_per_group = (a.trees.max_nodes + groups - 1) / groups;
  const dim3 grid(tiles, groups, n_seqs);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool vec = logits_stride % 8 == 0 && out_stride % 8 == 0 && aligned16(logits) && aligned16(out);
  if (dtype == SOPHIA_DTYPE_BF16) {
    if (vec)
      hipLaunchKernelGGL((adjust_logits_kernel<SOPHIA_DTYPE_BF16, true>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((adjust_logits_kernel<SOPHIA_DTYPE_BF16, false>), grid, dim3(256), 0, st, a);
  } else {
    if (vec)
      hipLaunchKernelGGL((adjust_logits_kernel<SOPHIA_DTYPE_F32, true>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((adjust_logits_kernel<SOPHIA_DTYPE_F32, false>), grid, dim3(256), 0, st, a);
  }
  return check_launch("adjust_logits");
}

extern "C" size_t sophia_tree_accept_workspace_size(int64_t rows, int vocab) {
  if (rows < 0 || vocab < 0) return 0;
  return static_cast<size_t>(rows) * argmax_parts(rows, vocab) * sizeof(f2);
}

extern "C" int sophia_tree_accept(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                                  const int64_t *tokens, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                                  int max_nodes, int32_t *path, int64_t path_stride, int32_t *n_path, int64_t *next_token,
                                  int64_t *chosen, void *workspace, size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype_ok(dtype), "tree_accept: dtype not supported");
  SOPHIA_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab >= 1 && vocab <= 1 << 30 && n_trees >= 0 && n_trees <= 65535,
                 "tree_accept: vocab must be 1..2^30, rows >= 0 and n_trees 0..65535");
  SOPHIA_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeNodes && path_stride >= max_nodes,
                 "tree_accept: max_nodes must be in [1, %d] and path rows at least as long", kTreeNodes);
  SOPHIA_REQUIRE(logits_stride >= vocab, "tree_accept: row stride smaller than a row");
  if (n_trees == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE((rows == 0 || (logits && tokens && parents && chosen)) && cu_nodes && path && n_path && next_token,
                 "tree_accept: NULL pointer");
  SOPHIA_REQUIRE(rows == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0 &&
                               workspace_bytes >= sophia_tree_accept_workspace_size(rows, vocab)),
                 "tree_accept: workspace too small");
  const int parts = argmax_parts(rows, vocab);
  const int tiles = (vocab + kTileV - 1) / kTileV;
  const int per_part = (tiles + parts - 1) / parts * kTileV;
  AcceptArgs a{{cu_nodes, parents, rows, max_nodes}, logits, logits_stride, vocab, tokens, parts, per_part,
               static_cast<f2 *>(workspace), path, path_stride, n_path, next_token, chosen};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool vec = logits_stride % 8 == 0 && aligned16(logits);
  // rows beyond the grid's y limit in further launches
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
    AcceptArgs p = a;
    const int esz = dtype == SOPHIA_DTYPE_BF16 ? 2 : 4;
    p.x = static_cast<const uint8_t *>(logits) + r0 * logits_stride * esz;
    p.part = a.part + r0 * parts;
    const dim3 grid(parts, static_cast<unsigned>(imin64(65535, rows - r0)));
    if (dtype == SOPHIA_DTYPE_BF16) {
      if (vec)
        hipLaunchKernelGGL((argmax_part_kernel<SOPHIA_DTYPE_BF16, true>), grid, dim3(256), 0, st, p);
      else
        hipLaunchKernelGGL((argmax_part_kernel<SOPHIA_DTYPE_BF16, false>), grid, dim3(256), 0, st, p);
    } else {
      if (vec)
        hipLaunchKernelGGL((argmax_part_kernel<SOPHIA_DTYPE_F32, true>), grid, dim3(256), 0, st, p);
      else
        hipLaunchKernelGGL((argmax_part_kernel<SOPHIA_DTYPE_F32, false>), grid, dim3(256), 0, st, p);
    }
  }
  const int64_t blocks = n_trees + (rows + 63) / 64;
  hipLaunchKernelGGL(tree_walk_kernel, dim3(static_cast<unsigned>(blocks)), dim3(64), 0, st, a, n_trees);
  return check_launch("tree_accept");
}
