// Logits of the next tokens: penalties, biases and masks on them, and the greedy
// walk along a tree of drafted tokens (include/sophia_draft.h).
//
// Both read every logit once and are bound by that.
//
// Adjust: a work-group takes a tile of the vocabulary for some rows of one
// sequence.  It counts the sequence's history into LDS (integer atomics, whose
// order does not matter), lays the biases of the tile beside the counts, and then
// streams its rows through both.  Tokens of a tree are few and mostly in other
// tiles, so a row's own ones are taken one by one, by the thread that has each.
// 362 rows of 24 trees, 65,536 tokens, bf16, histories of up to 4,000 tokens: 96 MB in
// 29 us (18.6 at the rate of a copy; about a third of a work-group's time is its
// setup); 8 rows in fp32: 4.2 MB in 5.3 us, latency.
//
// Accept: the chosen tokens of all rows in parts, then one wavefront per tree,
// whose lanes are the nodes, joins the parts and walks: a step is one ballot.  1,061
// rows of 64 trees, bf16: 139 MB in 22 us, 6.2 TB/s, and 4 for the walk; 7 rows 3.5
// and 2.4.  Rows off 16 bytes, one logit per lane at a time, are far from that: as many
// rows of 50,257 tokens 86 us with the walk, 1.2 TB/s.
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

// VEC: rows on 16-byte boundaries, a thread has kVec consecutive logits; else every
// 256th.  The same ones in every row: what is done to them stays in registers, and
// kRows rows are in flight together, the first of them while the history is counted.
constexpr int kRows = 4;
constexpr int kWords = 8;

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void adjust_logits_kernel(AdjustArgs a) {
  __shared__ __align__(16) uint32_t s_count[kTileV];
  __shared__ __align__(16) float s_bias[kTileV];
  __shared__ __align__(16) int s_first[kTileV];
  __shared__ int s_again;
  const int t = threadIdx.x, lane = t & 63;
  const int v0 = blockIdx.x * kTileV, seq = blockIdx.z;
  const int width = min(kTileV, a.vocab - v0);
  int64_t base = seq;
  int n = 1;
  if (a.trees.cu) n = tree_nodes(a.trees, seq, base);
  const int first = blockIdx.y * a.rows_per_group, last = min(n, first + a.rows_per_group);
  const int len = a.history ? max(0, min(a.history_len[seq], a.history_max)) : 0;
  const int prompt = a.history && a.prompt_len ? a.prompt_len[seq] : 0;
  const int64_t *hist = a.history + seq * a.history_stride;
  if (first >= last) return;

  // Everything that the setup needs is asked for before the logits, whose masks wait
  // for their numbers.
  int64_t word[kWords];   // tokens of the history, 256 apart
  const auto words = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) word[j] = hist[min(i0 + 256 * j + t, len - 1)] - v0;
  };
  if (len > 0) words(0);
  int64_t id = -1;
  int parent = -1;
  if (a.trees.cu) {
    if (lane < n) id = a.tokens[base + lane] - v0;
    parent = tree_parent(a.trees, base, n, lane);
  }
  const auto place = [&](int j) { return VEC ? kVec * t + j : t + 256 * j; };
  const bool whole = VEC ? kVec * t + kVec <= width : place(kVec - 1) < width;   // (the vocabulary's last logits)
  // Which mask the sequence's row `lane` has, or -1.
  int64_t mask_of = -1;
  if (a.allowed && lane < n) mask_of = a.allowed_rows ? a.allowed_rows[base + lane] : base + lane;
  const int mask_row = mask_of >= 0 && mask_of < a.n_masks ? static_cast<int>(mask_of) : -1;
  float x[kRows][kVec];
  uint32_t bits[kRows];   // of place(j): allowed
  const auto load = [&](int i, float (&r)[kVec], uint32_t &allow) {   // row min(i, last - 1)
    i = min(i, last - 1);
    const int m = __builtin_amdgcn_readlane(mask_row, i);
    allow = 0xffu;
    if (m >= 0) {
      const uint8_t *mask = reinterpret_cast<const uint8_t *>(a.allowed + static_cast<int64_t>(m) * a.mask_words) + v0 / 8;
      if (VEC) {
        allow = kVec * t < width ? mask[t] : 0u;
      } else {
        allow = 0;
#pragma unroll
        for (int j = 0; j < kVec; ++j) allow |= (place(j) < width ? mask[place(j) >> 3] >> (place(j) & 7) & 1u : 0u) << j;
      }
    }
    const int64_t at = (base + i) * a.x_stride + v0;
    if (VEC && whole) {
      const f4 lo = load4(a.x, at + kVec * t, DT), hi = load4(a.x, at + kVec * t + 4, DT);
#pragma unroll
      for (int j = 0; j < kVec; ++j) r[j] = j < 4 ? lo[j & 3] : hi[j & 3];
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) r[j] = place(j) < width ? load_elem(a.x, at + place(j), DT) : 0.f;
    }
  };
#pragma unroll
  for (int r = 0; r < kRows; ++r) load(first + r, x[r], bits[r]);

  // Of node `lane`: its token within this tile or -1, and its path; nodes whose token
  // lies in this tile.
  int tok = -1;
  uint64_t path = 0, in_tile = 0;
  if (a.trees.cu) {
    path = tree_paths(parent, n, lane, [](int, int) {});
    tok = id >= 0 && id < width ? static_cast<int>(id) : -1;
    in_tile = __ballot(tok >= 0);
  }
#pragma unroll
  for (int i = 0; i < kVec; i += 4) {
    *reinterpret_cast<u4 *>(&s_count[kVec * t + i]) = u4{0, 0, 0, 0};
    *reinterpret_cast<f4 *>(&s_bias[kVec * t + i]) = f4{0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<u4 *>(&s_first[kVec * t + i]) = u4{0x7fffffff, 0x7fffffff, 0x7fffffff, 0x7fffffff};
  }
  if (t == 0) s_again = 0;
  lds_barrier();
  for (int i0 = 0; i0 < len; i0 += kWords * 256) {
    if (i0 > 0) words(i0);
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const int i = i0 + 256 * j + t;
      if (i >= len || word[j] < 0 || word[j] >= width) continue;
      if (i < prompt)
        atomicOr(&s_count[word[j]], kSeen);
      else
        atomicAdd(&s_count[word[j]], 1u);
    }
  }
  if (a.bias_ids) {
    // The first entry of an id writes its bias; the others, if there are any, are
    // added in order, by one lane after the other.
    const int64_t *ids = a.bias_ids + static_cast<int64_t>(seq) * a.n_bias;
    const float *b = a.bias + static_cast<int64_t>(seq) * a.n_bias;
    const auto at = [&](int i) {
      const int64_t id = ids[i] - v0;
      return id >= 0 && id < width ? static_cast<int>(id) : -1;
    };
    for (int i = t; i < a.n_bias; i += 256) {
      const int p = at(i);
      if (p >= 0) atomicMin(&s_first[p], i);
    }
    lds_barrier();
    for (int i = t; i < a.n_bias; i += 256) {
      const int p = at(i);
      if (p < 0) continue;
      if (s_first[p] == i)
        s_bias[p] = b[i];
      else
        s_again = 1;
    }
    lds_barrier();
    if (s_again && t < 64)
      for (int i0 = 0; i0 < a.n_bias; i0 += 64) {
        const int i = i0 + lane, p = i < a.n_bias ? at(i) : -1;
        const bool again = p >= 0 && s_first[p] != i;
        const float v = again ? b[i] : 0.f;
        for (uint64_t todo = __ballot(again); todo; todo &= todo - 1)
          if (lane == __ffsll(static_cast<unsigned long long>(todo)) - 1) s_bias[p] += v;
      }
  }
  lds_barrier();
  const float rep = a.repetition ? a.repetition[seq] : 1.f, inv = 1.f / rep;
  const float pres = a.presence ? a.presence[seq] : 0.f;
  const float freq = a.frequency ? a.frequency[seq] : 0.f;
  // y = x f + add: f = 1 / rep or rep (by the sign of x) and add = bias - freq count -
  // pres (count > 0) where the token was seen, else f = 1 and add = bias.
  uint32_t count[kVec];
  float add[kVec];
  const auto addend = [&](uint32_t c, float bias) {
    const uint32_t made = c & ~kSeen;
    return made ? bias - (freq * static_cast<float>(made) + pres) : bias;
  };
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    count[j] = s_count[place(j)];
    add[j] = addend(count[j], s_bias[place(j)]);
  }
  for (int i0 = first; i0 < last; i0 += kRows) {
    if (i0 > first)
#pragma unroll
      for (int r = 0; r < kRows; ++r) load(i0 + r, x[r], bits[r]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = i0 + r;
      if (i >= last) break;
      const int64_t row = base + i;
      float y[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float f = count[j] ? (x[r][j] > 0.f ? inv : rep) : 1.f;
        y[j] = bits[r] >> j & 1 ? fmaf(x[r][j], f, add[j]) : -INFINITY;
      }
      // The tokens of the row's own path in this tile: theirs again, by the thread that has
      // each, with all nodes that have it.
      if (in_tile) {
        const uint64_t mine = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(path >> 32, i))) << 32 |
                              static_cast<uint32_t>(__builtin_amdgcn_readlane(path, i));
        for (uint64_t left = mine & in_tile; left;) {
          const int p = __builtin_amdgcn_readlane(tok, __ffsll(static_cast<unsigned long long>(left)) - 1);
          const uint64_t same = __ballot(tok == p) & mine;
          left &= ~same;
          if ((VEC ? p / kVec : p & 255) == t) {
            const float more = addend(s_count[p] + __popcll(same), s_bias[p]);
#pragma unroll
            for (int j = 0; j < kVec; ++j)
              if (place(j) == p && (bits[r] >> j & 1)) y[j] = fmaf(x[r][j], x[r][j] > 0.f ? inv : rep, more);
          }
        }
      }
      const int64_t at = row * a.y_stride + v0;
      if (VEC && whole) {
        store4(a.y, at + kVec * t, DT, f4{y[0], y[1], y[2], y[3]});
        store4(a.y, at + kVec * t + 4, DT, f4{y[4], y[5], y[6], y[7]});
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (place(j) < width) store_elem(a.y, at + place(j), DT, y[j]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
constexpr int kParts = 8;   // of a row's argmax, at most

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
  int none;                 // what a row without a value above -inf says
};

// The greater logit, of equal ones the lower index (of -inf any: join_parts).
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
  int at = 0x7fffffff;
  const auto see = [&](float v, int i) {
    if (v > best) {      // (never for NaN; indices rise, so an equal one is not lower)
      best = v;
      at = i;
    }
  };
  const auto see_any = [&](float v, int i) {
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };
  if constexpr (VEC) {
    // Four vectors in flight; the ones behind the last whole one are it again.
    const int whole = (v1 - v0) / kVec, end = v0 + kVec * whole;
    for (int i0 = v0 + kVec * t; i0 < end; i0 += 4 * kTileV) {
      f4 lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = min(i0 + kTileV * j, end - kVec);
        lo[j] = load4(a.x, xr + i, DT);
        hi[j] = load4(a.x, xr + i + 4, DT);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = min(i0 + kTileV * j, end - kVec);
#pragma unroll
        for (int c = 0; c < 4; ++c) see(lo[j][c], i + c);
#pragma unroll
        for (int c = 0; c < 4; ++c) see(hi[j][c], i + 4 + c);
      }
    }
    if (t < v1 - end) see_any(load_elem(a.x, xr + end + t, DT), end + t);   // the row's last logits
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
  f2 v[kParts];
#pragma unroll
  for (int p = 0; p < kParts; ++p) v[p] = a.part[row * a.parts + min(p, a.parts - 1)];   // the last one again
#pragma unroll
  for (int p = 0; p < kParts; ++p) better(best, at, v[p].x, __float_as_int(v[p].y));
  return best > -INFINITY ? at : a.none;
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
    if (want < 0) break;
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
// whole tiles each, and no more than the join loads at once.  us with 1,024, 2,048, 4,096
// and 8,192 of them (bf16, with the walk): 1,061 rows of 65,536 logits 34, 31, 30, 29; of
// 32,000 17.1, 16.3, 16.1, 18.7; 362 rows of 65,536 14.4, 14.3, 13.3, 13.3; 64 rows and
// fewer alike.
int argmax_parts(int64_t rows, int vocab) {
  const int64_t tiles = (static_cast<int64_t>(vocab) + kTileV - 1) / kTileV;
  const int64_t want = (4096 + rows - 1) / (rows > 0 ? rows : 1);
  return static_cast<int>(iclamp64(want, 1, imin64(tiles, kParts)));
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
  // Rows of a sequence per work-group: every one of them counts the history again,
  // but fewer than 1,536 of them leave the slow ones (a tile with the tokens that
  // repeat most) behind the others.  us with 768, 1,536 and 2,304: 24 trees of 8 to 24
  // nodes, 65,536 tokens, bf16, 38, 30, 35; 32,000 tokens 22, 24, 23; 8 trees of 24 to 64
  // nodes 41, 38, 39; in fp32, 128,256 tokens, 99, 89, 90; 64 trees of 16 to 24, which
  // have as many without a division, 81, 81, 82.
  const int64_t fill = static_cast<int64_t>(tiles) * n_seqs;
  const int groups = static_cast<int>(iclamp64((1536 + fill - 1) / fill, 1, (a.trees.max_nodes + kRows - 1) / kRows));
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

namespace {
int tree_accept(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab, const int64_t *tokens,
                const int32_t *cu_nodes, const int32_t *parents, int n_trees, int max_nodes, int32_t *path,
                int64_t path_stride, int32_t *n_path, int64_t *next_token, int64_t *chosen, int none, void *workspace,
                size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype_ok(dtype), "tree_accept: dtype not supported");
  SOPHIA_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab >= 1 && vocab <= 1 << 30 && n_trees >= 0 && n_trees <= 65535,
                 "tree_accept: vocab must be 1..2^30, rows >= 0 and n_trees 0..65535");
  SOPHIA_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeNodes && path_stride >= max_nodes,
                 "tree_accept: max_nodes must be in [1, %d] and path rows at least as long", kTreeNodes);
  SOPHIA_REQUIRE(logits_stride >= vocab, "tree_accept: row stride smaller than a row");
  if (n_trees == 0 && rows == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE((rows == 0 || (logits && tokens && parents && chosen)) &&
                     (n_trees == 0 || (cu_nodes && path && n_path && next_token)),
                 "tree_accept: NULL pointer");
  SOPHIA_REQUIRE(rows == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0 &&
                               workspace_bytes >= sophia_tree_accept_workspace_size(rows, vocab)),
                 "tree_accept: workspace too small");
  const int parts = argmax_parts(rows, vocab);
  const int tiles = (vocab + kTileV - 1) / kTileV;
  const int per_part = (tiles + parts - 1) / parts * kTileV;
  AcceptArgs a{{cu_nodes, parents, rows, max_nodes}, logits, logits_stride, vocab, tokens, parts, per_part,
               static_cast<f2 *>(workspace), path, path_stride, n_path, next_token, chosen, none};
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
}  // namespace

extern "C" int sophia_tree_accept(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                                  const int64_t *tokens, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                                  int max_nodes, int32_t *path, int64_t path_stride, int32_t *n_path, int64_t *next_token,
                                  int64_t *chosen, void *workspace, size_t workspace_bytes, void *stream) {
  return tree_accept(logits, logits_stride, dtype, rows, vocab, tokens, cu_nodes, parents, n_trees, max_nodes, path,
                     path_stride, n_path, next_token, chosen, 0, workspace, workspace_bytes, stream);
}

extern "C" int sophia_tree_accept_strict(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                                         const int64_t *tokens, const int32_t *cu_nodes, const int32_t *parents,
                                         int n_trees, int max_nodes, int32_t *path, int64_t path_stride, int32_t *n_path,
                                         int64_t *next_token, int64_t *chosen, void *workspace, size_t workspace_bytes,
                                         void *stream) {
  return tree_accept(logits, logits_stride, dtype, rows, vocab, tokens, cu_nodes, parents, n_trees, max_nodes, path,
                     path_stride, n_path, next_token, chosen, -1, workspace, workspace_bytes, stream);
}
