// Moves of cache slots and pages in place, as if all at once (include/sophia_pages.h).
//
// dst[i] <- src[i] for all i: a slot may be read by several moves and is written by at most
// one.  A move that reads a slot has to come before the one that writes it; each move has at
// most one such successor, so the moves are trees that end in one last move, or in a cycle, of
// which one slot's content is held in registers.  A first kernel (one work-group) finds the
// trees and orders each; in the second a thread has the same 16 bytes of every slot of some
// trees and moves them in that order, so nothing is copied twice and no thread waits for another.
// Moved bytes are read once and written once.
#include "common.hpp"

#include "../../include/sophia_pages.h"

namespace sophia {
namespace {

constexpr int kMoves = SOPHIA_MOVES;
constexpr int kPlanThreads = 1024;
constexpr int kHash = 2 * kMoves;

// A planned move.
struct Move {
  int32_t src, dst;         // slots, or pages
  int32_t flags;            // of its place in its tree
  int32_t tokens;           // taken along (a fork)
  int32_t src_page, dst_page;   // of the page that these fill in part (-1: none)
  int32_t held_tokens, held_page;   // kSave: the tokens and the source's page of the move at the end
};
constexpr int kFirst = 1;      // the first of its tree
constexpr int kSave = 2;       // what is in dst before is read at the end of the tree: held
constexpr int kFromSaved = 4;  // its source is what was held
static_assert(sizeof(Move) == 32, "two loads");

struct PlanArgs {
  const int32_t *src, *dst;
  int n;
  int64_t limit;            // slots, or pages
  const int64_t *cached;    // NULL: pages
  const int32_t *table;     // NULL: none
  int64_t table_stride;
  int max_pages, shift;
  int64_t n_pages;
  int32_t *count;
  Move *moves;
};

__global__ __launch_bounds__(kPlanThreads) void move_plan_kernel(PlanArgs a) {
  __shared__ int s_src[kMoves], s_dst[kMoves];
  // By slot: the last move that writes it.  Later the places of the trees' roots.
  __shared__ int s_key[kHash], s_by[kHash];
  __shared__ short s_next[kMoves], s_level[kMoves];   // the move that has to wait for this one; steps from the leaves
  __shared__ int s_readers[kMoves];                   // moves that have to come before
  __shared__ short s_end[kMoves];                     // of a cycle's first move: its last one
  __shared__ int s_left, s_total;
  const int t = threadIdx.x, n = a.n;
  for (int i = t; i < kHash; i += kPlanThreads) {
    s_key[i] = -1;
    s_by[i] = -1;
  }
  for (int i = t; i < n; i += kPlanThreads) {
    const int s = a.src[i], d = a.dst[i];
    const bool ok = s >= 0 && s < a.limit && d >= 0 && d < a.limit;
    s_src[i] = s;
    s_dst[i] = ok ? d : -1;
    s_next[i] = -1;
    s_level[i] = -1;
    s_readers[i] = 0;
  }
  if (t == 0) s_total = 0;
  __syncthreads();
  const auto hash = [](int slot) { return (static_cast<unsigned>(slot) * 2654435761u) >> (32 - 13); };
  static_assert(kHash == 1 << 13, "the hash's bits");
  for (int i = t; i < n; i += kPlanThreads) {
    if (s_dst[i] < 0) continue;
    unsigned h = hash(s_dst[i]);      // (half of the places stay free)
    for (;; h = (h + 1) & (kHash - 1)) {
      const int was = atomicCAS(&s_key[h], -1, s_dst[i]);
      if (was == -1 || was == s_dst[i]) break;
    }
    atomicMax(&s_by[h], i);
  }
  __syncthreads();
  const auto writer = [&](int slot) {
    for (unsigned h = hash(slot);; h = (h + 1) & (kHash - 1)) {
      if (s_key[h] == slot) return s_by[h];
      if (s_key[h] == -1) return -1;
    }
  };
  // What counts: the last move to a slot, if it changes it.
  for (int i = t; i < n; i += kPlanThreads) {
    const int d = s_dst[i];
    s_level[i] = d >= 0 && writer(d) == i && s_src[i] != d ? 0 : -1;
  }
  __syncthreads();
  for (int i = t; i < n; i += kPlanThreads) {
    if (s_level[i] < 0) continue;
    atomicAdd(&s_total, 1);
    const int next = writer(s_src[i]);
    if (next >= 0 && s_level[next] >= 0) {
      s_next[i] = static_cast<short>(next);
      atomicAdd(&s_readers[next], 1);
    }
  }
  __syncthreads();
  // Levels: a move comes after all that read its slot.  s_readers < 0: done.
  int level = 1;
  for (;; ++level) {
    if (t == 0) s_left = 0;
    __syncthreads();
    bool ready[kMoves / kPlanThreads];
#pragma unroll
    for (int k = 0; k < kMoves / kPlanThreads; ++k) {
      const int i = t + k * kPlanThreads;
      ready[k] = i < n && s_level[i] == 0 && s_readers[i] == 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMoves / kPlanThreads; ++k) {
      const int i = t + k * kPlanThreads;
      if (!ready[k]) continue;
      s_level[i] = static_cast<short>(level);
      s_left = 1;
      if (s_next[i] >= 0) atomicSub(&s_readers[s_next[i]], 1);
    }
    __syncthreads();
    if (s_left == 0) break;
    __syncthreads();
  }
  // What is left are cycles.  Each begins at its lowest move, whose slot's content is held, and
  // ends with the move that reads that slot, which waits for nobody any more.
  for (int i = t; i < n; i += kPlanThreads) s_readers[i] = 0;   // (now: the flags)
  __syncthreads();
  for (int i = t; i < n; i += kPlanThreads) {
    if (s_level[i] != 0) continue;
    bool lowest = true;
    for (int j = s_next[i]; j != i && lowest; j = s_next[j]) lowest = j > i;
    if (lowest) s_readers[i] = kSave;
  }
  __syncthreads();
  for (int i = t; i < n; i += kPlanThreads) {
    if (!(s_readers[i] & kSave)) continue;
    int at = level, j = i;
    for (;;) {
      const int next = s_next[j];
      s_level[j] = static_cast<short>(at++);
      if (next == i) break;
      j = next;
    }
    s_readers[j] |= kFromSaved;
    s_next[j] = -1;
    s_end[i] = static_cast<short>(j);
  }
  __syncthreads();
  // Each move's root, the last of its tree, by doubling; then the order: by root, then by level.
  short *s_root = reinterpret_cast<short *>(s_by);
  for (int i = t; i < n; i += kPlanThreads) s_root[i] = s_next[i] >= 0 ? s_next[i] : static_cast<short>(i);
  __syncthreads();
  for (int reach = 1; reach < n; reach *= 2) {
    short up[kMoves / kPlanThreads];
#pragma unroll
    for (int k = 0; k < kMoves / kPlanThreads; ++k) {
      const int i = t + k * kPlanThreads;
      if (i < n) up[k] = s_root[s_root[i]];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMoves / kPlanThreads; ++k) {
      const int i = t + k * kPlanThreads;
      if (i < n) s_root[i] = up[k];
    }
    __syncthreads();
  }
  const int total = s_total;
  // A key per move (root, level, move: 13 bits each; what does not count behind), sorted in place by
  // exchanges.  They lie where the hash was.
  int size = 1;
  while (size < n) size *= 2;
  uint64_t key[kMoves / kPlanThreads];
#pragma unroll
  for (int k = 0; k < kMoves / kPlanThreads; ++k) {
    const int i = t + k * kPlanThreads;
    key[k] = i < n && s_level[i] > 0
                 ? static_cast<uint64_t>(s_root[i]) << 32 | static_cast<uint64_t>(s_level[i]) << 16 | static_cast<uint64_t>(i)
                 : ~0ull;
  }
  __syncthreads();
  uint64_t *s_sort = reinterpret_cast<uint64_t *>(s_key);
  static_assert(sizeof(s_key) >= sizeof(uint64_t) * kMoves, "the keys fit");
#pragma unroll
  for (int k = 0; k < kMoves / kPlanThreads; ++k)
    if (t + k * kPlanThreads < size) s_sort[t + k * kPlanThreads] = key[k];
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int gap = run / 2; gap > 0; gap /= 2) {
      for (int p = t; p < size / 2; p += kPlanThreads) {
        const int lo = (p / gap) * 2 * gap + p % gap, hi = lo + gap;
        const bool up = (lo & run) == 0;
        const uint64_t x = s_sort[lo], y = s_sort[hi];
        if ((x > y) == up) {
          s_sort[lo] = y;
          s_sort[hi] = x;
        }
      }
      __syncthreads();
    }
  for (int p = t; p < total; p += kPlanThreads) {
    const uint64_t k = s_sort[p];
    const int i = static_cast<int>(k & 0xffff), root = static_cast<int>(k >> 32);
    Move m = {};
    m.src = s_src[i];
    m.dst = s_dst[i];
    m.flags = s_readers[i] | (p == 0 || static_cast<int>(s_sort[p - 1] >> 32) != root ? kFirst : 0);
    m.src_page = m.dst_page = m.held_page = -1;
    const auto tokens = [&](int move) { return a.cached ? static_cast<int>(iclamp64(a.cached[move], 0, 1 << 30)) : 0; };
    const auto page = [&](int slot, int count) {
      const int full = count >> a.shift;
      const int id = a.table && full < a.max_pages ? a.table[slot * a.table_stride + full] : -1;
      return id >= 0 && id < a.n_pages ? id : -1;
    };
    m.tokens = tokens(i);
    m.src_page = page(m.src, m.tokens);
    m.dst_page = page(m.dst, m.tokens);
    if (m.flags & kSave) {
      const int end = s_end[i];
      m.held_tokens = tokens(end);
      m.held_page = page(s_src[end], m.held_tokens);
    }
    a.moves[p] = m;
  }
  if (t == 0) *a.count = total;
}

// ---- the moves --------------------------------------------------------------------
enum Kind { kWhole, kLatents, kPageTail, kTable };
constexpr int kTensors = 2 * SOPHIA_FORK_KDA + 2 * SOPHIA_FORK_MLA + 1;
constexpr int kParts = 5;

struct Part {
  int kind, first, tensors;  // in `base`
  int chunks;                // work-groups per tensor
  int64_t stride, bytes;     // from slot (page) to slot, and of one
  int token_bytes;           // of a token (kLatents, kPageTail)
};

struct MoveArgs {
  const int32_t *count;
  const Move *moves;
  int shift;                 // of the pages
  int n_parts;
  int workers;               // that share the trees
  Part part[kParts];
  char *base[kTensors];
};
static_assert(sizeof(MoveArgs) <= 4000, "kernel arguments");

constexpr int kMoveThreads = 256, kChunk = 16 * kMoveThreads, kBatch = 8;

__global__ __launch_bounds__(kMoveThreads) void move_kernel(MoveArgs a) {
  int block = blockIdx.x, q = 0;
  while (q + 1 < a.n_parts && block >= a.part[q].tensors * a.part[q].chunks) {
    block -= a.part[q].tensors * a.part[q].chunks;
    ++q;
  }
  const Part p = a.part[q];
  char *base = a.base[p.first + block / p.chunks];
  const int64_t off = static_cast<int64_t>(block % p.chunks) * kChunk + 16 * threadIdx.x;
  const int total = *a.count;
  // This worker's trees: those that begin in its share of the list.
  const auto begin = [&](int w) {
    int at = static_cast<int>(static_cast<int64_t>(total) * w / a.workers);
    while (at < total && !(a.moves[at].flags & kFirst)) ++at;
    return at;
  };
  const int from = begin(blockIdx.y), to = begin(blockIdx.y + 1);
  // How many of the 16 bytes move with so many tokens (the ids of a table may end within them).
  const auto bytes = [&](int tokens) {
    switch (p.kind) {
      case kWhole:
        return off < p.bytes ? 16 : 0;
      case kLatents:
        return off < imin64(p.bytes, static_cast<int64_t>(tokens) * p.token_bytes) ? 16 : 0;
      case kPageTail:
        return off < static_cast<int64_t>(tokens & ((1 << a.shift) - 1)) * p.token_bytes ? 16 : 0;
      default:
        return static_cast<int>(iclamp64(imin64(p.bytes, 4ll * (tokens >> a.shift)) - off, 0, 16));
    }
  };
  const auto load = [&](int64_t slot, int n) {
    const char *at = base + slot * p.stride + off;
    u4 v = {0u, 0u, 0u, 0u};
    if (slot < 0) return v;
    if (p.kind != kTable) {
      if (n) v = *reinterpret_cast<const u4 *>(at);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * i < n) v[i] = reinterpret_cast<const uint32_t *>(at)[i];
    }
    return v;
  };
  const bool tail = p.kind == kPageTail;
  u4 held = {0u, 0u, 0u, 0u};
  for (int i0 = from; i0 < to; i0 += kBatch) {
    u4 v[kBatch];
    // All loads of a batch before its stores: what a batch reads is not written before it.
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i0 + k >= to) break;
      const Move m = a.moves[i0 + k];
      if (m.flags & kSave) held = load(tail ? m.held_page : m.dst, bytes(m.held_tokens));
      v[k] = m.flags & kFromSaved ? held : load(tail ? m.src_page : m.src, bytes(m.tokens));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i0 + k >= to) break;
      const Move m = a.moves[i0 + k];
      const int n = bytes(m.tokens);
      if (tail && (m.src_page < 0 || m.dst_page < 0)) continue;
      char *at = base + (tail ? m.dst_page : m.dst) * p.stride + off;
      if (p.kind != kTable) {
        if (n) *reinterpret_cast<u4 *>(at) = v[k];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * i < n) reinterpret_cast<uint32_t *>(at)[i] = v[k][i];
      }
    }
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace sophia

using namespace sophia;

namespace {
constexpr size_t kHeader = 64;   // of the workspace: the count

int run_moves(const char *what, PlanArgs plan, MoveArgs a, char *workspace, hipStream_t st) {
  plan.count = reinterpret_cast<int32_t *>(workspace);
  plan.moves = reinterpret_cast<Move *>(workspace + kHeader);
  a.count = plan.count;
  a.moves = plan.moves;
  int64_t blocks = 0;
  for (int i = 0; i < a.n_parts; ++i) blocks += static_cast<int64_t>(a.part[i].tensors) * a.part[i].chunks;
  if (blocks == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(blocks <= 0x7fffffff, "%s: too much work for one call", what);
  // Slots are large, and a thread each 16 bytes of them fills the chip; pages are small, and many.
  a.workers = static_cast<int>(iclamp64((2048 + blocks - 1) / blocks, 1, plan.n));
  hipLaunchKernelGGL(move_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, plan);
  hipLaunchKernelGGL(move_kernel, dim3(static_cast<unsigned>(blocks), a.workers), dim3(kMoveThreads), 0, st, a);
  return check_launch(what);
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
}  // namespace

extern "C" size_t sophia_move_workspace_size(int n) {
  return n < 1 || n > SOPHIA_MOVES ? 0 : kHeader + static_cast<size_t>(n) * sizeof(Move);
}

extern "C" int sophia_cache_fork(const int32_t *src, const int32_t *dst, const int64_t *cached, int n, int n_slots,
                                 float *const *states, int64_t state_elems, float *const *convs, int64_t conv_elems,
                                 int n_kda, float *const *mla, int64_t slot_stride, int max_seq, int n_mla,
                                 void *const *pools, int64_t page_stride, int64_t n_pages, int page_size, int n_pools,
                                 int32_t *table, int64_t table_stride, int max_pages, int rank, int pool_dtype,
                                 void *workspace, size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(n >= 0 && n <= SOPHIA_MOVES && n_slots >= 0, "cache_fork: moves must be 0..%d, slots >= 0", SOPHIA_MOVES);
  SOPHIA_REQUIRE(n_kda >= 0 && n_kda <= SOPHIA_FORK_KDA && n_mla >= 0 && n_mla <= SOPHIA_FORK_MLA && n_pools >= 0 &&
                     n_pools <= SOPHIA_FORK_MLA,
                 "cache_fork: at most %d KDA layers, %d MLA layers and %d pools", SOPHIA_FORK_KDA, SOPHIA_FORK_MLA,
                 SOPHIA_FORK_MLA);
  SOPHIA_REQUIRE(state_elems >= 0 && state_elems % 4 == 0 && conv_elems >= 0 && conv_elems % 4 == 0,
                 "cache_fork: slots of states and conv histories must be multiples of 4 values");
  SOPHIA_REQUIRE(n_mla == 0 || (max_seq >= 0 && rank > 0 && rank % 4 == 0 && slot_stride % 4 == 0 &&
                                slot_stride >= static_cast<int64_t>(max_seq) * rank),
                 "cache_fork: latents need a rank that is a multiple of 4 and a slot stride that holds a slot");
  const bool paged = table != nullptr;
  SOPHIA_REQUIRE(paged || n_pools == 0, "cache_fork: pools need their table");
  if (paged) {
    SOPHIA_REQUIRE(pool_dtype == SOPHIA_DTYPE_F32 || pool_dtype == SOPHIA_DTYPE_BF16, "cache_fork: dtype not supported");
    SOPHIA_REQUIRE(page_size >= 1 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
                   "cache_fork: page_size must be a power of two, at most 65536");
    SOPHIA_REQUIRE(max_pages >= 0 && table_stride >= max_pages && n_pages >= 0 && n_pages <= 0x7fffffff,
                   "cache_fork: the table's rows must hold max_pages entries");
    SOPHIA_REQUIRE(n_pools == 0 || (rank > 0 && rank % 8 == 0 && page_stride % 8 == 0 &&
                                    page_stride >= static_cast<int64_t>(page_size) * rank),
                   "cache_fork: pools need a rank and a page stride that are multiples of 8, and the stride to hold a page");
  }
  if (n == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(cached || (n_mla == 0 && !paged), "cache_fork: latents and pages need cached");
  SOPHIA_REQUIRE(src && dst && (n_kda == 0 || (states && (convs || conv_elems == 0))) && (n_mla == 0 || mla) &&
                     (n_pools == 0 || pools),
                 "cache_fork: NULL pointer");
  SOPHIA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= sophia_move_workspace_size(n),
                 "cache_fork: workspace too small");
  MoveArgs a = {};
  int at = 0;
  const auto chunks = [](int64_t bytes) { return static_cast<int>((bytes + kChunk - 1) / kChunk); };
  const auto add = [&](int kind, auto *const *list, int count, int64_t stride, int64_t bytes, int token_bytes) {
    if (count == 0 || bytes == 0) return true;
    a.part[a.n_parts++] = Part{kind, at, count, chunks(bytes), stride, bytes, token_bytes};
    for (int i = 0; i < count; ++i) {
      if (!list[i] || !aligned16(list[i])) return false;
      a.base[at++] = reinterpret_cast<char *>(const_cast<void *>(static_cast<const void *>(list[i])));
    }
    return true;
  };
  const int esz = pool_dtype == SOPHIA_DTYPE_F32 ? 4 : 2;
  bool ok = add(kWhole, states, n_kda, state_elems * 4, state_elems * 4, 0);
  ok = ok && (conv_elems == 0 || add(kWhole, convs, n_kda, conv_elems * 4, conv_elems * 4, 0));
  ok = ok && add(kLatents, mla, n_mla, slot_stride * 4, static_cast<int64_t>(max_seq) * rank * 4, rank * 4);
  ok = ok && (!paged || add(kPageTail, pools, n_pools, page_stride * esz, static_cast<int64_t>(page_size) * rank * esz, rank * esz));
  SOPHIA_REQUIRE(ok, "cache_fork: every layer's tensors must be there, 16-byte aligned");
  if (paged && max_pages > 0) {
    a.part[a.n_parts++] = Part{kTable, at, 1, chunks(4ll * max_pages), table_stride * 4, 4ll * max_pages, 0};
    a.base[at++] = reinterpret_cast<char *>(table);
  }
  a.shift = paged ? log2_of(page_size) : 0;
  const PlanArgs plan{src, dst, n, n_slots, cached, table, table_stride, max_pages, a.shift, n_pages, nullptr, nullptr};
  return run_moves("cache_fork", plan, a, static_cast<char *>(workspace), static_cast<hipStream_t>(stream));
}

extern "C" int sophia_page_copy(const int32_t *src, const int32_t *dst, int n, void *const *pools, int n_pools,
                                int64_t page_stride, int64_t page_elems, int64_t n_pages, int dtype, void *workspace,
                                size_t workspace_bytes, void *stream) {
  SOPHIA_REQUIRE(dtype == SOPHIA_DTYPE_F32 || dtype == SOPHIA_DTYPE_BF16, "page_copy: dtype not supported");
  SOPHIA_REQUIRE(n >= 0 && n <= SOPHIA_MOVES, "page_copy: moves must be 0..%d", SOPHIA_MOVES);
  SOPHIA_REQUIRE(n_pools >= 0 && n_pools <= SOPHIA_FORK_MLA, "page_copy: at most %d pools", SOPHIA_FORK_MLA);
  SOPHIA_REQUIRE(page_elems >= 0 && page_elems % 8 == 0 && page_stride % 8 == 0 && page_stride >= page_elems && n_pages >= 0 &&
                     n_pages <= 0x7fffffff,
                 "page_copy: pages and their stride must be multiples of 8 values, and the stride hold a page");
  if (n == 0 || n_pools == 0 || page_elems == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(src && dst && pools, "page_copy: NULL pointer");
  SOPHIA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= sophia_move_workspace_size(n),
                 "page_copy: workspace too small");
  const int esz = dtype == SOPHIA_DTYPE_F32 ? 4 : 2;
  MoveArgs a = {};
  a.n_parts = 1;
  a.part[0] = Part{kWhole, 0, n_pools, static_cast<int>((page_elems * esz + kChunk - 1) / kChunk), page_stride * esz,
                   page_elems * esz, 0};
  for (int i = 0; i < n_pools; ++i) {
    SOPHIA_REQUIRE(pools[i] && aligned16(pools[i]), "page_copy: every pool must be there, 16-byte aligned");
    a.base[i] = static_cast<char *>(pools[i]);
  }
  const PlanArgs plan{src, dst, n, n_pages, nullptr, nullptr, 0, 0, 0, 0, nullptr, nullptr};
  return run_moves("page_copy", plan, a, static_cast<char *>(workspace), static_cast<hipStream_t>(stream));
}
