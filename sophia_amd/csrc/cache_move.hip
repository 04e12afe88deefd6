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
constexpr int kFew = 64;      // so many moves each work-group plans by itself

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

// Move i, whose source and destination are given; of a cycle's first move also its last one.
__device__ __forceinline__ Move planned(const PlanArgs &a, int i, int src, int dst, int flags, int end, int end_src) {
  const auto tokens = [&](int move) { return a.cached ? static_cast<int>(iclamp64(a.cached[move], 0, 1 << 30)) : 0; };
  const auto page = [&](int slot, int count) {
    const int full = count >> a.shift;
    const int id = a.table && full < a.max_pages ? a.table[slot * a.table_stride + full] : -1;
    return id >= 0 && id < a.n_pages ? id : -1;
  };
  Move m = {};
  m.src = src;
  m.dst = dst;
  m.flags = flags;
  m.tokens = tokens(i);
  m.src_page = page(src, m.tokens);
  m.dst_page = page(dst, m.tokens);
  m.held_page = -1;
  if (flags & kSave) {
    m.held_tokens = tokens(end);
    m.held_page = page(end_src, m.held_tokens);
  }
  return m;
}

// At most 64 moves, planned by a wavefront: a move per lane, sets of moves as bits.  put(place, move)
// in any order; returns their number.
template <typename P>
__device__ __forceinline__ int plan_few(const PlanArgs &a, P put) {
  const int i = threadIdx.x & 63, n = a.n;
  const int src = i < n ? a.src[i] : -1, dst = i < n ? a.dst[i] : -1;
  const bool ok = src >= 0 && src < a.limit && dst >= 0 && dst < a.limit;
  const uint64_t all = __ballot(ok);
  const auto of = [](int v, int lane) { return __builtin_amdgcn_readlane(v, lane); };
  // The last move to this one's slot, and the last one to the slot that it reads.
  int last = i, writer = -1;
  for (uint64_t m = all; m; m &= m - 1) {
    const int j = __ffsll(static_cast<unsigned long long>(m)) - 1, d = of(dst, j);
    last = d == dst ? j : last;
    writer = d == src ? j : writer;
  }
  const bool active = ok && last == i && src != dst;
  const uint64_t live = __ballot(active);
  const int next = active && writer >= 0 && ((live >> writer) & 1) ? writer : -1;
  uint64_t readers = 0;       // the moves that have to come before
  for (uint64_t m = __ballot(next >= 0); m; m &= m - 1) {
    const int j = __ffsll(static_cast<unsigned long long>(m)) - 1;
    readers |= of(next, j) == i ? 1ull << j : 0;
  }
  // Levels; what is left are cycles, which take levels of their own one after the other.
  uint64_t left = live;
  int level = 0, flags = 0, end = 0, root = i, now = 0;
  for (uint64_t ready; (ready = __ballot(((left >> i) & 1) && !(readers & left))) != 0; left &= ~ready)
    if ((ready >> i) & 1) level = now++;
    else ++now;
  int up = next;
  for (uint64_t m = left; m;) {
    const int first = __ffsll(static_cast<unsigned long long>(m)) - 1;
    for (int j = first;;) {
      m &= ~(1ull << j);
      if (i == j) level = now;
      ++now;
      const int to = of(next, j);
      if (to == first) {
        if (i == j) flags |= kFromSaved, up = -1;
        if (i == first) flags |= kSave, end = j;
        break;
      }
      j = to;
    }
  }
  // Trees: each move's last one, by doubling.
  root = up >= 0 ? up : i;
#pragma unroll
  for (int r = 0; r < 6; ++r) root = __shfl(root, root, 64);
  const int key = root << 16 | level << 8 | i;   // (moves that read one slot have one level)
  int place = 0, same = 0;
  for (uint64_t m = live; m; m &= m - 1) {
    const int k = of(key, __ffsll(static_cast<unsigned long long>(m)) - 1);
    place += k < key;
    same += k < key && (k >> 16) == root;
  }
  const int end_src = __shfl(src, end, 64);
  if (active) put(place, planned(a, i, src, dst, flags | (same == 0 ? kFirst : 0), end, end_src));
  return __popcll(live);
}

__global__ __launch_bounds__(64) void move_plan_few_kernel(PlanArgs a) {
  const int total = plan_few(a, [&](int place, const Move &m) { a.moves[place] = m; });
  if (threadIdx.x == 0) *a.count = total;
}

// The same for more, by THREADS threads.
template <int N, int THREADS>
__global__ __launch_bounds__(THREADS) void move_plan_kernel(PlanArgs a) {
  constexpr int kEach = N / THREADS, kHash = 2 * N, kBits = __builtin_ctz(2 * N);
  static_assert(N == kEach * THREADS, "each thread has as many moves");
  __shared__ int s_src[N], s_dst[N], s_readers[N];   // s_readers: moves that have to come before; then places
  __shared__ short s_next[N];
  // By slot, the last move that writes it; later what is found of the trees.
  __shared__ int s_key[kHash], s_by[kHash];
  __shared__ int s_wave[THREADS / 64];
  int *const s_count = s_key;                        // of a root: moves of its tree, then the next one's place
  int *const s_first = s_key + N;                    // the first one's
  short *const s_jump = reinterpret_cast<short *>(s_by), *const s_low = s_jump + N, *const s_end = s_low + N;
  const int t = threadIdx.x, n = a.n;
  for (int i = t; i < kHash; i += THREADS) {
    s_key[i] = -1;
    s_by[i] = -1;
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    const int s = i < n ? a.src[i] : -1, d = i < n ? a.dst[i] : -1;
    s_src[i] = s;
    s_dst[i] = s >= 0 && s < a.limit && d >= 0 && d < a.limit ? d : -1;
    s_readers[i] = 0;
  }
  __syncthreads();
  const auto hash = [](int slot) { return (static_cast<unsigned>(slot) * 2654435761u) >> (32 - kBits); };
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS, d = s_dst[i];
    if (d < 0) continue;
    unsigned h = hash(d);      // (half of the places stay free)
    for (;; h = (h + 1) & (kHash - 1)) {
      const int was = atomicCAS(&s_key[h], -1, d);
      if (was == -1 || was == d) break;
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
  // What counts is the last move to a slot, if it changes it: so of a slot's writer too.
  bool active[kEach];
  int next[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS, d = s_dst[i];
    active[k] = d >= 0 && s_src[i] != d && writer(d) == i;
    const int w = active[k] ? writer(s_src[i]) : -1;
    next[k] = w >= 0 && s_src[w] != s_dst[w] ? w : -1;
    s_next[i] = static_cast<short>(next[k]);
    if (next[k] >= 0) atomicAdd(&s_readers[next[k]], 1);
  }
  __syncthreads();
  // By doubling: the move after 1, 2, 4 .. steps, and the lowest on the way.
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    s_jump[i] = static_cast<short>(next[k] >= 0 ? next[k] : i);
    s_low[i] = static_cast<short>(i);
  }
  __syncthreads();
  for (int reach = 1; reach < n; reach *= 2) {
    short jump[kEach], low[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = t + k * THREADS, j = s_jump[i];
      jump[k] = s_jump[j];
      low[k] = min(s_low[i], s_low[j]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      s_jump[t + k * THREADS] = jump[k];
      s_low[t + k * THREADS] = low[k];
    }
    __syncthreads();
  }
  // A tree's root is its last move, or the lowest move of the cycle that it ends in, which has that
  // cycle's first move.
  int root[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = s_jump[t + k * THREADS];
    root[k] = s_next[at] < 0 ? at : s_low[at];
    s_count[t + k * THREADS] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    s_low[t + k * THREADS] = 0;                      // (now: 1 + the root, of moves on a cycle)
    if (active[k]) atomicAdd(&s_count[root[k]], 1);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    if (!active[k] || next[k] < 0 || root[k] != i) continue;
    int j = i;
    for (;;) {
      s_low[j] = static_cast<short>(i + 1);
      const int to = s_next[j];
      if (to == i) break;
      j = to;
    }
    s_end[i] = static_cast<short>(j);
  }
  // Where the trees begin: a sum over the roots before, kEach neighbours per thread.
  int mine[kEach], sum = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    mine[k] = sum;
    sum += s_count[kEach * t + k];
  }
  int scan = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(scan, off, 64);
    if ((t & 63) >= off) scan += o;
  }
  if ((t & 63) == 63) s_wave[t >> 6] = scan;
  __syncthreads();
  int before = scan - sum, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < (t >> 6)) before += s_wave[w];
    total += s_wave[w];
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    s_count[kEach * t + k] = before + mine[k];
    s_first[kEach * t + k] = before + mine[k];
  }
  __syncthreads();
  // A move takes its place when all that read its slot have theirs.  Nobody waits for a cycle here, and of
  // what is on none there is always one that nothing is before: every thread comes to its end.
  bool waits[kEach], any = false;
  int place[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    waits[k] = active[k] && s_low[t + k * THREADS] == 0;
    any |= waits[k];
  }
  while (any) {
    any = false;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (!waits[k]) continue;
      if (__hip_atomic_load(&s_readers[t + k * THREADS], __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_WORKGROUP) == 0) {
        place[k] = __hip_atomic_fetch_add(&s_count[root[k]], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (next[k] >= 0) __hip_atomic_fetch_add(&s_readers[next[k]], -1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_WORKGROUP);
        waits[k] = false;
      } else {
        any = true;
      }
    }
  }
  __syncthreads();
  // Then the cycles.
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    if (!active[k] || next[k] < 0 || root[k] != i) continue;
    int at = s_count[i];
    for (int j = i;;) {
      s_readers[j] = at++;
      const int to = s_next[j];
      if (to == i) break;
      j = to;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    if (!active[k]) continue;
    int flags = 0, end = 0;
    if (s_low[i] != 0) {
      place[k] = s_readers[i];
      if (root[k] == i) {
        flags |= kSave;
        end = s_end[i];
      }
      if (next[k] == root[k]) flags |= kFromSaved;
    }
    if (place[k] == s_first[root[k]]) flags |= kFirst;
    a.moves[place[k]] = planned(a, i, s_src[i], s_dst[i], flags, end, s_src[end]);
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
  PlanArgs plan;
  int n_parts;
  int workers;               // that share the trees
  Part part[kParts];
  char *base[kTensors];
};
static_assert(sizeof(MoveArgs) <= 4000, "kernel arguments");

constexpr int kMoveThreads = 256, kChunk = 16 * kMoveThreads, kBatch = 8;

// FEW: at most kFew moves, planned here by the first wavefront; else a list of them, taken kFew at a time.
template <bool FEW>
__global__ __launch_bounds__(kMoveThreads) void move_kernel(MoveArgs a) {
  __shared__ Move s_moves[kFew + kBatch];
  __shared__ int s_total;
  int block = blockIdx.x, q = 0;
  while (q + 1 < a.n_parts && block >= a.part[q].tensors * a.part[q].chunks) {
    block -= a.part[q].tensors * a.part[q].chunks;
    ++q;
  }
  const Part p = a.part[q];
  char *base = a.base[p.first + block / p.chunks];
  const int64_t off = static_cast<int64_t>(block % p.chunks) * kChunk + 16 * threadIdx.x;
  if constexpr (FEW) {
    if (threadIdx.x < 64) {
      const int total = plan_few(a.plan, [&](int place, const Move &m) { s_moves[place] = m; });
      if (threadIdx.x == 0) s_total = total;
    }
    __syncthreads();
  }
  // This worker's trees: those that begin in its share of the list.
  const int total = FEW ? s_total : *a.plan.count;
  const Move *list = FEW ? s_moves : a.plan.moves;
  const auto begin = [&](int w) {
    int at = static_cast<int>(static_cast<int64_t>(total) * w / a.workers);
    while (at < total && !(list[at].flags & kFirst)) ++at;
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
        return off < static_cast<int64_t>(tokens & ((1 << a.plan.shift) - 1)) * p.token_bytes ? 16 : 0;
      default:
        return static_cast<int>(iclamp64(imin64(p.bytes, 4ll * (tokens >> a.plan.shift)) - off, 0, 16));
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
  const bool in = off < p.bytes;
  u4 held = {0u, 0u, 0u, 0u};
  // Moves [m, m + n) of s_moves: all loads before the stores, as what a batch reads is not written before it.
  const auto batch = [&](const Move *m, int n) {
    u4 v[kBatch];
    int flags = 0;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) flags |= k < n ? m[k].flags : 0;
    // Full batches without a branch between their loads, and past the caches: 48 slots in 28 layers 160 us in place of
    // 205 (of few moves, which the next step reads from the caches, 23 in place of 27 the other way round).
    if (p.kind == kWhole && n == kBatch && !(flags & (kSave | kFromSaved))) {
      if (!in) return;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) v[k] = __builtin_nontemporal_load(reinterpret_cast<const u4 *>(base + m[k].src * p.stride + off));
#pragma unroll
      for (int k = 0; k < kBatch; ++k) __builtin_nontemporal_store(v[k], reinterpret_cast<u4 *>(base + m[k].dst * p.stride + off));
      return;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k >= n) break;
      if (m[k].flags & kSave) held = load(tail ? m[k].held_page : m[k].dst, bytes(m[k].held_tokens));
      v[k] = m[k].flags & kFromSaved ? held : load(tail ? m[k].src_page : m[k].src, bytes(m[k].tokens));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k >= n) break;
      const int count = bytes(m[k].tokens);
      if (tail && (m[k].src_page < 0 || m[k].dst_page < 0)) continue;
      char *at = base + (tail ? m[k].dst_page : m[k].dst) * p.stride + off;
      if (p.kind != kTable) {
        if (count) *reinterpret_cast<u4 *>(at) = v[k];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * i < count) reinterpret_cast<uint32_t *>(at)[i] = v[k][i];
      }
    }
  };
  for (int i0 = from; i0 < to; i0 += kFew) {
    const int n = min(kFew, to - i0);
    if constexpr (!FEW) {
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * n; i += kMoveThreads)
        reinterpret_cast<u4 *>(s_moves)[i] = reinterpret_cast<const u4 *>(a.plan.moves + i0)[i];
      __syncthreads();
    }
    for (int i = 0; i < n; i += kBatch) batch(s_moves + (FEW ? i0 : 0) + i, min(kBatch, n - i));
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
  a.plan = plan;
  const auto blocks_of = [](const MoveArgs &m) {
    int64_t n = 0;
    for (int i = 0; i < m.n_parts; ++i) n += static_cast<int64_t>(m.part[i].tensors) * m.part[i].chunks;
    return n;
  };
  const int64_t blocks = blocks_of(a);
  if (blocks == 0) return SOPHIA_OK;
  SOPHIA_REQUIRE(blocks <= 0x7fffffff, "%s: too much work for one call", what);
  const dim3 threads(kMoveThreads);
  // Slots are large, and a thread for each 16 bytes of them fills the chip; pages are small, and many.
  a.workers = static_cast<int>(iclamp64((2048 + blocks - 1) / blocks, 1, plan.n));
  // Planned by each work-group itself: a launch less, where all run at once (24 pages in 7 layers 7.4 us in place of
  // 10), not where they come in turns and plan each time (48 slots in 28 layers 209 us in place of 201), and
  // not with a table, whose rows others may move while it is read for the plan.
  const bool table = a.part[a.n_parts - 1].kind == kTable;
  if (plan.n <= kFew && !table && blocks * a.workers <= 2048) {
    hipLaunchKernelGGL(move_kernel<true>, dim3(static_cast<unsigned>(blocks), a.workers), threads, 0, st, a);
    return check_launch(what);
  }
  if (plan.n <= kFew)
    hipLaunchKernelGGL(move_plan_few_kernel, dim3(1), dim3(64), 0, st, plan);
  else if (plan.n <= 512)
    hipLaunchKernelGGL((move_plan_kernel<512, 256>), dim3(1), dim3(256), 0, st, plan);
  else
    hipLaunchKernelGGL((move_plan_kernel<kMoves, 1024>), dim3(1), dim3(1024), 0, st, plan);
  hipLaunchKernelGGL(move_kernel<false>, dim3(static_cast<unsigned>(blocks), a.workers), threads, 0, st, a);
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
  const PlanArgs plan{src, dst, n, n_slots, cached, table, table_stride, max_pages, paged ? log2_of(page_size) : 0, n_pages, nullptr, nullptr};
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
