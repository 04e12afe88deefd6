// Moves of cache slots and pages in place, as if all at once (include/sophia_pages.h).
//
// dst[i] <- src[i] for all i: a slot may be read by several moves and is written by at most
// one.  A move that reads a slot has to come before the one that writes it; each move has at
// most one such successor, so the moves are trees that end in one last move, or in a cycle, of
// which one slot's content is held in registers.  A first kernel (one work-group) finds the
// trees and orders each; in the second a thread has the same 16 bytes of every slot of some
// trees and moves them in that order, so nothing is copied twice and no thread waits for another.
// Moved bytes are read once and written once, which is what bounds large calls: 48 slots in 28 layers, 943 MB read and
// written, 203 us with the plan (4.7 TB/s; a copy has 5.1), 3,000 pages in 7 layers 141 (4.9).  Trees are worked on
// at once, a tree of many moves in turn: 4,096 pages of one layer in three chains take 226 us, of their own 51 to 68.
#include "common.hpp"

#include "../../include/sophia_pages.h"

namespace sophia {
namespace {

constexpr int kMoves = SOPHIA_MOVES;
constexpr int kFew = 64;      // so many moves a work-group plans by itself, or takes from the list at a time

// A planned move.
struct Move {
  int32_t src, dst;         // slots, or pages
  int32_t flags;            // of its place in its tree, and where the next tree begins (<< kNext)
  int32_t tokens;           // taken along (a fork)
  int32_t src_page, dst_page;   // of the page that these fill in part (-1: none)
  int32_t held_tokens, held_page;   // kSave: the tokens and the source's page of the move at the end
};
constexpr int kFirst = 1;      // the first of its tree
constexpr int kSave = 2;       // what is in dst before is read at the end of the tree: held
constexpr int kFromSaved = 4;  // its source is what was held
constexpr int kNext = 3;
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

// The plan of at most N moves, by THREADS threads (the first of a work-group): put(place, move) in any order.  Returns their
// number to all.  Nothing in it waits for a move's turn, however long the chains (4,096 moves in three: 24 us).
// What bounds it is the latency of its steps: 3.1 us by a wavefront for 64 moves, its launch among them, 11 for 3,000 of which few
// depend on others.
template <int N, int THREADS, typename P>
__device__ __forceinline__ int plan(const PlanArgs &a, P put) {
  constexpr int kEach = N / THREADS, kHash = 2 * N, kBits = __builtin_ctz(2 * N);
  static_assert(N == kEach * THREADS, "each thread has as many moves");
  __shared__ int s_src[N], s_dst[N];
  __shared__ short s_next[N];
  // By slot, the last move that writes it; later what is found of the trees.
  __shared__ int s_key[kHash], s_by[kHash];
  __shared__ int s_wave[THREADS / 64];
  int *const s_count = s_key, *const s_first = s_key + N;   // of a root: its tree's moves, and their first place
  short *const s_jump = reinterpret_cast<short *>(s_by), *const s_low = s_jump + N, *const s_steps = s_low + N,
        *const s_end = s_steps + N;
  int *const s_level = s_by;                                 // moves of a tree's levels, then places
  const int t = threadIdx.x, n = a.n;
  // (What one wavefront writes to LDS it reads in its own order.)
  const auto sync = [] {
    if constexpr (THREADS > 64) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  const auto any = [&](bool v) {
    if constexpr (THREADS > 64) return __syncthreads_or(v) != 0;
    sync();
    return __any(v) != 0;
  };
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
  }
  sync();
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
  sync();
  const auto writer = [&](int slot) {
    for (unsigned h = hash(slot);; h = (h + 1) & (kHash - 1)) {
      if (s_key[h] == slot) return s_by[h];
      if (s_key[h] == -1) return -1;
    }
  };
  // What counts is the last move to a slot, if it changes it: so of a slot's writer too.
  bool active[kEach];
  int next[kEach];             // the move that has to come after
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS, d = s_dst[i];
    active[k] = d >= 0 && s_src[i] != d && writer(d) == i;
    const int w = active[k] ? writer(s_src[i]) : -1;
    next[k] = w >= 0 && s_src[w] != s_dst[w] ? w : -1;
    s_next[i] = static_cast<short>(next[k]);
  }
  sync();
  // By doubling: the move after 1, 2, 4 .. steps (its tree's last one, which stays), the steps to it, and the lowest
  // move before it.  On a cycle all are once round when nothing changes any more, or after n steps.
  const auto follow = [&] {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = t + k * THREADS;
      s_jump[i] = static_cast<short>(next[k] >= 0 ? next[k] : i);
      s_steps[i] = next[k] >= 0;
      s_low[i] = static_cast<short>(i);
    }
    sync();
    for (int reach = 1; reach < n; reach *= 2) {
      short jump[kEach], low[kEach], steps[kEach];
      bool moved = false;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int i = t + k * THREADS, j = s_jump[i];
        jump[k] = s_jump[j];
        low[k] = min(s_low[i], s_low[j]);
        steps[k] = static_cast<short>(s_steps[i] + s_steps[j]);
        moved |= jump[k] != j;
      }
      if (!any(moved)) break;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int i = t + k * THREADS;
        s_jump[i] = jump[k];
        s_low[i] = low[k];
        s_steps[i] = steps[k];
      }
      sync();
    }
  };
  follow();
  // A cycle is cut behind its lowest move, whose slot's content is held for the move that comes before it on the cycle:
  // a tree as the others.  On a cycle is what the steps from somewhere end at that is no last move.
  int flags[kEach], end[kEach];
  bool round = false;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    flags[k] = end[k] = 0;
    round |= s_next[s_jump[t + k * THREADS]] >= 0;
  }
  if (any(round)) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) s_end[t + k * THREADS] = -1;
    sync();
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = s_jump[t + k * THREADS];
      if (s_next[at] >= 0) s_end[at] = 0;                    // (marked)
    }
    sync();
    bool on[kEach];
    int lowest[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = t + k * THREADS;
      on[k] = s_end[i] == 0;
      lowest[k] = s_low[s_jump[i]];
    }
    sync();
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (!on[k] || next[k] != lowest[k]) continue;
      flags[k] |= kFromSaved;
      s_end[next[k]] = static_cast<short>(t + k * THREADS);
      next[k] = -1;
    }
    sync();
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (!on[k] || lowest[k] != t + k * THREADS) continue;
      flags[k] |= kSave;
      end[k] = s_end[lowest[k]];
    }
    sync();
    follow();
  }
  // Places: trees by their last moves, in each the moves with the most others after them first.  A tree of c moves has
  // at most c such levels, so the moves of all trees' levels are counted in n places, and the sums before them are places.
  int root[kEach], steps[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    root[k] = s_jump[t + k * THREADS];
    steps[k] = s_steps[t + k * THREADS];
    s_count[t + k * THREADS] = 0;
  }
  sync();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    s_level[t + k * THREADS] = 0;
    if (active[k]) atomicAdd(&s_count[root[k]], 1);
  }
  sync();
  // to[i] = the sum of from[0 .. i); kEach neighbours per thread.  Returns the sum of all.
  const auto sums = [&](const int *from, int *to) {
    int mine[kEach], sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      mine[k] = sum;
      sum += from[kEach * t + k];
    }
    int scan = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(scan, off, 64);
      if ((t & 63) >= off) scan += o;
    }
    if ((t & 63) == 63) s_wave[t >> 6] = scan;
    sync();
    int before = scan - sum, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < (t >> 6)) before += s_wave[w];
      total += s_wave[w];
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) to[kEach * t + k] = before + mine[k];
    sync();
    return total;
  };
  const int total = sums(s_count, s_first);
  int level[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    level[k] = s_first[root[k]] + s_count[root[k]] - 1 - steps[k];
    if (active[k]) atomicAdd(&s_level[level[k]], 1);
  }
  sync();
  sums(s_level, s_level);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = t + k * THREADS;
    if (!active[k]) continue;
    const int place = atomicAdd(&s_level[level[k]], 1);
    if (place == s_first[root[k]]) flags[k] |= kFirst;
    flags[k] |= (s_first[root[k]] + s_count[root[k]]) << kNext;
    put(place, planned(a, i, s_src[i], s_dst[i], flags[k], end[k], s_src[end[k]]));
  }
  return total;
}

template <int N, int THREADS>
__global__ __launch_bounds__(THREADS) void move_plan_kernel(PlanArgs a) {
  const int total = plan<N, THREADS>(a, [&](int place, const Move &m) { a.moves[place] = m; });
  if (threadIdx.x == 0) *a.count = total;
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
  int total;
  if constexpr (FEW) {
    if (threadIdx.x < 64) {
      const int found = plan<kFew, 64>(a.plan, [&](int place, const Move &m) { s_moves[place] = m; });
      if (threadIdx.x == 0) s_total = found;
    }
    __syncthreads();
    total = s_total;
  } else {
    total = *a.plan.count;
  }
  // This worker's trees: those that begin in its share of the list.
  const Move *list = FEW ? s_moves : a.plan.moves;
  const auto begin = [&](int w) {
    const int at = static_cast<int>(static_cast<int64_t>(total) * w / a.workers);
    if (at >= total) return total;
    const int flags = list[at].flags;
    return flags & kFirst ? at : flags >> kNext;
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
    // Full batches without a branch between their loads, and past the caches: 3,000 pages in 7 layers 128 us in place of 142,
    // 48 slots in 28 layers 160 in place of 205 where they were in the last cache before, the same where not (of
    // few moves, which the next step reads from the caches, 23 in place of 27 the other way round).
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
  // Planned by each work-group itself: a launch less, where all run at once (24 pages in 7 layers 6.3 us in place of
  // 8.8, 64 11.0 and 11.2), not where they come in turns and plan each time (48 slots in 28 layers 209 us in place of
  // 201), and not with a table, whose rows others may move while it is read for the plan.
  const bool table = a.part[a.n_parts - 1].kind == kTable;
  if (plan.n <= kFew && !table && blocks * a.workers <= 2048) {
    hipLaunchKernelGGL(move_kernel<true>, dim3(static_cast<unsigned>(blocks), a.workers), threads, 0, st, a);
    return check_launch(what);
  }
  // One wavefront, which waits for nobody, to 128 moves (65 pages of one layer 9.9 us in place of 11.4 by 256 threads; 200 16.4 and
  // 16.3, 400 20.0 and 15.0); 256 threads to 1,024 (700 pages 17.8 in place of 20.2 by 1,024 threads).
  if (plan.n <= 64)
    hipLaunchKernelGGL((move_plan_kernel<64, 64>), dim3(1), dim3(64), 0, st, plan);
  else if (plan.n <= 128)
    hipLaunchKernelGGL((move_plan_kernel<128, 64>), dim3(1), dim3(64), 0, st, plan);
  else if (plan.n <= 512)
    hipLaunchKernelGGL((move_plan_kernel<512, 256>), dim3(1), dim3(256), 0, st, plan);
  else if (plan.n <= 1024)
    hipLaunchKernelGGL((move_plan_kernel<1024, 256>), dim3(1), dim3(256), 0, st, plan);
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
