// New tokens of sequences and their latents' pages, as the kernels of
// include/sophia_pages.h read them.
#pragma once

#include "common.hpp"

namespace sophia {

struct Pages {
  const void *pages;        // [n_pages][page_stride]
  int64_t page_stride;
  int64_t n_pages;
  int shift;                // page_size = 1 << shift
  const int32_t *table;
  int64_t table_stride;
  int table_rows, max_pages;
  const int32_t *slots;     // NULL: s
  const int32_t *cu;
  const int64_t *kv_len;
  int n_seqs;
  int64_t rows;
};

// A sequence's rows (within the rows, whatever cu holds), the position of its first row (it
// may be negative) and the keys that its pages can hold.  The three loads have no branch
// between them, so they are under way together.
struct Sequence {
  int64_t base, slot;
  int n, pos0, keys;
};
__device__ __forceinline__ Sequence sequence(const Pages &p, int s) {
  const int64_t first = p.cu[s], end = p.cu[s + 1], kv = p.kv_len[s];
  Sequence q;
  q.slot = p.slots ? p.slots[s] : s;
  q.base = iclamp64(first, 0, p.rows);
  q.n = static_cast<int>(iclamp64(imin64(end, p.rows) - q.base, 0, 1 << 29));
  const int cap = p.max_pages << p.shift;      // (at most 2^29)
  // Beyond cap + n every row sees all keys that there can be, so nothing changes from there on.
  const int have = static_cast<int>(iclamp64(kv, 0, static_cast<int64_t>(cap) + q.n));
  q.pos0 = have - q.n;
  q.keys = q.slot >= 0 && q.slot < p.table_rows ? (have < cap ? have : cap) : 0;
  return q;
}

// The page of key j < keys of a sequence, or -1.
__device__ __forceinline__ int page_of(const Pages &p, int64_t slot, int j) {
  const int id = p.table[slot * p.table_stride + (j >> p.shift)];
  return id >= 0 && id < p.n_pages ? id : -1;
}

}  // namespace sophia
