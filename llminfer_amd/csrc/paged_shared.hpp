// Sequences that have their first keys in common, as the kernels of the paged
// attention see them (paged_gqa.hip, paged_tiles.hip): a group's shared keys
// with all rows of the group as columns, none of which is masked, and each
// sequence's own keys behind them. Both are sequences of a call to those
// kernels, so that one plan divides them; a row's partials of the two are
// joined by paged_shared_merge_kernel.
#pragma once

#include "paged_kv.hpp"

namespace llmi {

// Rows [row0, row0 + rows) over the keys from block `begin` to `end`: row i
// sees those up to past + i (step 1) or past (step 0, a group's shared keys).
struct SharedSeq {
  unsigned row0, rows, past;
  bool ok;
  unsigned begin, end, step, from; // from: the row of the table
  __device__ unsigned keys() const { return end; }
  __device__ unsigned first() const { return begin; }
  __device__ unsigned last(unsigned row) const { return past + step * row; }
  __device__ unsigned table(unsigned) const { return from; }
  __device__ bool joined() const { return begin != 0 || step == 0; }
};

// Sequences base .. base + sequences - 1 of `count` groups and then `all`
// sequences. Group i has sequences groups[i] .. groups[i + 1] - 1, whose first
// prefix[i] keys, in whole blocks, are read through its first one's table.
struct SharedView : PagedView {
  typedef SharedSeq Seq;
  const int32_t *groups, *prefix;
  unsigned count, all, base;
};

// A group's shared keys that are read as one: whole blocks.
__device__ __forceinline__ unsigned shared_keys(const SharedView &g, unsigned group) {
  return (unsigned)max(g.prefix[group], 0) & ~31u;
}

// The group of a sequence, by bisection (groups are in order); false if it is
// in none.
__device__ __forceinline__ bool shared_group(const SharedView &g, unsigned seq, unsigned &group) {
  unsigned lo = 0, hi = g.count; // groups[lo] <= seq < groups[hi], if any
  while (hi - lo > 1) {
    const unsigned mid = (lo + hi) / 2;
    if (g.groups[mid] <= (int)seq)
      lo = mid;
    else
      hi = mid;
  }
  group = lo;
  return g.groups[lo] <= (int)seq && (int)seq < g.groups[lo + 1];
}

// A sequence's own keys. One that is shorter than its group's prefix has no
// place.
__device__ __forceinline__ SharedSeq shared_own_keys(const SharedView &g, unsigned seq) {
  const PagedSeq p = paged_seq(static_cast<const PagedView &>(g), seq);
  SharedSeq q{p.row0, p.rows, p.past, p.ok, 0, p.past + p.rows, 1, seq};
  unsigned group;
  if (shared_group(g, seq, group)) {
    const int prefix = g.prefix[group];
    q.ok = q.ok && prefix <= (int)p.past;
    q.begin = q.ok ? shared_keys(g, group) / 32 : 0u;
  }
  return q;
}

// A group's shared keys, for all of its rows.
__device__ __forceinline__ SharedSeq shared_prefix_keys(const SharedView &g, unsigned group) {
  const int S = (int)g.all, T = (int)g.tokens;
  const int s0 = min(max(g.groups[group], 0), S), s1 = min(max(g.groups[group + 1], s0), S);
  const int lo = min(max(g.starts[s0], 0), T), hi = min(max(g.starts[s1], lo), T);
  const unsigned keys = shared_keys(g, group);
  // (more keys than a row of the table has: no sequence has a place)
  const bool any = s1 > s0 && keys && keys <= (unsigned)(g.tableStride * g.pageSize);
  return SharedSeq{(unsigned)lo, any ? (unsigned)(hi - lo) : 0u, keys - 1,       true, 0,
                   any ? keys : 0u, 0, (unsigned)s0};
}

__device__ __forceinline__ SharedSeq paged_seq(const SharedView &g, unsigned s) {
  s += g.base;
  return s < g.count ? shared_prefix_keys(g, s) : shared_own_keys(g, s - g.count);
}

__device__ __forceinline__ SharedSeq paged_from_lane(const SharedSeq &own, unsigned lane) {
  auto at = [&](unsigned x) { return (unsigned)__builtin_amdgcn_readlane((int)x, (int)lane); };
  SharedSeq q;
  q.row0 = at(own.row0);
  q.rows = at(own.rows);
  q.past = at(own.past);
  q.ok = at(own.ok) != 0;
  q.begin = at(own.begin);
  q.end = at(own.end);
  q.step = at(own.step);
  q.from = at(own.from);
  return q;
}

} // namespace llmi
