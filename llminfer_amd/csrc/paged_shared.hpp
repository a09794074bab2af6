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
// from: the row of the table. group: a sequence's, if it has shared keys.
struct SharedSeq {
  unsigned row0, rows, past;
  bool ok;
  unsigned begin, end, step, from, group;
  __device__ unsigned keys() const { return end; }
  __device__ unsigned first() const { return begin; }
  __device__ unsigned last(unsigned row) const { return past + step * row; }
  __device__ unsigned table(unsigned) const { return from; }
  __device__ bool joined() const { return begin != 0 || step == 0; }
};

// What the workgroups of a sequence leave for the join: its first piece, how
// many a unit has, its units (the last unit's pieces first), and the group whose
// partials are joined to them (+ 1; 0: none), for a group its first row. Of runs of
// blocks (paged_mixed.hip): the first of its blocks among all, the blocks of a unit,
// its first unit among all, the same, and for a group the columns of a unit; and in
// a note behind all others the blocks of a run of own keys, of one of shared keys,
// and whether units of these are parted anywhere (1) or at whole runs (0).
struct SharedNote {
  unsigned first, pieces, units, other, width, unused[3]; // (32 bytes)
};

// Sequences base .. base + sequences - 1 of `count` groups and then `all`
// sequences. Group i has sequences groups[i] .. groups[i + 1] - 1, whose first
// prefix[i] keys, in whole blocks, are read through its first one's table.
struct SharedView : PagedView {
  typedef SharedSeq Seq;
  const int32_t *groups, *prefix;
  SharedNote *notes; // [count + all], and one of the runs
  unsigned count, all, base;
};

// The groups' arrays, those of group `lane` in registers.
struct SharedGroups {
  int first, behind, prefix;
};
__device__ __forceinline__ SharedGroups shared_groups(const SharedView &g) {
  const unsigned i = min(threadIdx.x % 64, g.count - 1);
  return {g.groups[i], g.groups[i + 1], g.prefix[i]};
}

// Sequence s of the view (nothing past the last one), a different one in every
// lane; all lanes call it. Groups and sequences take the same steps, so that the
// loads of both are in flight together.
template <bool Few> // at most 64 groups, all of them in `lanes`
__device__ __forceinline__ SharedSeq shared_seq_of(const SharedView &g, const SharedGroups &lanes,
                                                   unsigned s) {
  const bool none = s >= g.sequences;
  const unsigned v = (none ? g.sequences - 1 : s) + g.base;
  const bool ofGroup = v < g.count;
  const unsigned seq = ofGroup ? 0u : v - g.count;
  auto group_of = [&](int mine, const int32_t *array, unsigned i) {
    return Few ? __shfl(mine, (int)i) : array[i];
  };
  // the last group that begins at or before the sequence, by bisection
  unsigned group = 0;
  for (unsigned n = g.count; n > 1; n -= n / 2)
    if (group_of(lanes.first, g.groups, group + n / 2) <= (int)seq)
      group += n / 2;
  group = ofGroup ? v : group;
  const int from = group_of(lanes.first, g.groups, group);
  const int to = group_of(lanes.behind, g.groups + 1, group);
  const int prefix = group_of(lanes.prefix, g.prefix, group);
  const int S = (int)g.all, T = (int)g.tokens;
  const int s0 = ofGroup ? min(max(from, 0), S) : (int)seq;
  const int s1 = ofGroup ? min(max(to, s0), S) : (int)seq + 1;
  const int lo = min(max(g.starts[s0], 0), T), hi = min(max(g.starts[s1], lo), T);
  const int past = g.past[seq];
  const unsigned keys = (unsigned)max(prefix, 0) & ~31u; // those that are read as one
  const long long most = (long long)g.tableStride * g.pageSize;
  SharedSeq q;
  q.row0 = (unsigned)lo;
  q.rows = none ? 0u : (unsigned)(hi - lo);
  q.step = ofGroup ? 0u : 1u;
  q.from = (unsigned)s0;
  q.group = group;
  if (ofGroup) {
    // (more keys than a row of the table has: no sequence has a place)
    const bool any = s1 > s0 && keys && keys <= most;
    q.rows = any ? q.rows : 0u;
    q.past = keys - 1;
    q.ok = true;
    q.begin = 0;
    q.end = any ? keys : 0u;
  } else {
    // one that is shorter than its group's prefix has no place
    const bool in = from <= (int)seq && (int)seq < to;
    q.past = (unsigned)past;
    q.ok = none || (past >= 0 && (long long)past + (hi - lo) <= most && !(in && prefix > past));
    q.begin = in && q.ok ? keys / 32 : 0u;
    q.end = q.past + (unsigned)(hi - lo);
  }
  return q;
}

__device__ __forceinline__ SharedSeq shared_seq(const SharedView &g, const SharedGroups &lanes,
                                                unsigned s) {
  return g.count <= 64 ? shared_seq_of<true>(g, lanes, s) : shared_seq_of<false>(g, lanes, s);
}

// The first 256 sequences, one a lane and member (no array, which would be in
// memory): most calls read the lengths once, all of them in flight.
struct SharedLanes {
  SharedGroups groups;
  SharedSeq a, b, c, d;
};
__device__ __forceinline__ SharedLanes paged_own(const SharedView &g) {
  const unsigned lane = threadIdx.x % 64;
  SharedLanes own;
  own.groups = shared_groups(g);
  if (g.sequences <= 64) {
    own.a = shared_seq(g, own.groups, lane);
    own.b = own.c = own.d = SharedSeq{0, 0, 0, true};
  } else if (g.count <= 64) {
    own.a = shared_seq_of<true>(g, own.groups, lane);
    own.b = shared_seq_of<true>(g, own.groups, 64 + lane);
    own.c = shared_seq_of<true>(g, own.groups, 128 + lane);
    own.d = shared_seq_of<true>(g, own.groups, 192 + lane);
  } else {
    own.a = shared_seq_of<false>(g, own.groups, lane);
    own.b = shared_seq_of<false>(g, own.groups, 64 + lane);
    own.c = shared_seq_of<false>(g, own.groups, 128 + lane);
    own.d = shared_seq_of<false>(g, own.groups, 192 + lane);
  }
  return own;
}
__device__ __forceinline__ const SharedSeq &paged_first(const SharedLanes &own) { return own.a; }

// `each(number of the 64, its sequences)` for all of them, in order, until it
// says true.
template <typename Each>
__device__ __forceinline__ void shared_chunks(const SharedView &g, const SharedLanes &own, Each each) {
  if (each(0u, own.a) || g.sequences <= 64)
    return;
  if (each(1u, own.b) || each(2u, own.c) || each(3u, own.d))
    return;
  for (unsigned c = 4; 64 * c < g.sequences; ++c)
    if (each(c, shared_seq(g, own.groups, 64 * c + threadIdx.x % 64)))
      return;
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
  q.group = at(own.group);
  return q;
}
__device__ __forceinline__ SharedSeq paged_seq_of(const SharedView &g, const SharedLanes &own,
                                                  unsigned seq) {
  if (seq < 64)
    return paged_from_lane(own.a, seq);
  if (seq < 128)
    return paged_from_lane(own.b, seq - 64);
  if (seq < 192)
    return paged_from_lane(own.c, seq - 128);
  if (seq < 256)
    return paged_from_lane(own.d, seq - 192);
  return paged_from_lane(shared_seq(g, own.groups, seq / 64 * 64 + threadIdx.x % 64), seq % 64);
}

template <typename Count>
__device__ __forceinline__ bool paged_find(const SharedView &g, const SharedLanes &own, unsigned u,
                                           Count count, unsigned &seq, unsigned &local,
                                           unsigned &before) {
  bool found = false;
  before = 0;
  shared_chunks(g, own, [&](unsigned c, const SharedSeq &q) {
    const unsigned n = count(q), sum = wave_scan(n);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(u - before < sum);
    if (!past) {
      before += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
      return false;
    }
    const int at = __builtin_ctzll(past);
    seq = 64 * c + (unsigned)at;
    before += (unsigned)__builtin_amdgcn_readlane((int)(sum - n), at);
    local = u - before;
    // (not so with starts out of order: a sum that wrapped)
    found = local < (unsigned)__builtin_amdgcn_readlane((int)n, at);
    return true;
  });
  return found;
}

// What the join needs of a sequence, left by its first workgroup of the first
// KV head. One without a place has its output already, and nothing to join.
__device__ __forceinline__ void leave_note(const PagedView &, const PagedSeq &, unsigned, unsigned,
                                           unsigned, unsigned) {}
__device__ __forceinline__ void leave_note(const SharedView &g, const SharedSeq &s, unsigned seq,
                                           unsigned first, unsigned pieces, unsigned units) {
  const bool join = s.ok && (s.joined() || pieces > 1);
  g.notes[g.base + seq] =
      SharedNote{first, join ? pieces : 0u, units,
                 s.step == 0 ? s.row0 : s.begin ? s.group + 1 : 0u, 0};
}

} // namespace llmi
