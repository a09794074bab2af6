// The pages of the paged 4-bit cache (paged_kv.hpp) as sequences come and go:
// children that share their parents' pages (fork), the pages that no sequence
// holds (free), chosen keys and values put side by side (move). No arithmetic,
// so bytes and latency are what there is to gain.
//
// In a loop: 64 children in pages of 256 keys of 4 heads of 256 (16 MB read, 20
// written) 7.4 us, 5 TB/s, the rate of a copy; 16 children of one prompt 3.8 to 4
// us, a launch with three dependent loads. The free ones of 400 thousand pages by
// 500 rows of up to 1031 13.0 us (traced: marks 7.5, join 2.8, list 3.7; the bytes
// would take 0.6), of 4096 by 16 rows 5.2 us. 8192 of 32749 keys of 4 heads of
// 256 moved between pages 10.8 us: every line of the source is touched, 41 MB, and
// 10 written, the rate of a copy; 6808 of 13 sequences' 8 heads of 128 9.2 us (23
// MB and 9), 42 accepted drafts of 16 sequences 4.4 us. Within the same pages a
// launch more and the rows once more through memory: 16.4, 14.1 and 7.6 us.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"

namespace llmi {
namespace {

// -------------------------------------------------------------------- fork

constexpr unsigned kForkThreads = 256;

struct ForkView {
  const int32_t *table, *past, *parent, *spare;
  int32_t *tableOut, *pastOut;
  unsigned pages, pageSize, kvHeads, sequences, tableStride;
};

// A workgroup copies one block of one head of a child's last page (contiguous, all
// of it in flight before it is stored); the first of a child writes its row of the
// table too. The others, of blocks without keys, leave at once: how full the page
// is only the device knows.
template <int D>
__global__ __launch_bounds__(kForkThreads) void paged_fork_kernel(ForkView g, uint4_t *pool,
                                                                  unsigned *invalid) {
  constexpr unsigned kWords = 40 * D / 16, kEach = (kWords + kForkThreads - 1) / kForkThreads;
  const unsigned blocks = g.pageSize / 32, parts = g.kvHeads * blocks;
  const unsigned child = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x;
  const unsigned parent = (unsigned)g.parent[child];
  const int spare = g.spare[child];
  const int held = parent < g.sequences ? g.past[parent] : -1;
  const bool ok = held >= 0 && (long long)held <= (long long)g.tableStride * g.pageSize;
  const unsigned length = ok ? (unsigned)held : 0u, whole = length / g.pageSize;
  const unsigned rest = length - whole * g.pageSize;
  const int32_t *row = g.table + (size_t)(ok ? parent : 0u) * g.tableStride;
  const bool taken = spare < 0; // the parent's pages as they are
  const unsigned from = ok && rest ? (unsigned)row[whole] : 0u;
  const bool fits = taken || ((unsigned)spare < g.pages && from < g.pages) ||
                    whole == g.tableStride; // (a full table needs no page)
  if (part == 0) {
    int32_t *to = g.tableOut + (size_t)child * g.tableStride;
    for (unsigned j = tid; j < g.tableStride; j += kForkThreads)
      to[j] = !ok                 ? -1
              : taken || j < whole ? row[j]
              : j == whole && fits ? spare
                                   : -1;
    if (tid == 0) {
      g.pastOut[child] = ok ? held : -1;
      if (invalid && !(ok && fits))
        atomicOr(invalid, kPagedPlace);
    }
  }
  const unsigned block = part % blocks, head = part / blocks;
  if (!ok || taken || !fits || 32 * block >= rest)
    return;
  const size_t at = ((size_t)head * blocks + block) * kWords;
  const size_t page = (size_t)g.kvHeads * blocks * kWords;
  const uint4_t *src = pool + from * page + at;
  uint4_t *dst = pool + (unsigned)spare * page + at, x[kEach];
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (tid + i * kForkThreads < kWords)
      x[i] = src[tid + i * kForkThreads];
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (tid + i * kForkThreads < kWords)
      dst[tid + i * kForkThreads] = x[i];
}

// -------------------------------------------------------------------- free

constexpr unsigned kFreeThreads = 1024;
constexpr unsigned kFreeWaves = kFreeThreads / 64;
constexpr unsigned kWindow = 1u << 19; // pages whose marks one workgroup has in LDS
constexpr unsigned kListed = 4096;     // pages whose entries one workgroup writes
constexpr unsigned kSmall = 8192;      // pages of a pool that one workgroup has alone
constexpr unsigned kMarkers = 32;      // workgroups that mark, at most
constexpr unsigned kSlots = 8;         // of a row that a lane has: 512 slots are a piece of it
constexpr unsigned kRows = 4;          // pieces that a wave has in flight

struct FreeView {
  const int32_t *table, *lengths;
  unsigned pages, pageSize, sequences, tableStride;
};

// The pages of window `window` that the tables name, as bits; this is workgroup
// `part` of `parts`. A wave takes 512 slots of a row at a time, four of these
// pieces of rows in flight.
__device__ __forceinline__ void mark_held(const FreeView &g, unsigned part, unsigned parts,
                                          unsigned window, uint32_t *marks, unsigned *invalid) {
  const unsigned tid = threadIdx.x, lane = tid % 64, first = window * kWindow;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const unsigned mine = min(kWindow, g.pages - first);
  const unsigned pieces = (g.tableStride + 64 * kSlots - 1) / (64 * kSlots); // of a row
  const unsigned all = g.sequences * pieces, step = parts * kFreeWaves;      // (< 2^31)
  bool lost = false;
  for (unsigned w = tid; w < (mine + 31) / 32; w += kFreeThreads)
    marks[w] = 0;
  __syncthreads();
  for (unsigned i0 = part * kFreeWaves + wave; i0 < all; i0 += kRows * step) {
    unsigned from[kRows], count[kRows]; // slots of the rows that hold pages
    size_t row[kRows];
    int page[kRows][kSlots];
#pragma unroll
    for (unsigned n = 0; n < kRows; ++n) {
      const unsigned i = min(i0 + n * step, all - 1), s = i / pieces;
      const int length = g.lengths[s];
      const bool bad = length < 0 || (long long)length > (long long)g.tableStride * g.pageSize;
      lost |= bad;
      // (a sequence that does not fit its row holds all of it)
      count[n] = i0 + n * step >= all ? 0u
                 : bad                ? g.tableStride
                                      : ((unsigned)length + g.pageSize - 1) / g.pageSize;
      from[n] = i % pieces * 64 * kSlots + lane;
      row[n] = (size_t)s * g.tableStride;
    }
#pragma unroll
    for (unsigned n = 0; n < kRows; ++n)
#pragma unroll
      for (unsigned k = 0; k < kSlots; ++k)
        if (from[n] + 64 * k < count[n])
          page[n][k] = g.table[row[n] + from[n] + 64 * k];
#pragma unroll
    for (unsigned n = 0; n < kRows; ++n)
#pragma unroll
      for (unsigned k = 0; k < kSlots; ++k) {
        if (from[n] + 64 * k >= count[n])
          continue;
        const unsigned x = (unsigned)page[n][k];
        lost |= x >= g.pages;
        if (x < g.pages && x - first < mine)
          atomicOr(&marks[(x - first) / 32], 1u << (x - first) % 32);
      }
  }
  if (lost && invalid)
    atomicOr(invalid, kPagedPlace);
  __syncthreads();
}

// Entries of the pages [first, first + count), `before` of the pages before
// them free: a free page at its rank, and for each other one a -1 from the end.
// word(i) has the marks of pages 32 i .. 32 i + 31.
template <unsigned Most, typename Word>
__device__ __forceinline__ void list_free(unsigned first, unsigned count, unsigned before,
                                          unsigned pages, int32_t *free, int32_t *number,
                                          Word word) {
  constexpr unsigned kGroups = Most / 64, kEach = kGroups / 64; // of 64 pages; of a lane
  static_assert(kEach * 4096 == Most, "whole groups a lane");
  __shared__ unsigned sBefore[kGroups + 1];
  const unsigned tid = threadIdx.x, lane = tid % 64;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const unsigned groups = (count + 63) / 64;
  auto held = [&](unsigned i) { // of group i; those behind the last page held
    const unsigned at = first / 32 + 2 * i, left = count - 64 * i;
    uint64_t x = word(at);
    if (left > 32)
      x |= (uint64_t)word(at + 1) << 32;
    return left < 64 ? x | ~0ull << left : x;
  };
  if (wave == 0) {
    unsigned n[kEach], sum = 0;
    for (unsigned j = 0; j < kEach; ++j) {
      const unsigned i = kEach * lane + j;
      n[j] = i < groups ? 64 - __builtin_popcountll(held(i)) : 0u;
      sum += n[j];
    }
    unsigned at = before + wave_scan(sum) - sum;
    for (unsigned j = 0; j < kEach; ++j) {
      sBefore[kEach * lane + j] = at;
      at += n[j];
    }
    if (lane == 63)
      sBefore[kGroups] = at;
  }
  __syncthreads();
  for (unsigned i = wave; i < groups; i += kFreeWaves) {
    const uint64_t x = held(i);
    const unsigned page = first + 64 * i + lane;
    const unsigned rank = sBefore[i] + (unsigned)__builtin_popcountll(~x & ((1ull << lane) - 1));
    if (64 * i + lane < count) {
      const bool isFree = !(x >> lane & 1);
      free[isFree ? rank : pages - 1 - (page - rank)] = isFree ? (int)page : -1;
    }
  }
  if (first + count == pages && tid == 0)
    *number = (int)sBefore[kGroups];
}

// All of a small pool in one workgroup.
__global__ __launch_bounds__(kFreeThreads) void paged_free_small_kernel(FreeView g, int32_t *free,
                                                                        int32_t *count,
                                                                        unsigned *invalid) {
  __shared__ uint32_t marks[kSmall / 32];
  mark_held(g, 0, 1, 0, marks, invalid);
  list_free<kSmall>(0, g.pages, 0, g.pages, free, count, [&](unsigned i) { return marks[i]; });
}

// Marks in up to 32 workgroups, each with bits of all pages in LDS, then joined, so
// that no memory has to be cleared and nothing is atomic but bits in LDS; the join
// and the list are launches of their own because a free page's rank needs all the
// marks before it (marks of eight workgroups joined by those that list: 24 us).
// The time goes by pieces of rows, not by slots: short rows are a piece each. One
// workgroup alone up to 8192 pages and 96 pieces, a round and a half of its waves
// (at 8192 pages, one workgroup and three launches: 65 rows of 256 7.4 and 10.1 us,
// 96 10.2 and 10.7, 127 11.3 and 11.0, 500 of 65 29 and 10.2); 32 pieces a marking
// workgroup, up to the most (1000 rows of 32 in 400 thousand pages: 12.2 us, 58 in
// one; 4000 of 16 15.3 and, in three, 74).
// What the launches leave each other: [part][words] marks, the words of a part
// whole 16 bytes, [words] of all of them and how many pages of each kListed are
// free.
struct FreeMarks {
  uint32_t *parts, *all, *count;
};
__host__ __device__ constexpr unsigned free_words(unsigned pages) {
  return (pages / 32 + 4) / 4 * 4;
}

__global__ __launch_bounds__(kFreeThreads) void paged_free_mark_kernel(FreeView g, uint32_t *out,
                                                                       unsigned *invalid) {
  __shared__ uint32_t marks[kWindow / 32];
  const unsigned window = blockIdx.y, words = free_words(g.pages);
  mark_held(g, blockIdx.x, gridDim.x, window, marks, invalid);
  uint32_t *to = out + (size_t)blockIdx.x * words + window * (kWindow / 32);
  const unsigned mine = min(kWindow, g.pages - window * kWindow);
  for (unsigned w = threadIdx.x; w < (mine + 31) / 32; w += kFreeThreads)
    to[w] = marks[w];
}

// The marks of all parts, kListed pages a workgroup: 16 bytes of every eighth
// part a thread.
constexpr unsigned kJoinThreads = kListed / 128 * 8;
__global__ __launch_bounds__(kJoinThreads) void paged_free_join_kernel(FreeMarks m, unsigned parts,
                                                                       unsigned pages) {
  constexpr unsigned kFours = kListed / 128;
  const unsigned words = free_words(pages), i = threadIdx.x % kFours, p0 = threadIdx.x / kFours;
  const unsigned at = 4 * (blockIdx.x * kFours + i), first = blockIdx.x * kListed + 128 * i;
  __shared__ uint4_t sMarks[8][kFours];
  uint4_t x = 0;
  if (at < words) {
#pragma unroll
    for (unsigned n = 0; n < kMarkers / 8; ++n) // (the last part again)
      x |= *reinterpret_cast<const uint4_t *>(m.parts + (size_t)min(p0 + 8 * n, parts - 1) * words + at);
  }
  sMarks[p0][i] = x;
  __syncthreads();
  if (threadIdx.x >= 64)
    return;
  unsigned n = 0;
  if (p0 == 0 && at < words) {
    for (unsigned p = 1; p < 8; ++p)
      x |= sMarks[p][i];
    *reinterpret_cast<uint4_t *>(m.all + at) = x;
    for (unsigned j = 0; j < 4; ++j) {
      const unsigned page = first + 32 * j, left = page < pages ? min(pages - page, 32u) : 0u;
      n += left - __builtin_popcount(left < 32 ? x[j] & ((1u << left) - 1) : x[j]);
    }
  }
  n = wave_scan(n);
  if (threadIdx.x == 63)
    m.count[blockIdx.x] = n;
}

// kListed pages a workgroup, behind the free ones of all before.
__global__ __launch_bounds__(kFreeThreads) void paged_free_list_kernel(FreeMarks m, unsigned pages,
                                                                       int32_t *free,
                                                                       int32_t *count) {
  const unsigned first = blockIdx.x * kListed, tid = threadIdx.x;
  __shared__ unsigned sFree[kFreeWaves];
  __shared__ uint32_t sWord[kListed / 32];
  const unsigned mine = min(kListed, pages - first);
  unsigned n = 0;
  for (unsigned i = tid; i < blockIdx.x; i += kFreeThreads)
    n += m.count[i];
  if (tid < (mine + 31) / 32)
    sWord[tid] = m.all[first / 32 + tid];
  n = wave_scan(n);
  if (tid % 64 == 63)
    sFree[tid / 64] = n;
  __syncthreads();
  n = 0;
  for (unsigned w = 0; w < kFreeWaves; ++w)
    n += sFree[w];
  list_free<kListed>(first, mine, n, pages, free, count,
                     [&](unsigned i) { return sWord[i - first / 32]; });
}

uint64_t free_pieces(const PagedFreeParams &p) {
  return (uint64_t)p.sequences * ((p.tableStride + 64 * kSlots - 1) / (64 * kSlots));
}
unsigned free_markers(const PagedFreeParams &p) {
  const uint64_t parts = free_pieces(p) / 32;
  return parts < 1 ? 1u : parts < kMarkers ? (unsigned)parts : kMarkers;
}
bool free_small(const PagedFreeParams &p) {
  return p.pages <= kSmall && free_pieces(p) <= 96;
}

// -------------------------------------------------------------------- move
//
// Within the same pages two launches, so that all rows are read before any is
// written: the first makes the blocks as they will be (which keys, in a word), the
// second puts them into their places. Between pages that are apart one launch
// does both. Codes and scales are laid out for the matrix instructions (paged_kv.hpp), so
// what moves is 16 bytes (8 at D 64) for 32 (16) channels of a key, but a
// nibble of a word for a channel of a value: a thread has four channels of eight
// keys, eight loads for a store.

constexpr unsigned kMoveThreads = 256;

// A block's 16-byte words: key codes, key scales, value codes, value scales.
template <int D> struct Words {
  static constexpr unsigned KEYS = D, SCALES = D / 4, ALL = 40 * D / 16;
  static_assert(ALL == 2 * (KEYS + SCALES), "the block's parts");
};

// The key of row `row` of the keys' tile t, and of slot e of the values' quad.
__device__ __forceinline__ unsigned key_of_row(unsigned t, unsigned row) {
  return row / 8 * 16 + 8 * t + row % 8;
}
__device__ __forceinline__ unsigned key_of_slot(unsigned quad, unsigned e) {
  return 16 * (quad / 2) + 4 * (quad % 2) + 8 * (e / 4) + e % 4;
}
__device__ __forceinline__ unsigned quad_of(unsigned key) { return key / 16 * 2 + key / 4 % 2; }
__device__ __forceinline__ unsigned slot_of(unsigned key) { return key / 8 % 2 * 4 + key % 4; }

// The bits of 32-bit word j of the block's 16-byte word c that belong to the
// keys of `live`.
template <int D> __device__ __forceinline__ uint32_t bits_of(unsigned c, unsigned j, uint32_t live) {
  using W = Words<D>;
  auto all = [&](unsigned key) { return live >> key & 1 ? ~0u : 0u; };
  if (c < W::KEYS) { // (a tile's are D / 2; at D 64 two rows a word)
    const unsigned t = c / (D / 2), row = D >= 128 ? c % 16 : c % 8 * 2 + j / 2;
    return all(key_of_row(t, row));
  }
  c -= W::KEYS;
  if (c < W::SCALES)
    return all(key_of_row(c / (D / 8), c % 4 * 4 + j));
  c -= W::SCALES;
  uint32_t bits = 0;
  if (c < W::KEYS) {
    for (unsigned e = 0; e < 8; ++e)
      bits |= live >> key_of_slot(c / 16 % 4, e) & 1 ? 15u << paged_nibble(e) : 0u;
    return bits;
  }
  c -= W::KEYS;
  for (unsigned e = 0; e < 2; ++e)
    bits |= live >> key_of_slot(c % 4, 2 * j + e) & 1 ? 0xFFFFu << 16 * e : 0u;
  return bits;
}

// Word c of a block, x in the bits of the keys of `live`.
template <int D>
__device__ __forceinline__ uint4_t with_keys(uint4_t old, uint4_t x, unsigned c, uint32_t live) {
#pragma unroll
  for (unsigned j = 0; j < 4; ++j) {
    const uint32_t bits = bits_of<D>(c, j, live);
    x[j] = (old[j] & ~bits) | (x[j] & bits);
  }
  return x;
}

// D threads: one has a word of key codes, one of value codes and perhaps one of
// scales, whose loads are all in flight together.
template <int D, bool APART>
__global__ __launch_bounds__(D) void paged_gather_kernel(
    uint8_t *pool, PagedView g, const int32_t *__restrict__ source,
    const int32_t *__restrict__ sourceTable, uint32_t *live, uint4_t *blocks, unsigned *invalid) {
  using W = Words<D>;
  PagedRun b;
  if (!paged_run(g, b))
    return;
  const unsigned tid = threadIdx.x, head = blockIdx.y;
  const size_t unit = (size_t)blockIdx.x * g.kvHeads + head;
  size_t target = 0;
  if (APART) {
    const bool placed = b.ok && paged_block(g, b.seq, b.base, head, target);
    if (!placed) {
      if (invalid && tid == 0)
        atomicOr(invalid, kPagedPlace);
      return;
    }
  }
  __shared__ const uint8_t *sBlock[32]; // of the keys of this block
  __shared__ unsigned sKey[32], sLive;
  if (tid < 64) {
    const bool mine = b.ok && tid >= b.first && tid < b.last;
    const int from = mine ? source[b.row + (tid - b.first)] : -1;
    PagedView of = g;
    of.table = sourceTable;
    size_t at = 0;
    const bool found = from >= 0 && (long long)from < (long long)g.tableStride * g.pageSize &&
                       paged_block(of, b.seq, (unsigned)from, head, at);
    if (tid < 32) {
      sBlock[tid] = pool + (found ? at : 0u); // (some block's, not put anywhere)
      sKey[tid] = found ? (unsigned)from % 32 : 0u;
    }
    const uint32_t keys = (uint32_t)__builtin_amdgcn_ballot_w64(found);
    if (tid == 0) {
      sLive = keys;
      if (!APART)
        live[unit] = keys;
      if (invalid && (!b.ok || __builtin_popcount(keys) != (int)(b.last - b.first)))
        atomicOr(invalid, kPagedPlace);
    }
  }
  __syncthreads();
  const uint32_t keys = sLive;
  if (!keys)
    return;
  uint4_t *to = APART ? reinterpret_cast<uint4_t *>(pool + target) : blocks + unit * W::ALL;
  uint4_t x[3] = {0, 0, 0}, y[8];
  unsigned from[8];
  { // key codes
    const unsigned t = tid / (D / 2), chunk = tid % (D / 2) / (D >= 128 ? 16 : 8);
    if constexpr (D >= 128) {
      const unsigned key = key_of_row(t, tid % 16), of = sKey[key];
      x[0] = *reinterpret_cast<const uint4_t *>(sBlock[key] + of / 8 % 2 * 8 * D +
                                                (chunk * 16 + paged_row(of)) * 16);
    } else {
#pragma unroll
      for (unsigned n = 0; n < 2; ++n) {
        const unsigned key = key_of_row(t, tid % 8 * 2 + n), of = sKey[key];
        const uint2 z = *reinterpret_cast<const uint2 *>(sBlock[key] + of / 8 % 2 * 8 * D +
                                                         (chunk * 16 + paged_row(of)) * 8);
        x[0][2 * n] = z.x;
        x[0][2 * n + 1] = z.y;
      }
    }
  }
  if (tid < W::SCALES) { // key scales
    const unsigned t = tid / (D / 8), group = tid % (D / 8) / 4;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const unsigned key = key_of_row(t, tid % 4 * 4 + j);
      x[2][j] = *reinterpret_cast<const uint32_t *>(sBlock[key] + paged_key_scale(D, sKey[key], group));
    }
  }
  // value codes: four channels of eight keys
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) {
    const unsigned key = key_of_slot(tid / 16 % 4, e);
    from[e] = sKey[key];
    y[e] = *reinterpret_cast<const uint4_t *>(
        sBlock[key] + paged_value_word(D, quad_of(from[e]), 64 * (tid / 64) + tid % 16));
  }
  if (tid >= W::SCALES && tid < 2 * W::SCALES) { // value scales
    const unsigned c = tid - W::SCALES, group = c / 8, bias = c / 4 % 2, quad = c % 4;
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned key = key_of_slot(quad, e), of = sKey[key];
      const uint32_t z = *reinterpret_cast<const uint16_t *>(
          sBlock[key] + paged_value_scale(D, quad_of(of), slot_of(of), group) + 64 * bias);
      x[2][e / 2] |= z << 16 * (e % 2);
    }
  }
#pragma unroll
  for (unsigned e = 0; e < 8; ++e)
    x[1] |= (y[e] >> paged_nibble(slot_of(from[e])) & 15u) << paged_nibble(e);
  // (a block's words: key codes, key scales, value codes, value scales)
  const unsigned at[3] = {tid, W::KEYS + W::SCALES + tid,
                          tid < W::SCALES ? W::KEYS + tid : 2 * W::KEYS + tid};
#pragma unroll
  for (unsigned i = 0; i < 3; ++i)
    if (i < 2 || tid < 2 * W::SCALES)
      to[at[i]] = APART && keys != ~0u ? with_keys<D>(to[at[i]], x[i], at[i], keys) : x[i];
}

template <int D>
__global__ __launch_bounds__(kMoveThreads) void paged_place_kernel(uint8_t *pool, PagedView g,
                                                                   const uint32_t *__restrict__ live,
                                                                   const uint4_t *__restrict__ blocks,
                                                                   unsigned *invalid) {
  using W = Words<D>;
  constexpr unsigned kEach = (W::ALL + kMoveThreads - 1) / kMoveThreads;
  PagedRun b;
  if (!paged_run(g, b) || !b.ok)
    return;
  const unsigned tid = threadIdx.x, head = blockIdx.y;
  const size_t unit = (size_t)blockIdx.x * g.kvHeads + head;
  const uint32_t keys = live[unit];
  size_t at;
  if (!paged_block(g, b.seq, b.base, head, at)) {
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  if (!keys)
    return;
  const uint4_t *from = blocks + unit * W::ALL;
  uint4_t *to = reinterpret_cast<uint4_t *>(pool + at), x[kEach];
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (tid + i * kMoveThreads < W::ALL)
      x[i] = from[tid + i * kMoveThreads];
  if (keys != ~0u) {
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) {
      const unsigned c = tid + i * kMoveThreads;
      if (c >= W::ALL)
        continue;
      x[i] = with_keys<D>(to[c], x[i], c, keys);
    }
  }
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (tid + i * kMoveThreads < W::ALL)
      to[tid + i * kMoveThreads] = x[i];
}

size_t move_units(const PagedKvParams &p) {
  return (size_t)paged_most_runs(p.tokens, p.sequences) * p.kvHeads;
}

} // namespace

hipError_t launch_paged_fork(const int32_t *table, const int32_t *past, const int32_t *parent,
                             const int32_t *spare, int32_t *tableOut, int32_t *pastOut, void *pool,
                             uint32_t *invalid, const PagedForkParams &p, hipStream_t stream) {
  const ForkView g{table,   past,       parent,    spare,       tableOut,     pastOut,
                   p.pages, p.pageSize, p.kvHeads, p.sequences, p.tableStride};
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(p.children * p.kvHeads * (p.pageSize / 32)), dim3(kForkThreads),
                       0, stream, g, static_cast<uint4_t *>(pool), invalid);
    return hipGetLastError();
  };
  return p.headDim == 256   ? run(paged_fork_kernel<256>)
         : p.headDim == 128 ? run(paged_fork_kernel<128>)
                            : run(paged_fork_kernel<64>);
}

unsigned paged_free_launches(const PagedFreeParams &p) { return free_small(p) ? 1 : 3; }
size_t paged_free_workspace_bytes(const PagedFreeParams &p) {
  const size_t lists = (p.pages + kListed - 1) / kListed;
  return free_small(p) ? 0 : 4 * ((free_markers(p) + 1) * (size_t)free_words(p.pages) + lists);
}
hipError_t launch_paged_free(const int32_t *table, const int32_t *lengths, int32_t *free,
                             int32_t *count, uint32_t *invalid, void *workspace,
                             const PagedFreeParams &p, hipStream_t stream) {
  const FreeView g{table, lengths, p.pages, p.pageSize, p.sequences, p.tableStride};
  if (free_small(p)) {
    hipLaunchKernelGGL(paged_free_small_kernel, dim3(1), dim3(kFreeThreads), 0, stream, g, free,
                       count, invalid);
    return hipGetLastError();
  }
  const unsigned parts = free_markers(p), windows = (p.pages + kWindow - 1) / kWindow;
  const unsigned lists = (p.pages + kListed - 1) / kListed;
  const size_t words = free_words(p.pages);
  uint32_t *marks = static_cast<uint32_t *>(workspace);
  const FreeMarks m{marks, marks + parts * words, marks + (parts + 1) * words};
  hipLaunchKernelGGL(paged_free_mark_kernel, dim3(parts, windows), dim3(kFreeThreads), 0, stream, g,
                     m.parts, invalid);
  if (hipError_t e = hipGetLastError())
    return e;
  hipLaunchKernelGGL(paged_free_join_kernel, dim3(lists), dim3(kJoinThreads), 0, stream, m, parts,
                     p.pages);
  if (hipError_t e = hipGetLastError())
    return e;
  hipLaunchKernelGGL(paged_free_list_kernel, dim3(lists), dim3(kFreeThreads), 0, stream, m, p.pages,
                     free, count);
  return hipGetLastError();
}

size_t paged_move_workspace_bytes(const PagedKvParams &p) {
  const size_t units = move_units(p);
  return units * 40 * p.headDim + (units * 4 + 15) / 16 * 16;
}
hipError_t launch_paged_move(const int32_t *source, const int32_t *sourceTable,
                             const int32_t *starts, const int32_t *past, const int32_t *table,
                             void *pool, uint32_t *invalid, void *workspace, const PagedKvParams &p,
                             hipStream_t stream) {
  const PagedView g = paged_view(p, starts, past, table);
  uint4_t *blocks = static_cast<uint4_t *>(workspace);
  uint32_t *live = reinterpret_cast<uint32_t *>(blocks + move_units(p) * (40 * p.headDim / 16));
  const dim3 grid(paged_most_runs(p.tokens, p.sequences), p.kvHeads);
  uint8_t *pages = static_cast<uint8_t *>(pool);
  const bool apart = sourceTable != nullptr;
  auto run = [&](auto move, auto gather, auto place) {
    hipLaunchKernelGGL(apart ? move : gather, grid, dim3(p.headDim), 0, stream, pages, g, source,
                       apart ? sourceTable : table, live, blocks, invalid);
    if (hipError_t e = hipGetLastError())
      return e;
    if (apart)
      return hipSuccess;
    hipLaunchKernelGGL(place, grid, dim3(kMoveThreads), 0, stream, pages, g, live, blocks, invalid);
    return hipGetLastError();
  };
  return p.headDim == 256   ? run(paged_gather_kernel<256, true>, paged_gather_kernel<256, false>,
                                  paged_place_kernel<256>)
         : p.headDim == 128 ? run(paged_gather_kernel<128, true>, paged_gather_kernel<128, false>,
                                  paged_place_kernel<128>)
                            : run(paged_gather_kernel<64, true>, paged_gather_kernel<64, false>,
                                  paged_place_kernel<64>);
}

} // namespace llmi
