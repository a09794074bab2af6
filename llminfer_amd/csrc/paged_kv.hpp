// The paged 4-bit KV cache on the device: where a pool keeps a key and a
// value, and the sequences of a call.
//
// A pool is [pages][kvHeads][pageSize / 32] blocks of 40 D bytes, a block the
// 32 keys of one KV head that follow each other, as the matrix instructions
// take them:
//   16 D  key codes    [t 2][D/128][quad 4][row 16][32 channels]   (D 64: 16)
//    4 D  key scales   [t 2][D/32][row 16]{scale, bias}            fp16
//   16 D  value codes  [D/64][quad 4][D%16 16][4][8 keys]
//    4 D  value scales [D/32]{scales, biases}[quad 4][8 keys]      fp16
// Key 16 m + 8 t + 4 h + v of a block is row 8 m + 4 h + v of the keys' tile
// t, and slot 4 t + v of the values' quad 2 m + h: the keys that a lane of
// the 16x16 score tiles holds are then the eight of one value word. Slot e of
// a word (for keys: channel 8 w + e of word w) is nibble e / 2 + 4 (e % 2),
// so that one mask gives two neighbours, 16 bits apart.
//
// A group is 32 channels of one key or value: scale s = fp16((max - min) /
// 15), bias b = fp16(min - 16 s), code = clamp(rint((x - b) / s) - 16, 0, 15),
// and a code stands for fp16((16 + code) s + b): with the 16 in it, the value
// is one packed fma on nibbles put behind the fp16 exponent of 16.
#pragma once

#include "hip_common.hpp"
#include "llminfer_hip.h"

namespace llmi {

constexpr float kPagedLimit = 16384.0f; // values are kept to +-this: 16 s and b stay finite

// invalid bits
constexpr unsigned kPagedValue = 1u; // a value not finite or past the limit
constexpr unsigned kPagedPlace = 2u; // a row whose place is not in its table or the pool

struct PagedView {
  const int32_t *starts, *past, *table;
  unsigned pages, pageSize, kvHeads, dim, sequences, tableStride, tokens;
};

inline PagedView paged_view(const PagedKvParams &p, const int32_t *starts, const int32_t *past,
                            const int32_t *table) {
  return PagedView{starts,     past,        table,         p.pages,  p.pageSize, p.kvHeads,
                   p.headDim, p.sequences, p.tableStride, p.tokens};
}

// Rows [row0, row0 + rows) of the call, at positions past + i. ok: they fit
// their table.
struct PagedSeq {
  unsigned row0, rows, past;
  bool ok;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedView &g, unsigned s) {
  const int T = (int)g.tokens;
  const int lo = min(max(g.starts[s], 0), T), hi = min(max(g.starts[s + 1], lo), T);
  const int past = g.past[s];
  const long long last = (long long)past + (hi - lo);
  PagedSeq q;
  q.row0 = (unsigned)lo;
  q.rows = (unsigned)(hi - lo);
  q.past = (unsigned)past;
  q.ok = past >= 0 && last <= (long long)g.tableStride * g.pageSize;
  return q;
}

// Byte offset of the block of position pos (a multiple of 32 below the
// table's end); false if its page is not in the pool.
__device__ __forceinline__ bool paged_block(const PagedView &g, unsigned s, unsigned pos,
                                            unsigned head, size_t &at) {
  const unsigned slot = pos / g.pageSize;
  const unsigned page = (unsigned)g.table[(size_t)s * g.tableStride + slot];
  const unsigned block = (pos - slot * g.pageSize) / 32;
  const bool ok = page < g.pages;
  at = (((size_t)(ok ? page : 0u) * g.kvHeads + head) * (g.pageSize / 32) + block) *
       (size_t)(40 * g.dim);
  return ok;
}

// Places in a block. `key` is 0..31, `word` channels 8 word .. 8 word + 7.
__host__ __device__ constexpr unsigned paged_row(unsigned key) {
  return (key >> 4) * 8 + (key & 7);
}
__device__ __forceinline__ unsigned paged_key_word(unsigned D, unsigned key, unsigned word) {
  const unsigned words = D >= 128 ? 4 : 2; // of a lane's chunk
  const unsigned chunk = word / words;
  return ((key >> 3) & 1) * 8 * D + (chunk / 4) * 256 * words +
         ((chunk % 4) * 16 + paged_row(key)) * 4 * words + 4 * (word % words);
}
__device__ __forceinline__ unsigned paged_key_scale(unsigned D, unsigned key, unsigned group) {
  return 16 * D + ((key >> 3) & 1) * 2 * D + (group * 16 + paged_row(key)) * 4;
}
// A value's, of the quad and slot that hold its key; the bias is 64 bytes
// behind the scale.
__device__ __forceinline__ unsigned paged_value_word(unsigned D, unsigned quad, unsigned channel) {
  return 20 * D + (channel / 64) * 1024 + (quad * 16 + channel % 16) * 16 + (channel / 16 % 4) * 4;
}
__device__ __forceinline__ unsigned paged_value_scale(unsigned D, unsigned quad, unsigned slot,
                                                      unsigned group) {
  return 36 * D + group * 128 + (quad * 8 + slot) * 2;
}
// Bit of slot e's nibble in its word.
__host__ __device__ constexpr unsigned paged_nibble(unsigned e) { return 4 * (e / 2) + 16 * (e % 2); }

// The mask of two nibbles and the exponent that they are put behind, in
// registers: as literals they would be two instructions and not one.
struct Nibbles {
  uint32_t mask = 0x03C003C0u, exponent = 0x4C004C00u;
  __device__ __forceinline__ Nibbles() {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(exponent));
  }
};

// The two values of slots 2 j and 2 j + 1 of a word, with their scales and biases.
template <int J>
__device__ __forceinline__ half2_t paged_pair(uint32_t word, half2_t scale, half2_t bias,
                                              const Nibbles &n) {
  // the nibble to mantissa bits 6..9 of an fp16 in [16, 32): 16 + code
  const uint32_t moved = J == 0 ? word << 6 : J == 1 ? word << 2 : J == 2 ? word >> 2 : word >> 6;
  const half2_t x = __builtin_bit_cast(half2_t, (moved & n.mask) | n.exponent);
  return __builtin_elementwise_fma(x, scale, bias);
}
// The eight values of a word, in the order of its slots.
__device__ __forceinline__ half8_t paged_eight(uint32_t u, half8_t scale, half8_t bias,
                                               const Nibbles &n) {
  const half2_t v0 = paged_pair<0>(u, half2_t{scale[0], scale[1]}, half2_t{bias[0], bias[1]}, n);
  const half2_t v1 = paged_pair<1>(u, half2_t{scale[2], scale[3]}, half2_t{bias[2], bias[3]}, n);
  const half2_t v2 = paged_pair<2>(u, half2_t{scale[4], scale[5]}, half2_t{bias[4], bias[5]}, n);
  const half2_t v3 = paged_pair<3>(u, half2_t{scale[6], scale[7]}, half2_t{bias[6], bias[7]}, n);
  return half8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}
// The same with one scale and bias, side by side in 32 bits.
__device__ __forceinline__ half8_t paged_eight(uint32_t u, half2_t both, const Nibbles &n) {
  const half_t s = both[0], b = both[1];
  return paged_eight(u, half8_t{s, s, s, s, s, s, s, s}, half8_t{b, b, b, b, b, b, b, b}, n);
}
__device__ __forceinline__ half_t paged_value(uint32_t word, unsigned e, half_t scale, half_t bias) {
  const half_t x = (half_t)(float)(16u + ((word >> paged_nibble(e)) & 15u));
  return __builtin_elementwise_fma(x, scale, bias);
}

// Sum over the wave's lanes up to this one (row shifts, then the rows' totals
// handed on).
template <int Ctrl, int Rows> __device__ __forceinline__ unsigned add_dpp(unsigned x) {
  return x + (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, Ctrl, Rows, 0xF, false);
}
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
  x = add_dpp<0x111, 0xF>(x); // row_shr 1, 2, 4, 8
  x = add_dpp<0x112, 0xF>(x);
  x = add_dpp<0x114, 0xF>(x);
  x = add_dpp<0x118, 0xF>(x);
  x = add_dpp<0x142, 0xA>(x); // row_bcast 15 into rows 1 and 3
  return add_dpp<0x143, 0xC>(x); // row_bcast 31 into rows 2 and 3
}

// The call's unit `u` of those that count(sequence) gives each sequence, in
// order: its sequence and its number there, the same scalars in every lane,
// and how many units come before the sequence's. Every lane of a full wave
// calls it; false past the last unit. `own` is paged_seq of sequence `lane`
// (nothing past the last one).
template <typename Count>
__device__ __forceinline__ bool paged_find(const PagedView &g, const PagedSeq &own, unsigned u,
                                           Count count, unsigned &seq, unsigned &local,
                                           unsigned &before) {
  const unsigned lane = threadIdx.x % 64;
  before = 0;
  PagedSeq q = own;
  for (unsigned s0 = 0; s0 < g.sequences; s0 += 64) {
    if (s0)
      q = s0 + lane < g.sequences ? paged_seq(g, s0 + lane) : PagedSeq{0, 0, 0, true};
    const unsigned n = count(q), sum = wave_scan(n);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(u - before < sum);
    if (past) {
      const int at = __builtin_ctzll(past);
      seq = s0 + (unsigned)at;
      before += (unsigned)__builtin_amdgcn_readlane((int)(sum - n), at);
      local = u - before;
      // (not so with starts out of order: a sum that wrapped)
      return local < (unsigned)__builtin_amdgcn_readlane((int)n, at);
    }
    before += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}
__device__ __forceinline__ PagedSeq paged_own(const PagedView &g) {
  const unsigned lane = threadIdx.x % 64;
  return lane < g.sequences ? paged_seq(g, lane) : PagedSeq{0, 0, 0, true};
}
// One of the sequences, the same in every lane.
__device__ __forceinline__ PagedSeq paged_seq_of(const PagedView &g, const PagedSeq &own,
                                                 unsigned seq) {
  if (seq >= 64)
    return paged_seq(g, seq);
  PagedSeq q;
  q.row0 = (unsigned)__builtin_amdgcn_readlane((int)own.row0, (int)seq);
  q.rows = (unsigned)__builtin_amdgcn_readlane((int)own.rows, (int)seq);
  q.past = (unsigned)__builtin_amdgcn_readlane((int)own.past, (int)seq);
  q.ok = __builtin_amdgcn_readlane((int)own.ok, (int)seq);
  return q;
}

} // namespace llmi
