// Appending to, and reading back from, the paged 4-bit cache (paged_kv.hpp).
//
// A block's part of a call (the rows of a sequence that lie in 32 keys of one
// KV head) is the work of a few workgroups: one for its values, the others
// each for some of its keys. A value word holds eight keys and is read, filled
// in and written back by the one workgroup that has them, without atomics; a
// key's words are its own.
//
// Traced, 2048 rows of 4 heads of 256 take 8.4 us (11 MB: 1.3 TB/s), 6357 rows of
// 8 heads of 128 in 13 sequences 17.6 us (34 MB: 1.9 TB/s). Bound by vector
// instructions, about 35 a value (converted, rotated, compared, quantized,
// transposed; 12 of the 17.6 us and 4 of the 8.4 if nothing else were), and by
// latency: lengths, table and rows, one load after the other. Reading them back
// takes 5.6 and 10.2 us (2.0 and 3.4 TB/s), the values' codes through two-byte
// writes to LDS.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "rope_rows.hpp"

namespace llmi {
namespace {

constexpr unsigned kThreads = 256;

struct AppendRows {
  unsigned keyToken, keyHead, valueToken, valueHead, half, layout, heads; // heads: of a workgroup
  float factor;
};

// Blocks that a sequence's rows touch.
__device__ __forceinline__ unsigned touched_blocks(const PagedSeq &q) {
  return q.rows ? (q.past % 32 + q.rows + 31) / 32 : 0u;
}
// At most as many units as that over any sequences: n rows touch at most
// (n + 62) / 32 blocks, and at most n.
unsigned most_units(unsigned tokens, unsigned sequences) {
  const uint64_t n = (uint64_t)tokens / 32 + 2 * (uint64_t)sequences;
  return (unsigned)(n < tokens ? n : tokens);
}

// Keys that one workgroup takes of a block: eight channels a thread.
constexpr unsigned keys_a_group(unsigned D) { return 8 * kThreads / D; }
constexpr unsigned key_groups(unsigned D) { return 32 / keys_a_group(D); }

// Eight neighbouring channels of a key or value, and what a group has in
// common: a thread's eight are a quarter of one.
struct Eight {
  float v[8];
};
__device__ __forceinline__ Eight eight_of(const uint16_t (&x)[8]) {
  Eight y;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y.v[e] = h2f(x[e]);
  return y;
}
__device__ __forceinline__ void ends_of(const Eight &x, float &lo, float &hi) {
  lo = fminf(fminf(x.v[0], x.v[1]), x.v[2]);
  hi = fmaxf(fmaxf(x.v[0], x.v[1]), x.v[2]);
#pragma unroll
  for (int e = 3; e < 7; e += 2) {
    lo = fminf(fminf(lo, x.v[e]), x.v[e + 1]);
    hi = fmaxf(fmaxf(hi, x.v[e]), x.v[e + 1]);
  }
  lo = fminf(lo, x.v[7]);
  hi = fmaxf(hi, x.v[7]);
}
// What the cache holds of values that are not finite or past the limit (lo
// and hi of the others are theirs); whether there were any: without their
// signs, the bits of fp16 values are in order, NaN behind the infinities.
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ bool keep(const uint16_t (&raw)[8], Eight &x, float &lo, float &hi) {
  static_assert(kPagedLimit == 16384.0f, "its bits below");
  ushort2_t most{0, 0};
#pragma unroll
  for (int e = 0; e < 8; e += 2)
    most = __builtin_elementwise_max(
        most, ushort2_t{(uint16_t)(raw[e] & 0x7FFFu), (uint16_t)(raw[e + 1] & 0x7FFFu)});
  if (max((unsigned)most[0], (unsigned)most[1]) <= 0x7400u)
    return false;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    x.v[e] = x.v[e] != x.v[e] ? 0.0f : __builtin_amdgcn_fmed3f(x.v[e], -kPagedLimit, kPagedLimit);
  ends_of(x, lo, hi);
  return true;
}

// A group's scale and bias. d / 15 as the product with 1 / 15 corrected by its
// exact remainder is the quotient rounded once (Markstein: the reciprocal is
// 1 / 15 rounded to nearest and nothing here underflows, d being 0 or at
// least 2^-24).
struct Group {
  half_t scale, bias;
  float s, b, inv;
};
__device__ __forceinline__ Group group_of(float low, float high) {
  constexpr float k15th = 1.0f / 15.0f;
  const float d = high - low, q = apart(d * k15th);
  Group g;
  g.scale = (half_t)apart(__builtin_fmaf(__builtin_fmaf(-15.0f, q, d), k15th, q));
  g.s = (float)g.scale;
  g.bias = (half_t)apart(__builtin_fmaf(-16.0f, g.s, low)); // (16 s is exact)
  g.b = (float)g.bias;
  g.inv = g.s > 0.0f ? __builtin_amdgcn_rcpf(g.s) : 0.0f;
  return g;
}
// The eight codes clamp(rint((x - b) / s) - 16, 0, 15), code e in nibble e / 2
// + 4 (e % 2). The quotients, clamped to [16, 31] first: as a product with the
// hardware's reciprocal they are within 2^-17 of the division's (at most 32,
// off by the reciprocal's step and two half steps of fp32), so where none of
// the eight lies within 2^-16 of a rounding border they stand, and else the
// divisions decide. Four codes are put together as a whole number of fp32.
__device__ __forceinline__ uint32_t codes_of(const Eight &x, const Group &g) {
  float q[8], r[8], border = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = __builtin_amdgcn_fmed3f(apart(x.v[e] - g.b) * g.inv, 16.0f, 31.0f);
    r[e] = __builtin_rintf(q[e]);
    border = fmaxf(border, fabsf(q[e] - r[e]));
  }
  if (border > 0.5f - 0x1p-16f && g.s > 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r[e] = __builtin_rintf(__builtin_amdgcn_fmed3f(__fdiv_rn(x.v[e] - g.b, g.s), 16.0f, 31.0f));
  }
  // 16 (1 + 16 + 256 + 4096) less: the 16s of the quotients
  uint32_t half[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    half[h] = (uint32_t)__builtin_fmaf(
        r[6 + h], 4096.0f,
        __builtin_fmaf(r[4 + h], 256.0f, __builtin_fmaf(r[2 + h], 16.0f, r[h] - 69904.0f)));
  return half[0] | half[1] << 16;
}

// Eight channels of a key, and those that they are rotated with. VEC: rows at
// 16 bytes, and a word's partners a word.
struct KeyPart {
  uint16_t own[8], other[8];
};
template <bool VEC>
__device__ __forceinline__ void load_eight(const uint16_t *__restrict__ x, uint16_t (&to)[8]) {
  *reinterpret_cast<uint4_t *>(to) = load_word<VEC>(x);
}
template <bool VEC>
__device__ __forceinline__ KeyPart load_key(const uint16_t *__restrict__ x, unsigned word,
                                            const AppendRows &p) {
  KeyPart k;
  const unsigned c0 = 8 * word;
  load_eight<VEC>(x + c0, k.own);
  const unsigned far = c0 >= 2 * p.half || p.layout ? c0 : c0 < p.half ? c0 + p.half : c0 - p.half;
  if (VEC || far == c0 || c0 + 8 <= p.half || (c0 >= p.half && c0 + 8 <= 2 * p.half)) {
    load_eight<VEC>(x + far, k.other);
    if (!VEC && p.layout)
#pragma unroll
      for (unsigned e = 0; e < 8; ++e)
        k.other[e] = k.own[e ^ 1];
  } else { // a word of both halves, or of the second and the rest
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned c = c0 + e;
      k.other[e] = x[c >= 2 * p.half ? c : c < p.half ? c + p.half : c - p.half];
    }
  }
  return k;
}

// `word` of key `key`: rotated, quantized (four neighbours have a group),
// stored; whether it had a value that the cache cannot hold.
template <int D, bool VEC>
__device__ __forceinline__ bool append_key(const KeyPart &k, unsigned word, unsigned key,
                                           const float2 *__restrict__ turns, uint8_t *block,
                                           const AppendRows &p) {
  const unsigned c0 = 8 * word;
  const uint16_t(&own)[8] = k.own, (&other)[8] = k.other;
  const bool low = c0 < p.half;
  uint16_t y[8];
#pragma unroll
  for (unsigned e = 0; e < 8; ++e)
    y[e] = own[e];
  if (VEC) {
    if (c0 < 2 * p.half) { // (all eight or none)
#pragma unroll
      for (unsigned e = 0; e < 8; ++e) {
        const float2 cs = turns[p.layout ? c0 / 2 + e / 2 : (low ? c0 : c0 - p.half) + e];
        const bool first = p.layout ? e % 2 == 0 : low;
        y[e] = turn(h2f(own[e]), h2f(p.layout ? own[e ^ 1] : other[e]), cs.x,
                    first ? -cs.y : cs.y);
      }
    }
  } else {
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned c = c0 + e;
      if (c < 2 * p.half) {
        const bool first = p.layout ? e % 2 == 0 : c < p.half;
        const float2 cs = turns[p.layout ? c / 2 : first ? c : c - p.half];
        y[e] = turn(h2f(own[e]), h2f(other[e]), cs.x, first ? -cs.y : cs.y);
      }
    }
  }
  Eight v = eight_of(y);
  float lo, hi;
  ends_of(v, lo, hi);
  const bool bad = keep(y, v, lo, hi);
  lo = fminf(lo, dpp<kDppXor1>(lo));
  hi = fmaxf(hi, dpp<kDppXor1>(hi));
  lo = fminf(lo, dpp<kDppXor2>(lo));
  hi = fmaxf(hi, dpp<kDppXor2>(hi));
  const Group g = group_of(lo, hi);
  *reinterpret_cast<uint32_t *>(block + paged_key_word(D, key, word)) = codes_of(v, g);
  if (word % 4 == 0)
    *reinterpret_cast<half2_t *>(block + paged_key_scale(D, key, word / 4)) =
        half2_t{g.scale, g.bias};
  return bad;
}

// Values: a wave has 64 channels of a quad's eight keys, lane slot + 8 c the
// channels 8 c .. 8 c + 7 of one key (a group is the lanes whose c / 4 is the
// same). Where the wave's eight lanes of a c have a word of channels each,
// the cache has a word of keys for each channel: a transposition of nibbles.
__device__ __forceinline__ unsigned value_key(unsigned quad) {
  const unsigned slot = threadIdx.x % 8;
  return 16 * (quad / 2) + 8 * (slot / 4) + 4 * (quad % 2) + slot % 4;
}
__device__ __forceinline__ uint32_t swapped(uint32_t mine, uint32_t theirs, bool upper,
                                            uint32_t low_mask, unsigned shift) {
  // the lower lane keeps its low parts and takes the other's to its high ones
  return upper ? (theirs >> shift & low_mask) | (mine & ~low_mask)
               : (mine & low_mask) | (theirs << shift & ~low_mask);
}
// Nibble n of lane i to nibble i of lane n, in each eight lanes.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  const unsigned i = threadIdx.x % 8;
  uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor1, 0xF, 0xF, false);
  x = swapped(x, other, i & 1, 0x0F0F0F0Fu, 4);
  other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor2, 0xF, 0xF, false);
  x = swapped(x, other, i & 2, 0x00FF00FFu, 8);
  // lane i ^ 4: the half row mirrored is i ^ 7, and that quad reversed i ^ 4
  other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppRowHalfMirror, 0xF, 0xF, false);
  other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)other, 0x1B, 0xF, 0xF, false);
  return swapped(x, other, i & 4, 0x0000FFFFu, 16);
}

template <int D>
__device__ __forceinline__ bool append_values(const uint16_t (&x)[8], unsigned quad, bool here,
                                              unsigned st, uint8_t *block) {
  const unsigned lane = threadIdx.x % 64, slot = lane % 8, c = lane / 8;
  Eight v = eight_of(x);
  float lo, hi;
  ends_of(v, lo, hi);
  const bool bad = keep(x, v, lo, hi) && here;
  lo = fminf(lo, row_ror<8>(lo));
  hi = fmaxf(hi, row_ror<8>(hi));
  LanePair p = pair16(lo);
  lo = fminf(p.a, p.b);
  p = pair16(hi);
  hi = fmaxf(p.a, p.b);
  const Group g = group_of(lo, hi);
  // Channel e is in nibble e / 2 + 4 (e % 2) of a word, and slot e of keys goes
  // there too: the lanes give their words in that order, and nibble n is
  // channel 2 (n % 4) + n / 4.
  const unsigned turned = 2 * (slot % 4) + slot / 4;
  uint32_t word = transposed((uint32_t)__builtin_amdgcn_ds_bpermute(
      (int)(4 * ((lane & 56u) + turned)), (int)codes_of(v, g)));
  const unsigned channel = 64 * st + 8 * c + turned;
  uint32_t *to = reinterpret_cast<uint32_t *>(block + paged_value_word(D, quad, channel));
  const unsigned long long all = __builtin_amdgcn_ballot_w64(here);
  if (~all) { // nibbles of keys that are here
    const unsigned long long there = all >> (lane & 56u);
    uint32_t mask = 0;
#pragma unroll
    for (unsigned e = 0; e < 8; ++e)
      mask |= there >> e & 1 ? 15u << paged_nibble(e) : 0u;
    if (mask != 0xFFFFFFFFu)
      word = (word & mask) | (*to & ~mask);
  }
  *to = word;
  if (here && c % 4 == 0) {
    half_t *s =
        reinterpret_cast<half_t *>(block + paged_value_scale(D, quad, slot, 2 * st + c / 4));
    s[0] = g.scale;
    s[32] = g.bias;
  }
  return bad;
}

// Where a workgroup's block lies in its sequence and in the call.
struct AppendBlock {
  unsigned seq, base, first, last, row; // keys [first, last) at position base, from row `row`
  bool ok;
};
__device__ __forceinline__ bool find_block(const PagedView &g, AppendBlock &b) {
  unsigned local, before;
  const PagedSeq own = paged_own(g);
  if (!paged_find(g, own, blockIdx.x, [](const PagedSeq &q) { return touched_blocks(q); }, b.seq,
                  local, before))
    return false;
  const PagedSeq q = paged_seq_of(g, own, b.seq);
  b.base = q.past / 32 * 32 + 32 * local;
  b.first = b.base < q.past ? q.past - b.base : 0u;
  b.last = min(32u, q.past + q.rows - b.base);
  b.row = q.row0 + (b.base + b.first - q.past);
  b.ok = q.ok;
  return true;
}

template <int D, bool VEC>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(
    const uint16_t *__restrict__ keys, const uint16_t *__restrict__ values, PagedView g,
    const float *__restrict__ freqs, uint8_t *pool, unsigned *invalid, AppendRows p) {
  extern __shared__ float2 sTurn[]; // [key of this workgroup][half]
  AppendBlock b;
  if (!find_block(g, b))
    return;
  // blockIdx.z: the values of one of this workgroup's heads (first: they take
  // longest), then groups of keys. Rows are loaded before the place they go
  // to is known.
  const unsigned tid = threadIdx.x, head0 = blockIdx.y * p.heads;
  const bool ofValues = blockIdx.z < p.heads;
  const unsigned part = blockIdx.z - p.heads;
  const unsigned first = ofValues ? b.first : max(b.first, keys_a_group(D) * part);
  const unsigned last = ofValues ? b.last : min(b.last, keys_a_group(D) * (part + 1));
  const unsigned head = head0 + (ofValues ? blockIdx.z : 0u);
  if (first >= last || head >= g.kvHeads)
    return;
  const size_t row = b.row + (first - b.first);
  size_t at = 0;
  bool bad = false;
  auto place = [&]() {
    const bool placed = b.ok && paged_block(g, b.seq, b.base, head, at);
    if (!placed && invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return placed;
  };
  if (ofValues) {
    // this wave's tasks (64 channels of a quad's keys) are wave, wave + 4, ...
    const uint16_t *x = values + row * p.valueToken + (size_t)head * p.valueHead + tid % 64 / 8 * 8;
    constexpr unsigned kTasks = 4 * (D / 64), kEach = kTasks / (kThreads / 64);
    uint16_t raw[kEach][8];
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) {
      const unsigned task = tid / 64 + i * (kThreads / 64), key = value_key(task / (D / 64));
      const unsigned from = key >= first && key < last ? key - first : 0u; // (some row of the call's)
      load_eight<VEC>(x + (size_t)from * p.valueToken + 64 * (task % (D / 64)), raw[i]);
    }
    if (!place())
      return;
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) {
      const unsigned task = tid / 64 + i * (kThreads / 64), key = value_key(task / (D / 64));
      const bool here = key >= first && key < last;
      if (__builtin_amdgcn_ballot_w64(here))
        bad |= append_values<D>(raw[i], task / (D / 64), here, task % (D / 64), pool + at);
    }
  } else {
    const unsigned heads = min(p.heads, g.kvHeads - head0);
    const unsigned k = tid / (D / 8), word = tid % (D / 8);
    const bool mine = k < last - first;
    const uint16_t *x = keys + (row + (mine ? k : 0u)) * p.keyToken + (size_t)head * p.keyHead;
    KeyPart next = load_key<VEC>(x, word, p);
    if (p.half) {
      const unsigned down = kThreads / p.half, right = kThreads % p.half;
      unsigned n = tid / p.half, pair = tid % p.half;
      while (n < last - first) {
        sTurn[n * p.half + pair] = rope_turn((int)(b.base + first + n), freqs[pair], p.factor);
        n += down;
        pair += right;
        if (pair >= p.half) {
          pair -= p.half;
          ++n;
        }
      }
    }
    if (!place())
      return;
    __syncthreads();
    const size_t nextHead = (size_t)(g.pageSize / 32) * (40 * D); // (of the same page)
    for (unsigned h = 0; h < heads; ++h) {
      const KeyPart now = next;
      if (h + 1 < heads)
        next = load_key<VEC>(x + (size_t)(h + 1) * p.keyHead, word, p);
      if (mine)
        bad |= append_key<D, VEC>(now, word, first + k, sTurn + k * p.half,
                                  pool + at + h * nextHead, p);
    }
  }
  if (invalid && __builtin_amdgcn_ballot_w64(bad) && tid % 64 == 0)
    atomicOr(invalid, kPagedValue);
}

// The cache's values of a block's rows, keys (blockIdx.z 0) or values: a lane
// decodes 16 bytes of codes as they lie, and the rows leave through LDS, 16
// bytes a thread.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(const uint8_t *__restrict__ pool,
                                                              PagedView g, uint16_t *keys,
                                                              uint16_t *values,
                                                              unsigned *invalid) {
  constexpr unsigned PITCH = D + 8;
  __shared__ __attribute__((aligned(16))) half_t sRow[32 * PITCH];
  AppendBlock b;
  if (!find_block(g, b))
    return;
  const unsigned head = blockIdx.y, tid = threadIdx.x, lane = tid % 64;
  size_t at = 0;
  const bool ok = b.ok && paged_block(g, b.seq, b.base, head, at);
  if (!ok && invalid && tid == 0)
    atomicOr(invalid, kPagedPlace);
  const uint8_t *block = pool + at;
  const Nibbles nibbles;
  if (ok && blockIdx.z == 0) {
    for (unsigned i = tid; i < 4 * D; i += kThreads) { // words: key, eight channels
      const unsigned key = i / (D / 8), word = i % (D / 8);
      const uint32_t w = *reinterpret_cast<const uint32_t *>(block + paged_key_word(D, key, word));
      const half2_t m =
          *reinterpret_cast<const half2_t *>(block + paged_key_scale(D, key, word / 4));
      *reinterpret_cast<half8_t *>(sRow + key * PITCH + 8 * word) = paged_eight(w, m, nibbles);
    }
  } else if (ok) {
    const unsigned quad = lane / 16, r = lane % 16;
    for (unsigned st = tid / 64; st < D / 64; st += kThreads / 64) {
      const uint4_t w =
          *reinterpret_cast<const uint4_t *>(block + paged_value_word(D, quad, 64 * st + r));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t *m = block + paged_value_scale(D, quad, 0, 2 * st + j / 2);
        const half8_t sc = *reinterpret_cast<const half8_t *>(m);
        const half8_t bi = *reinterpret_cast<const half8_t *>(m + 64);
#pragma unroll
        for (unsigned e = 0; e < 8; ++e)
          sRow[(16 * (quad / 2) + 8 * (e / 4) + 4 * (quad % 2) + e % 4) * PITCH + 64 * st +
               16 * j + r] = paged_value(w[j], e, sc[e], bi[e]);
      }
    }
  }
  __syncthreads();
  uint16_t *to = blockIdx.z ? values : keys;
  const uint32_t nan = 0x7E007E00u;
  for (unsigned i = tid; i < (b.last - b.first) * (D / 8); i += kThreads) {
    const unsigned k = i / (D / 8), c = 8 * (i % (D / 8));
    *reinterpret_cast<uint4_t *>(to + ((size_t)(b.row + k) * g.kvHeads + head) * D + c) =
        ok ? *reinterpret_cast<const uint4_t *>(sRow + (b.first + k) * PITCH + c)
           : uint4_t{nan, nan, nan, nan};
  }
}

} // namespace

hipError_t launch_paged_append(const uint16_t *keys, const uint16_t *values, const int32_t *starts,
                               const int32_t *past, const int32_t *table, const float *freqs,
                               void *pool, uint32_t *invalid, const PagedKvParams &p,
                               const PagedAppendParams &a, hipStream_t stream) {
  const PagedView g = paged_view(p, starts, past, table);
  const unsigned units = most_units(p.tokens, p.sequences), groups = key_groups(p.headDim);
  // A workgroup's turns serve as many heads as leave two workgroups a CU (6357
  // rows of 8 heads of 128, all of them rotated: 28.6 us with their reading
  // back, 34.3 with a head a workgroup).
  unsigned heads = 1;
  while (2 * heads <= p.kvHeads &&
         (uint64_t)units * groups * ((p.kvHeads + 2 * heads - 1) / (2 * heads)) >= 512)
    heads *= 2;
  const AppendRows r{a.keyTokenStride, a.keyHeadStride, a.valueTokenStride, a.valueHeadStride,
                     a.rotaryDim / 2,  a.layout,        heads,              a.factor};
  const dim3 grid(units, (p.kvHeads + heads - 1) / heads, groups + heads);
  const size_t lds = keys_a_group(p.headDim) * r.half * sizeof(float2);
  // (half % 8: a word's channels are all of one half, and their partners a word)
  const bool vec = (a.layout || r.half % 8 == 0) && r.half % 4 == 0 && aligned16(keys) &&
                   aligned16(values) &&
                   (a.keyTokenStride | a.keyHeadStride | a.valueTokenStride | a.valueHeadStride) %
                           8 == 0;
  auto run = [&](auto wide, auto any) {
    hipLaunchKernelGGL(vec ? wide : any, grid, dim3(kThreads), lds, stream, keys, values, g, freqs,
                       static_cast<uint8_t *>(pool), invalid, r);
    return hipGetLastError();
  };
  switch (p.headDim) {
  case 256:
    return run(paged_append_kernel<256, true>, paged_append_kernel<256, false>);
  case 128:
    return run(paged_append_kernel<128, true>, paged_append_kernel<128, false>);
  default:
    return run(paged_append_kernel<64, true>, paged_append_kernel<64, false>);
  }
}

hipError_t launch_paged_read(const void *pool, const int32_t *starts, const int32_t *past,
                             const int32_t *table, uint16_t *keys, uint16_t *values,
                             uint32_t *invalid, const PagedKvParams &p, hipStream_t stream) {
  const PagedView g = paged_view(p, starts, past, table);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(most_units(p.tokens, p.sequences), p.kvHeads, 2),
                       dim3(kThreads), 0, stream, static_cast<const uint8_t *>(pool), g, keys,
                       values, invalid);
    return hipGetLastError();
  };
  return p.headDim == 256   ? run(paged_read_kernel<256>)
         : p.headDim == 128 ? run(paged_read_kernel<128>)
                            : run(paged_read_kernel<64>);
}

} // namespace llmi
