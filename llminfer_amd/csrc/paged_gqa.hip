// Causal GQA over the paged 4-bit cache (paged_kv.hpp): a ragged batch of
// sequences, each with any number of new rows.
//
// For one sequence and KV head, the query rows of that head's group (token c /
// G, head c % G of column c) are columns of the score tiles, S^T = K Q^T with
// v_mfma_f32_16x16x32_f16, CG groups of 16 a unit. A workgroup takes one unit
// and a range of the keys; each of its waves its own blocks of 32 keys,
// without waiting for the others:
//  * a block is 40 D bytes in one piece, so it goes HBM -> LDS by DMA, 1 KB an
//    instruction, several blocks ahead and without a register;
//  * codes and scales lie in it as the matrix instructions want them: a lane
//    reads its 16 bytes of codes (a conflict-free 1 KB a wave), puts two
//    nibbles at a time behind the exponent of 16 and applies scale and bias
//    with one packed fma, which is the format's own rounding;
//  * a lane's scores are those of the eight keys whose values are one of its
//    words, so the weights go from the score tile into the O^T += V^T P^T
//    product as they are;
//  * the softmax reference moves only when a score would pass 2^15 of it.
// The weights exp2(s - reference) are rounded to fp16, the operand of the
// matrix product, a half step of each (2^-11 of it; below 2^-14, 2^-25 of the
// largest possible 2^15); their sum is of the same rounded weights, so that
// the rounding moves an output only between its values.
//
// Bound by memory from many or long sequences on: 48 tokens on up to 16385
// keys of 4 heads of 256, 577 MB, in 124 us (4.65 TB/s, the rate of a copy). A
// token on 32750 keys (42 MB) takes 18.7 us in its two launches, on 4097 keys
// 12.6 us: latencies of the lengths, the table, the first blocks, the joins.
// Keys are divided over workgroups by a plan that every workgroup makes for
// itself from the lengths in device memory (a captured call may be replayed on
// others); pagedGqaMerge joins the rows whose keys were divided.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "paged_plan.hpp"

#include <math.h>
#include <type_traits>

namespace llmi {
namespace {

constexpr unsigned kColumns = 16; // of a group
constexpr unsigned kCus = 256;

typedef __attribute__((address_space(3))) void lds_void_t;
constexpr int kBufferWord3 = 0x00020000; // gfx9 raw buffer descriptor, dword 3

__device__ __forceinline__ float4_t mfma16x16x32(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// On the host: most units and pieces a KV head that any lengths can give.
uint64_t most_units(const PagedKvParams &p, unsigned group, unsigned columns) {
  const uint64_t a = (uint64_t)p.tokens * ((group + columns - 1) / columns);
  const uint64_t b = (uint64_t)p.tokens * group / columns + p.sequences;
  return a < b ? a : b;
}
uint64_t most_pieces(const PagedKvParams &p, unsigned group, const SplitPlan &plan) {
  return plan.target + 1 + most_units(p, group, 1u << plan.shift);
}
// Units by the columns that a sequence has on average: 16 columns divide into
// most pieces and join least (one sequence, 4 KV heads of 256, 8000 keys, 32
// columns: 16.7 us, 19.8 with units of 32), more decode a key less often (64
// columns on 16000 keys of 8 heads: 31 us, 48 with 16); the units of
// paged_tiles.hip, decoded once, from 160 columns (192 on 31000 keys: 54 us, 84
// with 32; 128 on 8000: 35 and 26), or 384 at head_dim 128 (768 on 16000: 101
// and 131; 256 on 8000: 37 and 25), and from fewer in calls of many columns,
// which they fill the device with (24 sequences of 75 columns on average on
// 3000 keys: 48 us, 68). At head_dim 64, 16 columns up to 95 (64 on 8000 keys:
// 13.1 us, 15.4 with 64), 64 from there (128 on 31000: 23 us, 29).
// Pieces: as many as there are CUs (twice that at head_dim 64, where two
// workgroups share one); where single tokens have units enough that their
// different lengths count for more than the joining, up to six times as many,
// of 16 blocks at least (48 chats of up to 16385 keys: 125 us, 142 in one
// round; 12 chats of 8000: 25.7 us, 29.6 with at least 64 blocks).
struct GqaPlan {
  SplitPlan split;
  bool pooled; // eight pieces a unit or more, if the lengths give them
};
GqaPlan plan_for(const PagedKvParams &p, unsigned group) {
  const uint64_t all = (uint64_t)p.tokens * group, columns = all / p.sequences;
  const bool wide = p.headDim == 256, many = all * p.kvHeads >= (wide ? 2048u : 8192u);
  const bool tiles = p.headDim >= 128 && (columns >= (wide ? 160u : 384u) ||
                                          (many && columns >= (wide ? 48u : 96u)));
  const unsigned unit = tiles             ? paged_tiles_columns(p.headDim)
                        : p.headDim == 64 ? (columns < 96 ? 16 : 64)
                                          : (columns <= 32 ? 16 : 32);
  const unsigned cus = (kCus + p.kvHeads - 1) / p.kvHeads;
  const bool pooled = cus >= 8 * most_units(p, group, unit);
  const unsigned fill = unit == 16 && p.headDim == 64 ? 2 * cus : cus;
  const unsigned step = tiles ? 512 / p.headDim : unit == 16 && pooled ? 8 : 4;
  const bool rounds = unit == 16 && !pooled;
  return {{(unsigned)__builtin_ctz(unit), step, fill, rounds ? 6 * cus : fill,
           columns <= 16 ? 16u : 64u, tiles, unit > 16 || pooled},
          pooled};
}
// Whether some lengths that fit the table divide a unit's keys.
bool may_divide(const PagedKvParams &p, const SplitPlan &plan) {
  return (uint64_t)p.tableStride * p.pageSize > 32 * plan.step;
}

// ------------------------------------------------------------- the kernel

// W: waves of a workgroup. Eight where units have many pieces: the more of the
// keys that meet in one workgroup, the fewer partials there are to join (one
// token on 32750 keys: 18.1 us, 21.5 with four, two workgroups a CU); four
// otherwise, two workgroups a CU for single tokens, whose starts and ends then
// overlap (16 chats of 8000 keys: 33.7 us, 39.6 with eight).
template <int D, int CG, int W> struct Geo {
  static constexpr int BLOCK = 40 * D;               // bytes of a block
  static constexpr int LOADS = (BLOCK + 1023) / 1024; // 1-KB loads of one
  static constexpr int STAGE = 1024 * LOADS;
  // Blocks a wave has in LDS, and waves a SIMD.
  static constexpr int RING = CG == 1 ? (D == 256 ? 2 : D == 128 ? 4 : 3)
                                      : (D == 256 ? 3 : D == 128 ? 5 : 6);
  static constexpr int RESIDENT = CG > 1 ? 1 : D == 64 ? 4 : 2;
  static constexpr int CHUNKS = D >= 128 ? D / 128 : 1; // of a lane's key
  static constexpr int WORDS = D >= 128 ? 4 : 2;        // of a chunk
  static constexpr int TILES = D / 16;                  // output tiles
};

// The ring's buffers are variables of their own, so that the compiler sees
// that a wait for one need not be a wait for all. The first two also take the
// waves' partial outputs at the end, half of them each, and the columns' (m, l).
template <int D, int CG, int W, int I> __device__ __forceinline__ char *ring_buffer() {
  using Geom = Geo<D, CG, W>;
  constexpr int size = W * Geom::STAGE;
  static_assert(W / 2 * Geom::TILES * 1024 + W * CG * kColumns * 8 <= size, "room to join");
  __shared__ __attribute__((aligned(1024))) char buffer[size];
  return buffer;
}

// x, with y of the lanes Ctrl moves it from in the lanes of the banks.
constexpr int kRowShr4 = 0x114, kRowShr8 = 0x118, kRowShr12 = 0x11C;
template <int Ctrl, int Banks> __device__ __forceinline__ float shifted_in(float x, float y) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, x),
                                                               __builtin_bit_cast(int, y), Ctrl,
                                                               0xF, Banks, false));
}

template <int D, int CG, int W>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * W, 64 * W),
                          amdgpu_waves_per_eu(Geo<D, CG, W>::RESIDENT)))
void paged_gqa_kernel(const half_t *__restrict__ q, const uint8_t *__restrict__ pool, PagedView g,
                      half_t *out, unsigned *invalid, unsigned queryHeads, SplitPlan plan,
                      ScoreScale c, Partials parts) {
  using Geom = Geo<D, CG, W>;
  constexpr unsigned kUnit = CG * kColumns, kWaves = W;
  const unsigned G = queryHeads / g.kvHeads, kvh = blockIdx.y;
  const PagedSeq own = paged_own(g);
  const Split split = paged_split(g, own, G, plan);
  unsigned seq, local, before;
  if (!paged_find(g, own, blockIdx.x,
                  [&](const PagedSeq &s) { return split.units(s) * split.pieces(s); }, seq, local,
                  before))
    return;
  const PagedSeq s = paged_seq_of(g, own, seq);
  // (the last units first: they see most keys)
  const unsigned pieces = split.pieces(s), units = split.units(s);
  const unsigned unit = units - 1 - local / pieces, piece = local % pieces;
  const unsigned tid = threadIdx.x, lane = tid % 64, quad = lane / 16, r = lane % 16;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);

  // this lane's columns, one a group (past the unit's last: some row's, not written)
  const unsigned c0 = unit * kUnit, columns = min(kUnit, s.rows * G - c0);
  unsigned visible[CG]; // a column's last key
  size_t row[CG];
  auto token_of = [&](unsigned col) { return min((c0 + col) / G, s.rows - 1); };
  auto row_of = [&](unsigned col) {
    return ((size_t)(s.row0 + token_of(col)) * queryHeads + kvh * G + (c0 + col) % G) * D;
  };
#pragma unroll
  for (int j = 0; j < CG; ++j) {
    visible[j] = s.past + token_of(kColumns * j + r);
    row[j] = row_of(kColumns * j + r);
  }
  auto live = [&](int j) { return kColumns * j + r < columns; };
  if (!s.ok) { // no place for this sequence
    for (int j = 0; j < CG; ++j)
      if (live(j) && wave == 0)
        for (unsigned x = quad; x < D; x += 4)
          out[row[j] + x] = (half_t)NAN;
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  const unsigned least = s.past + c0 / G;                // the first column's last key
  const unsigned most = s.past + (c0 + columns - 1) / G; // the last column's
  // the keys that this wave has: to the sequence's end, or to a page that is not
  // in the pool, whose columns' outputs are NaN
  const unsigned whole = s.past + s.rows;
  unsigned end = whole;
  const unsigned length = split.length(s, pieces), b0 = min(piece * length, most / 32 + 1);
  const unsigned b1 = min(b0 + length, most / 32 + 1);
  const unsigned mine = b1 > b0 + wave ? (b1 - b0 - wave + kWaves - 1) / kWaves : 0u;

  // Block k of this wave is b0 + wave + kWaves k; a lane knows where one in 64 is.
  size_t place = 0;
  auto find_blocks = [&](unsigned k) {
    const unsigned b = b0 + wave + kWaves * (k + lane);
    bool lost = false;
    if (b < b1)
      lost = !paged_block(g, seq, 32 * b, kvh, place);
    if (const unsigned long long all = __builtin_amdgcn_ballot_w64(lost))
      end = min(end, 32 * (b0 + wave + kWaves * (k + (unsigned)__builtin_ctzll(all))));
  };
  // A block past the last is asked for with a descriptor of no bytes: it costs
  // no traffic, and the compiler's count of the loads in flight stays exact.
  auto issue = [&](unsigned k, char *buffer) {
    if (k % 64 == 0)
      find_blocks(k);
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)place, k % 64);
    const unsigned hi = __builtin_amdgcn_readlane((unsigned)(place >> 32), k % 64);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(pool + ((size_t)hi << 32 | lo)), (short)0, k < mine ? Geom::BLOCK : 0, kBufferWord3);
    char *to = buffer + wave * Geom::STAGE;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // this buffer's last reads are done
#pragma unroll
    for (int i = 0; i < Geom::LOADS; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(to + 1024 * i), 16,
                                               1024 * i + 16 * lane, 0, 0, 0);
  };

  // Q^T operands: the columns' channels as the key chunks have them.
  half8_t qv[CG][Geom::CHUNKS][Geom::WORDS];
#pragma unroll
  for (int j = 0; j < CG; ++j)
#pragma unroll
    for (int i = 0; i < Geom::CHUNKS; ++i)
#pragma unroll
      for (int w = 0; w < Geom::WORDS; ++w)
        qv[j][i][w] = with_sign(load8(q + row[j] + (4 * i + quad) * 8 * Geom::WORDS + 8 * w), c.sign);

  float m[CG], l[CG];
  float4_t o[CG][Geom::TILES];
#pragma unroll
  for (int j = 0; j < CG; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < Geom::TILES; ++i)
      o[j][i] = float4_t{0, 0, 0, 0};
  }

  const Nibbles nibbles;
  auto consume = [&](unsigned k, char *buffer) {
    char *block = buffer + wave * Geom::STAGE;
    const unsigned base = 32 * (b0 + wave + kWaves * k);
    // The slots behind the last key hold anything (what is in page 0 from a
    // missing page on), and 0 times that may be NaN: their values' scales and
    // biases become 0. (A lane has one slot's scale or bias in every group.)
    const unsigned slot = lane % 8, behind = 16 * (lane / 16 % 2) + 8 * (slot / 4) +
                                             4 * (lane / 8 % 2) + slot % 4;
    if (base + 32 > end) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the block is there, before it is changed
      if (base + behind >= end) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          *reinterpret_cast<half_t *>(block + 36 * D + 128 * i + 2 * lane) = (half_t)0;
      }
    }
    float4_t acc[2][CG];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < CG; ++j)
        acc[t][j] = float4_t{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < Geom::CHUNKS; ++i) {
      uint32_t word[2][Geom::WORDS];
      half2_t both[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char *at = block + t * 8 * D + i * 1024 + lane * 4 * Geom::WORDS;
        if constexpr (Geom::WORDS == 4) {
          const uint4_t v = *reinterpret_cast<const uint4_t *>(at);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            word[t][w] = v[w];
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(at);
          word[t][0] = v.x, word[t][1] = v.y;
        }
        const unsigned group = D >= 128 ? 4 * i + quad : quad / 2;
        both[t] = *reinterpret_cast<const half2_t *>(block + 16 * D + t * 2 * D +
                                                     (group * 16 + r) * 4);
      }
#pragma unroll
      for (int w = 0; w < Geom::WORDS; ++w) {
        half8_t key[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
          key[t] = paged_eight(word[t][w], both[t], nibbles);
#pragma unroll
        for (int j = 0; j < CG; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[t][j] = mfma16x16x32(key[t], qv[j][i][w], acc[t][j]);
        }
      }
    }
    float x[CG][8];
#pragma unroll
    for (int j = 0; j < CG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[j][e] = scaled_score(acc[e / 4][j][e % 4], c.c);
    // key of slot 4 t + v of this lane
    const unsigned first = base + 16 * (quad / 2) + 4 * (quad % 2);
    if (base + 31 > least) {
#pragma unroll
      for (int j = 0; j < CG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[j][e] = first + 8 * (e / 4) + e % 4 <= visible[j] ? x[j][e] : -INFINITY;
    }
    float top[CG];
    bool raise = false;
#pragma unroll
    for (int j = 0; j < CG; ++j) {
      top[j] = x[j][0];
#pragma unroll
      for (int e = 1; e < 8; ++e)
        top[j] = fmaxf(top[j], x[j][e]);
      raise |= top[j] - m[j] > kPagedRaise;
    }
    if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
      for (int j = 0; j < CG; ++j) {
        LanePair p = pair16(top[j]);
        const float half = fmaxf(p.a, p.b);
        p = pair32(half);
        const float all = fmaxf(p.a, p.b);
        const float to = all - m[j] > kPagedRaise ? all - kPagedHeadroom : m[j];
        const float alpha = m[j] == to ? 1.0f : fast_exp2(m[j] - to);
        m[j] = to;
        l[j] *= alpha;
#pragma unroll
        for (int i = 0; i < Geom::TILES; ++i)
          o[j][i] *= alpha;
      }
    }
    half8_t w[CG];
    const half8_t ones{1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int j = 0; j < CG; ++j) {
      const float ref = m[j] == -INFINITY ? 0.0f : m[j]; // nothing seen yet: weights 0
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[j][e] = (half_t)fast_exp2(x[j][e] - ref);
      l[j] = dot8(w[j], ones, l[j]);
    }
#pragma unroll
    for (int st = 0; st < D / 64; ++st) {
      const uint4_t word = *reinterpret_cast<const uint4_t *>(block + 20 * D + st * 1024 + lane * 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char *at = block + 36 * D + (2 * st + half) * 128 + quad * 16;
        const half8_t sc = *reinterpret_cast<const half8_t *>(at);
        const half8_t bi = *reinterpret_cast<const half8_t *>(at + 64);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t u = word[2 * half + n];
          const half8_t value = paged_eight(u, sc, bi, nibbles);
#pragma unroll
          for (int j = 0; j < CG; ++j)
            o[j][4 * st + 2 * half + n] = mfma16x16x32(value, w[j], o[j][4 * st + 2 * half + n]);
        }
      }
    }
  };

  // R blocks in flight, their buffers known at compile time.
  constexpr int R = Geom::RING;
  static_assert(R >= 2 && R <= 6, "the buffers below");
  auto buffer = [&](int i) -> char * {
    switch (i % R) {
    case 0:
      return ring_buffer<D, CG, W, 0>();
    case 1:
      return ring_buffer<D, CG, W, 1>();
    case 2:
      return ring_buffer<D, CG, W, (R > 2 ? 2 : 0)>();
    case 3:
      return ring_buffer<D, CG, W, (R > 3 ? 3 : 0)>();
    case 4:
      return ring_buffer<D, CG, W, (R > 4 ? 4 : 0)>();
    default:
      return ring_buffer<D, CG, W, (R > 5 ? 5 : 0)>();
    }
  };
#pragma unroll
  for (int i = 0; i < R - 1; ++i)
    issue(i, buffer(i));
  unsigned k = 0;
  for (; k + R <= mine; k += R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      issue(k + i + R - 1, buffer(i + R - 1));
      consume(k + i, buffer(i));
    }
  }
#pragma unroll
  for (int i = 0; i < R - 1; ++i)
    if (k + i < mine)
      consume(k + i, buffer(i));

  // Join the waves: (m, l) of the columns, then each wave its output tiles.
  auto out_of = [&](unsigned w) { // wave w's tiles
    return reinterpret_cast<float4_t *>(
        (w < kWaves / 2 ? ring_buffer<D, CG, W, 0>() : ring_buffer<D, CG, W, 1>()) +
        w % (kWaves / 2) * Geom::TILES * 1024);
  };
  float *sM = reinterpret_cast<float *>(ring_buffer<D, CG, W, 1>() +
                                       kWaves / 2 * Geom::TILES * 1024);
  float *sL = sM + kWaves * kUnit;
  __syncthreads(); // the ring's blocks are done with
  if (end < whole && invalid && lane == 0)
    atomicOr(invalid, kPagedPlace);
#pragma unroll
  for (int j = 0; j < CG; ++j) {
    LanePair p = pair16(l[j]);
    const float half = p.a + p.b;
    p = pair32(half);
    if (quad == 0) {
      const bool lost = visible[j] >= end;
      sM[wave * kUnit + kColumns * j + r] = lost ? 0.0f : m[j];
      sL[wave * kUnit + kColumns * j + r] = lost ? NAN : p.a + p.b;
    }
  }
  // Up to 16 / F columns of a group, a token's heads, are in every F-th four
  // lanes: F tiles go side by side, lane r with column r % (16 / F) of tile
  // F i + r / (16 / F) (a token's four heads on 4097 keys: 8.6 us, 9.7 with F 1).
  auto join = [&](auto factor, const int j) {
    constexpr unsigned F = decltype(factor)::value, kCols = kColumns / F;
    constexpr unsigned kTiles = Geom::TILES / F;
#pragma unroll
    for (unsigned i = 0; i < kTiles; ++i) {
      float4_t y = o[j][F * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F == 2)
          y[e] = shifted_in<kRowShr8, 0xC>(y[e], o[j][2 * i + 1][e]);
        if constexpr (F == 4) {
          y[e] = shifted_in<kRowShr4, 2>(y[e], o[j][4 * i + 1][e]);
          y[e] = shifted_in<kRowShr8, 4>(y[e], o[j][4 * i + 2][e]);
          y[e] = shifted_in<kRowShr12, 8>(y[e], o[j][4 * i + 3][e]);
        }
      }
      out_of(wave)[i * 64 + lane] = y;
    }
    __syncthreads();
    const unsigned at = r % kCols, col = kColumns * j + at;
    float top = sM[col], sum = 0.0f, a[kWaves];
#pragma unroll
    for (unsigned w = 1; w < kWaves; ++w)
      top = fmaxf(top, sM[w * kUnit + col]);
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w) {
      const float mw = sM[w * kUnit + col];
      a[w] = mw == -INFINITY ? 0.0f : fast_exp2(mw - top);
      sum += sL[w * kUnit + col] * a[w];
    }
    const size_t part = ((size_t)blockIdx.x * g.kvHeads + kvh) * kUnit + col;
    const float scale = pieces == 1 ? 1.0f / sum : 1.0f;
    const size_t to = F == 1 ? row[j] : row_of(col);
    for (unsigned i = wave; i < kTiles; i += kWaves) {
      float4_t y{0, 0, 0, 0};
#pragma unroll
      for (unsigned w = 0; w < kWaves; ++w)
        y += out_of(w)[i * 64 + lane] * a[w];
      if (col >= columns)
        continue;
      const unsigned channel = 16 * (F * i + r / kCols) + 4 * quad;
      if (pieces == 1)
        *reinterpret_cast<half4_t *>(out + to + channel) =
            half4_t{(half_t)(y[0] * scale), (half_t)(y[1] * scale), (half_t)(y[2] * scale),
                    (half_t)(y[3] * scale)};
      else
        *reinterpret_cast<float4_t *>(parts.o + part * D + channel) = y;
    }
    if (pieces > 1 && wave == 0 && lane < kCols && col < columns)
      *reinterpret_cast<float2 *>(parts.ml + 2 * part) = make_float2(top, sum);
  };
  if constexpr (CG == 1) {
    if (columns <= 4)
      return join(std::integral_constant<unsigned, 4>(), 0);
    if (columns <= 8)
      return join(std::integral_constant<unsigned, 2>(), 0);
  }
#pragma unroll
  for (int j = 0; j < CG; ++j) {
    if (j)
      __syncthreads(); // the group before is done with
    join(std::integral_constant<unsigned, 1>(), j);
  }
}

// Joins the rows whose keys were divided. An item is such a row's query head,
// the work of W waves, each every W-th piece, a lane D/64 channels; items are
// taken in turn, so that a call without any costs one round of workgroups.
// W: 8 where units have many pieces or few columns, 1 otherwise.
constexpr unsigned kMergeThreads = 512;
constexpr unsigned kMergeGroups = 1024; // workgroups: four a CU
template <int D, int W>
__global__ __launch_bounds__(kMergeThreads) void paged_gqa_merge_kernel(
    PagedView g, half_t *out, unsigned queryHeads, SplitPlan plan, unsigned most, Partials parts) {
  constexpr int N = D / 64;
  constexpr unsigned kItems = kMergeThreads / 64 / W; // of a workgroup
  typedef float vec __attribute__((ext_vector_type(N)));
  typedef _Float16 halves __attribute__((ext_vector_type(N)));
  const unsigned G = queryHeads / g.kvHeads, unit = 1u << plan.shift;
  const PagedSeq own = paged_own(g);
  const Split split = paged_split(g, own, G, plan);
  const unsigned lane = threadIdx.x % 64;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  __shared__ float sM[W], sL[W];
  __shared__ vec sY[W][64];
  // (W > 1: the same item in every wave, so all of them leave together)
  for (unsigned item = blockIdx.x * kItems + wave / W;; item += gridDim.x * kItems) {
    unsigned seq, local, before, pieceBefore = 0;
    if (!paged_find(g, own, item,
                    [&](const PagedSeq &s) {
                      return s.ok && split.pieces(s) > 1 ? s.rows * queryHeads : 0u;
                    },
                    seq, local, before))
      return;
    for (unsigned s0 = 0; s0 <= seq; s0 += 64) { // pieces of the sequences before
      const PagedSeq o = s0 ? (s0 + lane < g.sequences ? paged_seq(g, s0 + lane)
                                                       : PagedSeq{0, 0, 0, true})
                            : own;
      const unsigned n = split.units(o) * split.pieces(o), sum = wave_scan(n);
      const int at = seq - s0 < 64 ? (int)(seq - s0) : 63;
      pieceBefore += (unsigned)__builtin_amdgcn_readlane((int)(seq - s0 < 64 ? sum - n : sum), at);
    }
    const PagedSeq s = paged_seq_of(g, own, seq);
    const unsigned pieces = split.pieces(s), h = local % queryHeads, row = local / queryHeads;
    const unsigned column = row * G + h % G, kvh = h / G;
    const unsigned first = pieceBefore + (split.units(s) - 1 - column / unit) * pieces;
    if (first >= most || pieces > most - first) // starts out of order: more pieces than the rows can have
      return;
    const size_t at = ((size_t)first * g.kvHeads + kvh) * unit + column % unit;
    const size_t step = (size_t)g.kvHeads * unit;
    const float2 *ml = reinterpret_cast<const float2 *>(parts.ml) + at;
    const vec *po = reinterpret_cast<const vec *>(parts.o + at * D) + lane;
    float m = -INFINITY, l = 0.0f;
    vec y = 0.0f;
    // `count` of this wave's pieces at a time, all of them in flight at once
    auto take = [&](auto count, unsigned i0) {
      constexpr unsigned kCount = decltype(count)::value;
      float2 x[kCount];
      vec o[kCount];
#pragma unroll
      for (unsigned n = 0; n < kCount; ++n) {
        const unsigned i = min(i0 + W * n, pieces - 1);
        x[n] = ml[step * i];
        o[n] = po[step * i * 64];
      }
      float to = m;
#pragma unroll
      for (unsigned n = 0; n < kCount; ++n) {
        x[n].x = i0 + W * n < pieces ? x[n].x : -INFINITY;
        to = fmaxf(to, x[n].x);
      }
      const float a = m == -INFINITY ? 0.0f : fast_exp2(m - to);
      l *= a;
      y *= a;
#pragma unroll
      for (unsigned n = 0; n < kCount; ++n)
        if (x[n].x != -INFINITY) {
          const float b = fast_exp2(x[n].x - to);
          l += x[n].y * b;
          y += o[n] * b;
        }
      m = to;
    };
    unsigned i = wave % W;
    for (; i + 4 * W < pieces; i += 8 * W)
      take(std::integral_constant<unsigned, 8>(), i);
    if (i < pieces)
      take(std::integral_constant<unsigned, 4>(), i);
    if (W > 1) {
      sM[wave] = m;
      sL[wave] = l;
      sY[wave][lane] = y;
      __syncthreads();
      m = sM[0];
      for (unsigned w = 1; w < W; ++w)
        m = fmaxf(m, sM[w]);
      l = 0.0f;
      y = 0.0f;
      for (unsigned w = 0; w < W; ++w) {
        const float a = sM[w] == -INFINITY ? 0.0f : fast_exp2(sM[w] - m);
        l += sL[w] * a;
        y += sY[w][lane] * a;
      }
      __syncthreads();
    }
    if (wave % W == 0) {
      halves z;
      for (int i = 0; i < N; ++i)
        z[i] = (half_t)(y[i] / l);
      reinterpret_cast<halves *>(out + ((size_t)(s.row0 + row) * queryHeads + h) * D)[lane] = z;
    }
  }
}

size_t partial_columns(const PagedKvParams &p, unsigned group, const SplitPlan &plan) {
  return (size_t)most_pieces(p, group, plan) * p.kvHeads << plan.shift;
}

} // namespace

bool paged_gqa_tiled(const PagedKvParams &p, unsigned queryHeads) {
  return (1u << plan_for(p, queryHeads / p.kvHeads).split.shift) > 64;
}
bool paged_gqa_joins(const PagedKvParams &p, unsigned queryHeads) {
  return may_divide(p, plan_for(p, queryHeads / p.kvHeads).split);
}
bool paged_gqa_launchable(const PagedKvParams &p, unsigned queryHeads) {
  const unsigned group = queryHeads / p.kvHeads;
  const uint64_t rows = (uint64_t)p.tokens * queryHeads;
  return rows <= 0x7fffffffull &&
         (most_pieces(p, group, plan_for(p, group).split)) * p.kvHeads < (1u << 22);
}

size_t paged_gqa_workspace_bytes(const PagedKvParams &p, unsigned queryHeads) {
  const unsigned group = queryHeads / p.kvHeads;
  if (!paged_gqa_joins(p, queryHeads))
    return 0;
  return 4 * (p.headDim + 2) * partial_columns(p, group, plan_for(p, group).split);
}

hipError_t launch_paged_gqa(const uint16_t *q, const int32_t *starts, const int32_t *past,
                            const int32_t *table, const void *pool, uint16_t *out,
                            uint32_t *invalid, void *workspace, const PagedKvParams &p,
                            unsigned queryHeads, float scale, hipStream_t stream) {
  const unsigned group = queryHeads / p.kvHeads;
  const GqaPlan both = plan_for(p, group);
  const SplitPlan &plan = both.split;
  const unsigned unit = 1u << plan.shift, pieces = (unsigned)most_pieces(p, group, plan);
  const PagedView g = paged_view(p, starts, past, table);
  float *ws = static_cast<float *>(workspace);
  const Partials parts{ws + partial_columns(p, group, plan) * p.headDim, ws};
  half_t *to = reinterpret_cast<half_t *>(out);
  const half_t *from = reinterpret_cast<const half_t *>(q);
  const uint8_t *pages = static_cast<const uint8_t *>(pool);
  const ScoreScale c = score_scale(scale);
  auto attend = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(pieces, p.kvHeads), dim3(64 * plan.step), 0,
                       stream, from, pages, g, to, invalid, queryHeads, plan, c, parts);
    return hipGetLastError();
  };
  auto by_columns = [&](auto one, auto pooled, auto more) {
    return attend(unit > 16 ? more : both.pooled ? pooled : one);
  };
  hipError_t e;
  if (unit > 64)
    e = launch_paged_tiles(from, pages, g, to, invalid, queryHeads, plan, c, parts, pieces, stream);
  else if (p.headDim == 256)
    e = by_columns(paged_gqa_kernel<256, 1, 4>, paged_gqa_kernel<256, 1, 8>,
                   paged_gqa_kernel<256, 2, 4>);
  else if (p.headDim == 128)
    e = by_columns(paged_gqa_kernel<128, 1, 4>, paged_gqa_kernel<128, 1, 8>,
                   paged_gqa_kernel<128, 2, 4>);
  else
    e = by_columns(paged_gqa_kernel<64, 1, 4>, paged_gqa_kernel<64, 1, 8>,
                   paged_gqa_kernel<64, 4, 4>);
  if (e != hipSuccess)
    return e;
  if (!may_divide(p, plan))
    return e;
  const bool wide = both.pooled || unit <= 64;
  auto merge = [&](auto few, auto many) {
    const unsigned each = wide ? 1 : kMergeThreads / 64;
    const uint64_t groups = ((uint64_t)p.tokens * queryHeads + each - 1) / each;
    const unsigned grid = (unsigned)(groups < kMergeGroups ? groups : kMergeGroups);
    if (wide)
      hipLaunchKernelGGL(few, dim3(grid), dim3(kMergeThreads), 0, stream, g, to, queryHeads, plan,
                         pieces, parts);
    else
      hipLaunchKernelGGL(many, dim3(grid), dim3(kMergeThreads), 0, stream, g, to, queryHeads, plan,
                         pieces, parts);
    return hipGetLastError();
  };
  return p.headDim == 256   ? merge(paged_gqa_merge_kernel<256, 8>, paged_gqa_merge_kernel<256, 1>)
         : p.headDim == 128 ? merge(paged_gqa_merge_kernel<128, 8>, paged_gqa_merge_kernel<128, 1>)
                            : merge(paged_gqa_merge_kernel<64, 8>, paged_gqa_merge_kernel<64, 1>);
}

} // namespace llmi
