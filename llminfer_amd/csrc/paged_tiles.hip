// Causal GQA over the paged 4-bit cache for sequences of many rows: tiles of
// keys and values decoded once for all of a workgroup's columns.
//
// A workgroup has 128 columns of a KV head (256 at head_dim 128), eight waves:
// wave w the 32-column tiles of column wave w % 4, and of the keys of a step
// the half w / 4. A step is 512 / D blocks of 32 keys:
//  * every thread decodes 16 bytes of key codes and 16 of value codes of the
//    next step into LDS, as fp16 operands of v_mfma_f32_32x32x16_f16 in the
//    order in which a wave reads them (1 KB, conflict-free), while
//  * the matrix products of this one run: S^T = K Q^T with the columns in the
//    lanes, and O^T += V^T P^T, whose weights are the score tile's registers
//    as they are (the slots of a value word are the keys of a lane's eight);
//  * codes and scales go HBM -> LDS by DMA two steps ahead, each wave those
//    that its own threads decode, so that no register holds them and only
//    the decoded tiles need the workgroup's barrier, one a step.
// The halves of the keys are joined at the end through the tiles' memory.
//
// 2048 tokens of 16 heads of 256 on 4096 keys take 131 us (traced, after some
// hundred passes; the first take 138 and more; 134 to 138 in their call with
// the join's launch, by the card), 103 GFLOP; the last units see 4096 keys and
// the first 2080, and the kernel takes the time of the last ones: 128 blocks at
// 0.97 us, 1.1 PFLOP/s while all of them run. Bound by the products and the
// vector instructions of a SIMD's two waves, which overlap little: 99 and 78
// thousand cycles of the 208 thousand that a SIMD's workgroups run (half of the
// vector instructions decode, without them the kernel takes 64 % of its time;
// LDS is busy for 86 thousand).
// At head_dim 128 the kernel has more than its 256 registers hold: addresses are
// reloaded from scratch between a step's DMA loads, each reload a wait for all
// loads before it. SQ_WAIT_ANY is 56 million in seven ragged messages (125 us
// traced, 127 to 131 in their call) and 28 million in the call above, whose
// products are more.
// Of a short call (61 tokens on 16472 keys: 30 us inside the kernel) 6 us are
// the plan, the table and the first blocks, 5 the joining and the partials.
#include "hip_common.hpp"
#include "paged_kv.hpp"
#include "paged_plan.hpp"

#include <math.h>
#include <type_traits>

namespace llmi {
namespace {

constexpr unsigned kThreads = 512;

template <int D> struct Tiles {
  static constexpr int CT = 256 / D;       // 32-column tiles of a wave
  static constexpr int UNIT = 128 * CT;    // columns of a workgroup
  static constexpr int BLOCKS = 512 / D;   // of a step
  static constexpr int EACH = BLOCKS / 2;  // of a half
  static constexpr int BLOCKB = 64 * D;    // bytes of a decoded block
  static constexpr int STEPS = D / 16;     // products over the channels
  static constexpr int OUT = D / 32;       // output tiles
};

// Decoded keys [block][D/8][key 32][8 channels] and values [block][D/32]
// [quad 4][channel 32][8 keys], two buffers each, variables of their own.
template <int I> __device__ __forceinline__ char *tile_buffer() {
  __shared__ __attribute__((aligned(1024))) char buffer[32768];
  return buffer;
}

// The call's piece `u` with the sequences of the longest pieces first (up to 64
// sequences; in their order otherwise), so that workgroups which start late
// have little to do (seven messages of 41 to 110 blocks, 296 workgroups:
// 174 us in order, 130 longest first).
__device__ __forceinline__ bool find_longest(const PagedView &g, const PagedSeq &own,
                                             const Split &split, unsigned u, unsigned &seq,
                                             unsigned &local, unsigned &number) {
  unsigned before;
  if (g.sequences == 1 || g.sequences > 64) {
    number = u;
    return paged_find(g, own, u,
                      [&](const PagedSeq &s) { return split.units(s) * split.pieces(s); }, seq,
                      local, before);
  }
  const unsigned lane = threadIdx.x % 64;
  const unsigned pieces = split.pieces(own), length = split.length(own, pieces);
  const unsigned n = split.units(own) * pieces;
  unsigned ahead = 0;
  for (unsigned j = 0; j < g.sequences; ++j) {
    const unsigned lj = (unsigned)__builtin_amdgcn_readlane((int)length, (int)j);
    const unsigned nj = (unsigned)__builtin_amdgcn_readlane((int)n, (int)j);
    ahead += lj > length || (lj == length && j < lane) ? nj : 0u;
  }
  const unsigned long long here =
      __builtin_amdgcn_ballot_w64(lane < g.sequences && u - ahead < n);
  if (!here)
    return false;
  const int at = __builtin_ctzll(here);
  seq = (unsigned)at;
  local = u - (unsigned)__builtin_amdgcn_readlane((int)ahead, at);
  number = (unsigned)__builtin_amdgcn_readlane((int)(wave_scan(n) - n), at) + local;
  return true;
}

constexpr unsigned kRaw = 2560; // bytes of a wave's part of a step
__device__ __forceinline__ char *raw_buffer() {
  __shared__ __attribute__((aligned(1024))) char buffer[kThreads / 64 * kRaw];
  return buffer;
}

typedef __attribute__((address_space(3))) void lds_void_t;
constexpr int kBufferWord3 = 0x00020000; // gfx9 raw buffer descriptor, dword 3

// The order that the scheduler gives a run of products, N operands read from
// LDS and CT products for each: some reads ahead of the first, then one after
// each operand's products.
template <int N, int CT> __device__ __forceinline__ void reads_ahead() {
  constexpr int kMfma = 0x008, kRead = 0x100, kAhead = CT == 1 ? 4 : 3;
  __builtin_amdgcn_sched_group_barrier(kRead, kAhead, 0);
#pragma unroll
  for (int i = 0; i < N - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, CT, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, CT * kAhead, 0);
}

template <int D>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads),
                          amdgpu_waves_per_eu(2, 2)))
void paged_tiles_kernel(const half_t *__restrict__ q, const uint8_t *__restrict__ pool,
                        PagedView g, half_t *out, unsigned *invalid, unsigned queryHeads,
                        SplitPlan plan, ScoreScale c, Partials parts) {
  using T = Tiles<D>;
  constexpr int CT = T::CT;
  const unsigned G = queryHeads / g.kvHeads, kvh = blockIdx.x % g.kvHeads;
  const PagedSeq own = paged_own(g);
  const Split split = paged_split(g, own, G, plan);
  unsigned seq, local, number; // number: of this piece, for its partials
  if (!find_longest(g, own, split, blockIdx.x / g.kvHeads, seq, local, number) ||
      number >= gridDim.x / g.kvHeads) // (starts out of order: more pieces than the rows can have)
    return;
  const PagedSeq s = paged_seq_of(g, own, seq);
  const unsigned pieces = split.pieces(s), units = split.units(s);
  const unsigned unit = units - 1 - local / pieces, piece = local % pieces;
  const unsigned tid = threadIdx.x, lane = tid % 64, r = lane % 32, hi = lane / 32;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const unsigned half = wave / 4, tile0 = wave % 4 * CT;

  // this lane's columns (past the unit's last: some row's, not written)
  const unsigned c0 = unit * T::UNIT, columns = min((unsigned)T::UNIT, s.rows * G - c0);
  unsigned visible[CT]; // a column's last key
  size_t row[CT];
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const unsigned col = c0 + 32 * (tile0 + j) + r, token = min(col / G, s.rows - 1);
    visible[j] = s.past + token;
    row[j] = ((size_t)(s.row0 + token) * queryHeads + kvh * G + col % G) * D;
  }
  auto live = [&](int j) { return 32 * (tile0 + j) + r < columns; };
  if (!s.ok) { // no place for this sequence
    for (int j = 0; j < CT; ++j)
      if (live(j) && half == 0)
        for (unsigned x = hi; x < D; x += 2)
          out[row[j] + x] = (half_t)NAN;
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  const unsigned least = s.past + c0 / G;                // the first column's last key
  const unsigned most = s.past + (c0 + columns - 1) / G; // the last column's
  // the keys that this wave decodes: to the sequence's end, or to a page that is
  // not in the pool, whose columns' outputs are NaN
  const unsigned whole = s.past + s.rows;
  unsigned end = whole;
  const unsigned length = split.length(s, pieces), b0 = min(piece * length, most / 32 + 1);
  const unsigned b1 = min(b0 + length, most / 32 + 1);
  const unsigned steps = (b1 - b0 + T::BLOCKS - 1) / T::BLOCKS;

  // ---- decoding: this thread's 16 bytes of codes of a step's block
  __shared__ unsigned sEnd; // the least of the waves'
  if (tid == 0)
    sEnd = whole;
  const unsigned slot = __builtin_amdgcn_readfirstlane(tid / D), unit16 = tid % D;
  size_t place = 0;
  auto block_of = [&](unsigned n) { return min(b0 + T::BLOCKS * n + slot, b1 - 1); };
  const Nibbles nibbles;
  // A wave's part of a step: 1 KB of key codes and of value codes, and the
  // scales and biases of both, a word a lane (of its 64 keys' groups, and of
  // its 64 channels).
  char *raw = raw_buffer() + kRaw * wave;
  auto fetch = [&](unsigned n) { // (n < steps; a block past the last again)
    if (n % 64 == 0) {           // where the next 64 steps' blocks are, one a lane
      const bool lost = !paged_block(g, seq, 32 * block_of(n + lane), kvh, place);
      if (const unsigned long long all = __builtin_amdgcn_ballot_w64(lost))
        end = min(end, 32 * block_of(n + (unsigned)__builtin_ctzll(all)));
    }
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)place, n % 64);
    const unsigned up = __builtin_amdgcn_readlane((unsigned)(place >> 32), n % 64);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(pool + ((size_t)up << 32 | lo)), (short)0, 40 * D, kBufferWord3);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the part before has been read
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)raw, 16, 16 * unit16, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(raw + 1024), 16,
                                             20 * D + 16 * unit16, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(raw + 2048), 4,
                                             16 * D + 4 * unit16, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(raw + 2304), 4,
                                             36 * D + 4 * unit16, 0, 0, 0);
  };
  const unsigned quad = unit16 / 16 % 4, rr = unit16 % 16;
  const unsigned keyAt = slot * T::BLOCKB + (unit16 % (D / 2) / 16) * 2048 +
                         (16 * (rr / 8) + 8 * (unit16 / (D / 2)) + rr % 8) * 16;
  const unsigned valueAt = slot * T::BLOCKB + (unit16 / 64) * 4096 + quad * 512 + rr * 16;
  // The wave's part of step n has come. Behind the last key lies anything (what
  // is in page 0 from a missing page on), and 0 times that may be NaN: those
  // slots' scales and biases become 0 (a lane has two slots of one quad).
  auto arrived = [&](unsigned n) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned base = 32 * block_of(n);
    if (base + 32 > end) {
      const unsigned sq = lane / 4 % 4, e = lane % 4 * 2;
      const unsigned at = base + 16 * (sq / 2) + 4 * (sq % 2) + 8 * (e / 4) + e % 4;
      half_t *mine = reinterpret_cast<half_t *>(raw + 2304) + 2 * lane;
      if (at >= end)
        mine[0] = (half_t)0;
      if (at + 1 >= end)
        mine[1] = (half_t)0;
    }
  };
  auto decode_keys = [&](char *to) {
    const uint4_t keyCodes = *reinterpret_cast<const uint4_t *>(raw + 16 * lane);
    const half2_t keyScale = *reinterpret_cast<const half2_t *>(raw + 2048 + 4 * lane);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      *reinterpret_cast<half8_t *>(to + keyAt + 512 * w) =
          paged_eight(keyCodes[w], keyScale, nibbles);
  };
  auto decode_values = [&](char *to) {
    const uint4_t valueCodes = *reinterpret_cast<const uint4_t *>(raw + 1024 + 16 * lane);
    const uint32_t *mine = reinterpret_cast<const uint32_t *>(raw + 2304);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const half8_t sc = *reinterpret_cast<const half8_t *>(mine + 32 * p + 4 * quad);
      const half8_t bi = *reinterpret_cast<const half8_t *>(mine + 32 * p + 16 + 4 * quad);
#pragma unroll
      for (int w = 0; w < 2; ++w)
        *reinterpret_cast<half8_t *>(to + valueAt + 2048 * p + 256 * w) =
            paged_eight(valueCodes[2 * p + w], sc, bi, nibbles);
    }
  };

  // ---- the products: Q^T operands, outputs
  half8_t qv[CT][T::STEPS];
#pragma unroll
  for (int j = 0; j < CT; ++j)
#pragma unroll
    for (int n = 0; n < T::STEPS; ++n)
      qv[j][n] = with_sign(load8(q + row[j] + 16 * n + 8 * hi), c.sign);
  float m[CT], l[CT];
  float16_t o[CT][T::OUT];
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < T::OUT; ++i)
      o[j][i] = float16_t{0};
  }
  auto consume = [&](auto wide, unsigned b, const char *keys,
                     const char *values) __attribute__((always_inline)) {
    constexpr bool kWide = decltype(wide)::value;
    // before the other wave's decoding, where both could go on: 2048 tokens on
    // 4096 keys in 138 us, 144 without, 143 with only the scores' products ahead
    __builtin_amdgcn_s_setprio(1);
    const unsigned base = 32 * b;
    float16_t x[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j)
      x[j] = float16_t{0};
#pragma unroll
    for (int n = 0; n < T::STEPS; ++n) {
      const half8_t key = *reinterpret_cast<const half8_t *>(keys + 1024 * n + 16 * lane);
#pragma unroll
      for (int j = 0; j < CT; ++j)
        x[j] = mfma32x32x16(key, qv[j][n], x[j]);
    }
    reads_ahead<T::STEPS, CT>();
    if constexpr (kWide)
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          x[j][v] = scaled_score(x[j][v], c.c);
    if (base + 31 > least) {
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          x[j][v] = base + mfma_c_row(v, hi) <= visible[j] ? x[j][v] : -INFINITY;
    }
    float top[CT];
    bool raise = false;
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      top[j] = x[j][0];
#pragma unroll
      for (int v = 1; v < 16; ++v)
        top[j] = fmaxf(top[j], x[j][v]);
      if constexpr (!kWide)
        top[j] *= c.c;
      raise |= top[j] - m[j] > kPagedRaise;
    }
    if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const LanePair p = pair32(top[j]);
        const float all = fmaxf(p.a, p.b);
        const float to = all - m[j] > kPagedRaise ? all - kPagedHeadroom : m[j];
        const float alpha = m[j] == to ? 1.0f : fast_exp2(m[j] - to);
        m[j] = to;
        l[j] *= alpha;
#pragma unroll
        for (int i = 0; i < T::OUT; ++i)
          o[j][i] *= alpha;
      }
    }
    half8_t w[CT][2];
    const half8_t ones{1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      const float ref = m[j] == -INFINITY ? 0.0f : m[j]; // nothing seen yet: weights 0
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[j][e / 8][e % 8] = (half_t)fast_exp2(kWide ? x[j][e] - ref : fmaf(x[j][e], c.c, -ref));
      l[j] = dot8(w[j][0], ones, l[j]);
      l[j] = dot8(w[j][1], ones, l[j]);
    }
#pragma unroll
    for (int i = 0; i < T::OUT; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const half8_t value =
            *reinterpret_cast<const half8_t *>(values + 2048 * i + 1024 * n + 16 * lane);
#pragma unroll
        for (int j = 0; j < CT; ++j)
          o[j][i] = mfma32x32x16(value, w[j][n], o[j][i]);
      }
    reads_ahead<2 * T::OUT, CT>();
    __builtin_amdgcn_s_setprio(0);
  };

  // Whether a score may be past 2^22: |q| summed, times the largest value that an
  // append leaves (kPagedLimit and its roundings, below 1/64 of it). Below it
  // the fma shifts the exponents of a row by 2^-2 at most, all by the same, and
  // its weights stay below 2^15.5. At head_dim 128 both are there, a loop each
  // (seven ragged messages: 127 us, 135 with the rounded products alone); at 256
  // the rounded products alone are faster (2048 tokens on 4096 keys: 135 us, 141
  // with both on the same card).
  constexpr bool kBoth = D == 128;
  bool wide = !kBoth;
  __shared__ unsigned sWide[kThreads / 64];
  if (steps) {
    fetch(0);
#pragma unroll
    for (int j = 0; j < (kBoth ? CT : 0); ++j) {
      const half8_t ones{1, 1, 1, 1, 1, 1, 1, 1};
      float all = 0.0f;
#pragma unroll
      for (int n = 0; n < T::STEPS; ++n)
        all = dot8(__builtin_elementwise_abs(qv[j][n]), ones, all);
      const LanePair p = pair32(all);
      wide |= !((p.a + p.b) * (c.c * (kPagedLimit * 1.015625f)) < 0x1p22f);
    }
    if (kBoth && lane == 0)
      sWide[wave] = __builtin_amdgcn_ballot_w64(wide) != 0;
    arrived(0);
    decode_keys(tile_buffer<0>());
    decode_values(tile_buffer<2>());
    if (kBoth) { // the workgroup's waves take the same loop, for its barriers
      lds_sync();
      wide = __builtin_amdgcn_ballot_w64(sWide[lane % (kThreads / 64)] != 0);
    }
    if (steps > 1)
      fetch(1);
  }
  auto step = [&](auto wide, unsigned n, const char *keys, const char *values, char *nextKeys,
                  char *nextValues) __attribute__((always_inline)) {
    lds_sync(); // step n is decoded, and step n - 1's tiles are done with
    auto decode = [&]() {
      if (n + 1 < steps) {
        arrived(n + 1);
        decode_keys(nextKeys);
        decode_values(nextValues);
        if (n + 2 < steps)
          fetch(n + 2);
      }
    };
    // The two waves of a SIMD (the halves of the keys) take turns: one decodes
    // while the other's products run.
    if (half == 0)
      decode();
#pragma unroll
    for (int i = 0; i < T::EACH; ++i) {
      const unsigned at = half * T::EACH + i, b = b0 + T::BLOCKS * n + at;
      if (b < b1)
        consume(wide, b, keys + at * T::BLOCKB, values + at * T::BLOCKB);
    }
    if (half == 1)
      decode();
  };
  auto all_steps = [&](auto wide) __attribute__((always_inline)) {
    for (unsigned n = 0; n < steps; n += 2) {
      step(wide, n, tile_buffer<0>(), tile_buffer<2>(), tile_buffer<1>(), tile_buffer<3>());
      if (n + 1 < steps)
        step(wide, n + 1, tile_buffer<1>(), tile_buffer<3>(), tile_buffer<0>(), tile_buffer<2>());
    }
  };
  if (wide)
    all_steps(std::true_type());
  else if constexpr (kBoth)
    all_steps(std::false_type());

  // ---- join the halves of the keys
  if (end < whole && lane == 0) { // a page that is not in the pool
    atomicMin(&sEnd, end);
    if (invalid)
      atomicOr(invalid, kPagedPlace);
  }
  __shared__ float sM[T::UNIT], sL[T::UNIT];
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const LanePair p = pair32(l[j]);
    l[j] = p.a + p.b;
  }
  __syncthreads();
  // a wave's 128 output registers, 32 KB, a buffer each
  float4_t *mine = reinterpret_cast<float4_t *>(wave % 4 == 0   ? tile_buffer<0>()
                                                : wave % 4 == 1 ? tile_buffer<1>()
                                                : wave % 4 == 2 ? tile_buffer<2>()
                                                                : tile_buffer<3>());
  if (half == 1) {
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      if (hi == 0) {
        sM[32 * (tile0 + j) + r] = m[j];
        sL[32 * (tile0 + j) + r] = l[j];
      }
#pragma unroll
      for (int i = 0; i < T::OUT; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          mine[((j * T::OUT + i) * 4 + v) * 64 + lane] =
              float4_t{o[j][i][4 * v], o[j][i][4 * v + 1], o[j][i][4 * v + 2], o[j][i][4 * v + 3]};
    }
  }
  __syncthreads();
  if (half == 1)
    return;
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const unsigned col = 32 * (tile0 + j) + r;
    const bool lost = visible[j] >= sEnd;
    const float other = sM[col], top = lost ? 0.0f : fmaxf(m[j], other);
    const float a = m[j] == -INFINITY ? 0.0f : fast_exp2(m[j] - top);
    const float b = other == -INFINITY ? 0.0f : fast_exp2(other - top);
    const float sum = lost ? NAN : l[j] * a + sL[col] * b;
    const size_t part = ((size_t)number * g.kvHeads + kvh) * T::UNIT + col;
    const float inv = 1.0f / sum;
    if (!live(j))
      continue;
#pragma unroll
    for (int i = 0; i < T::OUT; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float4_t z = mine[((j * T::OUT + i) * 4 + v) * 64 + lane];
        float4_t y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = o[j][i][4 * v + e] * a + z[e] * b;
        const unsigned at = 32 * i + 8 * v + 4 * hi;
        if (pieces == 1)
          *reinterpret_cast<half4_t *>(out + row[j] + at) =
              half4_t{(half_t)(y[0] * inv), (half_t)(y[1] * inv), (half_t)(y[2] * inv),
                      (half_t)(y[3] * inv)};
        else
          *reinterpret_cast<float4_t *>(parts.o + part * D + at) = y;
      }
    if (pieces > 1 && hi == 0)
      *reinterpret_cast<float2 *>(parts.ml + 2 * part) = make_float2(top, sum);
  }
}

} // namespace

unsigned paged_tiles_columns(unsigned headDim) { return 128 * (256 / headDim); }

hipError_t launch_paged_tiles(const half_t *q, const uint8_t *pool, const PagedView &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, SplitPlan plan, ScoreScale c,
                              Partials parts, unsigned pieces, hipStream_t stream) {
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(pieces * g.kvHeads), dim3(kThreads), 0, stream, q, pool, g, out,
                       invalid, queryHeads, plan, c, parts);
    return hipGetLastError();
  };
  return g.dim == 256 ? run(paged_tiles_kernel<256>) : run(paged_tiles_kernel<128>);
}

} // namespace llmi
