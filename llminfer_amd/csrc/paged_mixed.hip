// Causal GQA of groups of sequences behind shared keys, in one launch: some
// workgroups have tiles of a group's shared keys, with all its rows as columns
// (paged_tiles.hpp: bound by the matrix cores), the waves of the others the
// sequences' own keys, sixteen columns a unit (bound by memory and decoding), so
// that both run at once. The partials of the two are joined by
// paged_shared_merge_kernel.
//
// A workgroup of either kind takes a CU's LDS, so the plan gives each kind as many
// CUs as make them end together, and own keys go by waves and not by workgroups:
// a wave with a run of blocks waits for no other, and its runs are of equal
// length whatever the sequences' are (pieces by workgroups, joined in LDS: 12 us
// each, five of them waiting; 48 chats 57 us, 44 with runs). Shared keys go by
// workgroups, which begin a unit in 8 us: a run of blocks each, of one unit where
// there are fewer units than workgroups, else wherever the runs part them (900
// sequences of 8 heads of 128, 29 units for 32 workgroups a KV head, behind 4096
// keys: 156 us, 411 with whole units of as many blocks each).
//
// 48 sequences of 16 / 4 heads of 256, 16384 shared keys and up to 1024 of their
// own, 13.3 GFLOP, take 38 us here and 41.5 with the join (paged_gqa: 137 to 142).
// Tiles, 48 of a KV head's 64 workgroups, 22 blocks each: 7 us until the first
// block is there (plan 2, table, block, one after the other), 1 us a block, 4 to
// join the halves and write 22 MB of partials. A step of two blocks is 3800 cycles
// of a SIMD with two waves, whose own take 1200 of decoding each, 1030 and 1050 of
// products (512 and 512 of them the matrix cores'; LDS gives 192 KB a step and
// takes 64, 2000 cycles of its own) and 660 of softmax; no wave waits for loads.
// Own keys, 8 blocks a wave: 2.2 us a block of 10 KB, two waves a SIMD, bound by
// decoding (550 instructions a block). Matrix instructions take 16 % of the
// time, vector instructions 32 %, waves wait for 43 %. Six groups at head_dim 128:
// 45 us with the join, own keys 1.2 us a block; two of 187 rows in all at 64:
// 42 us, tiles 2.9 us a step of eight blocks, of which a wave's softmax is 2300 to
// 3000 of 6600 cycles. At 256 a lane has all of its 256 registers; at 128 and 64 it
// has 166 and 129: there the tiles' 128 KB of LDS, the same at every width, leave
// room for two waves a SIMD only, which keep the vector units active for 48 % of
// their cycles and the matrix cores for 14 to 17 %.
#include "paged_tiles.hpp"

namespace llmi {
namespace {

constexpr unsigned kColumns = 16; // of a unit of own keys
constexpr unsigned kWaves = kMixedWaves;
static_assert(kWaves == kThreads / 64, "the tiles' waves");
constexpr unsigned kTileColumns = 128; // of a unit of shared keys, at most
constexpr unsigned kLeastRun = 2; // blocks

__device__ __forceinline__ float4_t mfma16x16x32(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A scalar, also where the compiler does not see that it is one.
__device__ __forceinline__ unsigned uniform(unsigned x) {
  return (unsigned)__builtin_amdgcn_readfirstlane((int)x);
}

// What a wave loads of a block into registers: the key codes and scales as the
// matrix instructions take them, a lane's its own. The values' half of the block
// goes by DMA to LDS (both halves in registers spill, both in LDS leave no room
// for a second block), two blocks a wave: codes in the tiles' buffers 0 and 1,
// scales in 2 and 3, so that a wait for one block is none for the other.
template <int D> struct OwnBlock {
  static constexpr int CHUNKS = D >= 128 ? D / 128 : 1; // of a lane's key
  static constexpr int WORDS = D >= 128 ? 4 : 2;        // of a chunk
  uint32_t key[2][CHUNKS][WORDS], scale[2][CHUNKS];
};

// Blocks [b0, b1) of a sequence's own keys with the columns of unit `unit`, by one
// wave, which waits for no other. As paged_gqa_kernel, which has the arithmetic.
template <int D>
__device__ __forceinline__ void own_piece(const half_t *__restrict__ q,
                                          const uint8_t *__restrict__ pool, const SharedView &g,
                                          half_t *out, unsigned *invalid, unsigned queryHeads,
                                          ScoreScale c, const Partials &parts, const SharedSeq &s,
                                          unsigned kvh, unsigned unit, unsigned b0, unsigned b1,
                                          bool direct, unsigned number) {
  using Block = OwnBlock<D>;
  constexpr int TILES = D / 16;
  const unsigned G = queryHeads / g.kvHeads;
  unsigned tid = threadIdx.x;
  asm volatile("" : "+v"(tid)); // (as in tiles_piece)
  __builtin_assume(tid < kThreads);
  const unsigned lane = tid % 64, quad = lane / 16, r = lane % 16;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const unsigned c0 = unit * kColumns, columns = min(kColumns, s.rows * G - c0);
  auto token_of = [&](unsigned col) { return min((c0 + col) / G, s.rows - 1); };
  auto row_of = [&](unsigned col) {
    return ((size_t)(s.row0 + token_of(col)) * queryHeads + kvh * G + (c0 + col) % G) * D;
  };
  const unsigned visible = s.last(token_of(r)); // this lane's column's last key
  const size_t row = row_of(r);
  if (!s.ok) { // no place for this sequence
    if (r < columns)
#pragma unroll 1
      for (unsigned x = quad; x < D; x += 4)
        out[row + x] = (half_t)NAN;
    if (invalid && lane == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  const unsigned least = s.last(c0 / G), most = s.last((c0 + columns - 1) / G);
  // the keys that this wave has: to the sequence's end, or to a page that is not
  // in the pool, whose columns' outputs are NaN
  const unsigned whole = s.keys();
  unsigned end = whole;
  b1 = min(b1, most / 32 + 1);
  const unsigned mine = b1 > b0 ? b1 - b0 : 0u;

  // A lane knows where one block in 64 is.
  size_t place = 0;
  auto find_blocks = [&](unsigned k) {
    const unsigned b = b0 + k + lane;
    bool lost = false;
    if (b < b1)
      lost = !paged_block(g, s.from, 32 * b, kvh, place);
    if (const unsigned long long all = __builtin_amdgcn_ballot_w64(lost))
      end = min(end, 32 * (b0 + k + (unsigned)__builtin_ctzll(all)));
  };
  // (a block past the last is asked for with a descriptor of no bytes)
  auto issue = [&](unsigned k, Block &block, char *values, char *scales) {
    if (k % 64 == 0)
      find_blocks(k);
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)place, k % 64);
    const unsigned hi = __builtin_amdgcn_readlane((unsigned)(place >> 32), k % 64);
    const size_t at0 = reinterpret_cast<size_t>(pool) + ((size_t)hi << 32 | lo);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void *)((size_t)uniform((unsigned)(at0 >> 32)) << 32 | uniform((unsigned)at0)), (short)0,
        uniform(k < mine ? 40 * D : 0), kBufferWord3);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // this buffer's last reads are done
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (lds_void_t *)(values + 16 * D * wave + 1024 * i), 16, 20 * D + 1024 * i + 16 * lane,
          0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(scales + 1024 * wave), 16,
                                             36 * D + 16 * lane, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < Block::CHUNKS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = t * 8 * D + i * 1024 + lane * 4 * Block::WORDS;
        if constexpr (Block::WORDS == 4) {
          const uint4_t v = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            block.key[t][i][w] = v[w];
        } else {
          typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
          const uint2_t v = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
          block.key[t][i][0] = v[0], block.key[t][i][1] = v[1];
        }
        const unsigned group = D >= 128 ? 4 * i + quad : quad / 2;
        block.scale[t][i] = __builtin_amdgcn_raw_buffer_load_b32(
            rs, 16 * D + t * 2 * D + (group * 16 + r) * 4, 0, 0);
      }
  };

  half8_t qv[Block::CHUNKS][Block::WORDS];
#pragma unroll
  for (int i = 0; i < Block::CHUNKS; ++i)
#pragma unroll
    for (int w = 0; w < Block::WORDS; ++w)
      qv[i][w] = with_sign(load8(q + row + (4 * i + quad) * 8 * Block::WORDS + 8 * w), c.sign);
  float m = -INFINITY, l = 0.0f;
  float4_t o[TILES];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
    o[i] = float4_t{0, 0, 0, 0};
  const Nibbles nibbles;
  auto consume = [&](unsigned k, const Block &block, char *values,
                     char *scales) __attribute__((always_inline)) {
    values += 16 * D * wave;
    scales += 1024 * wave;
    const unsigned base = 32 * (b0 + k);
    float4_t acc[2] = {float4_t{0, 0, 0, 0}, float4_t{0, 0, 0, 0}};
#pragma unroll
    for (int i = 0; i < Block::CHUNKS; ++i)
#pragma unroll
      for (int w = 0; w < Block::WORDS; ++w)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          acc[t] = mfma16x16x32(paged_eight(block.key[t][i][w],
                                            __builtin_bit_cast(half2_t, block.scale[t][i]), nibbles),
                                qv[i][w], acc[t]);
    // (no decoding ahead of its use past these: it would take the registers that
    // the block in flight has)
    __builtin_amdgcn_sched_barrier(0);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = scaled_score(acc[e / 4][e % 4], c.c);
    const unsigned first = base + 16 * (quad / 2) + 4 * (quad % 2); // key of slot 4 t + v
    if (base + 31 > least) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = first + 8 * (e / 4) + e % 4 <= visible ? x[e] : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
      top = fmaxf(top, x[e]);
    if (__builtin_amdgcn_ballot_w64(top - m > kPagedRaise)) {
      LanePair p = pair16(top);
      const float two = fmaxf(p.a, p.b);
      p = pair32(two);
      const float all = fmaxf(p.a, p.b);
      const float to = all - m > kPagedRaise ? all - kPagedHeadroom : m;
      const float alpha = m == to ? 1.0f : fast_exp2(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
        o[i] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.0f : m; // nothing seen yet: weights 0
    half8_t w;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e] = (half_t)fast_exp2(x[e] - ref);
    l = dot8(w, half8_t{1, 1, 1, 1, 1, 1, 1, 1}, l);
    // The slots behind the last key hold anything, and 0 times that may be NaN:
    // their values' scales and biases become 0. (A lane has one slot's scale or
    // bias in every group.)
    if (base + 32 > end) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the block is there, before it is changed
      const unsigned slot = lane % 8;
      const unsigned behind = 16 * (lane / 16 % 2) + 8 * (slot / 4) + 4 * (lane / 8 % 2) + slot % 4;
      if (base + behind >= end) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          *reinterpret_cast<half_t *>(scales + 128 * i + 2 * lane) = (half_t)0;
      }
    }
#pragma unroll
    for (int st = 0; st < D / 64; ++st) {
      __builtin_amdgcn_sched_barrier(0);
      const uint4_t word = *reinterpret_cast<const uint4_t *>(values + st * 1024 + lane * 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char *at = scales + (2 * st + half) * 128 + quad * 16;
        const half8_t sc = *reinterpret_cast<const half8_t *>(at);
        const half8_t bi = *reinterpret_cast<const half8_t *>(at + 64);
#pragma unroll
        for (int n = 0; n < 2; ++n)
          o[4 * st + 2 * half + n] =
              mfma16x16x32(paged_eight(word[2 * half + n], sc, bi, nibbles), w,
                           o[4 * st + 2 * half + n]);
      }
    }
  };
  Block a, b;
  issue(0, a, tile_buffer<0>(), tile_buffer<2>());
  unsigned k = 0;
  for (; k + 2 <= mine; k += 2) {
    issue(k + 1, b, tile_buffer<1>(), tile_buffer<3>());
    consume(k, a, tile_buffer<0>(), tile_buffer<2>());
    issue(k + 2, a, tile_buffer<0>(), tile_buffer<2>());
    consume(k + 1, b, tile_buffer<1>(), tile_buffer<3>());
  }
  if (k < mine)
    consume(k, a, tile_buffer<0>(), tile_buffer<2>());

  if (end < whole && invalid && lane == 0)
    atomicOr(invalid, kPagedPlace);
  LanePair p = pair16(l);
  const float half = p.a + p.b;
  p = pair32(half);
  const bool lost = visible >= end;
  const float sum = lost ? NAN : p.a + p.b;
  if (r >= columns)
    return;
  const size_t part = ((size_t)number * g.kvHeads + kvh) * kColumns + r;
  const float scale = 1.0f / sum;
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const unsigned channel = 16 * i + 4 * quad;
    if (direct)
      *reinterpret_cast<half4_t *>(out + row + channel) =
          half4_t{(half_t)(o[i][0] * scale), (half_t)(o[i][1] * scale), (half_t)(o[i][2] * scale),
                  (half_t)(o[i][3] * scale)};
    else
      *reinterpret_cast<float4_t *>(parts.o + part * D + channel) = o[i];
  }
  if (!direct && quad == 0)
    *reinterpret_cast<float2 *>(parts.ml + 2 * part) = make_float2(lost ? 0.0f : m, sum);
}

// The two divisions. The blocks of all units of shared keys, one after the other,
// are cut into runs, one for each of `workers` workgroups a KV head, those of all
// units of own keys into runs, one for each wave of the other workgroups; a unit's
// pieces are where its blocks lie in them. whole: units of shared keys begin with
// a run, so that each workgroup has blocks of one unit and begins once.
struct Mixed {
  unsigned workers, sharedRun, ownRun;
  bool whole;
};
__device__ __forceinline__ unsigned own_units(const SharedSeq &q, unsigned group) {
  return q.step ? (q.rows * group + kColumns - 1) / kColumns : 0u;
}
__device__ __forceinline__ unsigned tile_units(const SharedSeq &q, unsigned group) {
  return q.step ? 0u : (q.rows * group + kTileColumns - 1) / kTileColumns;
}
// Blocks of a unit of shared keys in the runs.
__device__ __forceinline__ unsigned tile_blocks(const SharedSeq &q, const Mixed &x) {
  const unsigned n = Split::blocks(q);
  return x.whole ? (n + x.sharedRun - 1) / x.sharedRun * x.sharedRun : n;
}
// (the host sees to it that the blocks of all units of a kind are no more than 2^31)
__device__ __forceinline__ Mixed mixed_split(const SharedView &g, const SharedLanes &lanes,
                                             unsigned group, const MixedPlan &plan) {
  unsigned shared = 0, own = 0, units = 0, tiles = 0;
  shared_chunks(g, lanes, [&](unsigned, const SharedSeq &q) {
    const unsigned n = own_units(q, group), t = tile_units(q, group), blocks = Split::blocks(q);
    shared += t * blocks;
    own += n * blocks;
    units += n;
    tiles += t;
    return false;
  });
  auto all = [](unsigned n) { return uniform((unsigned)__builtin_amdgcn_readlane((int)wave_scan(n), 63)); };
  shared = all(shared);
  own = all(own);
  units = all(units);
  tiles = all(tiles);
  const float a = (float)(shared + tiles * plan.again) * plan.sharedCost;
  const float b = (float)own * plan.ownCost + (float)units * plan.ownFixed;
  unsigned workers = 0;
  if (shared) {
    workers = max(1u, uniform((unsigned)ceilf((float)plan.cus * a / (a + b) - 0.5f)));
    workers = own ? min(workers, plan.cus - 1) : plan.cus;
  }
  Mixed x{workers, plan.step, 1, false};
  if (workers) {
    auto steps = [&](unsigned n) { return uniform((n + plan.step - 1) / plan.step * plan.step); };
    const unsigned even = steps((shared + workers - 1) / workers);
    // whole runs a unit: longer ones until there are no more than workgroups
    unsigned n = 0, run = even;
    for (int i = 0; i < 5; ++i) {
      n = 0;
      shared_chunks(g, lanes, [&](unsigned c, const SharedSeq &q) { // (the groups come first)
        n += tile_units(q, group) * ((Split::blocks(q) + run - 1) / run);
        return 64 * (c + 1) >= g.count;
      });
      n = all(n);
      if (n <= workers)
        break;
      run = steps(max(run + 1, (unsigned)fminf((float)run * (float)n / (float)workers, 0x1p30f)));
    }
    x.whole = n <= workers && run <= even + plan.again;
    x.sharedRun = x.whole ? run : even;
    x.workers = x.whole ? n : (shared + even - 1) / even;
  }
  const unsigned waves = max(kWaves * (plan.cus - x.workers), 1u);
  x.ownRun = max(uniform((own + waves - 1) / waves), kLeastRun);
  return x;
}

// The sequence whose units have block `at` of a kind, each units(q) units of
// blocks(q) blocks: its first block and its first unit among all; false behind the
// last.
template <typename Units, typename Blocks>
__device__ __forceinline__ bool find_block(const SharedView &g, const SharedLanes &lanes,
                                           Units unitsOf, Blocks blocksOf, unsigned at,
                                           unsigned &seq, unsigned &firstBlock,
                                           unsigned &firstUnit) {
  bool found = false;
  firstBlock = firstUnit = 0;
  shared_chunks(g, lanes, [&](unsigned c, const SharedSeq &q) {
    const unsigned units = unitsOf(q), n = units * blocksOf(q);
    const unsigned blocks = wave_scan(n), sum = wave_scan(units);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(at - firstBlock < blocks);
    if (!past) {
      firstBlock += (unsigned)__builtin_amdgcn_readlane((int)blocks, 63);
      firstUnit += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
      return false;
    }
    const int lane = __builtin_ctzll(past);
    seq = 64 * c + (unsigned)lane;
    firstBlock += (unsigned)__builtin_amdgcn_readlane((int)(blocks - n), lane);
    firstUnit += (unsigned)__builtin_amdgcn_readlane((int)(sum - units), lane);
    found = at - firstBlock < (unsigned)__builtin_amdgcn_readlane((int)n, lane);
    return true;
  });
  return found;
}

// A run of the blocks of a kind, taken unit by unit: each(s, seq, unit, first block
// of the piece in its unit, blocks of the piece, of the unit, first block and unit
// of the sequence), until it says false. s: the sequence, one of the first
// `sequences` of the view (the groups come first).
template <typename Units, typename Blocks, typename Count, typename Next,
          typename Each>
__device__ __forceinline__ void each_piece(const SharedView &g, const SharedLanes &lanes,
                                           Units unitsOf, Blocks blocksOf, Count sequences,
                                           unsigned at, unsigned run, Next next, Each each) {
  unsigned seq, firstBlock, firstUnit;
  const unsigned stop = at + run;
  if (!find_block(g, lanes, unitsOf, blocksOf, at, seq, firstBlock, firstUnit))
    return;
  seq = uniform(seq);
  firstBlock = uniform(firstBlock);
  firstUnit = uniform(firstUnit);
  SharedSeq s = paged_from_lane(paged_seq_of(g, lanes, seq), 0);
  while (true) {
    const unsigned units = uniform(unitsOf(s)), blocks = uniform(blocksOf(s));
    while (at < stop && at - firstBlock < units * blocks) {
      const unsigned unit = uniform((at - firstBlock) / blocks);
      const unsigned b0 = uniform(at - firstBlock - unit * blocks);
      const unsigned length = uniform(min(blocks - b0, stop - at));
      if (!each(s, seq, unit, b0, length, blocks, firstBlock, firstUnit))
        return;
      at += length;
    }
    if (at >= stop || ++seq >= sequences())
      return;
    firstBlock += units * blocks;
    firstUnit += units;
    s = next(seq);
  }
}

struct MixedArgs {
  const half_t *q;
  const uint8_t *pool;
  SharedView g;
  half_t *out;
  unsigned *invalid;
  unsigned queryHeads;
  MixedPlan plan;
  ScoreScale c;
  Partials shared, rest;
  unsigned mostShared, mostOwn;
};
// The arguments, read again: kept in registers over the pieces of a run they and
// what comes of them fill the scalar ones, and with these full the compiler takes
// no operand of the tiles' products ahead (16 drafts: 56 us, 52.6 so; six groups
// 48 and 44).
__device__ __forceinline__ MixedArgs mixed_args() {
  auto at = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const MixedArgs *)at;
}

template <int D>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads),
                          amdgpu_waves_per_eu(2, 2)))
void paged_mixed_kernel(MixedArgs args) {
  const unsigned G = args.queryHeads / args.g.kvHeads, kvh = blockIdx.x % args.g.kvHeads;
  const unsigned me = blockIdx.x / args.g.kvHeads;
  const SharedLanes lanes = paged_own(args.g);
  const Mixed x = mixed_split(args.g, lanes, G, args.plan);
  if (blockIdx.x == 0 && threadIdx.x == 0)
    args.g.notes[args.g.count + args.g.all] =
        SharedNote{x.ownRun, x.sharedRun, x.whole ? 0u : 1u, 0, 0};
  if (me < x.workers) {
    bool again = false;
    each_piece(
        args.g, lanes, [&](const SharedSeq &q) {
          const MixedArgs a = mixed_args();
          return tile_units(q, a.queryHeads / a.g.kvHeads);
        },
        [&](const SharedSeq &q) { return tile_blocks(q, x); }, [&] { return mixed_args().g.count; }, me * x.sharedRun,
        x.sharedRun,
        [&](unsigned seq) {
          const MixedArgs a = mixed_args();
          return paged_from_lane(shared_seq(a.g, shared_groups(a.g), seq), 0);
        },
        [&](const SharedSeq &s, unsigned seq, unsigned unit, unsigned b0, unsigned length,
            unsigned blocks, unsigned firstBlock, unsigned firstUnit) {
          if (again)
            __syncthreads(); // the piece before is done with its LDS
          again = true;
          const MixedArgs a = mixed_args();
          const unsigned group = a.queryHeads / a.g.kvHeads, head = blockIdx.x % a.g.kvHeads;
          const unsigned number = (x.whole ? 0u : firstUnit + unit) + blockIdx.x / a.g.kvHeads;
          if (number >= a.mostShared) // (starts out of order: more than the rows can have)
            return false;
          // (units of as many columns each, in whole tiles)
          const unsigned units = tile_units(s, group), each = (s.rows * group + units - 1) / units;
          const unsigned width = uniform((each + 31) & ~31u);
          if (unit == 0 && b0 == 0 && head == 0 && threadIdx.x == 0)
            a.g.notes[seq] = SharedNote{firstBlock, blocks, firstUnit, s.row0, width};
          tiles_piece<D, 1, false>(a.q, a.pool, a.g, a.out, a.invalid, a.queryHeads, a.c, a.shared,
                                   s, seq, head, unit, width, b0,
                                   uniform(min(length, Split::blocks(s) - b0)), false,
                                   uniform(number));
          return !x.whole;
        });
    return;
  }
  // this wave's run of own blocks
  const unsigned worker = uniform((me - x.workers) * kWaves + threadIdx.x / 64);
  each_piece(
      args.g, lanes, [&](const SharedSeq &q) { return own_units(q, G); },
      [&](const SharedSeq &q) { return Split::blocks(q); }, [&] { return args.g.sequences; }, worker * x.ownRun,
      x.ownRun,
      [&](unsigned seq) { return paged_from_lane(shared_seq(args.g, lanes.groups, seq), 0); },
      [&](const SharedSeq &s, unsigned seq, unsigned unit, unsigned b0, unsigned length,
          unsigned blocks, unsigned firstBlock, unsigned firstUnit) {
        const unsigned number = worker + firstUnit + unit;
        if (number >= args.mostOwn)
          return false;
        if (unit == 0 && b0 == 0 && kvh == 0 && threadIdx.x % 64 == 0)
          args.g.notes[seq] = SharedNote{firstBlock, s.ok ? blocks : 0u, firstUnit,
                                         s.begin ? s.group + 1 : 0u, 0};
        own_piece<D>(args.q, args.pool, args.g, args.out, args.invalid, args.queryHeads, args.c,
                     args.rest, s, kvh, unit, s.begin + b0, s.begin + b0 + length,
                     length == blocks && !s.joined(), number);
        return true;
      });
}

} // namespace

hipError_t launch_paged_mixed(const half_t *q, const uint8_t *pool, const SharedView &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, const MixedPlan &plan,
                              ScoreScale c, Partials shared, Partials rest, unsigned mostShared,
                              unsigned mostOwn, hipStream_t stream) {
  const MixedArgs args{q, pool, g, out, invalid, queryHeads, plan, c, shared, rest, mostShared,
                       mostOwn};
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(plan.cus * g.kvHeads), dim3(kThreads), 0, stream, args);
    return hipGetLastError();
  };
  return g.dim == 256   ? run(paged_mixed_kernel<256>)
         : g.dim == 128 ? run(paged_mixed_kernel<128>)
                        : run(paged_mixed_kernel<64>);
}

} // namespace llmi
