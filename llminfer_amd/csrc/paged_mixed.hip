// Causal GQA of groups of sequences behind shared keys, in one launch: some
// workgroups have tiles of a group's shared keys, with all its rows as columns
// (paged_tiles.hpp: bound by the matrix cores), the others the sequences' own
// keys, sixteen columns a unit (bound by memory), so that both run at once. The
// partials of the two are joined by paged_shared_merge_kernel.
#include "paged_tiles.hpp"

namespace llmi {
namespace {

constexpr unsigned kColumns = 16; // of a unit of own keys
constexpr unsigned kWaves = kThreads / 64;

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

// Unit `unit` of a sequence's own keys over its piece `piece` of `pieces`: a wave
// has every eighth block of 32 keys. As paged_gqa_kernel, which has the
// arithmetic.
template <int D>
__device__ __forceinline__ void own_piece(const half_t *__restrict__ q,
                                          const uint8_t *__restrict__ pool, const SharedView &g,
                                          half_t *out, unsigned *invalid, unsigned queryHeads,
                                          const Split &split, ScoreScale c, const Partials &parts,
                                          const SharedSeq &s, unsigned kvh, unsigned unit,
                                          unsigned piece, unsigned pieces, unsigned number) {
  using Block = OwnBlock<D>;
  constexpr int TILES = D / 16;
  const unsigned G = queryHeads / g.kvHeads;
  const unsigned tid = threadIdx.x, lane = tid % 64, quad = lane / 16, r = lane % 16;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const unsigned c0 = unit * kColumns, columns = min(kColumns, s.rows * G - c0);
  auto token_of = [&](unsigned col) { return min((c0 + col) / G, s.rows - 1); };
  auto row_of = [&](unsigned col) {
    return ((size_t)(s.row0 + token_of(col)) * queryHeads + kvh * G + (c0 + col) % G) * D;
  };
  const unsigned visible = s.last(token_of(r)); // this lane's column's last key
  const size_t row = row_of(r);
  if (!s.ok) { // no place for this sequence
    if (r < columns && wave == 0)
#pragma unroll 1
      for (unsigned x = quad; x < D; x += 4)
        out[row + x] = (half_t)NAN;
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  const unsigned least = s.last(c0 / G), most = s.last((c0 + columns - 1) / G);
  // the keys that this wave has: to the sequence's end, or to a page that is not
  // in the pool, whose columns' outputs are NaN
  const unsigned whole = s.keys(), length = split.length(s, pieces);
  unsigned end = whole;
  const unsigned b0 = min(s.first() + piece * length, most / 32 + 1);
  const unsigned b1 = min(b0 + length, most / 32 + 1);
  const unsigned mine = b1 > b0 + wave ? (b1 - b0 - wave + kWaves - 1) / kWaves : 0u;

  // Block k of this wave is b0 + wave + kWaves k; a lane knows where one in 64 is.
  size_t place = 0;
  auto find_blocks = [&](unsigned k) {
    const unsigned b = b0 + wave + kWaves * (k + lane);
    bool lost = false;
    if (b < b1)
      lost = !paged_block(g, s.from, 32 * b, kvh, place);
    if (const unsigned long long all = __builtin_amdgcn_ballot_w64(lost))
      end = min(end, 32 * (b0 + wave + kWaves * (k + (unsigned)__builtin_ctzll(all))));
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
    const unsigned base = 32 * (b0 + wave + kWaves * k);
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
  for (unsigned k = 0; k < mine; k += 2) {
    issue(k + 1, b, tile_buffer<1>(), tile_buffer<3>());
    consume(k, a, tile_buffer<0>(), tile_buffer<2>());
    issue(k + 2, a, tile_buffer<0>(), tile_buffer<2>());
    if (k + 1 < mine)
      consume(k + 1, b, tile_buffer<1>(), tile_buffer<3>());
  }

  // Join the waves: (m, l) of the columns, then each wave its output tiles.
  auto out_of = [&](unsigned w) { // wave w's tiles
    return reinterpret_cast<float4_t *>((w / 2 == 0   ? tile_buffer<0>()
                                         : w / 2 == 1 ? tile_buffer<1>()
                                         : w / 2 == 2 ? tile_buffer<2>()
                                                      : tile_buffer<3>()) +
                                        w % 2 * TILES * 1024);
  };
  __shared__ float sM[kWaves * kColumns], sL[kWaves * kColumns];
  __syncthreads(); // the blocks are done with
  if (end < whole && invalid && lane == 0)
    atomicOr(invalid, kPagedPlace);
  LanePair p = pair16(l);
  const float half = p.a + p.b;
  p = pair32(half);
  if (quad == 0) {
    const bool lost = visible >= end;
    sM[wave * kColumns + r] = lost ? 0.0f : m;
    sL[wave * kColumns + r] = lost ? NAN : p.a + p.b;
  }
#pragma unroll
  for (int i = 0; i < TILES; ++i)
    out_of(wave)[i * 64 + lane] = o[i];
  __syncthreads();
  float top = sM[r], sum = 0.0f, by[kWaves];
#pragma unroll
  for (unsigned w = 1; w < kWaves; ++w)
    top = fmaxf(top, sM[w * kColumns + r]);
#pragma unroll
  for (unsigned w = 0; w < kWaves; ++w) {
    const float mw = sM[w * kColumns + r];
    by[w] = mw == -INFINITY ? 0.0f : fast_exp2(mw - top);
    sum += sL[w * kColumns + r] * by[w];
  }
  const size_t part = ((size_t)number * g.kvHeads + kvh) * kColumns + r;
  const bool direct = pieces == 1 && !s.joined();
  const float scale = direct ? 1.0f / sum : 1.0f;
  if (r >= columns)
    return;
  for (unsigned i = wave; i < TILES; i += kWaves) {
    float4_t y{0, 0, 0, 0};
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w)
      y += out_of(w)[i * 64 + lane] * by[w];
    const unsigned channel = 16 * i + 4 * quad;
    if (direct)
      *reinterpret_cast<half4_t *>(out + row + channel) =
          half4_t{(half_t)(y[0] * scale), (half_t)(y[1] * scale), (half_t)(y[2] * scale),
                  (half_t)(y[3] * scale)};
    else
      *reinterpret_cast<float4_t *>(parts.o + part * D + channel) = y;
  }
  if (!direct && wave == 0 && quad == 0)
    *reinterpret_cast<float2 *>(parts.ml + 2 * part) = make_float2(top, sum);
}

// The two divisions: of the groups' shared keys over `workers` workgroups a KV
// head, of the sequences' own keys over the others.
struct Mixed {
  Split shared, own;
  unsigned workers;
};
__device__ __forceinline__ float wave_sum(float x) {
  x = group_sum<16>(x);
  LanePair p = pair16(x);
  x = p.a + p.b;
  p = pair32(x);
  return p.a + p.b;
}
__device__ __forceinline__ Mixed mixed_split(const SharedView &g, const SharedLanes &lanes,
                                             unsigned group, const MixedPlan &plan) {
  Mixed x{Split{group, plan.shift, plan.step, plan.step, 0.0f, true},
          Split{group, 4, kWaves, kWaves, 0.0f, false}, 0};
  float shared = 0.0f, own = 0.0f, units = 0.0f;
  shared_chunks(g, lanes, [&](unsigned, const SharedSeq &q) {
    if (q.step == 0)
      shared += lane_blocks(x.shared, q);
    else {
      own += lane_blocks(x.own, q);
      units += (float)x.own.units(q);
    }
    return false;
  });
  shared = wave_sum(shared);
  own = wave_sum(own);
  units = wave_sum(units);
  auto whole = [](float v) { // (below 2^30: no table has more blocks)
    return (unsigned)__builtin_amdgcn_readfirstlane((int)fminf(ceilf(v), 0x1p30f));
  };
  const float a = shared * plan.sharedCost, b = own * plan.ownCost + units * plan.ownFixed;
  const float cus = (float)plan.cus;
  unsigned workers = shared == 0.0f ? 0u : max(1u, whole(cus * a / (a + b) - 0.5f));
  workers = b == 0.0f ? plan.cus : min(workers, plan.cus - 1);
  auto take = [](Split &s, unsigned chunk) {
    const unsigned steps = (chunk + s.step - 1) & ~(s.step - 1);
    s.chunk = (unsigned)__builtin_amdgcn_readfirstlane((int)(steps ? steps : s.step));
    s.inv = __builtin_amdgcn_rcpf((float)s.chunk);
  };
  take(x.shared, whole(shared * 1.0001f / (float)max(workers, 1u)));
  // Every unit's last piece is rounded up: longer ones until each has a
  // workgroup, undivided units at last (the host sees to it that they fit).
  auto pieces = [&](bool undivided) {
    unsigned n = 0;
    shared_chunks(g, lanes, [&](unsigned, const SharedSeq &q) {
      if (q.step == 0)
        n += x.shared.units(q) * (undivided ? 1u : x.shared.pieces(q));
      return false;
    });
    return (unsigned)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
  };
  unsigned n = pieces(false);
  for (int i = 0; i < 4 && n > workers; ++i) {
    take(x.shared, max(x.shared.chunk + 1, (unsigned)fminf((float)x.shared.chunk * (float)n /
                                                               (float)max(workers, 1u), 0x1p30f)));
    n = pieces(false);
  }
  if (n > workers) {
    take(x.shared, 1u << 30);
    n = pieces(true);
  }
  x.workers = workers = min(n, plan.cus);
  // own keys: as many pieces as the other workgroups, but of 16 blocks at least,
  // and in up to four rounds where they would be longer than 64
  const float rest = (float)max(plan.cus - workers, 1u), even = own * 1.0001f / rest;
  take(x.own, max(16u, whole(fminf(even, fmaxf(64.0f, even * 0.25f)))));
  return x;
}

template <int D, int CT>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads),
                          amdgpu_waves_per_eu(2, 2)))
void paged_mixed_kernel(const half_t *__restrict__ q, const uint8_t *__restrict__ pool,
                        SharedView g, half_t *out, unsigned *invalid, unsigned queryHeads,
                        MixedPlan plan, ScoreScale c, Partials shared, Partials rest,
                        unsigned mostShared, unsigned mostOwn) {
  const unsigned G = queryHeads / g.kvHeads, kvh = blockIdx.x % g.kvHeads;
  const unsigned me = blockIdx.x / g.kvHeads;
  SharedLanes lanes = paged_own(g);
  Mixed x = mixed_split(g, lanes, G, plan);
  // piece u of shared or of own keys: whether there is one, and where
  SharedSeq s;
  unsigned seq, unit, piece, pieces;
  auto find = [&](const Split &split, unsigned step, unsigned u, unsigned most) {
    unsigned local, before;
    if (u >= most || // (starts out of order make more pieces than the rows can have)
        !paged_find(g, lanes, u,
                    [&](const SharedSeq &q) {
                      return q.step == step ? split.units(q) * split.pieces(q) : 0u;
                    },
                    seq, local, before))
      return false;
    seq = uniform(seq);
    local = uniform(local);
    s = paged_from_lane(paged_seq_of(g, lanes, seq), 0);
    pieces = uniform(split.pieces(s));
    const unsigned units = split.units(s);
    unit = units - 1 - local / pieces;
    piece = local % pieces;
    if (local == 0 && kvh == 0 && threadIdx.x == 0)
      leave_note(g, s, seq, before, pieces, units);
    return true;
  };
  if (me < x.workers) {
    if (find(x.shared, 0, me, mostShared))
      tiles_piece<D, CT>(q, pool, g, out, invalid, queryHeads, x.shared, c, shared, s, seq, kvh,
                         unit, piece, pieces, me);
    return;
  }
  for (unsigned u = me - x.workers; find(x.own, 1, u, mostOwn); u += plan.cus - x.workers) {
    own_piece<D>(q, pool, g, out, invalid, queryHeads, x.own, c, rest, s, kvh, unit, piece, pieces,
                 u);
    __syncthreads(); // done with its LDS
    // (made again for the next: kept, the lengths would need registers that the
    // pieces have none of)
    lanes = paged_own(g);
    x = mixed_split(g, lanes, G, plan);
  }
}

} // namespace

hipError_t launch_paged_mixed(const half_t *q, const uint8_t *pool, const SharedView &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, const MixedPlan &plan,
                              ScoreScale c, Partials shared, Partials rest, unsigned mostShared,
                              unsigned mostOwn, hipStream_t stream) {
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(plan.cus * g.kvHeads), dim3(kThreads), 0, stream, q, pool, g,
                       out, invalid, queryHeads, plan, c, shared, rest, mostShared, mostOwn);
    return hipGetLastError();
  };
  if (g.dim == 256)
    return run(paged_mixed_kernel<256, 1>);
  if (g.dim == 128)
    return plan.shift == 8 ? run(paged_mixed_kernel<128, 2>) : run(paged_mixed_kernel<128, 1>);
  return plan.shift == 8 ? run(paged_mixed_kernel<64, 2>) : run(paged_mixed_kernel<64, 1>);
}

} // namespace llmi
