// Causal GQA over the paged 4-bit cache (paged_kv.hpp): a ragged batch of
// sequences, each with any number of new rows.
//
// The 16-column kernel: for one sequence and KV head, the query rows of that
// head's group (token c / G, head c % G of column c) are 16 columns of the
// score tiles, S^T = K Q^T with v_mfma_f32_16x16x32_f16. A workgroup takes a
// range of the keys; each of its waves its own blocks of 32 keys, without
// waiting for the others:
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
// Keys are divided over workgroups by a plan that every workgroup makes for
// itself from the lengths in device memory (a captured call may be replayed on
// others); pagedGqaMerge joins the rows whose keys were divided.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"

#include <math.h>

namespace llmi {
namespace {

constexpr unsigned kColumns = 16;
constexpr unsigned kWaves = 4;
constexpr unsigned kTargetGroups = 256; // workgroups to fill: one a CU
constexpr float kRaise = 15.0f;   // raise m when a weight would pass 2^15
constexpr float kHeadroom = 7.0f; // after a raise the largest weight is 2^7

typedef __attribute__((address_space(3))) void lds_void_t;
constexpr int kBufferWord3 = 0x00020000; // gfx9 raw buffer descriptor, dword 3

__device__ __forceinline__ float4_t mfma16x16x32(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------- the plan

// Units (column blocks) of a sequence, blocks of 32 keys it holds (one where
// it has no place, for the workgroup that says so), and how its keys are
// divided: pieces of `chunk` blocks.
struct Split {
  unsigned group, chunk;
  __device__ unsigned units(const PagedSeq &q) const {
    return (unsigned)(((uint64_t)q.rows * group + kColumns - 1) / kColumns);
  }
  __device__ static unsigned blocks(const PagedSeq &q) {
    return q.ok ? (q.past + q.rows + 31) / 32 : 1u;
  }
  __device__ unsigned pieces(const PagedSeq &q) const { return (blocks(q) + chunk - 1) / chunk; }
};

// The chunk for which the call's blocks make about `target` pieces: a
// multiple of the waves, at least one block each.
__device__ __forceinline__ Split paged_split(const PagedView &g, unsigned group, unsigned target) {
  Split s{group, kWaves};
  const unsigned lane = threadIdx.x % 64;
  uint64_t all = 0;
  for (unsigned s0 = 0; s0 < g.sequences; s0 += 64)
    if (s0 + lane < g.sequences) {
      const PagedSeq q = paged_seq(g, s0 + lane);
      all += (uint64_t)s.units(q) * Split::blocks(q);
    }
  for (int d = 1; d < 64; d *= 2)
    all += __shfl_xor(all, d);
  const uint64_t chunk = (all + target - 1) / target;
  const unsigned whole = (unsigned)((chunk + kWaves - 1) / kWaves * kWaves);
  s.chunk = (unsigned)__builtin_amdgcn_readfirstlane((int)(whole ? whole : kWaves));
  return s;
}

// On the host: most units and pieces a KV head that any lengths can give.
uint64_t most_units(const PagedKvParams &p, unsigned group) {
  const uint64_t a = (uint64_t)p.tokens * ((group + kColumns - 1) / kColumns);
  const uint64_t b = (uint64_t)p.tokens * group / kColumns + p.sequences;
  return a < b ? a : b;
}
unsigned target_pieces(const PagedKvParams &p) {
  return (kTargetGroups + p.kvHeads - 1) / p.kvHeads;
}
uint64_t most_pieces(const PagedKvParams &p, unsigned group) {
  return target_pieces(p) + most_units(p, group);
}

// ------------------------------------------------------------- the kernel

template <int D> struct Geo {
  static constexpr int BLOCK = 40 * D;               // bytes of a block
  static constexpr int LOADS = (BLOCK + 1023) / 1024; // 1-KB loads of one
  static constexpr int STAGE = 1024 * LOADS;
  static constexpr int RING = D == 256 ? 3 : D == 128 ? 5 : 6;
  static constexpr int CHUNKS = D >= 128 ? D / 128 : 1; // of a lane's key
  static constexpr int WORDS = D >= 128 ? 4 : 2;        // of a chunk
  static constexpr int TILES = D / 16;                  // output tiles
};

// The ring's buffers are variables of their own, so that the compiler sees
// that a wait for one need not be a wait for all; the first also takes the
// waves' partial outputs at the end.
template <int D, int I> __device__ __forceinline__ char *ring_buffer() {
  constexpr int stage = kWaves * Geo<D>::STAGE, joined = kWaves * Geo<D>::TILES * 1024;
  __shared__ __attribute__((aligned(1024))) char buffer[I == 0 && joined > stage ? joined : stage];
  return buffer;
}

// Where the output or the partial of a workgroup goes.
struct Partials {
  float *ml, *o; // [piece][KV head][column]{m, l}, [piece][KV head][column][D]
};

template <int D>
__global__ __launch_bounds__(64 * kWaves) void paged_gqa_kernel(
    const half_t *__restrict__ q, const uint8_t *__restrict__ pool, PagedView g, half_t *out,
    unsigned *invalid, unsigned queryHeads, unsigned target, float c, Partials parts) {
  using Geom = Geo<D>;
  const unsigned G = queryHeads / g.kvHeads, kvh = blockIdx.y;
  const Split split = paged_split(g, G, target);
  unsigned seq, local;
  if (!paged_find(g, blockIdx.x,
                  [&](const PagedSeq &s) { return split.units(s) * split.pieces(s); }, seq, local))
    return;
  const PagedSeq s = paged_seq(g, seq);
  const unsigned pieces = split.pieces(s), unit = local / pieces, piece = local % pieces;
  const unsigned tid = threadIdx.x, lane = tid % 64, quad = lane / 16, r = lane % 16;
  const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64);

  // this lane's column (past the unit's last: some row's, not written)
  const unsigned c0 = unit * kColumns, columns = min(kColumns, s.rows * G - c0), col = c0 + r;
  const unsigned token = min(col / G, s.rows - 1), head = kvh * G + col % G;
  const bool live = r < columns;
  const size_t row = ((size_t)(s.row0 + token) * queryHeads + head) * D;
  if (!s.ok) { // no place for this sequence
    if (live && wave == 0)
      for (unsigned x = quad; x < D; x += 4)
        out[row + x] = (half_t)NAN;
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  const unsigned visible = s.past + token;              // the column's last key
  const unsigned least = s.past + c0 / G;               // the first column's
  const unsigned most = s.past + (c0 + columns - 1) / G; // the last column's
  const unsigned end = s.past + s.rows;
  const unsigned b0 = min(piece * split.chunk, most / 32 + 1);
  const unsigned b1 = min(b0 + split.chunk, most / 32 + 1);
  const unsigned mine = b1 > b0 + wave ? (b1 - b0 - wave + kWaves - 1) / kWaves : 0u;

  // Block k of this wave is b0 + wave + 4 k; a lane knows where one in 64 is.
  size_t place = 0;
  bool bad = false;
  auto find_blocks = [&](unsigned k) {
    const unsigned b = b0 + wave + kWaves * (k + lane);
    if (b < b1)
      bad |= !paged_block(g, seq, 32 * b, kvh, place);
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

  // Q^T operands: this column's channels as the key chunks have them.
  half8_t qv[Geom::CHUNKS][Geom::WORDS];
#pragma unroll
  for (int i = 0; i < Geom::CHUNKS; ++i)
#pragma unroll
    for (int w = 0; w < Geom::WORDS; ++w)
      qv[i][w] = load8(q + row + (4 * i + quad) * 8 * Geom::WORDS + 8 * w);

  float m = -INFINITY, l = 0.0f;
  float4_t o[Geom::TILES];
#pragma unroll
  for (int i = 0; i < Geom::TILES; ++i)
    o[i] = float4_t{0, 0, 0, 0};

  auto consume = [&](unsigned k, char *buffer) {
    char *block = buffer + wave * Geom::STAGE;
    const unsigned base = 32 * (b0 + wave + kWaves * k);
    // The slots behind the sequence's last key hold anything, and 0 times that
    // may be NaN: their values' scales and biases become 0. (A lane has one
    // slot's scale or bias in every group.)
    const unsigned slot = lane % 8, behind = 16 * (lane / 16 % 2) + 8 * (slot / 4) +
                                             4 * (lane / 8 % 2) + slot % 4;
    if (base + 32 > end) {
      if (base + behind >= end) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          *reinterpret_cast<half_t *>(block + 36 * D + 128 * i + 2 * lane) = (half_t)0;
      }
    }
    float x[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float4_t acc{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < Geom::CHUNKS; ++i) {
        uint32_t word[Geom::WORDS];
        const char *at = block + t * 8 * D + i * 1024 + lane * 4 * Geom::WORDS;
        if constexpr (Geom::WORDS == 4) {
          const uint4_t v = *reinterpret_cast<const uint4_t *>(at);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            word[w] = v[w];
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(at);
          word[0] = v.x, word[1] = v.y;
        }
        const unsigned group = D >= 128 ? 4 * i + quad : quad / 2;
        const half2_t sb = *reinterpret_cast<const half2_t *>(block + 16 * D + t * 2 * D +
                                                              (group * 16 + r) * 4);
        const half2_t sc{sb[0], sb[0]}, bi{sb[1], sb[1]};
#pragma unroll
        for (int w = 0; w < Geom::WORDS; ++w) {
          const half2_t k0 = paged_pair<0>(word[w], sc, bi), k1 = paged_pair<1>(word[w], sc, bi);
          const half2_t k2 = paged_pair<2>(word[w], sc, bi), k3 = paged_pair<3>(word[w], sc, bi);
          acc = mfma16x16x32(half8_t{k0[0], k0[1], k1[0], k1[1], k2[0], k2[1], k3[0], k3[1]},
                             qv[i][w], acc);
        }
      }
#pragma unroll
      for (int v = 0; v < 4; ++v)
        x[4 * t + v] = acc[v] * c;
    }
    // key of slot 4 t + v of this lane
    const unsigned first = base + 16 * (quad / 2) + 4 * (quad % 2);
    if (base + 31 > least) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = first + 8 * (e / 4) + e % 4 <= visible ? x[e] : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
      top = fmaxf(top, x[e]);
    if (__builtin_amdgcn_ballot_w64(top > m + kRaise)) {
      LanePair p = pair16(top);
      top = fmaxf(p.a, p.b);
      p = pair32(top);
      top = fmaxf(p.a, p.b);
      const float to = top > m + kRaise ? top - kHeadroom : m;
      const float alpha = m == to ? 1.0f : fast_exp2(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < Geom::TILES; ++i)
        o[i] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.0f : m; // nothing seen yet: weights 0
    half8_t w;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e] = (half_t)fast_exp2(x[e] - ref);
    const half8_t ones{1, 1, 1, 1, 1, 1, 1, 1};
    l = dot8(w, ones, l);
#pragma unroll
    for (int st = 0; st < D / 64; ++st) {
      const uint4_t word = *reinterpret_cast<const uint4_t *>(block + 20 * D + st * 1024 + lane * 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char *at = block + 36 * D + (2 * st + half) * 128 + quad * 16;
        const half8_t sc = *reinterpret_cast<const half8_t *>(at);
        const half8_t bi = *reinterpret_cast<const half8_t *>(at + 64);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u = word[2 * half + j];
          const half2_t v0 = paged_pair<0>(u, half2_t{sc[0], sc[1]}, half2_t{bi[0], bi[1]});
          const half2_t v1 = paged_pair<1>(u, half2_t{sc[2], sc[3]}, half2_t{bi[2], bi[3]});
          const half2_t v2 = paged_pair<2>(u, half2_t{sc[4], sc[5]}, half2_t{bi[4], bi[5]});
          const half2_t v3 = paged_pair<3>(u, half2_t{sc[6], sc[7]}, half2_t{bi[6], bi[7]});
          o[4 * st + 2 * half + j] =
              mfma16x16x32(half8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]}, w,
                           o[4 * st + 2 * half + j]);
        }
      }
    }
  };

  // R blocks in flight, their buffers known at compile time.
  constexpr int R = Geom::RING;
  static_assert(R >= 3 && R <= 6, "the buffers below");
  auto buffer = [&](int i) -> char * {
    switch (i % R) {
    case 0:
      return ring_buffer<D, 0>();
    case 1:
      return ring_buffer<D, 1>();
    case 2:
      return ring_buffer<D, 2>();
    case 3:
      return ring_buffer<D, (R > 3 ? 3 : 0)>();
    case 4:
      return ring_buffer<D, (R > 4 ? 4 : 0)>();
    default:
      return ring_buffer<D, (R > 5 ? 5 : 0)>();
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
  __shared__ float sM[kWaves][kColumns], sL[kWaves][kColumns];
  LanePair p = pair16(l);
  l = p.a + p.b;
  p = pair32(l);
  l = p.a + p.b;
  if (__builtin_amdgcn_ballot_w64(bad)) {
    l = NAN; // a page that is not in the pool
    if (invalid && lane == 0)
      atomicOr(invalid, kPagedPlace);
  }
  if (quad == 0) {
    sM[wave][r] = m;
    sL[wave][r] = l;
  }
  __syncthreads(); // (the ring's blocks are done with)
  float4_t *sO = reinterpret_cast<float4_t *>(ring_buffer<D, 0>());
#pragma unroll
  for (int i = 0; i < Geom::TILES; ++i)
    sO[(wave * Geom::TILES + i) * 64 + lane] = o[i];
  __syncthreads();
  float top = sM[0][r], sum = 0.0f, a[kWaves];
#pragma unroll
  for (unsigned w = 1; w < kWaves; ++w)
    top = fmaxf(top, sM[w][r]);
#pragma unroll
  for (unsigned w = 0; w < kWaves; ++w) {
    a[w] = sM[w][r] == -INFINITY ? 0.0f : fast_exp2(sM[w][r] - top);
    sum += sL[w][r] * a[w]; // (a wave's NaN stays: its m is a number, or every page was bad)
  }
  const size_t part = ((size_t)blockIdx.x * g.kvHeads + kvh) * kColumns + r;
  const float scale = pieces == 1 ? 1.0f / sum : 1.0f;
  for (unsigned i = wave; i < (unsigned)Geom::TILES; i += kWaves) {
    float4_t y{0, 0, 0, 0};
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w)
      y += sO[(w * Geom::TILES + i) * 64 + lane] * a[w];
    if (!live)
      continue;
    if (pieces == 1)
      *reinterpret_cast<half4_t *>(out + row + 16 * i + 4 * quad) =
          half4_t{(half_t)(y[0] * scale), (half_t)(y[1] * scale), (half_t)(y[2] * scale),
                  (half_t)(y[3] * scale)};
    else
      *reinterpret_cast<float4_t *>(parts.o + part * D + 16 * i + 4 * quad) = y;
  }
  if (pieces > 1 && wave == 0 && quad == 0 && live)
    *reinterpret_cast<float2 *>(parts.ml + 2 * part) = make_float2(top, sum);
}

// One workgroup a row, query head and 64 channels: four waves, each every
// fourth piece.
constexpr unsigned kMergeWaves = 4;
template <int D>
__global__ __launch_bounds__(64 * kMergeWaves) void paged_gqa_merge_kernel(
    PagedView g, half_t *out, unsigned queryHeads, unsigned target, Partials parts) {
  const unsigned G = queryHeads / g.kvHeads;
  const Split split = paged_split(g, G, target);
  unsigned seq, local;
  if (!paged_find(g, blockIdx.x, [](const PagedSeq &s) { return s.rows; }, seq, local))
    return;
  const PagedSeq s = paged_seq(g, seq);
  const unsigned pieces = split.pieces(s);
  if (!s.ok || pieces == 1)
    return;
  const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = blockIdx.y;
  const unsigned column = local * G + h % G, kvh = h / G;
  // the number of the first piece of this column's unit
  unsigned first = 0;
  for (unsigned s0 = 0; s0 < seq; s0 += 64)
    if (s0 + lane < seq) {
      const PagedSeq o = paged_seq(g, s0 + lane);
      first += split.units(o) * split.pieces(o);
    }
  for (int d = 1; d < 64; d *= 2)
    first += __shfl_xor(first, d);
  first += column / kColumns * pieces;
  const float *ml = parts.ml + 2 * (((size_t)first * g.kvHeads + kvh) * kColumns + column % kColumns);
  const float *po = parts.o + (((size_t)first * g.kvHeads + kvh) * kColumns + column % kColumns) * D +
                    64 * blockIdx.z + lane;
  const size_t step = (size_t)g.kvHeads * kColumns;
  float m = -INFINITY, l = 0.0f, y = 0.0f;
  for (unsigned i = wave; i < pieces; i += kMergeWaves) {
    const float mi = ml[2 * step * i], li = ml[2 * step * i + 1], oi = po[step * i * D];
    const float to = fmaxf(m, mi);
    const float a = m == -INFINITY ? 0.0f : fast_exp2(m - to);
    const float b = mi == -INFINITY ? 0.0f : fast_exp2(mi - to);
    l = l * a + li * b;
    y = y * a + oi * b;
    m = to;
  }
  __shared__ float sM[kMergeWaves], sL[kMergeWaves], sY[kMergeWaves][64];
  sM[wave] = m;
  sL[wave] = l;
  sY[wave][lane] = y;
  __syncthreads();
  if (wave)
    return;
  float top = sM[0];
  for (unsigned w = 1; w < kMergeWaves; ++w)
    top = fmaxf(top, sM[w]);
  l = y = 0.0f;
  for (unsigned w = 0; w < kMergeWaves; ++w) {
    const float a = sM[w] == -INFINITY ? 0.0f : fast_exp2(sM[w] - top);
    l += sL[w] * a;
    y += sY[w][lane] * a;
  }
  out[((size_t)(s.row0 + local) * queryHeads + h) * D + 64 * blockIdx.z + lane] = (half_t)(y / l);
}

size_t partials_floats(const PagedKvParams &p, unsigned group, unsigned dim) {
  return (size_t)most_pieces(p, group) * p.kvHeads * kColumns * dim;
}

} // namespace

size_t paged_gqa_workspace_bytes(const PagedKvParams &p, unsigned queryHeads) {
  const unsigned group = queryHeads / p.kvHeads;
  return 4 * (partials_floats(p, group, p.headDim) + partials_floats(p, group, 2));
}

hipError_t launch_paged_gqa(const uint16_t *q, const int32_t *starts, const int32_t *past,
                            const int32_t *table, const void *pool, uint16_t *out,
                            uint32_t *invalid, void *workspace, const PagedKvParams &p,
                            unsigned queryHeads, float scale, hipStream_t stream) {
  const unsigned group = queryHeads / p.kvHeads, target = target_pieces(p);
  const PagedView g = paged_view(p, starts, past, table);
  float *ws = static_cast<float *>(workspace);
  const Partials parts{ws + partials_floats(p, group, p.headDim), ws};
  half_t *to = reinterpret_cast<half_t *>(out);
  auto run = [&](auto kernel, auto merge) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)most_pieces(p, group), p.kvHeads), dim3(64 * kWaves),
                       0, stream, reinterpret_cast<const half_t *>(q),
                       static_cast<const uint8_t *>(pool), g, to, invalid, queryHeads, target,
                       scale * kLog2e, parts);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
      return e;
    hipLaunchKernelGGL(merge, dim3(p.tokens, queryHeads, p.headDim / 64), dim3(64 * kMergeWaves),
                       0, stream, g, to, queryHeads, target, parts);
    return hipGetLastError();
  };
  return p.headDim == 256   ? run(paged_gqa_kernel<256>, paged_gqa_merge_kernel<256>)
         : p.headDim == 128 ? run(paged_gqa_kernel<128>, paged_gqa_merge_kernel<128>)
                            : run(paged_gqa_kernel<64>, paged_gqa_merge_kernel<64>);
}

} // namespace llmi
