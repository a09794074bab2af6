// Appending to, and reading back from, the paged 4-bit cache (paged_kv.hpp).
//
// A block's part of a call (the rows of a sequence that lie in 32 keys of one
// KV head) is the work of a few workgroups: one for its values, the others
// each for some of its keys. A value word holds eight keys and is read, filled
// in and written back by the one workgroup that has them, without atomics; a
// key's words are its own.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "rope_rows.hpp"

namespace llmi {
namespace {

constexpr unsigned kThreads = 256;

struct AppendRows {
  unsigned keyToken, keyHead, valueToken, valueHead, half, layout;
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

// The value as the cache takes it; sets `bad` for one that it cannot hold.
__device__ __forceinline__ float kept(float x, bool &bad) {
  bad |= !(fabsf(x) <= kPagedLimit);
  return x != x ? 0.0f : fminf(fmaxf(x, -kPagedLimit), kPagedLimit);
}

struct Group {
  half_t scale, bias;
  float s, b;
};
__device__ __forceinline__ Group group_of(float low, float high) {
  Group g;
  g.scale = f16_of(__fdiv_rn(__fsub_rn(high, low), 15.0f));
  g.s = (float)g.scale;
  g.bias = f16_of(__fsub_rn(low, mul32(16.0f, g.s)));
  g.b = (float)g.bias;
  return g;
}
// clamp(rint((x - b) / s) - 16, 0, 15). The quotient as a product with the
// hardware's reciprocal is within 2^-17 of the exact one (at most 32, off by
// three half steps of fp32 and the reciprocal's one); where that could change
// the rounding, the division decides.
struct Coder {
  float s, b, inv;
  __device__ explicit Coder(const Group &g)
      : s(g.s), b(g.b), inv(g.s > 0.0f ? __builtin_amdgcn_rcpf(g.s) : 0.0f) {}
  __device__ uint32_t operator()(float x) const {
    const float d = __fsub_rn(x, b);
    float q = mul32(d, inv);
    const float r = __builtin_rintf(q);
    // a scale below 2^-14 (fp16's subnormals) has quotients past 32: divided too
    if (fabsf(fabsf(q - r) - 0.5f) < 0x1p-12f || s < 0x1p-14f)
      q = s > 0.0f ? __fdiv_rn(d, s) : 0.0f;
    return (uint32_t)fminf(fmaxf(__builtin_rintf(q) - 16.0f, 0.0f), 15.0f);
  }
};

__device__ __forceinline__ float row_min(float x) { // over the 16 lanes of a row
  x = fminf(x, row_ror<1>(x));
  x = fminf(x, row_ror<2>(x));
  x = fminf(x, row_ror<4>(x));
  return fminf(x, row_ror<8>(x));
}
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, row_ror<1>(x));
  x = fmaxf(x, row_ror<2>(x));
  x = fmaxf(x, row_ror<4>(x));
  return fmaxf(x, row_ror<8>(x));
}

// Keys that one workgroup takes of a block: eight channels a thread.
constexpr unsigned keys_a_group(unsigned D) { return 8 * kThreads / D; }
constexpr unsigned key_groups(unsigned D) { return 32 / keys_a_group(D); }

// VEC: eight channels of a key, and those that they are rotated with, are
// each one 16-byte load.
template <int D, bool VEC>
__device__ __forceinline__ bool append_keys(const uint16_t *__restrict__ x, unsigned word,
                                            unsigned key,
                                            const float2 *__restrict__ turn, uint8_t *block,
                                            const AppendRows &p) {
  uint16_t own[8], other[8];
  const unsigned c0 = 8 * word;
  const bool turned = c0 < 2 * p.half; // (VEC: all eight or none)
  const bool low = c0 < p.half;
  if constexpr (VEC) {
    *reinterpret_cast<uint4_t *>(own) = *reinterpret_cast<const uint4_t *>(x + c0);
    const unsigned far = !turned || p.layout ? c0 : low ? c0 + p.half : c0 - p.half;
    *reinterpret_cast<uint4_t *>(other) = *reinterpret_cast<const uint4_t *>(x + far);
  } else {
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned c = c0 + e;
      own[e] = x[c];
      other[e] = x[c >= 2 * p.half ? c : p.layout ? c ^ 1u : c < p.half ? c + p.half : c - p.half];
    }
  }
  bool bad = false;
  float v[8];
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) {
    const unsigned c = c0 + e;
    uint16_t y = own[e];
    if (VEC ? turned : c < 2 * p.half) {
      if (p.layout) {
        const float2 cs = turn[c / 2];
        const uint16_t with = VEC ? own[e ^ 1] : other[e];
        y = e % 2 == 0 ? turn_x(h2f(y), h2f(with), cs) : turn_y(h2f(with), h2f(y), cs);
      } else {
        const bool first = VEC ? low : c < p.half;
        const float2 cs = turn[first ? c : c - p.half];
        y = first ? turn_x(h2f(y), h2f(other[e]), cs) : turn_y(h2f(other[e]), h2f(y), cs);
      }
    }
    v[e] = kept(h2f(y), bad);
  }
  // four neighbours have a group
  float lo = v[0], hi = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fminf(lo, v[e]);
    hi = fmaxf(hi, v[e]);
  }
  lo = fminf(lo, dpp<kDppXor1>(lo));
  hi = fmaxf(hi, dpp<kDppXor1>(hi));
  lo = fminf(lo, dpp<kDppXor2>(lo));
  hi = fmaxf(hi, dpp<kDppXor2>(hi));
  const Group grp = group_of(lo, hi);
  const Coder code(grp);
  uint32_t packed = 0;
#pragma unroll
  for (unsigned e = 0; e < 8; ++e)
    packed |= code(v[e]) << paged_nibble(e);
  *reinterpret_cast<uint32_t *>(block + paged_key_word(D, key, word)) = packed;
  if (word % 4 == 0)
    *reinterpret_cast<half2_t *>(block + paged_key_scale(D, key, word / 4)) =
        half2_t{grp.scale, grp.bias};
  return bad;
}

// Values of keys [first, last) of a block, 64 channels from 64 st on: a lane
// has four of them (16 apart) for the eight keys of its quad.
template <int D>
__device__ __forceinline__ bool append_values(const uint16_t *__restrict__ x, size_t stride,
                                              unsigned first, unsigned last, unsigned st,
                                              uint8_t *block) {
  const unsigned lane = threadIdx.x % 64, quad = lane / 16, r = lane % 16;
  auto key_of = [&](unsigned e) { return 16 * (quad / 2) + 8 * (e / 4) + 4 * (quad % 2) + e % 4; };
  auto here = [&](unsigned e) { return key_of(e) >= first && key_of(e) < last; };
  uint16_t raw[8][4] = {};
#pragma unroll
  for (unsigned e = 0; e < 8; ++e)
    if (here(e)) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        raw[e][w] = x[(key_of(e) - first) * stride + 64 * st + 16 * w + r];
    }
  uint32_t word[4] = {0, 0, 0, 0}, mask = 0;
  bool bad = false;
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) {
    if (!__builtin_amdgcn_ballot_w64(here(e)))
      continue;
    float v[4];
#pragma unroll
    for (int w = 0; w < 4; ++w)
      v[w] = kept(h2f(raw[e][w]), bad);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Group grp = group_of(row_min(fminf(v[2 * half], v[2 * half + 1])),
                                 row_max(fmaxf(v[2 * half], v[2 * half + 1])));
      const Coder code(grp);
      word[2 * half] |= code(v[2 * half]) << paged_nibble(e);
      word[2 * half + 1] |= code(v[2 * half + 1]) << paged_nibble(e);
      if (here(e) && r == 0) {
        half_t *s =
            reinterpret_cast<half_t *>(block + paged_value_scale(D, key_of(e), 2 * st + half));
        s[0] = grp.scale;
        s[32] = grp.bias;
      }
    }
    mask |= here(e) ? 15u << paged_nibble(e) : 0u;
  }
  if (mask) {
    uint4_t *to = reinterpret_cast<uint4_t *>(block + 20 * D + st * 1024 + lane * 16);
    uint4_t w{word[0], word[1], word[2], word[3]};
    if (mask != 0xFFFFFFFFu) {
      const uint4_t old = *to;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (w[j] & mask) | (old[j] & ~mask);
    }
    *to = w;
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
  const unsigned head = blockIdx.y, tid = threadIdx.x;
  const bool ofValues = blockIdx.z == key_groups(D);
  // this workgroup's keys [first, last)
  const unsigned first = ofValues ? b.first : max(b.first, keys_a_group(D) * blockIdx.z);
  const unsigned last = ofValues ? b.last : min(b.last, keys_a_group(D) * (blockIdx.z + 1));
  if (first >= last)
    return;
  size_t at = 0;
  if (!b.ok || !paged_block(g, b.seq, b.base, head, at)) {
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  uint8_t *block = pool + at;
  const size_t row = b.row + (first - b.first);
  bool bad = false;
  if (ofValues) {
    const uint16_t *x = values + row * p.valueToken + (size_t)head * p.valueHead;
    for (unsigned st = tid / 64; st < D / 64; st += kThreads / 64)
      bad |= append_values<D>(x, p.valueToken, first, last, st, block);
  } else {
    for (unsigned i = tid; i < (last - first) * p.half; i += kThreads) {
      const unsigned k = i / p.half;
      sTurn[i] = rope_turn((int)(b.base + first + k), freqs[i - k * p.half], p.factor);
    }
    __syncthreads();
    const unsigned k = tid / (D / 8), word = tid % (D / 8);
    if (k < last - first) {
      const uint16_t *x = keys + (row + k) * p.keyToken + (size_t)head * p.keyHead;
      bad = append_keys<D, VEC>(x, word, first + k, sTurn + k * p.half, block, p);
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
  if (ok && blockIdx.z == 0) {
    for (unsigned i = tid; i < 4 * D; i += kThreads) { // words: key, eight channels
      const unsigned key = i / (D / 8), word = i % (D / 8);
      const uint32_t w = *reinterpret_cast<const uint32_t *>(block + paged_key_word(D, key, word));
      const half2_t m =
          *reinterpret_cast<const half2_t *>(block + paged_key_scale(D, key, word / 4));
      const half2_t sc{m[0], m[0]}, bi{m[1], m[1]};
      const half2_t v0 = paged_pair<0>(w, sc, bi), v1 = paged_pair<1>(w, sc, bi);
      const half2_t v2 = paged_pair<2>(w, sc, bi), v3 = paged_pair<3>(w, sc, bi);
      *reinterpret_cast<half8_t *>(sRow + key * PITCH + 8 * word) =
          half8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
    }
  } else if (ok) {
    const unsigned quad = lane / 16, r = lane % 16;
    for (unsigned st = tid / 64; st < D / 64; st += kThreads / 64) {
      const uint4_t w = *reinterpret_cast<const uint4_t *>(block + 20 * D + st * 1024 + lane * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t *m = block + 36 * D + (2 * st + j / 2) * 128 + quad * 16;
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
  const AppendRows r{a.keyTokenStride,   a.keyHeadStride,  a.valueTokenStride,
                     a.valueHeadStride, a.rotaryDim / 2, a.layout, a.factor};
  const dim3 grid(most_units(p.tokens, p.sequences), p.kvHeads, key_groups(p.headDim) + 1);
  const size_t lds = keys_a_group(p.headDim) * r.half * sizeof(float2);
  // (half % 8: a word's channels are all of one half, and their partners a word)
  const bool vec = (a.layout || r.half % 8 == 0) && r.half % 4 == 0 && aligned16(keys) &&
                   (a.keyTokenStride | a.keyHeadStride) % 8 == 0;
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
