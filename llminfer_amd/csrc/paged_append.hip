// Appending to, and reading back from, the paged 4-bit cache (paged_kv.hpp).
//
// A workgroup makes one block's part of the call: the rows of a sequence that
// lie in 32 keys of one KV head. Nobody else writes that block, so a value
// word, which holds eight keys, is read, filled in and written back without
// atomics.
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
__device__ __forceinline__ uint32_t code_of(float x, const Group &g) {
  if (!(g.s > 0.0f))
    return 0;
  const float step = __builtin_rintf(__fdiv_rn(__fsub_rn(x, g.b), g.s)) - 16.0f;
  return (uint32_t)fminf(fmaxf(step, 0.0f), 15.0f);
}

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

template <int D>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(
    const uint16_t *__restrict__ keys, const uint16_t *__restrict__ values, PagedView g,
    const float *__restrict__ freqs, uint8_t *pool, unsigned *invalid, AppendRows p) {
  extern __shared__ float2 sTurn[]; // [rows of this block][half]
  unsigned seq, local, before;
  const PagedSeq own = paged_own(g);
  if (!paged_find(g, own, blockIdx.x, [](const PagedSeq &q) { return touched_blocks(q); }, seq,
                  local, before))
    return;
  const PagedSeq q = paged_seq_of(g, own, seq);
  const unsigned head = blockIdx.y, tid = threadIdx.x;
  // keys [first, last) of the block at position base, from the call's row `row`
  const unsigned base = q.past / 32 * 32 + 32 * local;
  const unsigned first = base < q.past ? q.past - base : 0u;
  const unsigned last = min(32u, q.past + q.rows - base), n = last - first;
  const unsigned row = q.row0 + (base + first - q.past);
  size_t at = 0;
  if (!q.ok || !paged_block(g, seq, base, head, at)) {
    if (invalid && tid == 0)
      atomicOr(invalid, kPagedPlace);
    return;
  }
  uint8_t *block = pool + at;
  for (unsigned i = tid; i < n * p.half; i += kThreads)
    sTurn[i] = rope_turn((int)(base + first + i / p.half), freqs[i % p.half], p.factor);
  __syncthreads();
  bool bad = false;

  // Keys: a thread has 8 channels of one, four neighbours a group.
  constexpr unsigned W = D / 8;
  for (unsigned i = tid; i < n * W; i += kThreads) {
    const unsigned r = i / W, word = i % W, key = first + r;
    const uint16_t *x = keys + (size_t)(row + r) * p.keyToken + (size_t)head * p.keyHead;
    float v[8];
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned c = 8 * word + e;
      uint16_t y = x[c];
      if (c < 2 * p.half) {
        const unsigned pair = p.layout ? c / 2 : c < p.half ? c : c - p.half;
        const bool low = p.layout ? c % 2 == 0 : c < p.half;
        const unsigned other = p.layout ? c ^ 1u : low ? c + p.half : c - p.half;
        const float2 cs = sTurn[r * p.half + pair];
        y = low ? turn_x(h2f(y), h2f(x[other]), cs) : turn_y(h2f(x[other]), h2f(y), cs);
      }
      v[e] = kept(h2f(y), bad);
    }
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
    uint32_t packed = 0;
#pragma unroll
    for (unsigned e = 0; e < 8; ++e)
      packed |= code_of(v[e], grp) << paged_nibble(e);
    *reinterpret_cast<uint32_t *>(block + paged_key_word(D, key, word)) = packed;
    if (word % 4 == 0)
      *reinterpret_cast<half2_t *>(block + paged_key_scale(D, key, word / 4)) =
          half2_t{grp.scale, grp.bias};
  }

  // Values: a wave takes 64 channels, a lane four of them (16 apart) for the
  // eight keys of its quad.
  const unsigned lane = tid % 64, quad = lane / 16, r = lane % 16;
  for (unsigned st = tid / 64; st < D / 64; st += kThreads / 64) {
    uint32_t word[4] = {0, 0, 0, 0}, mask = 0;
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      const unsigned key = 16 * (quad / 2) + 8 * (e / 4) + 4 * (quad % 2) + e % 4;
      const bool here = key >= first && key < last;
      if (!__builtin_amdgcn_ballot_w64(here))
        continue;
      const uint16_t *x = values + (size_t)(row + (here ? key - first : 0u)) * p.valueToken +
                          (size_t)head * p.valueHead + 64 * st + r;
      float v[4];
      bool off = false;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        v[w] = kept(h2f(x[16 * w]), off);
      bad |= off && here;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Group grp = group_of(row_min(fminf(v[2 * half], v[2 * half + 1])),
                                   row_max(fmaxf(v[2 * half], v[2 * half + 1])));
        word[2 * half] |= code_of(v[2 * half], grp) << paged_nibble(e);
        word[2 * half + 1] |= code_of(v[2 * half + 1], grp) << paged_nibble(e);
        if (here && r == 0) {
          half_t *s = reinterpret_cast<half_t *>(block + paged_value_scale(D, key, 2 * st + half));
          s[0] = grp.scale;
          s[32] = grp.bias;
        }
      }
      mask |= here ? 15u << paged_nibble(e) : 0u;
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
  }
  if (invalid && __builtin_amdgcn_ballot_w64(bad) && lane == 0)
    atomicOr(invalid, kPagedValue);
}

// A thread reads 8 channels of one row's key or value.
__global__ __launch_bounds__(kThreads) void paged_read_kernel(const uint8_t *__restrict__ pool,
                                                              PagedView g, uint16_t *keys,
                                                              uint16_t *values,
                                                              unsigned *invalid) {
  unsigned seq, local, before;
  const PagedSeq own = paged_own(g);
  if (!paged_find(g, own, blockIdx.x, [](const PagedSeq &q) { return touched_blocks(q); }, seq,
                  local, before))
    return;
  const PagedSeq q = paged_seq_of(g, own, seq);
  const unsigned head = blockIdx.y, tid = threadIdx.x, W = g.dim / 8;
  const unsigned base = q.past / 32 * 32 + 32 * local;
  const unsigned first = base < q.past ? q.past - base : 0u;
  const unsigned last = min(32u, q.past + q.rows - base);
  const unsigned row = q.row0 + (base + first - q.past);
  size_t at = 0;
  const bool ok = q.ok && paged_block(g, seq, base, head, at);
  if (!ok && invalid && tid == 0)
    atomicOr(invalid, kPagedPlace);
  const uint8_t *block = pool + at;
  for (unsigned i = tid; i < (last - first) * W; i += kThreads) {
    const unsigned r = i / W, word = i % W, key = first + r, group = word / 4;
    const half_t nan = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
    half8_t k, v;
    if (ok) {
      const uint32_t kw = *reinterpret_cast<const uint32_t *>(block + paged_key_word(g.dim, key, word));
      const half2_t km = *reinterpret_cast<const half2_t *>(block + paged_key_scale(g.dim, key, group));
      const half_t *vm =
          reinterpret_cast<const half_t *>(block + paged_value_scale(g.dim, key, group));
#pragma unroll
      for (unsigned e = 0; e < 8; ++e) {
        k[e] = paged_value(kw, e, km[0], km[1]);
        const uint32_t vw = *reinterpret_cast<const uint32_t *>(
            block + paged_value_word(g.dim, key, 8 * word + e));
        v[e] = paged_value(vw, paged_slot(key), vm[0], vm[32]);
      }
    } else {
      k = half8_t{nan, nan, nan, nan, nan, nan, nan, nan};
      v = k;
    }
    const size_t to = ((size_t)(row + r) * g.kvHeads + head) * g.dim + 8 * word;
    *reinterpret_cast<half8_t *>(keys + to) = k;
    *reinterpret_cast<half8_t *>(values + to) = v;
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
  const dim3 grid(most_units(p.tokens, p.sequences), p.kvHeads);
  const size_t lds = 32 * (a.rotaryDim / 2) * sizeof(float2);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, stream, keys, values, g, freqs,
                       static_cast<uint8_t *>(pool), invalid, r);
    return hipGetLastError();
  };
  return p.headDim == 256   ? run(paged_append_kernel<256>)
         : p.headDim == 128 ? run(paged_append_kernel<128>)
                            : run(paged_append_kernel<64>);
}

hipError_t launch_paged_read(const void *pool, const int32_t *starts, const int32_t *past,
                             const int32_t *table, uint16_t *keys, uint16_t *values,
                             uint32_t *invalid, const PagedKvParams &p, hipStream_t stream) {
  hipLaunchKernelGGL(paged_read_kernel, dim3(most_units(p.tokens, p.sequences), p.kvHeads),
                     dim3(kThreads), 0, stream, static_cast<const uint8_t *>(pool),
                     paged_view(p, starts, past, table), keys, values, invalid);
  return hipGetLastError();
}

} // namespace llmi
