// Rotary embedding of rows at positions of their own: half or interleaved
// pairs, any part of the head, given frequencies, strided rows.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "rope_rows.hpp"

namespace llmi {
namespace {

constexpr unsigned kThreads = 256;
constexpr unsigned kTurns = 1024; // cos/sin pairs that a token may have

struct RopeRows {
  unsigned heads, dim, half, layout;
  unsigned inToken, inHead, outToken, outHead;
  float factor;
};

// A row in parts: eight pairs a part (two 16-byte words of the row, side by
// side where pairs are interleaved), then eight channels a part that are
// copied; the last of either may have fewer where the row is not VEC.
struct Parts {
  unsigned turned, all;
  __host__ __device__ Parts(unsigned half, unsigned dim)
      : turned((half + 7) / 8), all(turned + (dim - 2 * half + 7) / 8) {}
};

// A workgroup takes a token and the heads of blockIdx.y: its cosines and sines
// once, into LDS, then the rows of all its heads, `across` threads to a row. A
// thread owns whole pairs, so a row may be rotated in place.
// Bound by the rows' bytes: 16381 tokens of 16 heads of 256, 64 rotated, pass
// in 55 us, a copy of as many bytes in 56; 2048 tokens of 16 heads of 128 in 5.0
// (5.9 with four tokens a workgroup). VEC: whole 16-byte words; else words at any
// element (186 of the 256 rotated: 62 us warm, 77 channel by channel; 192, VEC: 42).
template <bool VEC>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(
    const uint16_t *in, const int *__restrict__ positions, const float *__restrict__ freqs,
    uint16_t *out, unsigned headBlock, unsigned across, RopeRows p) {
  __shared__ float2 sTurn[kTurns];
  const unsigned t = blockIdx.x;
  const unsigned h0 = blockIdx.y * headBlock, h1 = min(h0 + headBlock, p.heads);
  const int position = p.half ? positions[t] : 0;
  for (unsigned i = threadIdx.x; i < p.half; i += kThreads)
    sTurn[i] = rope_turn(position, freqs[i], p.factor);
  __syncthreads();
  const Parts parts(p.half, p.dim);
  const unsigned down = kThreads / across, y = threadIdx.x / across;
  if (y >= down)
    return;
  for (unsigned part = threadIdx.x % across; part < parts.all; part += across)
    for (unsigned h = h0 + y; h < h1; h += down) {
      const uint16_t *x = in + (size_t)t * p.inToken + (size_t)h * p.inHead;
      uint16_t *z = out + (size_t)t * p.outToken + (size_t)h * p.outHead;
      if (part >= parts.turned) {
        unsigned c = 2 * p.half + 8 * (part - parts.turned);
        if (!VEC && c + 8 > p.dim) {
          if (p.dim - 2 * p.half < 8) {
            for (; c < p.dim; ++c)
              z[c] = x[c];
            continue;
          }
          c = p.dim - 8; // some of them by the part before as well
        }
        store_word<VEC>(z + c, load_word<VEC>(x + c));
        continue;
      }
      // (the last part: eight pairs with those before it, which others write)
      unsigned pair = 8 * part, skip = 0;
      if (!VEC && pair + 8 > p.half) {
        if (p.half < 8) {
          for (; pair < p.half; ++pair) {
            const unsigned a = p.layout ? 2 * pair : pair, b = p.layout ? a + 1 : a + p.half;
            const float s = h2f(x[a]), w = h2f(x[b]);
            z[a] = turn_x(s, w, sTurn[pair]);
            z[b] = turn_y(s, w, sTurn[pair]);
          }
          continue;
        }
        skip = pair - (p.half - 8);
        pair -= skip;
      }
      const unsigned a = p.layout ? 2 * pair : pair, b = p.layout ? a + 8 : a + p.half;
      const uint4_t u = load_word<VEC>(x + a), v = load_word<VEC>(x + b);
      uint16_t e[16], f[16];
      *reinterpret_cast<uint4_t *>(e) = u;
      *reinterpret_cast<uint4_t *>(e + 8) = v;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 cs = sTurn[pair + i];
        const float s = h2f(p.layout ? e[2 * i] : e[i]);
        const float w = h2f(p.layout ? e[2 * i + 1] : e[8 + i]);
        const uint16_t s1 = turn_x(s, w, cs), w1 = turn_y(s, w, cs);
        f[i] = s1; // the turned pairs apart; put side by side below
        f[8 + i] = w1;
      }
      if (!VEC && skip) {
#pragma unroll
        for (unsigned i = 1; i < 8; ++i)
          if (i >= skip) {
            z[p.layout ? a + 2 * i : a + i] = f[i];
            z[p.layout ? a + 2 * i + 1 : b + i] = f[8 + i];
          }
        continue;
      }
      uint4_t lo, hi;
      if (p.layout) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = f[i] | (uint32_t)f[8 + i] << 16;
          hi[i] = f[4 + i] | (uint32_t)f[12 + i] << 16;
        }
      } else {
        lo = *reinterpret_cast<uint4_t *>(f);
        hi = *reinterpret_cast<uint4_t *>(f + 8);
      }
      store_word<VEC>(z + a, lo);
      store_word<VEC>(z + b, hi);
    }
}

} // namespace

bool rope_rows_supported(unsigned rotaryDim) { return rotaryDim / 2 <= kTurns; }

hipError_t launch_rope_rows(const uint16_t *input, const int32_t *positions, const float *freqs,
                            uint16_t *output, const RopeRowsParams &p, hipStream_t stream) {
  const unsigned half = p.rotaryDim / 2;
  // a call of few tokens: its heads over several workgroups, four at least in each
  unsigned headBlock = p.heads;
  while (p.tokens * ((p.heads + headBlock - 1) / headBlock) < 256 && headBlock > 4)
    headBlock = (headBlock + 1) / 2;
  const RopeRows r{p.heads,  p.headDim,          half,
                   p.layout, p.inputTokenStride, p.inputHeadStride,
                   p.outputTokenStride, p.outputHeadStride, p.factor};
  const unsigned strides = p.inputTokenStride | p.inputHeadStride | p.outputTokenStride |
                           p.outputHeadStride;
  const bool vec = half % 8 == 0 && p.headDim % 8 == 0 && strides % 8 == 0 && aligned16(input) &&
                   aligned16(output);
  const dim3 grid(p.tokens, (p.heads + headBlock - 1) / headBlock);
  const unsigned parts = Parts(half, p.headDim).all;
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, input, positions, freqs, output,
                       headBlock, parts < kThreads ? parts : kThreads, r);
    return hipGetLastError();
  };
  return run(vec ? rope_rows_kernel<true> : rope_rows_kernel<false>);
}

} // namespace llmi
