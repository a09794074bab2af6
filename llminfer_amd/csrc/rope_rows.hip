// Rotary embedding of rows at positions of their own: half or interleaved
// pairs, any part of the head, given frequencies, strided rows.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "rope_rows.hpp"

namespace llmi {
namespace {

constexpr unsigned kThreads = 256;
constexpr unsigned kTurns = 1024; // cos/sin pairs that a workgroup keeps

struct RopeRows {
  unsigned heads, dim, half, layout;
  unsigned inToken, inHead, outToken, outHead;
  float factor;
};

// A workgroup takes `block` tokens and the heads of blockIdx.y: their cosines
// and sines once, into LDS, then the rows of all its heads. A thread owns
// whole pairs, so that a row may be rotated in place.
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(
    const uint16_t *in, const int *__restrict__ positions, const float *__restrict__ freqs,
    uint16_t *out, unsigned tokens, unsigned block, unsigned headBlock, RopeRows p) {
  __shared__ float2 sTurn[kTurns];
  const unsigned t0 = blockIdx.x * block, count = min(block, tokens - t0);
  const unsigned h0 = blockIdx.y * headBlock, heads = min(headBlock, p.heads - h0);
  for (unsigned i = threadIdx.x; i < count * p.half; i += kThreads)
    sTurn[i] = rope_turn(positions[t0 + i / p.half], freqs[i % p.half], p.factor);
  __syncthreads();
  const unsigned rest = p.dim - 2 * p.half, items = p.half + rest;
  for (unsigned i = threadIdx.x; i < count * heads * items; i += kThreads) {
    const unsigned item = i % items, row = i / items, h = h0 + row % heads, t = row / heads;
    const uint16_t *x = in + (size_t)(t0 + t) * p.inToken + (size_t)h * p.inHead;
    uint16_t *y = out + (size_t)(t0 + t) * p.outToken + (size_t)h * p.outHead;
    if (item < p.half) {
      const unsigned a = p.layout ? 2 * item : item, b = p.layout ? a + 1 : a + p.half;
      const float2 cs = sTurn[t * p.half + item];
      const float u = h2f(x[a]), v = h2f(x[b]);
      y[a] = turn_x(u, v, cs);
      y[b] = turn_y(u, v, cs);
    } else {
      const unsigned c = p.half + item;
      y[c] = x[c];
    }
  }
}

} // namespace

bool rope_rows_supported(unsigned rotaryDim) { return rotaryDim / 2 <= kTurns; }

hipError_t launch_rope_rows(const uint16_t *input, const int32_t *positions, const float *freqs,
                            uint16_t *output, const RopeRowsParams &p, hipStream_t stream) {
  const unsigned half = p.rotaryDim / 2;
  unsigned block = half ? kTurns / half : 16;
  block = block > 4 ? 4 : block;
  const RopeRows r{p.heads,          p.headDim,         half,
                   p.layout,         p.inputTokenStride, p.inputHeadStride,
                   p.outputTokenStride, p.outputHeadStride, p.factor};
  hipLaunchKernelGGL(rope_rows_kernel, dim3((p.tokens + block - 1) / block, 1), dim3(kThreads), 0,
                     stream, input, positions, freqs, output, p.tokens, block, p.heads, r);
  return hipGetLastError();
}

} // namespace llmi
