// Causal GQA over the paged 4-bit cache (paged_kv.hpp): a ragged batch of
// sequences, each with any number of new rows.
#include "hip_common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"

#include <math.h>

namespace llmi {
namespace {

// One wave a row and query head: a block of 32 keys at a time, a lane half a
// key's channels for the scores, then D/64 channels for the sum, with the
// running maximum and sum of the softmax.
__global__ __launch_bounds__(64) void paged_gqa_rows_kernel(
    const half_t *__restrict__ q, const uint8_t *__restrict__ pool, PagedView g, half_t *out,
    unsigned *invalid, unsigned queryHeads, float scale) {
  unsigned seq, local;
  if (!paged_find(g, blockIdx.x, [](const PagedSeq &s) { return s.rows; }, seq, local))
    return;
  const PagedSeq s = paged_seq(g, seq);
  const unsigned h = blockIdx.y, head = h / (queryHeads / g.kvHeads), lane = threadIdx.x;
  const unsigned D = g.dim, visible = s.past + local + 1, key = lane / 2;
  const half_t *x = q + ((size_t)(s.row0 + local) * queryHeads + h) * D;
  half_t *y = out + ((size_t)(s.row0 + local) * queryHeads + h) * D;
  float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
  bool ok = s.ok;
  for (unsigned base = 0; ok && base < visible; base += 32) {
    size_t at;
    ok = paged_block(g, seq, base, head, at);
    if (!ok)
      break;
    const uint8_t *block = pool + at;
    float score = 0.0f;
    for (unsigned word = lane % 2 * (D / 16); word < (lane % 2 + 1) * (D / 16); ++word) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(block + paged_key_word(D, key, word));
      const half2_t sb =
          *reinterpret_cast<const half2_t *>(block + paged_key_scale(D, key, word / 4));
      for (unsigned e = 0; e < 8; ++e)
        score = fmaf((float)x[8 * word + e], (float)paged_value(w, e, sb[0], sb[1]), score);
    }
    score += __shfl_xor(score, 1);
    score = base + key < visible ? score * scale : -INFINITY;
    float top = score;
    for (int d = 2; d < 64; d *= 2)
      top = fmaxf(top, __shfl_xor(top, d));
    const float mNew = fmaxf(m, top);
    const float p = expf(score - mNew), alpha = expf(m - mNew);
    m = mNew;
    float sum = p;
    for (int d = 2; d < 64; d *= 2)
      sum += __shfl_xor(sum, d);
    l = l * alpha + sum;
    for (unsigned c = 0; c < D / 64; ++c)
      o[c] *= alpha;
    const unsigned keys = min(32u, visible - base);
    for (unsigned k = 0; k < keys; ++k) {
      const float pk = __shfl(p, (int)(2 * k));
      for (unsigned c = 0; c < D / 64; ++c) {
        const unsigned ch = 64 * c + lane;
        const uint32_t w = *reinterpret_cast<const uint32_t *>(block + paged_value_word(D, k, ch));
        const half_t *sb =
            reinterpret_cast<const half_t *>(block + paged_value_scale(D, k, ch / 32));
        o[c] = fmaf(pk, (float)paged_value(w, paged_slot(k), sb[0], sb[32]), o[c]);
      }
    }
  }
  if (!ok && invalid && lane == 0)
    atomicOr(invalid, kPagedPlace);
  for (unsigned c = 0; c < D / 64; ++c)
    y[64 * c + lane] = (half_t)(ok ? o[c] / l : NAN);
}

} // namespace

size_t paged_gqa_workspace_bytes(const PagedKvParams &, unsigned) { return 0; }

hipError_t launch_paged_gqa(const uint16_t *q, const int32_t *starts, const int32_t *past,
                            const int32_t *table, const void *pool, uint16_t *out,
                            uint32_t *invalid, void *, const PagedKvParams &p,
                            unsigned queryHeads, float scale, hipStream_t stream) {
  hipLaunchKernelGGL(paged_gqa_rows_kernel, dim3(p.tokens, queryHeads), dim3(64), 0, stream,
                     reinterpret_cast<const half_t *>(q), static_cast<const uint8_t *>(pool),
                     paged_view(p, starts, past, table), reinterpret_cast<half_t *>(out), invalid,
                     queryHeads, scale);
  return hipGetLastError();
}

} // namespace llmi
