// C ABI of the HIP backend: validation, kernel selection, workspace sizing
// and status reporting. Declarations and contracts: include/llminfer_hip.h.
#include "llminfer_hip.h"
#include "capi_internal.hpp"
#include "kernels.hpp"
#include "rope_gate.hpp"

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

namespace llmi {

namespace {
thread_local char g_error[512] = "";
} // namespace

int fail(int status, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof g_error, fmt, ap);
  va_end(ap);
  return status;
}

int launched(hipError_t err, const char *what) {
  if (err == hipSuccess)
    return LLMI_HIP_OK;
  return fail(LLMI_HIP_LAUNCH_FAILED, "%s: %s", what, hipGetErrorString(err));
}

// Mirrors the reference lowering's 32-bit element-index limit
// (lib/Backend/Metal/MetalExecutionPlan.cpp:32-40).
static bool fits32(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t ab = a * b;
  if (a && ab / a != b)
    return false;
  uint64_t abc = ab * c;
  if (ab && abc / ab != c)
    return false;
  return abc <= 0xffffffffull;
}

// Whether no two rows of tokens x heads rows of `dim` elements overlap, the
// heads of a token inside its stride or the tokens of a head inside its.
static bool strides_apart(uint64_t tokens, uint64_t tokenStride, uint64_t heads,
                          uint64_t headStride, uint64_t dim) {
  if (tokens == 1 || heads == 1)
    return (tokens == 1 || tokenStride >= dim) && (heads == 1 || headStride >= dim);
  return (headStride >= dim && tokenStride >= (heads - 1) * headStride + dim) ||
         (tokenStride >= dim && headStride >= (tokens - 1) * tokenStride + dim);
}

int check_gqa(const GqaParams &p) {
  if (p.tokens == 0 || p.queryHeads == 0 || p.kvHeads == 0 || p.headDim == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "CausalGqa: tokens, heads and head_dim must be positive");
  if (p.queryHeads % p.kvHeads)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "CausalGqa: query heads %u not a multiple of KV heads %u",
                p.queryHeads, p.kvHeads);
  uint64_t rows = (uint64_t)p.past + p.tokens;
  if (!fits32(p.tokens, p.queryHeads, p.headDim) ||
      !fits32(rows, p.kvHeads, p.headDim))
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "CausalGqa: tensor exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

int check_delta(const GraphDeltaParams &p) {
  if (!p.tokens || !p.keyHeads || !p.keyDim || !p.valueHeads || !p.valueDim)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "DeltaUpdate: every dimension must be positive");
  if (p.valueHeads % p.keyHeads)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "DeltaUpdate: value heads %u not a multiple of key heads %u",
                p.valueHeads, p.keyHeads);
  if (!fits32(p.tokens, p.keyHeads, p.keyDim) ||
      !fits32(p.tokens, p.valueHeads, p.valueDim) ||
      !fits32(p.valueHeads, p.keyDim, p.valueDim))
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "DeltaUpdate: tensor exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

GqaKernel select_gqa(const GqaParams &p) {
  GqaShape s{p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past};
  if (p.tokens == 1 && decode_supported(s))
    return GqaKernel::Decode;
  if (p.tokens > 1 && prefill_supported(s))
    return GqaKernel::Prefill;
  if (generic_supported(s))
    return GqaKernel::Generic;
  return GqaKernel::None;
}

DeltaKernel select_delta(const GraphDeltaParams &p) {
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  if (p.tokens > 1 && delta_chunked_supported(s))
    return DeltaKernel::Chunked;
  if (delta_recurrent_supported(s))
    return DeltaKernel::Recurrent;
  return DeltaKernel::Generic;
}

} // namespace llmi

using namespace llmi;

// normRope / rmsNorm / partialRope as one row shape. Rows per tile (one
// wave each): about 2048 tiles (two waves per SIMD on 256 CUs), but at least
// 8 rows once there are 4096 rows, since the sequential sum costs a tile the
// same whatever its row count, and 2 for a decode step's few rows, where the
// wave's latency is what counts (a sweep of 1..32 on MI355X: q 2048x16 rows
// best at 16, k 2048x4 at 4-8, decode 16 rows at 2).
RopeShape rope_shape(unsigned rows, unsigned heads, unsigned D, unsigned rot,
                     unsigned stride, unsigned past, unsigned out_row0, float eps,
                     float theta, bool norm) {
  unsigned rw = (rows + 2047) / 2048;
  unsigned lo = rows >= 4096 ? 8 : 2;
  rw = rw < lo ? lo : rw > 64 ? 64 : rw;
  return RopeShape{rows, heads, D, rot, stride, past, out_row0, eps, theta, norm, rw};
}

int check_rope(const char *what, uint64_t rows, unsigned heads, unsigned D,
               unsigned rot, uint64_t in_extent, uint64_t out_rows) {
  if (rows && heads == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: heads == 0", what);
  if (rot % 2 || rot > D)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "%s: rotary width %u must be even and <= width %u", what, rot, D);
  if (!fits32(rows, in_extent, 1) || !fits32(out_rows, D, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: exceeds the 32-bit index range", what);
  return LLMI_HIP_OK;
}

int rope_kernel_name_index(const RopeShape &s) {
  return norm_rope_tiled(s, nullptr, nullptr) ? 0 : norm_rope_wide_rows(s) ? 2 : 1;
}

static const char *rope_kernel_name(const RopeShape &s, const char *tile, const char *rows,
                                    const char *wide) {
  const int i = rope_kernel_name_index(s);
  return i == 0 ? tile : i == 2 ? wide : rows;
}

extern "C" {

int llmi_hip_norm_rope(const uint16_t *input, const float *weight, uint16_t *output,
                       RopeParams p, void *stream) {
  uint64_t rows = (uint64_t)p.tokens * p.heads;
  if (rows == 0 || p.headDim == 0)
    return LLMI_HIP_OK;
  if (!input || !weight || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "normRope: null buffer");
  if (int st = check_rope("normRope", rows, p.heads, p.headDim, p.rotaryDim,
                          p.headStride > p.headDim ? p.headStride : p.headDim,
                          ((uint64_t)p.outputStart + p.tokens) * p.heads))
    return st;
  if ((uint64_t)p.past + p.tokens > 0xffffffffull)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "normRope: past + tokens overflows");
  RopeShape s = rope_shape((unsigned)rows, p.heads, p.headDim, p.rotaryDim, p.headStride,
                           p.past, p.outputStart * p.heads, p.epsilon, p.theta, true);
  return launched(launch_norm_rope(input, weight, output, s,
                                   static_cast<hipStream_t>(stream)),
                  "normRope");
}

int llmi_hip_rms_norm(const uint16_t *input, const float *weight, uint16_t *output,
                      RowParams p, void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!input || !weight || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rmsNorm: null buffer");
  if (int st = check_rope("rmsNorm", p.rows, 1, p.width, 0, p.width, p.rows))
    return st;
  RopeShape s = rope_shape(p.rows, 1, p.width, 0, p.width, 0, 0, p.epsilon, 0.0f, true);
  return launched(launch_norm_rope(input, weight, output, s,
                                   static_cast<hipStream_t>(stream)),
                  "rmsNorm");
}

int llmi_hip_partial_rope(const uint16_t *input, uint16_t *output, PartialRopeParams p,
                          void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!input || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "partialRope: null buffer");
  if (int st = check_rope("partialRope", p.rows, p.heads, p.width, p.rotaryWidth,
                          p.width, p.rows))
    return st;
  if ((uint64_t)p.past + p.rows / p.heads > 0xffffffffull)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "partialRope: past + tokens overflows");
  RopeShape s = rope_shape(p.rows, p.heads, p.width, p.rotaryWidth, p.width, p.past, 0,
                           0.0f, p.theta, false);
  return launched(launch_norm_rope(input, nullptr, output, s,
                                   static_cast<hipStream_t>(stream)),
                  "partialRope");
}

int llmi_hip_sigmoid_mul(const uint16_t *gate, const uint16_t *input, uint16_t *output,
                         ElementParams p, void *stream) {
  if (p.count == 0)
    return LLMI_HIP_OK;
  if (!gate || !input || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "sigmoidMul: null buffer");
  return launched(launch_sigmoid_mul(gate, input, output, p.count,
                                     static_cast<hipStream_t>(stream)),
                  "sigmoidMul");
}

int llmi_hip_causal_conv(const uint16_t *input, const uint16_t *weight, uint16_t *history,
                         uint16_t *output, ConvParams p, void *stream) {
  if (p.tokens == 0 || p.channels == 0)
    return LLMI_HIP_OK;
  if (!causal_conv_supported(p.kernelSize))
    return fail(LLMI_HIP_UNSUPPORTED, "causalConv: kernel size %u (1..8 supported)",
                p.kernelSize);
  if (!input || !weight || !output || (p.kernelSize > 1 && !history))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "causalConv: null buffer");
  if (!fits32(p.tokens, p.channels, 1) || !fits32(p.channels, p.kernelSize, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "causalConv: exceeds the 32-bit index range");
  return launched(launch_causal_conv(input, weight, history, output, p.tokens, p.channels,
                                     p.kernelSize, p.applySilu ? 1u : 0u,
                                     static_cast<hipStream_t>(stream)),
                  "causalConv");
}

int llmi_hip_l2_norm(const uint16_t *input, float *output, L2Params p, void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!input || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "l2NormF32: null buffer");
  if (!fits32(p.rows, p.width, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "l2NormF32: exceeds the 32-bit index range");
  return launched(launch_l2_norm(input, output, p.rows, p.width, p.epsilon, p.scale,
                                 static_cast<hipStream_t>(stream)),
                  "l2NormF32");
}

int llmi_hip_delta_gates(const uint16_t *a, const uint16_t *b, const float *a_log,
                         const float *dt_bias, float *beta, float *decay, RowParams p,
                         void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!a || !b || !a_log || !dt_bias || !beta || !decay)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "deltaGates: null buffer");
  if (!fits32(p.rows, p.width, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "deltaGates: exceeds the 32-bit index range");
  return launched(launch_delta_gates(a, b, a_log, dt_bias, beta, decay, p.rows, p.width,
                                     static_cast<hipStream_t>(stream)),
                  "deltaGates");
}

// ------------------------------------------------------ W8A8 projections

int llmi_hip_quantize_activation(const uint16_t *input, int8_t *quantized, float *scales,
                                 uint32_t *invalid, QuantizeParams p, void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!input || !quantized || !scales)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "quantizeActivation: null buffer");
  if (p.groups != (p.width + 31) / 32)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "quantizeActivation: %u groups for width %u (32-element groups: %u)",
                p.groups, p.width, (p.width + 31) / 32);
  if (!fits32(p.rows, p.groups, 32) || !fits32(p.rows, p.width, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "quantizeActivation: exceeds the 32-bit index range");
  if (!aligned16(quantized))
    return fail(LLMI_HIP_UNSUPPORTED, "quantizeActivation: quantized rows not 16-byte aligned");
  return launched(launch_quantize_activation(input, quantized, scales, invalid, p.rows, p.width,
                                             p.groups, static_cast<hipStream_t>(stream)),
                  "quantizeActivation");
}

static int check_linear_w8(const LinearW8Params &p) {
  if (p.epilogue > LLMI_LINEAR_DELTA_DECAY)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: unknown epilogue %u", p.epilogue);
  if (p.epilogue == LLMI_LINEAR_SIGMOID_COLUMNS && p.epilogueBlock == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: sigmoid columns need a block width");
  if (p.groups == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: no groups");
  if ((uint64_t)p.firstRow + p.columns > p.outputWidth)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "linearW8A8: columns %u from %u past the output width %u", p.columns,
                p.firstRow, p.outputWidth);
  if (!fits32(p.rows, p.groups, 32) || !fits32(p.columns, p.groups, 32) ||
      !fits32(p.rows, p.outputWidth, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

int llmi_hip_linear_w8a8(const int8_t *activation, const float *act_scales,
                         const int8_t *weight, const uint16_t *weight_scales, void *output,
                         const void *aux, const float *bias, LinearW8Params p, void *stream) {
  if (p.rows == 0 || p.columns == 0)
    return LLMI_HIP_OK;
  if (int rc = check_linear_w8(p))
    return rc;
  if (!activation || !act_scales || !weight || !weight_scales || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: null buffer");
  if (p.epilogue == LLMI_LINEAR_SILU_MUL && !aux)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: SiluMul needs its multiplier (aux)");
  if (p.epilogue == LLMI_LINEAR_DELTA_DECAY && (!aux || !bias))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearW8A8: the decay needs A_log (aux) and bias");
  if (!aligned16(activation) || !aligned16(weight))
    return fail(LLMI_HIP_UNSUPPORTED,
                "linearW8A8: activation and weight rows must be 16-byte aligned");
  const W8Shape s{p.outputWidth, p.firstRow, p.groups, p.rows, p.columns, p.epilogue,
                  p.epilogueBlock};
  return launched(launch_linear_w8a8(activation, act_scales, weight, weight_scales, output, aux,
                                     bias, s, static_cast<hipStream_t>(stream)),
                  linear_w8a8_kernel(p.rows));
}

int llmi_hip_embedding_w8(const uint32_t *ids, const int8_t *weight, const uint16_t *scales,
                          uint16_t *output, GroupedEmbedParams p, void *stream) {
  if (p.tokens == 0 || p.hidden == 0 || p.rowCount == 0)
    return LLMI_HIP_OK;
  if (!ids || !weight || !scales || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "embeddingW8: null buffer");
  if (p.groups < (p.hidden + 31) / 32)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "embeddingW8: %u groups for hidden %u", p.groups,
                p.hidden);
  if (!fits32(p.tokens, p.hidden, 1) || !fits32(p.rowCount, p.groups, 32))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "embeddingW8: exceeds the 32-bit index range");
  return launched(launch_embedding_w8(ids, weight, scales, output, p.tokens, p.hidden,
                                      p.firstRow, p.rowCount, p.groups,
                                      static_cast<hipStream_t>(stream)),
                  "embeddingW8");
}

int llmi_hip_embedding(const uint32_t *ids, const uint16_t *weight, uint16_t *output,
                       EmbedParams p, void *stream) {
  if (p.tokens == 0 || p.hidden == 0 || p.rowCount == 0)
    return LLMI_HIP_OK;
  if (!ids || !weight || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "embedding: null buffer");
  if (!fits32(p.tokens, p.hidden, 1) || !fits32(p.rowCount, p.hidden, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "embedding: exceeds the 32-bit index range");
  return launched(launch_embedding(ids, weight, output, p.tokens, p.hidden, p.firstRow,
                                   p.rowCount, static_cast<hipStream_t>(stream)),
                  "embedding");
}

static int elementwise(ElementwiseKind kind, const char *name, const uint16_t *a,
                       const uint16_t *b, uint16_t *out, ElementParams p, void *stream) {
  if (p.count == 0)
    return LLMI_HIP_OK;
  if (!a || !out || (kind != ElementwiseKind::Silu && !b))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: null buffer", name);
  return launched(launch_elementwise(kind, a, b, out, p.count, static_cast<hipStream_t>(stream)),
                  name);
}

int llmi_hip_residual_add(const uint16_t *a, const uint16_t *b, uint16_t *out, ElementParams p,
                          void *stream) {
  return elementwise(ElementwiseKind::Add, "residualAdd", a, b, out, p, stream);
}

int llmi_hip_swiglu(const uint16_t *gate, const uint16_t *up, uint16_t *out, ElementParams p,
                    void *stream) {
  return elementwise(ElementwiseKind::SwiGlu, "swiGlu", gate, up, out, p, stream);
}

int llmi_hip_silu(const uint16_t *in, uint16_t *out, ElementParams p, void *stream) {
  return elementwise(ElementwiseKind::Silu, "siluF16", in, nullptr, out, p, stream);
}

int llmi_hip_multiply(const uint16_t *a, const uint16_t *b, uint16_t *out, ElementParams p,
                      void *stream) {
  return elementwise(ElementwiseKind::Multiply, "multiplyF16", a, b, out, p, stream);
}

static int check_add_norm_quantize(const RowParams &p) {
  if (p.width > kAddNormQuantizeMax)
    return fail(LLMI_HIP_UNSUPPORTED, "addRmsNormQuantize: width %u (at most %u)", p.width,
                kAddNormQuantizeMax);
  if (!fits32(p.rows, (p.width + 31) / 32 * 32, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "addRmsNormQuantize: exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

int llmi_hip_add_rms_norm_quantize(const uint16_t *a, const uint16_t *b, uint16_t *sum_out,
                                   const float *weight, int8_t *q, float *scales,
                                   uint32_t *invalid, RowParams p, void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (int rc = check_add_norm_quantize(p))
    return rc;
  if (!a || !weight || !q || !scales || (b && !sum_out))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "addRmsNormQuantize: null buffer");
  if (!aligned16(q))
    return fail(LLMI_HIP_UNSUPPORTED, "addRmsNormQuantize: quantized rows not 16-byte aligned");
  return launched(launch_add_norm_quantize(a, b, sum_out, weight, q, scales, invalid, p.rows,
                                           p.width, p.epsilon, static_cast<hipStream_t>(stream)),
                  b ? "addRmsNormQuantize" : "rmsNormQuantize");
}

static int check_norm_linear(const NormLinearParams &p) {
  const RowParams &n = p.norm;
  if (n.rows != 1 || n.width == 0 || n.width > kNormLinearMaxWidth)
    return fail(LLMI_HIP_UNSUPPORTED, "addRmsNormLinearW8A8: one row of at most %u (%u x %u)",
                kNormLinearMaxWidth, n.rows, n.width);
  if (p.count == 0 || p.count > kNormLinearMax)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "addRmsNormLinearW8A8: %u projections (1 to %u)",
                p.count, kNormLinearMax);
  const unsigned groups = (n.width + 31) / 32;
  unsigned wgs = 0;
  for (unsigned k = 0; k < p.count; ++k) {
    const LinearW8Params &l = p.linear[k];
    if (int rc = check_linear_w8(l))
      return rc;
    if (l.rows != 1 || l.groups != groups || l.columns == 0)
      return fail(LLMI_HIP_INVALID_ARGUMENT,
                  "addRmsNormLinearW8A8: projection %u takes %u rows of %u groups and %u "
                  "columns (one row of %u groups, at least one column)",
                  k, l.rows, l.groups, l.columns, groups);
    wgs += norm_linear_workgroups(l.columns);
  }
  if (wgs > kNormLinearMaxWgs)
    return fail(LLMI_HIP_UNSUPPORTED, "addRmsNormLinearW8A8: %u workgroups (at most %u)", wgs,
                kNormLinearMaxWgs);
  return LLMI_HIP_OK;
}

int llmi_hip_add_rms_norm_linear_w8a8(const uint16_t *a, const uint16_t *b, uint16_t *sum_out,
                                      const float *weight, int8_t *q, float *scales,
                                      uint32_t *invalid,
                                      const llmi_hip_norm_projection *projections,
                                      NormLinearParams p, void *stream) {
  if (int rc = check_norm_linear(p))
    return rc;
  if (!a || !weight || !projections || (b && !sum_out))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "addRmsNormLinearW8A8: null buffer");
  if (q && !aligned16(q))
    return fail(LLMI_HIP_UNSUPPORTED, "addRmsNormLinearW8A8: quantized row not 16-byte aligned");
  NormLinearProj proj[kNormLinearMax];
  for (unsigned k = 0; k < p.count; ++k) {
    const llmi_hip_norm_projection &x = projections[k];
    const LinearW8Params &l = p.linear[k];
    if (!x.weight || !x.weight_scales || !x.output)
      return fail(LLMI_HIP_INVALID_ARGUMENT, "addRmsNormLinearW8A8: projection %u: null buffer",
                  k);
    if (!aligned16(x.weight))
      return fail(LLMI_HIP_UNSUPPORTED,
                  "addRmsNormLinearW8A8: projection %u: weight rows not 16-byte aligned", k);
    bool mate = false; // computed by the lanes of projection k - 1
    if (l.epilogue == LLMI_LINEAR_SILU_MUL) {
      if (!x.aux)
        return fail(LLMI_HIP_INVALID_ARGUMENT,
                    "addRmsNormLinearW8A8: projection %u: SiluMul needs its multiplier (aux)", k);
      mate = k > 0 && x.aux == projections[k - 1].output;
      // (projection k - 1 has no epilogue, so it is nobody's mate itself)
      if (mate && (p.norm.width > kNormLinearPairedWidth ||
                   p.linear[k - 1].epilogue != LLMI_LINEAR_NONE ||
                   p.linear[k - 1].columns != l.columns))
        return fail(LLMI_HIP_UNSUPPORTED,
                    "addRmsNormLinearW8A8: projection %u: a SwiGLU multiplier computed in the "
                    "call must be the previous projection's output, with no epilogue, the same "
                    "columns and width <= %u",
                    k, kNormLinearPairedWidth);
      for (unsigned j = 0; j < p.count; ++j)
        if (j + 1 != k && projections[j].output == x.aux)
          return fail(LLMI_HIP_UNSUPPORTED,
                      "addRmsNormLinearW8A8: projection %u: its SwiGLU multiplier is another "
                      "projection's output",
                      k);
    }
    if (l.epilogue == LLMI_LINEAR_DELTA_DECAY && (!x.aux || !x.bias))
      return fail(LLMI_HIP_INVALID_ARGUMENT,
                  "addRmsNormLinearW8A8: projection %u: the decay needs A_log (aux) and bias", k);
    if (!x.conv_weight != !x.conv_history)
      return fail(LLMI_HIP_INVALID_ARGUMENT,
                  "addRmsNormLinearW8A8: projection %u: a convolution needs its weight and its "
                  "history",
                  k);
    if (x.conv_weight && (l.epilogue != LLMI_LINEAR_NONE || l.firstRow != 0 ||
                          l.columns != l.outputWidth))
      return fail(LLMI_HIP_UNSUPPORTED,
                  "addRmsNormLinearW8A8: projection %u: a convolution takes the whole row of a "
                  "projection with no epilogue",
                  k);
    proj[k] = {x.weight, x.weight_scales, x.output, x.aux, x.bias,
               W8Shape{l.outputWidth, l.firstRow, l.groups, l.rows, l.columns, l.epilogue,
                       l.epilogueBlock},
               false, x.conv_weight, x.conv_history};
    if (mate) {
      if (proj[k - 1].cw)
        return fail(LLMI_HIP_UNSUPPORTED,
                    "addRmsNormLinearW8A8: projection %u: a SwiGLU multiplier has no "
                    "convolution",
                    k);
      proj[k - 1].paired = true;
    }
  }
  return launched(launch_add_norm_linear(a, b, sum_out, weight, q, scales, invalid, p.norm.width,
                                         p.norm.epsilon, proj, p.count,
                                         static_cast<hipStream_t>(stream)),
                  b ? "addRmsNormLinearW8A8" : "rmsNormLinearW8A8");
}

int llmi_hip_gated_rms_norm_activated_quantize(const uint16_t *x, const float *gate,
                                               const float *weight, uint16_t *out, int8_t *q,
                                               float *scales, uint32_t *invalid, RowParams p,
                                               void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!x || !gate || !weight || !out || !q || !scales)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gatedRmsNormQuantize: null buffer");
  if (!fits32(p.rows, p.width, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gatedRmsNormQuantize: exceeds the 32-bit index range");
  if (!gated_rms_norm_quantize_supported(p.width, x, gate, out, q))
    return fail(LLMI_HIP_UNSUPPORTED,
                "gatedRmsNormQuantize: width %u (a multiple of 32, at most 256) or an unaligned "
                "buffer",
                p.width);
  return launched(launch_gated_rms_norm_quantize(x, gate, weight, out, q, scales, invalid, p.rows,
                                                 p.width, p.epsilon,
                                                 static_cast<hipStream_t>(stream)),
                  "gatedRmsNormQuantize");
}

static int check_view(const HalfViewParams &p) {
  uint64_t last = p.offset;
  for (int d = 0; d < 3; ++d) {
    if (p.dims[d] == 0)
      return fail(LLMI_HIP_INVALID_ARGUMENT, "copyHalfView: zero extent on axis %d", d);
    last += (uint64_t)(p.dims[d] - 1) * p.strides[d];
  }
  if ((uint64_t)p.dims[0] * p.dims[1] * p.dims[2] != p.count)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "copyHalfView: count %u is not the view's extent",
                p.count);
  if (last > UINT32_MAX)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "copyHalfView: exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

int llmi_hip_copy_half_view(const uint16_t *src, uint16_t *out, HalfViewParams p, void *stream) {
  if (p.count == 0)
    return LLMI_HIP_OK;
  if (int rc = check_view(p))
    return rc;
  if (!src || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "copyHalfView: null buffer");
  return launched(launch_copy_half_view(src, out, p, static_cast<hipStream_t>(stream)),
                  "copyHalfView");
}

static int check_linear_f16(const LinearParams &p) {
  if (p.epilogue > LLMI_LINEAR_DELTA_DECAY)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: unknown epilogue %u", p.epilogue);
  if (p.epilogue == LLMI_LINEAR_SIGMOID_COLUMNS && p.epilogueBlock == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: sigmoid columns need a block width");
  if (p.inputWidth == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: zero input width");
  if ((uint64_t)p.firstRow + p.rowCount > p.outputWidth)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "linearF16: columns %u from %u past the output width %u", p.rowCount,
                p.firstRow, p.outputWidth);
  if (!fits32(p.tokens, p.inputWidth, 1) || !fits32(p.rowCount, p.inputWidth, 1) ||
      !fits32(p.tokens, p.outputWidth, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: exceeds the 32-bit index range");
  return LLMI_HIP_OK;
}

int llmi_hip_linear_f16(const uint16_t *input, const uint16_t *weight, void *output,
                        const void *aux, const float *bias, LinearParams p, void *stream) {
  if (p.tokens == 0 || p.rowCount == 0)
    return LLMI_HIP_OK;
  if (int rc = check_linear_f16(p))
    return rc;
  if (!input || !weight || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: null buffer");
  if (p.epilogue == LLMI_LINEAR_SILU_MUL && !aux)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: SiluMul needs its multiplier (aux)");
  if (p.epilogue == LLMI_LINEAR_DELTA_DECAY && (!aux || !bias))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "linearF16: the decay needs A_log (aux) and bias");
  return launched(launch_linear_f16(input, weight, output, aux, bias, p,
                                    static_cast<hipStream_t>(stream)),
                  "linearF16");
}

static int gated_norm(const uint16_t *input, const void *gate, bool activated,
                      const float *weight, uint16_t *output, RowParams p, void *stream) {
  if (p.rows == 0 || p.width == 0)
    return LLMI_HIP_OK;
  if (!input || !gate || !weight || !output)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gatedRmsNorm: null buffer");
  if (!fits32(p.rows, p.width, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gatedRmsNorm: exceeds the 32-bit index range");
  return launched(launch_gated_rms_norm(input, gate, activated, weight, output, p.rows,
                                        p.width, p.epsilon, static_cast<hipStream_t>(stream)),
                  "gatedRmsNorm");
}

int llmi_hip_gated_rms_norm(const uint16_t *input, const uint16_t *gate, const float *weight,
                            uint16_t *output, RowParams p, void *stream) {
  return gated_norm(input, gate, false, weight, output, p, stream);
}

int llmi_hip_gated_rms_norm_activated(const uint16_t *input, const float *gate,
                                      const float *weight, uint16_t *output, RowParams p,
                                      void *stream) {
  return gated_norm(input, gate, true, weight, output, p, stream);
}

int llmi_hip_cache_append(const uint16_t *src, uint16_t *cache, CacheParams p,
                          void *stream) {
  if (p.count && (!src || !cache))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "cacheAppend: null buffer");
  if ((uint64_t)p.offset + p.count > 0xffffffffull)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "cacheAppend: offset + count exceeds the 32-bit index range");
  return launched(launch_cache_append(src, cache, p.count, p.offset,
                                      static_cast<hipStream_t>(stream)),
                  "cacheAppend");
}

int llmi_hip_kv_append(const uint16_t *k_src, const uint16_t *v_src,
                       uint16_t *k_cache, uint16_t *v_cache, CacheParams p,
                       void *stream) {
  if (p.count && (!k_src || !v_src || !k_cache || !v_cache))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "KvAppend: null buffer");
  if ((uint64_t)p.offset + p.count > 0xffffffffull)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "KvAppend: offset + count exceeds the 32-bit index range");
  return launched(launch_kv_append(k_src, v_src, k_cache, v_cache, p.count,
                                   p.offset, static_cast<hipStream_t>(stream)),
                  "kvAppend");
}

size_t llmi_hip_gqa_workspace_bytes(GqaParams p) {
  if (check_gqa(p) != LLMI_HIP_OK)
    return 0;
  if (select_gqa(p) == GqaKernel::Decode)
    return decode_workspace_bytes(
        {p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past});
  if (select_gqa(p) == GqaKernel::Prefill)
    return prefill_workspace_bytes(
        {p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past});
  return 0;
}

} // extern "C"

namespace llmi {

// Whether a prefill divides its keys: its shape calls for it and the caller
// brought the workspace (callers without one get the undivided kernels).
static bool run_prefill_split(const GqaShape &s, const void *workspace, size_t bytes) {
  return workspace && aligned16(workspace) && prefill_split(s) &&
         bytes >= prefill_workspace_bytes(s);
}

// CausalGqa with an optional fused KvAppend (k_new/v_new non-null).
int run_gqa(const uint16_t *q, const uint16_t *k_new, const uint16_t *v_new,
            uint16_t *k_cache, uint16_t *v_cache, uint16_t *out,
            const GqaParams &p, void *workspace, size_t workspace_bytes,
            void *stream) {
  if (int st = check_gqa(p))
    return st;
  if (!q || !k_cache || !v_cache || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "CausalGqa: null buffer");
  const bool fused = k_new || v_new;
  if (fused && (!k_new || !v_new))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "KvAppend: null buffer");
  GqaShape s{p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past};
  hipStream_t st = static_cast<hipStream_t>(stream);
  GqaKernel kind = select_gqa(p);
  if (kind == GqaKernel::None)
    return fail(LLMI_HIP_UNSUPPORTED, "CausalGqa: head_dim %u is not supported",
                p.headDim);
  if (kind == GqaKernel::Decode) {
    size_t need = decode_workspace_bytes(s);
    if (need && (!workspace || workspace_bytes < need))
      return fail(LLMI_HIP_WORKSPACE,
                  "CausalGqa: decode needs a %zu-byte workspace, got %zu",
                  need, workspace ? workspace_bytes : (size_t)0);
    return launched(launch_gqa_decode(q, k_cache, v_cache, k_new, v_new, out,
                                      workspace, s, st),
                    "gqaDecodeSplitK");
  }
  if (fused) {
    unsigned row = p.kvHeads * p.headDim;
    int r = launched(launch_kv_append(k_new, v_new, k_cache, v_cache,
                                      p.tokens * row, p.past * row, st),
                     "kvAppend");
    if (r != LLMI_HIP_OK)
      return r;
  }
  if (kind == GqaKernel::Prefill && run_prefill_split(s, workspace, workspace_bytes))
    return launched(launch_gqa_prefill_split(q, k_cache, v_cache, out, workspace, s, nullptr, 0, st),
                    "gqaPrefillMfma");
  if (kind == GqaKernel::Prefill)
    return launched(launch_gqa_prefill(q, k_cache, v_cache, out, s, st),
                    "gqaPrefillMfma");
  return launched(launch_gqa_generic(q, k_cache, v_cache, out, s, st),
                  "gqaGeneric");
}

} // namespace llmi

extern "C" {

int llmi_hip_causal_gqa(const uint16_t *q, const uint16_t *k_cache,
                        const uint16_t *v_cache, uint16_t *out, GqaParams p,
                        void *workspace, size_t workspace_bytes, void *stream) {
  // The caches are only read on this path; the kernels take them non-const
  // because the fused variant writes the new rows.
  return run_gqa(q, nullptr, nullptr, const_cast<uint16_t *>(k_cache),
                 const_cast<uint16_t *>(v_cache), out, p, workspace,
                 workspace_bytes, stream);
}

int llmi_hip_kv_append_causal_gqa(const uint16_t *q, const uint16_t *k_new,
                                  const uint16_t *v_new, uint16_t *k_cache,
                                  uint16_t *v_cache, uint16_t *out, GqaParams p,
                                  void *workspace, size_t workspace_bytes,
                                  void *stream) {
  if (!k_new || !v_new)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "KvAppend: null buffer");
  return run_gqa(q, k_new, v_new, k_cache, v_cache, out, p, workspace,
                 workspace_bytes, stream);
}

static int gated_attention(const uint16_t *q_proj, const uint16_t *k_proj,
                           const uint16_t *v_new, const float *q_weight, const float *k_weight,
                           uint16_t *k_cache, uint16_t *v_cache, uint16_t *out, GqaParams p,
                           unsigned rotary_dim, float epsilon, float theta, void *workspace,
                           size_t workspace_bytes, bool activated, void *stream) {
  if (int st = check_gqa(p))
    return st;
  if (!q_proj || !k_proj || !v_new || !q_weight || !k_weight || !k_cache || !v_cache || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gated attention: null buffer");
  if (rotary_dim % 2 || rotary_dim > p.headDim)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "gated attention: rotary width %u must be even and <= head_dim %u",
                rotary_dim, p.headDim);
  if (!fits32((uint64_t)p.tokens * p.queryHeads, 2 * p.headDim, 1))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "gated attention: exceeds the 32-bit index range");
  GqaShape s{p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past};
  hipStream_t st = static_cast<hipStream_t>(stream);
  GatedRows ga;
  ga.qproj = reinterpret_cast<const _Float16 *>(q_proj);
  ga.kproj = reinterpret_cast<const _Float16 *>(k_proj);
  ga.vnew = reinterpret_cast<const _Float16 *>(v_new);
  ga.qw = q_weight;
  ga.kw = k_weight;
  ga.rot = rotary_dim;
  ga.eps = epsilon;
  ga.activated = activated ? 1u : 0u;
  const unsigned half = rotary_dim / 2;
  if (half > 256)
    return fail(LLMI_HIP_UNSUPPORTED, "gated attention: rotary width %u", rotary_dim);
  memcpy(ga.freqs, host_freqs(theta, rotary_dim).v, sizeof(float) * half);
  if (decode_gated_supported(s, rotary_dim)) {
    size_t need = decode_workspace_bytes(s);
    if (need && (!workspace || workspace_bytes < need))
      return fail(LLMI_HIP_WORKSPACE,
                  "gated attention: decode needs a %zu-byte workspace, got %zu", need,
                  workspace ? workspace_bytes : (size_t)0);
    return launched(launch_gqa_decode_gated(k_cache, v_cache, out, workspace, s, ga, st),
                    "gqaDecodeGated");
  }
  if (p.tokens > 1 && prefill_gated_supported(s, rotary_dim)) {
    const unsigned row = p.kvHeads * p.headDim;
    RopeShape ks = rope_shape(p.tokens * p.kvHeads, p.kvHeads, p.headDim, rotary_dim,
                              p.headDim, p.past, p.past * p.kvHeads, epsilon, theta, true);
    // The normalised query rows go through the output: each is read back only
    // by the wave that then writes it, or before the merge writes any.
    RopeShape qs = rope_shape(p.tokens * p.queryHeads, p.queryHeads, p.headDim, rotary_dim,
                              2 * p.headDim, p.past, 0, epsilon, theta, true);
    int r = launched(launch_attention_rows(q_proj, q_weight, out, qs, k_proj, k_weight, k_cache,
                                           ks, v_new, v_cache + (size_t)p.past * row,
                                           p.tokens * row, st),
                     "normRope");
    if (r == LLMI_HIP_OK && run_prefill_split(s, workspace, workspace_bytes))
      r = launched(launch_gqa_prefill_split(out, k_cache, v_cache, out, workspace, s, q_proj,
                                            ga.activated, st),
                   "gqaPrefillGated");
    else if (r == LLMI_HIP_OK)
      r = launched(launch_gqa_prefill_gated(out, k_cache, v_cache, out, s, q_proj, ga.activated,
                                            st),
                   "gqaPrefillGated");
    return r;
  }
  return fail(LLMI_HIP_UNSUPPORTED,
              "gated attention: no fused kernel for T %u, heads %u/%u, head_dim %u, rotary %u",
              p.tokens, p.queryHeads, p.kvHeads, p.headDim, rotary_dim);
}

int llmi_hip_gated_attention(const uint16_t *q_proj, const uint16_t *k_proj,
                             const uint16_t *v_new, const float *q_weight,
                             const float *k_weight, uint16_t *k_cache, uint16_t *v_cache,
                             uint16_t *out, GqaParams p, unsigned rotary_dim, float epsilon,
                             float theta, void *workspace, size_t workspace_bytes,
                             void *stream) {
  return gated_attention(q_proj, k_proj, v_new, q_weight, k_weight, k_cache, v_cache, out, p,
                         rotary_dim, epsilon, theta, workspace, workspace_bytes, false, stream);
}

int llmi_hip_gated_attention_activated(const uint16_t *q_proj, const uint16_t *k_proj,
                                       const uint16_t *v_new, const float *q_weight,
                                       const float *k_weight, uint16_t *k_cache,
                                       uint16_t *v_cache, uint16_t *out, GqaParams p,
                                       unsigned rotary_dim, float epsilon, float theta,
                                       void *workspace, size_t workspace_bytes, void *stream) {
  return gated_attention(q_proj, k_proj, v_new, q_weight, k_weight, k_cache, v_cache, out, p,
                         rotary_dim, epsilon, theta, workspace, workspace_bytes, true, stream);
}

size_t llmi_hip_delta_workspace_bytes(GraphDeltaParams p) {
  if (check_delta(p) != LLMI_HIP_OK)
    return 0;
  if (select_delta(p) == DeltaKernel::Chunked)
    return delta_chunked_workspace_bytes(
        {p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim});
  return 0;
}

int llmi_hip_delta_update(const float *q, const float *k, const uint16_t *v,
                          const float *beta, const float *decay, float *state,
                          uint16_t *out, GraphDeltaParams p, void *workspace,
                          size_t workspace_bytes, void *stream) {
  if (int st = check_delta(p))
    return st;
  if (!q || !k || !v || !beta || !decay || !state || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "DeltaUpdate: null buffer");
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (select_delta(p)) {
  case DeltaKernel::Chunked: {
    size_t need = delta_chunked_workspace_bytes(s);
    if (need && (!workspace || workspace_bytes < need))
      return fail(LLMI_HIP_WORKSPACE,
                  "DeltaUpdate: chunked form needs a %zu-byte workspace", need);
    return launched(launch_delta_chunked(q, k, v, beta, decay, state, out,
                                         workspace, s, st),
                    "deltaChunkedWy");
  }
  case DeltaKernel::Recurrent:
    return launched(
        launch_delta_recurrent(q, k, v, beta, decay, state, out, s, st),
        "deltaRecurrent");
  case DeltaKernel::Generic:
    return launched(launch_delta_generic(q, k, v, beta, decay, state, out, s, st),
                    "deltaGeneric");
  }
  return fail(LLMI_HIP_UNSUPPORTED, "DeltaUpdate: unsupported shape");
}

int llmi_hip_l2_norm_delta_update(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                  const float *beta, const float *decay, float *state,
                                  uint16_t *out, GraphDeltaParams p, float epsilon,
                                  float q_scale, void *workspace, size_t workspace_bytes,
                                  void *stream) {
  if (int st = check_delta(p))
    return st;
  if (!q || !k || !v || !beta || !decay || !state || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "L2Norm+DeltaUpdate: null buffer");
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (select_delta(p)) {
  case DeltaKernel::Chunked: {
    size_t need = delta_chunked_workspace_bytes(s);
    if (need && (!workspace || workspace_bytes < need))
      return fail(LLMI_HIP_WORKSPACE,
                  "L2Norm+DeltaUpdate: chunked form needs a %zu-byte workspace", need);
    return launched(launch_delta_chunked_qk16(q, k, v, beta, decay, state, out, workspace,
                                              epsilon, q_scale, s, st),
                    "deltaChunkedWy");
  }
  case DeltaKernel::Recurrent:
    return launched(launch_delta_recurrent_qk16(q, k, v, beta, decay, state, out, epsilon,
                                                q_scale, s, st),
                    "deltaRecurrent");
  case DeltaKernel::Generic:
    break;
  }
  return fail(LLMI_HIP_UNSUPPORTED,
              "L2Norm+DeltaUpdate: dk %u, dv %u have no fused kernel (dk 64 or 128, dv a "
              "multiple of 16)",
              p.keyDim, p.valueDim);
}

int llmi_hip_l2_norm_delta_gated_norm(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                      const float *beta, const float *decay, float *state,
                                      const uint16_t *gate, const float *norm_weight,
                                      uint16_t *out, GraphDeltaParams p, float qk_epsilon,
                                      float q_scale, float norm_epsilon, void *workspace,
                                      size_t workspace_bytes, void *stream) {
  if (int st = check_delta(p))
    return st;
  if (!q || !k || !v || !beta || !decay || !state || !gate || !norm_weight || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "L2Norm+DeltaUpdate+GatedRmsNorm: null buffer");
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (select_delta(p) == DeltaKernel::Chunked) {
    // The scan's norm reads and writes 16-byte row pieces of out and gate.
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(gate)) & 15u)
      return fail(LLMI_HIP_UNSUPPORTED,
                  "L2Norm+DeltaUpdate+GatedRmsNorm: out and gate must be 16-byte aligned");
    size_t need = delta_chunked_workspace_bytes(s);
    if (!workspace || workspace_bytes < need)
      return fail(LLMI_HIP_WORKSPACE,
                  "L2Norm+DeltaUpdate+GatedRmsNorm: chunked form needs a %zu-byte workspace",
                  need);
    if (!delta_chunked_norm_resident(s))
      return fail(LLMI_HIP_UNSUPPORTED,
                  "L2Norm+DeltaUpdate+GatedRmsNorm: %u x %u scan workgroups do not fit on the "
                  "device at once",
                  p.valueHeads, p.valueDim / 16);
    return launched(launch_delta_chunked_gated_norm(q, k, v, beta, decay, state, gate,
                                                    norm_weight, out, workspace, qk_epsilon,
                                                    q_scale, norm_epsilon, s, st),
                    "deltaChunkedWy+gatedRmsNorm");
  }
  if (delta_recurrent_norm_supported(s))
    return launched(launch_delta_recurrent_gated_norm(q, k, v, beta, decay, state, gate,
                                                      norm_weight, out, qk_epsilon, q_scale,
                                                      norm_epsilon, s, st),
                    "deltaRecurrent+gatedRmsNorm");
  return fail(LLMI_HIP_UNSUPPORTED,
              "L2Norm+DeltaUpdate+GatedRmsNorm: T %u, dk %u, dv %u have no fused kernel "
              "(chunked: dk 128, T >= 32; recurrent: dk 64 or 128, dv 64 or 128, T <= %u)",
              p.tokens, p.keyDim, p.valueDim, kRecNormMaxT);
}

int llmi_hip_l2_norm_delta_gated_norm_status(const void *workspace, size_t workspace_bytes,
                                             GraphDeltaParams p, void *stream) {
  if (int st = check_delta(p))
    return st;
  // Only the chunked form waits for other workgroups.
  if (select_delta(p) != DeltaKernel::Chunked)
    return LLMI_HIP_OK;
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  if (!workspace || workspace_bytes < delta_chunked_workspace_bytes(s))
    return fail(LLMI_HIP_WORKSPACE, "GatedRmsNorm status: workspace smaller than the call's");
  bool gave_up = false;
  if (int st = launched(delta_chunked_wait_status(workspace, s, static_cast<hipStream_t>(stream),
                                                  &gave_up),
                        "GatedRmsNorm status"))
    return st;
  if (gave_up)
    return fail(LLMI_HIP_LAUNCH_FAILED,
                "L2Norm+DeltaUpdate+GatedRmsNorm: the scan's arrival wait gave up; the "
                "normalised rows are not trustworthy");
  return LLMI_HIP_OK;
}

int llmi_hip_l2_norm_delta_gated_norm_activated_quantize(
    const uint16_t *q, const uint16_t *k, const uint16_t *v, const float *beta,
    const float *decay, float *state, const float *gate, const float *norm_weight,
    uint16_t *out, int8_t *quantized, float *scales, uint32_t *invalid, GraphDeltaParams p,
    float qk_epsilon, float q_scale, float norm_epsilon, void *stream) {
  if (int st = check_delta(p))
    return st;
  if (!q || !k || !v || !beta || !decay || !state || !gate || !norm_weight || !out ||
      !quantized || !scales)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "L2Norm+DeltaUpdate+GatedRmsNormQuantize: null buffer");
  DeltaShape s{p.tokens, p.keyHeads, p.keyDim, p.valueHeads, p.valueDim};
  if (!delta_recurrent_norm_supported(s))
    return fail(LLMI_HIP_UNSUPPORTED,
                "L2Norm+DeltaUpdate+GatedRmsNormQuantize: T %u, dk %u, dv %u have no fused "
                "kernel (dk 64 or 128, dv 64 or 128, T <= %u)",
                p.tokens, p.keyDim, p.valueDim, kRecNormMaxT);
  // The norm writes 16-byte pieces of out and 8-byte pieces of quantized.
  if (!aligned16(out) || !aligned16(quantized))
    return fail(LLMI_HIP_UNSUPPORTED,
                "L2Norm+DeltaUpdate+GatedRmsNormQuantize: out and quantized must be 16-byte "
                "aligned");
  return launched(launch_delta_recurrent_gated_norm_quantize(
                      q, k, v, beta, decay, state, gate, norm_weight, out, quantized, scales,
                      invalid, qk_epsilon, q_scale, norm_epsilon, s,
                      static_cast<hipStream_t>(stream)),
                  "deltaRecurrent+gatedRmsNormQuantize");
}

unsigned llmi_hip_set_arrival_wait_limit(unsigned polls) {
  return delta_chunked_wait_limit(polls);
}

int llmi_hip_workspace_init(void *workspace, size_t bytes, void *stream) {
  if (!bytes)
    return LLMI_HIP_OK;
  if (!workspace)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "workspace_init: null workspace");
  return launched(hipMemsetAsync(workspace, 0, bytes,
                                 static_cast<hipStream_t>(stream)),
                  "workspace_init");
}

// ------------------------------------------- rotary rows, paged 4-bit cache

int llmi_hip_rope(const uint16_t *input, const int32_t *positions, const float *freqs,
                  uint16_t *output, RopeRowsParams p, void *stream) {
  if (p.tokens == 0 || p.heads == 0 || p.headDim == 0)
    return LLMI_HIP_OK;
  if (!input || !output || (p.rotaryDim && (!positions || !freqs)))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rope: null buffer");
  if (p.rotaryDim % 2 || p.rotaryDim > p.headDim)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rope: rotary width %u must be even and <= width %u",
                p.rotaryDim, p.headDim);
  if (p.layout > LLMI_ROPE_INTERLEAVED)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rope: unknown layout %u", p.layout);
  if (!rope_rows_supported(p.rotaryDim))
    return fail(LLMI_HIP_UNSUPPORTED, "rope: rotary width %u", p.rotaryDim);
  if (!strides_apart(p.tokens, p.outputTokenStride, p.heads, p.outputHeadStride, p.headDim))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rope: the output's rows overlap");
  if (!fits32(p.tokens, p.heads, p.headDim) || p.tokens >= 1u << 24)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "rope: exceeds the 32-bit index range or 2^24 tokens");
  return launched(launch_rope_rows(input, positions, freqs, output, p,
                                   static_cast<hipStream_t>(stream)),
                  "ropeRows");
}

int llmi_hip_rope_frequencies(RopeScalingParams p, float *freqs, float *factor) {
  if (!freqs || !factor)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "ropeFrequencies: null buffer");
  if (p.rotaryDim % 2)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "ropeFrequencies: rotary width %u is odd", p.rotaryDim);
  if (!rope_rows_supported(p.rotaryDim))
    return fail(LLMI_HIP_UNSUPPORTED, "ropeFrequencies: rotary width %u", p.rotaryDim);
  if (p.scaling > LLMI_ROPE_SCALING_BANDS)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "ropeFrequencies: unknown scaling %u", p.scaling);
  const bool ramp = p.scaling == LLMI_ROPE_SCALING_YARN || p.scaling == LLMI_ROPE_SCALING_BANDS;
  if (!(p.theta > 0.0f) || (p.scaling && !(p.scale > 0.0f)) ||
      (ramp && !(p.originalPositions > 0.0f && p.highTurns > p.lowTurns)))
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "ropeFrequencies: theta, scale and the original positions must be positive and "
                "the turns in order");
  double theta = p.theta;
  if (p.scaling == LLMI_ROPE_SCALING_NTK && p.rotaryDim > 2)
    theta *= pow((double)p.scale, (double)p.rotaryDim / (p.rotaryDim - 2));
  for (unsigned i = 0; i < p.rotaryDim / 2; ++i) {
    double f = pow(theta, -2.0 * i / p.rotaryDim);
    if (p.scaling == LLMI_ROPE_SCALING_LINEAR)
      f /= p.scale;
    if (ramp) {
      const double turns = p.originalPositions * f / 6.283185307179586;
      double keep = (turns - p.lowTurns) / ((double)p.highTurns - p.lowTurns);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = keep * f + (1.0 - keep) * f / p.scale;
    }
    freqs[i] = (float)f;
  }
  *factor = p.scaling == LLMI_ROPE_SCALING_YARN && p.scale > 1.0f
                ? (float)(0.1 * log((double)p.scale) + 1.0)
                : 1.0f;
  return LLMI_HIP_OK;
}

// The pool's and the sequences' shape; buffers as the caller lists them.
static int check_paged(const char *what, const PagedKvParams &p, const int32_t *starts,
                       const int32_t *past, const int32_t *table, const void *pool) {
  if (p.headDim != 64 && p.headDim != 128 && p.headDim != 256)
    return fail(LLMI_HIP_UNSUPPORTED, "%s: head_dim %u (64, 128 or 256)", what, p.headDim);
  if (p.pageSize == 0 || p.pageSize % 32)
    return fail(LLMI_HIP_UNSUPPORTED, "%s: page size %u is no multiple of 32", what, p.pageSize);
  if (p.pages == 0 || p.kvHeads == 0 || p.tableStride == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: pages, heads and table must not be empty", what);
  if ((uint64_t)p.tableStride * p.pageSize > 0x7fffffffull || p.pages > 0x7fffffffu ||
      p.tokens >= 1u << 22 || p.sequences >= 1u << 22 || p.kvHeads > 65535u)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: exceeds the 31-bit range of positions and pages, "
                "2^22 rows or sequences, or 65535 heads", what);
  if (!starts || !past || !table || !pool)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: null buffer", what);
  if (!aligned16(pool))
    return fail(LLMI_HIP_UNSUPPORTED, "%s: pool not 16-byte aligned", what);
  return LLMI_HIP_OK;
}

int llmi_hip_paged_append(const uint16_t *keys, const uint16_t *values, const int32_t *starts,
                          const int32_t *past, const int32_t *table, const float *freqs,
                          void *pool, uint32_t *invalid, PagedKvParams p, PagedAppendParams a,
                          void *stream) {
  if (p.tokens == 0 || p.sequences == 0)
    return LLMI_HIP_OK;
  if (int rc = check_paged("pagedAppend", p, starts, past, table, pool))
    return rc;
  if (!keys || !values || (a.rotaryDim && !freqs))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedAppend: null buffer");
  if (a.rotaryDim % 2 || a.rotaryDim > p.headDim || a.layout > LLMI_ROPE_INTERLEAVED)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "pagedAppend: rotary width %u (even, <= %u) or layout %u", a.rotaryDim, p.headDim,
                a.layout);
  return launched(launch_paged_append(keys, values, starts, past, table, freqs, pool, invalid, p,
                                      a, static_cast<hipStream_t>(stream)),
                  "pagedAppend");
}

int llmi_hip_paged_read(const void *pool, const int32_t *starts, const int32_t *past,
                        const int32_t *table, uint16_t *keys, uint16_t *values,
                        uint32_t *invalid, PagedKvParams p, void *stream) {
  if (p.tokens == 0 || p.sequences == 0)
    return LLMI_HIP_OK;
  if (int rc = check_paged("pagedRead", p, starts, past, table, pool))
    return rc;
  if (!keys || !values)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedRead: null buffer");
  if (!aligned16(keys) || !aligned16(values))
    return fail(LLMI_HIP_UNSUPPORTED, "pagedRead: rows not 16-byte aligned");
  return launched(launch_paged_read(pool, starts, past, table, keys, values, invalid, p,
                                    static_cast<hipStream_t>(stream)),
                  "pagedRead");
}

static int check_paged_heads(const PagedGqaParams &p) {
  if (p.kv.headDim != 64 && p.kv.headDim != 128 && p.kv.headDim != 256)
    return fail(LLMI_HIP_UNSUPPORTED, "pagedGqa: head_dim %u (64, 128 or 256)", p.kv.headDim);
  if (p.queryHeads == 0 || p.kv.kvHeads == 0 || p.queryHeads % p.kv.kvHeads ||
      p.queryHeads > 65535u)
    return fail(LLMI_HIP_INVALID_ARGUMENT,
                "pagedGqa: query heads %u not a multiple of KV heads %u (at most 65535)",
                p.queryHeads, p.kv.kvHeads);
  return LLMI_HIP_OK;
}

int llmi_hip_paged_gqa(const uint16_t *q, const int32_t *starts, const int32_t *past,
                       const int32_t *table, const void *pool, uint16_t *out, uint32_t *invalid,
                       PagedGqaParams p, void *workspace, size_t workspace_bytes, void *stream) {
  if (p.kv.tokens == 0 || p.kv.sequences == 0)
    return LLMI_HIP_OK;
  if (int rc = check_paged("pagedGqa", p.kv, starts, past, table, pool))
    return rc;
  if (int rc = check_paged_heads(p))
    return rc;
  if (!q || !out)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedGqa: null buffer");
  if (!aligned16(q) || !aligned16(out))
    return fail(LLMI_HIP_UNSUPPORTED, "pagedGqa: rows not 16-byte aligned");
  if (!paged_gqa_launchable(p.kv, p.queryHeads))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedGqa: too many rows and heads for one call");
  const uintptr_t from = reinterpret_cast<uintptr_t>(q), to = reinterpret_cast<uintptr_t>(out);
  const size_t bytes = (size_t)p.kv.tokens * p.queryHeads * p.kv.headDim * 2;
  if (from < to + bytes && to < from + bytes)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedGqa: out overlaps q");
  const size_t need = paged_gqa_workspace_bytes(p.kv, p.queryHeads);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(LLMI_HIP_WORKSPACE, "pagedGqa: workspace of %zu bytes, %zu needed (16-byte "
                "aligned)", workspace ? workspace_bytes : 0, need);
  return launched(launch_paged_gqa(q, starts, past, table, pool, out, invalid, workspace, p.kv,
                                   p.queryHeads, p.scale, static_cast<hipStream_t>(stream)),
                  "pagedGqa");
}

size_t llmi_hip_paged_gqa_workspace_bytes(PagedGqaParams p) {
  if (p.kv.tokens == 0 || p.kv.sequences == 0 || check_paged_heads(p) ||
      !paged_gqa_launchable(p.kv, p.queryHeads))
    return 0;
  return paged_gqa_workspace_bytes(p.kv, p.queryHeads);
}

static int check_workspace(const char *what, const void *workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need || !aligned16(workspace)))
    return fail(LLMI_HIP_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what,
                workspace ? bytes : 0, need);
  return LLMI_HIP_OK;
}
// Whether two ranges of memory have bytes in common.
static bool overlap(const void *a, size_t aBytes, const void *b, size_t bBytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + bBytes && y < x + aBytes;
}

int llmi_hip_paged_gqa_shared(const uint16_t *q, const int32_t *starts, const int32_t *past,
                              const int32_t *table, const int32_t *groups, const int32_t *prefix,
                              const void *pool, uint16_t *out, uint32_t *invalid,
                              PagedSharedParams p, void *workspace, size_t workspace_bytes,
                              void *stream) {
  const PagedKvParams &kv = p.gqa.kv;
  if (p.groups == 0)
    return llmi_hip_paged_gqa(q, starts, past, table, pool, out, invalid, p.gqa, workspace,
                              workspace_bytes, stream);
  if (kv.tokens == 0 || kv.sequences == 0)
    return LLMI_HIP_OK;
  const char *what = "pagedGqaShared";
  if (int rc = check_paged(what, kv, starts, past, table, pool))
    return rc;
  if (int rc = check_paged_heads(p.gqa))
    return rc;
  if (!q || !out || !groups || !prefix)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: null buffer", what);
  if (!aligned16(q) || !aligned16(out))
    return fail(LLMI_HIP_UNSUPPORTED, "%s: rows not 16-byte aligned", what);
  if (p.groups >= 1u << 22 || !paged_shared_launchable(kv, p.gqa.queryHeads, p.groups))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: too many rows, heads or groups for one call", what);
  const size_t bytes = (size_t)kv.tokens * p.gqa.queryHeads * kv.headDim * 2;
  if (overlap(q, bytes, out, bytes))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: out overlaps q", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes,
                               paged_shared_workspace_bytes(kv, p.gqa.queryHeads, p.groups)))
    return rc;
  return launched(launch_paged_gqa_shared(q, starts, past, table, groups, prefix, pool, out, invalid,
                                          workspace, kv, p.gqa.queryHeads, p.gqa.scale, p.groups,
                                          static_cast<hipStream_t>(stream)),
                  what);
}

size_t llmi_hip_paged_gqa_shared_workspace_bytes(PagedSharedParams p) {
  if (p.groups == 0)
    return llmi_hip_paged_gqa_workspace_bytes(p.gqa);
  if (p.gqa.kv.tokens == 0 || p.gqa.kv.sequences == 0 || check_paged_heads(p.gqa) ||
      p.groups >= 1u << 22 || !paged_shared_launchable(p.gqa.kv, p.gqa.queryHeads, p.groups))
    return 0;
  return paged_shared_workspace_bytes(p.gqa.kv, p.gqa.queryHeads, p.groups);
}

int llmi_hip_paged_fork(const int32_t *table, const int32_t *past, const int32_t *parent,
                        const int32_t *spare, int32_t *tableOut, int32_t *pastOut, void *pool,
                        uint32_t *invalid, PagedForkParams p, void *stream) {
  if (p.children == 0)
    return LLMI_HIP_OK;
  const char *what = "pagedFork";
  if (p.sequences == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: no sequences to continue", what);
  const PagedKvParams kv{p.pages,     p.pageSize,    p.kvHeads, p.headDim,
                         p.sequences, p.tableStride, 1};
  if (int rc = check_paged(what, kv, past, past, table, pool))
    return rc;
  if (!parent || !spare || !tableOut || !pastOut)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: null buffer", what);
  if (p.children >= 1u << 22 || !fits32(256 * (uint64_t)p.children, p.kvHeads, p.pageSize / 32))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: too many children, heads or blocks for one call",
                what);
  const size_t row = (size_t)p.tableStride * 4, tableBytes = p.sequences * row;
  const size_t outBytes = p.children * row, n = (size_t)p.children * 4;
  const size_t pastBytes = (size_t)p.sequences * 4;
  const struct {
    const void *at;
    size_t bytes;
  } in[] = {{table, tableBytes}, {past, pastBytes}, {parent, n}, {spare, n}};
  for (const auto &x : in)
    if (overlap(x.at, x.bytes, tableOut, outBytes) || overlap(x.at, x.bytes, pastOut, n))
      return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: an output overlaps an input", what);
  if (overlap(tableOut, outBytes, pastOut, n))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "%s: the outputs overlap", what);
  return launched(launch_paged_fork(table, past, parent, spare, tableOut, pastOut, pool, invalid, p,
                                    static_cast<hipStream_t>(stream)),
                  what);
}

static int check_free(const PagedFreeParams &p) {
  if (p.pageSize == 0 || p.pageSize % 32)
    return fail(LLMI_HIP_UNSUPPORTED, "pagedFree: page size %u is no multiple of 32", p.pageSize);
  if (p.pages == 0 || p.tableStride == 0)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedFree: pages and table must not be empty");
  if (p.pages > 0x7fffffffu || (uint64_t)p.tableStride * p.pageSize > 0x7fffffffull ||
      (uint64_t)p.sequences * p.tableStride > 0x7fffffffull)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedFree: exceeds the 31-bit range of pages, "
                "positions or entries");
  return LLMI_HIP_OK;
}

int llmi_hip_paged_free(const int32_t *table, const int32_t *lengths, int32_t *free, int32_t *count,
                        uint32_t *invalid, PagedFreeParams p, void *workspace,
                        size_t workspace_bytes, void *stream) {
  if (int rc = check_free(p))
    return rc;
  if ((p.sequences && (!table || !lengths)) || !free || !count)
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedFree: null buffer");
  const size_t entries = (size_t)p.sequences * p.tableStride * 4, out = (size_t)p.pages * 4;
  if (overlap(table, entries, free, out) || overlap(lengths, (size_t)p.sequences * 4, free, out) ||
      overlap(table, entries, count, 4) || overlap(lengths, (size_t)p.sequences * 4, count, 4) ||
      overlap(free, out, count, 4))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedFree: an output overlaps another buffer");
  if (int rc = check_workspace("pagedFree", workspace, workspace_bytes,
                               paged_free_workspace_bytes(p)))
    return rc;
  return launched(launch_paged_free(table, lengths, free, count, invalid, workspace, p,
                                    static_cast<hipStream_t>(stream)),
                  "pagedFree");
}

size_t llmi_hip_paged_free_workspace_bytes(PagedFreeParams p) {
  return check_free(p) ? 0 : paged_free_workspace_bytes(p);
}

int llmi_hip_paged_move(const int32_t *source, const int32_t *sourceTable, const int32_t *starts,
                        const int32_t *past, const int32_t *table, void *pool, uint32_t *invalid,
                        PagedMoveParams p, void *workspace, size_t workspace_bytes, void *stream) {
  if (p.kv.tokens == 0 || p.kv.sequences == 0)
    return LLMI_HIP_OK;
  if (int rc = check_paged("pagedMove", p.kv, starts, past, table, pool))
    return rc;
  if (!source || (p.apart && !sourceTable))
    return fail(LLMI_HIP_INVALID_ARGUMENT, "pagedMove: null buffer");
  if (int rc = check_workspace("pagedMove", workspace, workspace_bytes,
                               llmi_hip_paged_move_workspace_bytes(p)))
    return rc;
  return launched(launch_paged_move(source, p.apart ? sourceTable : nullptr, starts, past, table,
                                    pool, invalid, workspace, p.kv,
                                    static_cast<hipStream_t>(stream)),
                  "pagedMove");
}

size_t llmi_hip_paged_move_workspace_bytes(PagedMoveParams p) {
  const unsigned dim = p.kv.headDim;
  if (p.apart || p.kv.tokens == 0 || p.kv.sequences == 0 || (dim != 64 && dim != 128 && dim != 256))
    return 0;
  return paged_move_workspace_bytes(p.kv);
}

// Whether a supported CausalGqa is a prefill that divides its keys.
static bool prefill_merges(const GqaParams &p) {
  return select_gqa(p) == GqaKernel::Prefill &&
         prefill_split({p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past});
}

unsigned llmi_hip_dispatch_count(int op, const void *params) {
  if (!params)
    return 0;
  switch (op) {
  case LLMI_HIP_OP_KV_APPEND:
    return 1;
  case LLMI_HIP_OP_CAUSAL_GQA: {
    const GqaParams &p = *static_cast<const GqaParams *>(params);
    if (check_gqa(p) || select_gqa(p) == GqaKernel::None)
      return 0;
    if (select_gqa(p) == GqaKernel::Decode)
      return decode_launches({p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past});
    return prefill_merges(p) ? 2 : 1;
  }
  case LLMI_HIP_OP_KV_APPEND_CAUSAL_GQA: {
    const GqaParams &p = *static_cast<const GqaParams *>(params);
    if (check_gqa(p))
      return 0;
    switch (select_gqa(p)) {
    case GqaKernel::Decode:
      return decode_launches({p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past});
    case GqaKernel::None:
      return 0;
    default:
      return prefill_merges(p) ? 3 : 2;
    }
  }
  case LLMI_HIP_OP_DELTA_UPDATE: {
    const GraphDeltaParams &p = *static_cast<const GraphDeltaParams *>(params);
    if (check_delta(p))
      return 0;
    return select_delta(p) == DeltaKernel::Chunked ? delta_chunked_dispatches() : 1;
  }
  case LLMI_HIP_OP_NORM_ROPE: {
    const RopeParams &p = *static_cast<const RopeParams *>(params);
    return p.tokens && p.heads && p.headDim ? 1 : 0;
  }
  case LLMI_HIP_OP_RMS_NORM: {
    const RowParams &p = *static_cast<const RowParams *>(params);
    return p.rows && p.width ? 1 : 0;
  }
  case LLMI_HIP_OP_PARTIAL_ROPE: {
    const PartialRopeParams &p = *static_cast<const PartialRopeParams *>(params);
    return p.rows && p.width ? 1 : 0;
  }
  case LLMI_HIP_OP_SIGMOID_MUL:
    return static_cast<const ElementParams *>(params)->count ? 1 : 0;
  case LLMI_HIP_OP_CAUSAL_CONV: {
    const ConvParams &p = *static_cast<const ConvParams *>(params);
    return p.tokens && p.channels && causal_conv_supported(p.kernelSize) ? 1 : 0;
  }
  case LLMI_HIP_OP_L2_NORM: {
    const L2Params &p = *static_cast<const L2Params *>(params);
    return p.rows && p.width ? 1 : 0;
  }
  case LLMI_HIP_OP_QUANTIZE_ACTIVATION: {
    const QuantizeParams &p = *static_cast<const QuantizeParams *>(params);
    return p.rows && p.width && p.groups == (p.width + 31) / 32 ? 1 : 0;
  }
  case LLMI_HIP_OP_LINEAR_W8A8: {
    const LinearW8Params &p = *static_cast<const LinearW8Params *>(params);
    return p.rows && p.columns && check_linear_w8(p) == LLMI_HIP_OK ? 1 : 0;
  }
  case LLMI_HIP_OP_EMBEDDING_W8: {
    const GroupedEmbedParams &p = *static_cast<const GroupedEmbedParams *>(params);
    return p.tokens && p.hidden && p.rowCount && p.groups >= (p.hidden + 31) / 32 ? 1 : 0;
  }
  case LLMI_HIP_OP_EMBEDDING: {
    const EmbedParams &p = *static_cast<const EmbedParams *>(params);
    return p.tokens && p.hidden && p.rowCount ? 1 : 0;
  }
  case LLMI_HIP_OP_RESIDUAL_ADD:
  case LLMI_HIP_OP_SWIGLU:
  case LLMI_HIP_OP_SILU:
  case LLMI_HIP_OP_MULTIPLY:
    return static_cast<const ElementParams *>(params)->count ? 1 : 0;
  case LLMI_HIP_OP_COPY_HALF_VIEW: {
    const HalfViewParams &p = *static_cast<const HalfViewParams *>(params);
    return p.count && check_view(p) == LLMI_HIP_OK ? 1 : 0;
  }
  case LLMI_HIP_OP_ADD_RMS_NORM_QUANTIZE: {
    const RowParams &p = *static_cast<const RowParams *>(params);
    return p.rows && p.width && check_add_norm_quantize(p) == LLMI_HIP_OK ? 1 : 0;
  }
  case LLMI_HIP_OP_ADD_RMS_NORM_LINEAR_W8A8:
    return check_norm_linear(*static_cast<const NormLinearParams *>(params)) == LLMI_HIP_OK ? 1
                                                                                          : 0;
  case LLMI_HIP_OP_LINEAR_F16: {
    const LinearParams &p = *static_cast<const LinearParams *>(params);
    return p.tokens && p.rowCount && check_linear_f16(p) == LLMI_HIP_OK ? 1 : 0;
  }
  case LLMI_HIP_OP_DELTA_GATES: {
    const RowParams &p = *static_cast<const RowParams *>(params);
    return p.rows && p.width ? 1 : 0;
  }
  case LLMI_HIP_OP_GATED_RMS_NORM: {
    const RowParams &p = *static_cast<const RowParams *>(params);
    return p.rows && p.width ? 1 : 0;
  }
  case LLMI_HIP_OP_ROPE: {
    const RopeRowsParams &p = *static_cast<const RopeRowsParams *>(params);
    return p.tokens && p.heads && p.headDim ? 1 : 0;
  }
  case LLMI_HIP_OP_PAGED_APPEND:
  case LLMI_HIP_OP_PAGED_READ: {
    const PagedKvParams &p = *static_cast<const PagedKvParams *>(params);
    return p.tokens && p.sequences ? 1 : 0;
  }
  case LLMI_HIP_OP_PAGED_GQA: {
    const PagedGqaParams &p = *static_cast<const PagedGqaParams *>(params);
    if (!p.kv.tokens || !p.kv.sequences || check_paged_heads(p))
      return 0;
    return 1u + paged_gqa_joins(p.kv, p.queryHeads);
  }
  case LLMI_HIP_OP_PAGED_GQA_SHARED: {
    const PagedSharedParams &p = *static_cast<const PagedSharedParams *>(params);
    if (!p.groups)
      return llmi_hip_dispatch_count(LLMI_HIP_OP_PAGED_GQA, &p.gqa);
    if (!p.gqa.kv.tokens || !p.gqa.kv.sequences || check_paged_heads(p.gqa))
      return 0;
    return paged_shared_launches(p.gqa.kv, p.gqa.queryHeads, p.groups);
  }
  case LLMI_HIP_OP_PAGED_FORK:
    return static_cast<const PagedForkParams *>(params)->children ? 1 : 0;
  case LLMI_HIP_OP_PAGED_FREE: {
    const PagedFreeParams &p = *static_cast<const PagedFreeParams *>(params);
    return check_free(p) ? 0 : paged_free_launches(p);
  }
  case LLMI_HIP_OP_PAGED_MOVE: {
    const PagedMoveParams &p = *static_cast<const PagedMoveParams *>(params);
    return !p.kv.tokens || !p.kv.sequences ? 0 : p.apart ? 1 : 2;
  }
  case LLMI_HIP_OP_GATED_ATTENTION: {
    // Launches for a rotary width the kernels take (a multiple of 16).
    const GqaParams &p = *static_cast<const GqaParams *>(params);
    if (check_gqa(p))
      return 0;
    GqaShape s{p.tokens, p.queryHeads, p.kvHeads, p.headDim, p.past};
    if (decode_gated_supported(s, 16))
      return decode_launches(s);
    if (p.tokens < 2 || !prefill_gated_supported(s, 16))
      return 0;
    return prefill_split(s) ? 3 : 2;
  }
  }
  return 0;
}

const char *llmi_hip_kernel_name(int op, const void *params, unsigned index) {
  if (index >= llmi_hip_dispatch_count(op, params))
    return nullptr;
  switch (op) {
  case LLMI_HIP_OP_KV_APPEND:
    return "kvAppend";
  case LLMI_HIP_OP_KV_APPEND_CAUSAL_GQA:
    if (select_gqa(*static_cast<const GqaParams *>(params)) != GqaKernel::Decode)
      return index == 0 ? "kvAppend"
                        : llmi_hip_kernel_name(LLMI_HIP_OP_CAUSAL_GQA, params, index - 1);
    return llmi_hip_kernel_name(LLMI_HIP_OP_CAUSAL_GQA, params, index);
  case LLMI_HIP_OP_CAUSAL_GQA:
    switch (select_gqa(*static_cast<const GqaParams *>(params))) {
    case GqaKernel::Decode:
      return index == 0 ? "gqaDecodeSplitK" : "gqaDecodeMerge";
    case GqaKernel::Prefill:
      return index == 0 ? "gqaPrefillMfma" : "gqaPrefillMerge";
    case GqaKernel::Generic:
      return "gqaGeneric";
    case GqaKernel::None:
      return nullptr;
    }
    return nullptr;
  case LLMI_HIP_OP_DELTA_UPDATE:
    switch (select_delta(*static_cast<const GraphDeltaParams *>(params))) {
    case DeltaKernel::Chunked:
      return delta_chunked_kernel_name(index);
    case DeltaKernel::Recurrent:
      return "deltaRecurrent";
    case DeltaKernel::Generic:
      return "deltaGeneric";
    }
    return nullptr;
  // The tile kernels need 16-byte aligned buffers as well; these names
  // assume them (torch allocations are).
  case LLMI_HIP_OP_NORM_ROPE: {
    const RopeParams &p = *static_cast<const RopeParams *>(params);
    RopeShape s = rope_shape(p.tokens * p.heads, p.heads, p.headDim, p.rotaryDim,
                             p.headStride, p.past, 0, 0, 0, true);
    return rope_kernel_name(s, "normRopeTile", "normRopeRows", "normRopeWide");
  }
  case LLMI_HIP_OP_RMS_NORM: {
    const RowParams &p = *static_cast<const RowParams *>(params);
    RopeShape s = rope_shape(p.rows, 1, p.width, 0, p.width, 0, 0, 0, 0, true);
    return rope_kernel_name(s, "normRopeTile", "normRopeRows", "normRopeWide");
  }
  case LLMI_HIP_OP_PARTIAL_ROPE: {
    const PartialRopeParams &p = *static_cast<const PartialRopeParams *>(params);
    RopeShape s = rope_shape(p.rows, p.heads, p.width, p.rotaryWidth, p.width, 0, 0, 0,
                             0, false);
    return rope_kernel_name(s, "partialRopeTile", "partialRopeRows", "partialRopeWide");
  }
  case LLMI_HIP_OP_CAUSAL_CONV:
    return "causalConv";
  case LLMI_HIP_OP_L2_NORM:
    return l2_norm_tiled(static_cast<const L2Params *>(params)->width, nullptr, nullptr)
               ? "l2NormTile"
               : "l2NormRows";
  case LLMI_HIP_OP_DELTA_GATES:
    return "deltaGates";
  case LLMI_HIP_OP_QUANTIZE_ACTIVATION:
    return "quantizeActivation";
  case LLMI_HIP_OP_LINEAR_W8A8:
    return linear_w8a8_kernel(static_cast<const LinearW8Params *>(params)->rows);
  case LLMI_HIP_OP_EMBEDDING_W8:
    return "embeddingW8";
  case LLMI_HIP_OP_EMBEDDING:
    return "embedding";
  case LLMI_HIP_OP_RESIDUAL_ADD:
    return "residualAdd";
  case LLMI_HIP_OP_SWIGLU:
    return "swiGlu";
  case LLMI_HIP_OP_SILU:
    return "siluF16";
  case LLMI_HIP_OP_MULTIPLY:
    return "multiplyF16";
  case LLMI_HIP_OP_COPY_HALF_VIEW:
    return "copyHalfView";
  case LLMI_HIP_OP_LINEAR_F16:
    return "linearF16";
  case LLMI_HIP_OP_ADD_RMS_NORM_QUANTIZE:
    return "addRmsNormQuantize";
  case LLMI_HIP_OP_ADD_RMS_NORM_LINEAR_W8A8:
    return "addRmsNormLinearW8A8";
  case LLMI_HIP_OP_GATED_RMS_NORM: {
    const unsigned width = static_cast<const RowParams *>(params)->width;
    return width % 8 == 0 && width <= 256 ? "gatedRmsNormTile" : "gatedRmsNormRows";
  }
  case LLMI_HIP_OP_SIGMOID_MUL:
    return sigmoid_mul_vectorised(static_cast<const ElementParams *>(params)->count,
                                  nullptr, nullptr, nullptr)
               ? "sigmoidMulVec"
               : "sigmoidMulScalar";
  case LLMI_HIP_OP_ROPE:
    return "ropeRows";
  case LLMI_HIP_OP_PAGED_APPEND:
    return "pagedAppend";
  case LLMI_HIP_OP_PAGED_READ:
    return "pagedRead";
  case LLMI_HIP_OP_PAGED_GQA:
    return index ? "pagedGqaMerge"
           : paged_gqa_tiled(static_cast<const PagedGqaParams *>(params)->kv,
                             static_cast<const PagedGqaParams *>(params)->queryHeads)
               ? "pagedGqaTiles"
               : "pagedGqaSplit";
  case LLMI_HIP_OP_PAGED_GQA_SHARED: {
    const PagedSharedParams &p = *static_cast<const PagedSharedParams *>(params);
    if (!p.groups)
      return llmi_hip_kernel_name(LLMI_HIP_OP_PAGED_GQA, &p.gqa, index);
    return paged_shared_kernel(p.gqa.kv, p.gqa.queryHeads, p.groups, index);
  }
  case LLMI_HIP_OP_PAGED_FORK:
    return "pagedFork";
  case LLMI_HIP_OP_PAGED_FREE:
    return llmi_hip_dispatch_count(op, params) == 1 ? "pagedFree"
           : index == 0                             ? "pagedFreeMark"
           : index == 1                             ? "pagedFreeJoin"
                                                    : "pagedFreeList";
  case LLMI_HIP_OP_PAGED_MOVE:
    return index                                                 ? "pagedPlace"
           : static_cast<const PagedMoveParams *>(params)->apart ? "pagedMove"
                                                                 : "pagedGather";
  case LLMI_HIP_OP_GATED_ATTENTION:
    if (static_cast<const GqaParams *>(params)->tokens == 1)
      return index == 0 ? "gqaDecodeGated" : "gqaDecodeMergeGated";
    if (index == 0) // (for 16-byte aligned rows apart from the outputs)
      return "attentionRows";
    if (llmi_hip_dispatch_count(op, params) == 2)
      return "gqaPrefillGated";
    return index == 1 ? "gqaPrefillMfma" : "gqaPrefillMergeGated";
  }
  return nullptr;
}

const char *llmi_hip_status_string(int status) {
  switch (status) {
  case LLMI_HIP_OK:
    return "ok";
  case LLMI_HIP_INVALID_ARGUMENT:
    return "invalid argument";
  case LLMI_HIP_UNSUPPORTED:
    return "unsupported";
  case LLMI_HIP_WORKSPACE:
    return "workspace missing or too small";
  case LLMI_HIP_LAUNCH_FAILED:
    return "launch failed";
  case LLMI_HIP_NO_DEVICE:
    return "no device";
  }
  return "unknown status";
}

const char *llmi_hip_last_error(void) { return g_error; }

const char *llmi_hip_build_info(void) {
  return "llminfer-hip 0.1 gfx950";
}

} // extern "C"
