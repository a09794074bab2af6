// What the kernels of the paged attention share: the plan that divides a
// call's keys over workgroups, made by each of them from the lengths in device
// memory, and where partial outputs go.
#pragma once

#include "hip_common.hpp"
#include "paged_kv.hpp"
#include "paged_shared.hpp"

namespace llmi {

constexpr float kPagedRaise = 15.0f;   // raise m when a weight would pass 2^15
constexpr float kPagedHeadroom = 7.0f; // after a raise the largest weight is 2^7

// The softmax scale as the kernels take it: exp2 of positive multiples of the
// scores, so that their largest is the largest weight's, with the sign given
// to the queries; 0 as a multiple that leaves every score 0.
struct ScoreScale {
  float c;
  uint32_t sign; // of two fp16 values
};
inline ScoreScale score_scale(float scale) {
  const float c = __builtin_fabsf(scale * kLog2e);
  return {c > 1e-30f || c != c ? c : 1e-30f, scale < 0.0f ? 0x80008000u : 0u};
}
// A score in those multiples, rounded, as the reference m is made of it. The fma
// of the score, c and -m keeps what that rounding lost, 32 at 2^29, and the
// largest weight would leave fp16 at either end: the weights take the rounded
// product less m, exact where it counts.
__device__ __forceinline__ float scaled_score(float x, float c) {
  x *= c;
  asm("" : "+v"(x)); // no fma of it
  return x;
}
__device__ __forceinline__ half8_t with_sign(half8_t x, uint32_t sign) {
  return __builtin_bit_cast(half8_t, __builtin_bit_cast(uint4_t, x) ^ sign);
}

// How a call's work is divided: a sequence's rows into units of `columns`
// columns, and the blocks of 32 keys that it holds (one where it has no place,
// for the workgroup that says so) into equal pieces of about `chunk` blocks:
// at most chunk, or (nearest) at most 1.5 of it, for a kernel whose pieces
// cost more to join than some workgroups' longer time.
struct Split {
  unsigned group, shift, step, chunk; // units of 2^shift columns, whole steps of blocks
  float inv;                    // 1 / chunk
  bool nearest;
  template <typename Seq> __device__ unsigned units(const Seq &q) const {
    return (unsigned)(((uint64_t)q.rows * group + (1u << shift) - 1) >> shift);
  }
  template <typename Seq> __device__ static unsigned blocks(const Seq &q) {
    return q.ok ? (q.keys() + 31) / 32 - q.first() : 1u;
  }
  // (x + round) / chunk by the reciprocal, corrected by its remainder: at most
  // as many pieces as the host planned for, so off by one at most
  template <typename Seq> __device__ unsigned pieces(const Seq &q) const {
    const unsigned x = blocks(q) + (nearest ? chunk / 2 : chunk - 1);
    unsigned n = (unsigned)((float)x * inv);
    const int rest = (int)(x - n * chunk);
    n = rest < 0 ? n - 1 : rest >= (int)chunk ? n + 1 : n;
    return n ? n : 1u;
  }
  // blocks of a piece: whole steps of the kernels
  template <typename Seq> __device__ unsigned length(const Seq &q, unsigned pieces) const {
    const unsigned each = (blocks(q) + pieces - 1) / pieces;
    return (each + step - 1) & ~(step - 1);
  }
};

// How the host asks for it: `fill` pieces a KV head fill the device, and at
// most `target`, some rounds of that, are made where pieces then still have
// `whole` blocks. step (a power of two): the blocks that a workgroup takes at
// a time. alone: workgroups have a CU each, so that pieces past
// `fill` would wait for the others.
struct SplitPlan {
  unsigned shift, step, fill, target, whole, nearest, alone;
};

// The chunk, whole steps, for which the call has at most plan.target pieces
// more than units. (The fp32 sum is exact below 2^24, and off by less than
// the 1.0001 above; every workgroup and the merge add in the same order.)
template <typename Seq>
__device__ __forceinline__ float lane_blocks(const Split &s, const Seq &q) {
  return (float)s.units(q) * (float)Split::blocks(q);
}
__device__ __forceinline__ float all_blocks(const Split &s, const PagedView &g,
                                            const PagedSeq &own) {
  const unsigned lane = threadIdx.x % 64;
  float all = lane_blocks(s, own);
  for (unsigned s0 = 64; s0 < g.sequences; s0 += 64)
    if (s0 + lane < g.sequences)
      all += lane_blocks(s, paged_seq(g, s0 + lane));
  return all;
}
__device__ __forceinline__ float all_blocks(const Split &s, const SharedView &g,
                                            const SharedLanes &own) {
  float all = 0.0f;
  shared_chunks(g, own, [&](unsigned, const SharedSeq &q) {
    all += lane_blocks(s, q);
    return false;
  });
  return all;
}
template <typename View, typename Own>
__device__ __forceinline__ Split paged_split(const View &g, const Own &lanes, unsigned group,
                                             const SplitPlan &plan) {
  Split s{group, plan.shift, plan.step, plan.step, 0.0f, plan.nearest != 0};
  const auto &own = paged_first(lanes);
  float all = group_sum<16>(all_blocks(s, g, lanes));
  LanePair p = pair16(all);
  all = p.a + p.b;
  p = pair32(all);
  all = p.a + p.b;
  all = all < 16777216.0f ? all : all * 1.0001f;
  // (below 2^30: no table has more blocks)
  const unsigned least = (unsigned)fminf(ceilf(all / (float)plan.target), 0x1p30f);
  const unsigned one = (unsigned)fminf(ceilf(all / (float)plan.fill), 0x1p30f); // of a single round
  auto take = [&](unsigned chunk) {
    const unsigned steps = (chunk + s.step - 1) & ~(s.step - 1);
    s.chunk = (unsigned)__builtin_amdgcn_readfirstlane((int)(steps ? steps : s.step));
    s.inv = __builtin_amdgcn_rcpf((float)s.chunk);
  };
  take(max(least, min(one, plan.whole)));
  // Every unit's last piece is rounded up, and a few pieces more than fill the
  // device would be a second round: longer ones, where one round can be (160
  // columns on 31000 keys at head_dim 128, units of 32: 36 us, 52 without).
  if (plan.alone && g.sequences <= 64) {
    auto total = [&](unsigned x) {
      return g.sequences == 1 ? (unsigned)__builtin_amdgcn_readfirstlane((int)x)
                              : (unsigned)__builtin_amdgcn_readlane((int)wave_scan(x), 63);
    };
    const unsigned units = s.units(own);
    if (total(units) <= plan.fill)
      for (int i = 0; i < 4; ++i) {
        const unsigned n = total(units * s.pieces(own));
        if (n <= plan.fill)
          break;
        take(max(s.chunk + 1, (unsigned)fminf((float)s.chunk * (float)n / (float)plan.fill,
                                              0x1p30f)));
      }
  }
  return s;
}

// Where the output or the partial of a workgroup goes.
struct Partials {
  float *ml, *o; // [piece][KV head][column]{m, l}, [piece][KV head][column][D]
};

// The kernel for sequences of many rows (paged_tiles.hip): columns of its
// units, and its launch.
unsigned paged_tiles_columns(unsigned headDim);
template <typename View>
hipError_t launch_paged_tiles(const half_t *q, const uint8_t *pool, const View &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, SplitPlan plan, ScoreScale c,
                              Partials parts, unsigned pieces, hipStream_t stream);

// The kernel for groups with many rows in all and sequences with few
// (paged_mixed.hip): whole steps of blocks, `cus` workgroups a KV head, the blocks
// of shared keys whose time a workgroup loses by beginning a second time, and the
// time that a block of a unit of shared keys, a block of a unit of own keys and a
// unit of own keys take of a workgroup.
constexpr unsigned kMixedWaves = 8; // of a workgroup
struct MixedPlan {
  unsigned step, cus, again;
  float sharedCost, ownCost, ownFixed;
};
hipError_t launch_paged_mixed(const half_t *q, const uint8_t *pool, const SharedView &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, const MixedPlan &plan,
                              ScoreScale c, Partials shared, Partials rest, unsigned mostShared,
                              unsigned mostOwn, hipStream_t stream);

} // namespace llmi
