// Causal GQA over the paged 4-bit cache for sequences of many rows: tiles of
// keys and values decoded once for all of a workgroup's columns.
//
// A workgroup has 128 columns of a KV head (256 at head_dim 128), eight waves:
// wave w the 32-column tiles of column wave w % 4, and of the keys of a step
// the half w / 4. A step is 512 / D blocks of 32 keys:
//  * every thread decodes 16 bytes of key codes and 16 of value codes of the
//    next step into LDS, as fp16 operands of v_mfma_f32_32x32x16_f16 in the
//    order in which a wave reads them (1 KB, conflict-free), while
//  * the matrix products of this one run: S^T = K Q^T with the columns in the
//    lanes, and O^T += V^T P^T, whose weights are the score tile's registers
//    as they are (the slots of a value word are the keys of a lane's eight);
//  * codes and scales go HBM -> LDS by DMA two steps ahead, each wave those
//    that its own threads decode, so that no register holds them and only
//    the decoded tiles need the workgroup's barrier, one a step.
// The halves of the keys are joined at the end through the tiles' memory.
//
// 2048 tokens of 16 heads of 256 on 4096 keys take 131 us (traced, after some
// hundred passes; the first take 138 and more; 134 to 138 in their call with
// the join's launch, by the card), 103 GFLOP; the last units see 4096 keys and
// the first 2080, and the kernel takes the time of the last ones: 128 blocks at
// 0.97 us, 1.1 PFLOP/s while all of them run. Bound by the products and the
// vector instructions of a SIMD's two waves, which overlap little: 99 and 78
// thousand cycles of the 208 thousand that a SIMD's workgroups run (half of the
// vector instructions decode, without them the kernel takes 64 % of its time;
// LDS is busy for 86 thousand).
// At head_dim 128 the kernel has more than its 256 registers hold: addresses are
// reloaded from scratch between a step's DMA loads, each reload a wait for all
// loads before it. SQ_WAIT_ANY is 56 million in seven ragged messages (125 us
// traced, 127 to 131 in their call) and 28 million in the call above, whose
// products are more.
// Of a short call (61 tokens on 16472 keys: 30 us inside the kernel) 6 us are
// the plan, the table and the first blocks, 5 the joining and the partials.
#include "paged_tiles.hpp"

namespace llmi {
namespace {

// The call's piece `u` with the sequences of the longest pieces first (up to 64
// sequences; in their order otherwise), so that workgroups which start late
// have little to do (seven messages of 41 to 110 blocks, 296 workgroups:
// 174 us in order, 130 longest first).
template <typename View, typename Own>
__device__ __forceinline__ bool find_longest(const View &g, const Own &lanes, const Split &split,
                                             unsigned u, unsigned &seq, unsigned &local,
                                             unsigned &number) {
  const auto &own = paged_first(lanes);
  unsigned before;
  if (g.sequences == 1 || g.sequences > 64) {
    number = u;
    return paged_find(g, lanes, u,
                      [&](const auto &s) { return split.units(s) * split.pieces(s); }, seq,
                      local, before);
  }
  const unsigned lane = threadIdx.x % 64;
  const unsigned pieces = split.pieces(own), length = split.length(own, pieces);
  const unsigned n = split.units(own) * pieces;
  unsigned ahead = 0;
  for (unsigned j = 0; j < g.sequences; ++j) {
    const unsigned lj = (unsigned)__builtin_amdgcn_readlane((int)length, (int)j);
    const unsigned nj = (unsigned)__builtin_amdgcn_readlane((int)n, (int)j);
    ahead += lj > length || (lj == length && j < lane) ? nj : 0u;
  }
  const unsigned long long here =
      __builtin_amdgcn_ballot_w64(lane < g.sequences && u - ahead < n);
  if (!here)
    return false;
  const int at = __builtin_ctzll(here);
  seq = (unsigned)at;
  local = u - (unsigned)__builtin_amdgcn_readlane((int)ahead, at);
  number = (unsigned)__builtin_amdgcn_readlane((int)(wave_scan(n) - n), at) + local;
  return true;
}

template <int D, typename View>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads),
                          amdgpu_waves_per_eu(2, 2)))
void paged_tiles_kernel(const half_t *__restrict__ q, const uint8_t *__restrict__ pool,
                        View g, half_t *out, unsigned *invalid, unsigned queryHeads,
                        SplitPlan plan, ScoreScale c, Partials parts) {
  const unsigned G = queryHeads / g.kvHeads, kvh = blockIdx.x % g.kvHeads;
  const auto own = paged_own(g);
  const Split split = paged_split(g, own, G, plan);
  unsigned seq, local, number; // number: of this piece, for its partials
  if (!find_longest(g, own, split, blockIdx.x / g.kvHeads, seq, local, number) ||
      number >= gridDim.x / g.kvHeads) // (starts out of order: more pieces than the rows can have)
    return;
  const auto s = paged_seq_of(g, own, seq);
  const unsigned pieces = split.pieces(s), units = split.units(s);
  const unsigned unit = units - 1 - local / pieces, piece = local % pieces;
  if (local == 0 && kvh == 0 && threadIdx.x == 0)
    leave_note(g, s, seq, number, pieces, units);
  const unsigned length = split.length(s, pieces);
  tiles_piece<D, 256 / D, true>(q, pool, g, out, invalid, queryHeads, c, parts, s, seq, kvh,
                                unit, Tiles<D, 256 / D>::UNIT, s.first() + piece * length, length,
                                pieces == 1, number);
}

} // namespace

unsigned paged_tiles_columns(unsigned headDim) { return 128 * (256 / headDim); }

template <typename View>
hipError_t launch_paged_tiles(const half_t *q, const uint8_t *pool, const View &g, half_t *out,
                              unsigned *invalid, unsigned queryHeads, SplitPlan plan, ScoreScale c,
                              Partials parts, unsigned pieces, hipStream_t stream) {
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(pieces * g.kvHeads), dim3(kThreads), 0, stream, q, pool, g, out,
                       invalid, queryHeads, plan, c, parts);
    return hipGetLastError();
  };
  return g.dim == 256 ? run(paged_tiles_kernel<256, View>) : run(paged_tiles_kernel<128, View>);
}
template hipError_t launch_paged_tiles<PagedView>(const half_t *, const uint8_t *,
                                                  const PagedView &, half_t *, unsigned *, unsigned,
                                                  SplitPlan, ScoreScale, Partials, unsigned,
                                                  hipStream_t);
template hipError_t launch_paged_tiles<SharedView>(const half_t *, const uint8_t *,
                                                   const SharedView &, half_t *, unsigned *,
                                                   unsigned, SplitPlan, ScoreScale, Partials,
                                                   unsigned, hipStream_t);

} // namespace llmi
