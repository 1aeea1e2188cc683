// Launch of one tcgen05 forward instantiation (fa_sm100.cuh).
#pragma once
#include <atomic>

#include "../../include/mfa.h"
#include "fa_sm100.cuh"
#include "host.cuh"

namespace mfa {

// Tiles per CTA of the tcgen05 kernel fa_fwd_sm100<DP, *, GEN> (its default template argument).
template <int DP, int GEN>
constexpr int sm100_tiles() {
  return DefaultTiles<DP, DefaultCG<GEN, DP>::value, GEN>::value;
}

// SHORT: the one-tile, one-column-group kPack instantiation (sm100_short). SINK: the kSink one.
// ONE: one tile per CTA (without SHORT, only where there is one column group).
template <int DP, bool BF16, int GEN, bool SHORT, bool SINK, bool ONE = SHORT>
int launch_sm100(const Sm100Args& args, int dev, int64_t grid, cudaStream_t st) {
  constexpr int CG = SHORT ? 1 : DefaultCG<GEN, DP>::value;
  constexpr int TILES = ONE ? 1 : sm100_tiles<DP, GEN>();
  auto k = fa_fwd_sm100<DP, BF16, GEN, CG, TILES, SHORT, SINK>;
  using R = sm100::Roles<CG, TILES>;
  constexpr int KBN = sm100::BlockKeys<DP, GEN, CG, TILES, SHORT>::value;
  const int smem = (int)sm100::Cfg<DP, TILES, KBN>::SMEM;
  // The kernel re-splits its registers with setmaxnreg assuming exactly kLaunchRegs per thread
  // at launch; a build that launched with fewer would make setmaxnreg.inc wait forever.
  static std::atomic<int> launch_regs{-1};
  int regs = launch_regs.load(std::memory_order_relaxed);
  if (regs < 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, k) != cudaSuccess) return MFA_ERR_CUDA;
    regs = fa.numRegs;
    launch_regs.store(regs, std::memory_order_relaxed);
  }
  if (regs != R::kLaunchRegs) return MFA_ERR_UNSUPPORTED;
  if (ensure_smem(k, dev, smem) != cudaSuccess) return MFA_ERR_CUDA;
  k<<<(unsigned)grid, R::kThreads, smem, st>>>(args);
  return MFA_OK;
}

// The instantiation for run-time choices; `wide` is D > 64, `gen` the score transform (kBias),
// `one` whether a kSink launch of long rows takes one tile per CTA (sm100_sink_one).
template <int DP, bool BF16, int GEN, bool SINK>
int launch_sm100_gen(const Sm100Args& args, int dev, bool short_rows, bool one, int64_t grid,
                     cudaStream_t st) {
  if (short_rows) return launch_sm100<DP, BF16, GEN, true, SINK>(args, dev, grid, st);
  if constexpr (SINK && sm100_tiles<DP, GEN>() == 2 && DefaultCG<GEN, DP>::value == 1)
    if (one) return launch_sm100<DP, BF16, GEN, false, SINK, true>(args, dev, grid, st);
  return launch_sm100<DP, BF16, GEN, false, SINK>(args, dev, grid, st);
}
template <bool SINK>
int launch_sm100_rt(const Sm100Args& args, int dev, bool wide, bool bf16, int gen, bool short_rows,
                    bool one, int64_t grid, cudaStream_t st) {
#define MFA_SM100_G(DP, BF, G) \
  launch_sm100_gen<DP, BF, G, SINK>(args, dev, short_rows, one, grid, st)
#define MFA_SM100(DP, BF)                                                   \
  (gen == 2 ? MFA_SM100_G(DP, BF, 2)                                        \
            : gen == 1 ? MFA_SM100_G(DP, BF, 1) : MFA_SM100_G(DP, BF, 0))
  if (wide) return bf16 ? MFA_SM100(128, true) : MFA_SM100(128, false);
  return bf16 ? MFA_SM100(64, true) : MFA_SM100(64, false);
#undef MFA_SM100
#undef MFA_SM100_G
}

// The instantiations whose first keys stay visible left of the window, compiled in sink_fwd.cu.
int launch_sm100_sink(const Sm100Args& args, int dev, bool wide, bool bf16, int gen,
                      bool short_rows, bool one, int64_t grid, cudaStream_t st);

}  // namespace mfa
