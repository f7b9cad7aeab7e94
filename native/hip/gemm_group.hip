// Grouped (ragged by expert) and block-scaled fp8 matrix products: the dispatch and the C entry.
// The mathematics and the modes: group_common.h. Kernels: group_tile.h.
#include "group_tile.h"

namespace {

template <class C>
int launch_tile_regs(const GroupArgs& g, hipStream_t s) {
  const long long tiles_n = ((long long)g.cols + C::BN - 1) / C::BN;
  const long long tiles_m = g.mode == kModeWgrad ? ((long long)g.rows + C::BM - 1) / C::BM * g.experts
                                                 : group_tile_bound(g.rows, g.experts, g.offsets != nullptr, C::BM);
  const long long grid = tiles_m * tiles_n;
  if (grid > 0x7fffffff) return (int)hipErrorInvalidValue;
  if (grid == 0) return 0;
  hipLaunchKernelGGL((group_tile_regs<C>), dim3((unsigned)grid), dim3(C::THREADS), 0, s, g);
  return (int)hipGetLastError();
}

template <int DT>
int dispatch16(const GroupArgs& g, hipStream_t s) {
  switch (g.mode) {
    case kModeForward: return launch_tile_regs<TileCfg<DT, kScaleNone, false, false, 128, 128, 2, 2>>(g, s);
    case kModeDgrad: return launch_tile_regs<TileCfg<DT, kScaleNone, false, true, 128, 128, 2, 2>>(g, s);
    case kModeWgrad: return launch_tile_regs<TileCfg<DT, kScaleNone, true, true, 128, 128, 2, 2>>(g, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace

extern "C" {

int amdgo_gemm_group(const GroupArgs* args, hipStream_t s) {
  if (!args) return (int)hipErrorInvalidValue;
  const GroupArgs& g = *args;
  if (g.rows < 0 || g.cols < 0 || g.red < 0 || g.experts < 1) return (int)hipErrorInvalidValue;
  if (g.rows == 0 || g.cols == 0) return 0;
  if (g.dtype == kFp8) {
    if (g.mode != kModeForward) return (int)hipErrorInvalidValue;
    if (g.scale == kScaleF32) return launch_tile_regs<TileCfg<kFp8, kScaleF32, false, false, 128, 128, 2, 2>>(g, s);
    if (g.scale == kScaleE8) return launch_tile_regs<TileCfg<kFp8, kScaleE8, false, false, 128, 128, 2, 2>>(g, s);
    return (int)hipErrorInvalidValue;
  }
  if (g.scale != kScaleNone) return (int)hipErrorInvalidValue;
  if (g.dtype == kBf16) return dispatch16<kBf16>(g, s);
  if (g.dtype == kFp16) return dispatch16<kFp16>(g, s);
  return (int)hipErrorInvalidValue;
}

}  // extern "C"
