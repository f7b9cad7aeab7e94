// Grouped (ragged by expert) and block-scaled fp8 matrix products: the dispatch and the C entry.
// The mathematics and the modes: group_common.h. Kernels: group_tile.h.
#include "group_tile.h"

namespace {

template <class C>
long long tile_grid(const GroupArgs& g) {
  const long long tiles_n = ((long long)g.cols + C::BN - 1) / C::BN;
  const long long tiles_m = g.mode == kModeWgrad ? ((long long)g.rows + C::BM - 1) / C::BM * g.experts
                                                 : group_tile_bound(g.rows, g.experts, g.offsets != nullptr, C::BM);
  return tiles_m * tiles_n;
}

template <class C, bool DMA>
int launch_tile(const GroupArgs& g, hipStream_t s) {
  const long long grid = tile_grid<C>(g);
  if (grid > 0x7fffffff) return (int)hipErrorInvalidValue;
  if (grid == 0) return 0;
  if constexpr (DMA) hipLaunchKernelGGL((group_tile_dma<C>), dim3((unsigned)grid), dim3(C::THREADS), 0, s, g);
  else hipLaunchKernelGGL((group_tile_regs<C>), dim3((unsigned)grid), dim3(C::THREADS), 0, s, g);
  return (int)hipGetLastError();
}

// Whether every 16-byte chunk that a tile reads is whole and aligned, and a tile's lane offsets fit a buffer's
// 2 GiB: what LDS-DMA needs. (A K-major operand's chunks lie along the reduction, a reduction-major one's along
// its rows.)
bool dma_ready(const GroupArgs& g) {
  const long long es = g.dtype == kFp8 ? 1 : 2;
  const bool a_tr = g.mode == kModeWgrad, b_tr = g.mode != kModeForward;
  const auto fits = [&](const void* p, long long ld, long long batch, bool tr, long long width) {
    return (((uintptr_t)p | (uintptr_t)(ld * es) | (uintptr_t)(batch * es) | (uintptr_t)((tr ? width : g.red) * es)) & 15) == 0 &&
           ld * es * 256 + width * es < 0x7fffffffll;
  };
  if (!fits(g.a, g.lda, 0, a_tr, g.rows) || !fits(g.b, g.ldb, g.b_expert, b_tr, g.cols)) return false;
  return g.scale == kScaleNone || (g.as_row * 4 * 256 < 0x7fffffffll && g.bs_row * 4 * 4 < 0x7fffffffll);
}

// 256 x 256 tiles (one workgroup a CU) once the groups fill them and the grid fills the CUs, else 128 x 128
// (two a CU, so that one's prologue and epilogue run under the other's loop).
template <int DT, int SC, bool ATR, bool BTR>
int dispatch_tile(const GroupArgs& g, hipStream_t s) {
  using Small = TileCfg<DT, SC, ATR, BTR, 128, 128, 2, 2, 128, 2>;
  using Large = TileCfg<DT, SC, ATR, BTR, 256, 256, 2, 4, 128, 2>;
  if (!dma_ready(g)) return launch_tile<TileCfg<DT, SC, ATR, BTR, 128, 128, 2, 2>, false>(g, s);
  const long long per_group = g.mode == kModeWgrad ? g.rows : g.rows / g.experts;
  if (per_group > 128 && tile_grid<Large>(g) >= 256) return launch_tile<Large, true>(g, s);
  return launch_tile<Small, true>(g, s);
}

template <int DT>
int dispatch16(const GroupArgs& g, hipStream_t s) {
  switch (g.mode) {
    case kModeForward: return dispatch_tile<DT, kScaleNone, false, false>(g, s);
    case kModeDgrad: return dispatch_tile<DT, kScaleNone, false, true>(g, s);
    case kModeWgrad: return dispatch_tile<DT, kScaleNone, true, true>(g, s);
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
    if (g.scale == kScaleF32) return dispatch_tile<kFp8, kScaleF32, false, false>(g, s);
    if (g.scale == kScaleE8) return dispatch_tile<kFp8, kScaleE8, false, false>(g, s);
    return (int)hipErrorInvalidValue;
  }
  if (g.scale != kScaleNone) return (int)hipErrorInvalidValue;
  if (g.dtype == kBf16) return dispatch16<kBf16>(g, s);
  if (g.dtype == kFp16) return dispatch16<kFp16>(g, s);
  return (int)hipErrorInvalidValue;
}

}  // extern "C"
