// Grouped (ragged by expert) and block-scaled fp8 matrix products: the dispatch and the C entry.
// The mathematics and the modes: group_common.h. Kernels: group_tile.h, group_skinny.h.
#include "group_skinny.h"
#include "memory_reach.h"

#include <stddef.h>

namespace {

template <class C>
long long tile_grid(const GroupArgs& g) {
  const long long tiles_n = ((long long)g.cols + C::BN - 1) / C::BN;
  const long long tiles_m = g.mode == kModeWgrad ? ((long long)g.rows + C::BM - 1) / C::BM * g.experts
                                                 : group_tile_bound(g.rows, g.experts, g.offsets != nullptr, C::BM);
  return tiles_m * tiles_n;
}

enum TileKernel { kTileDma, kTilePingPong };

template <class C, TileKernel KERNEL>
int launch_tile(const GroupArgs& g, hipStream_t s) {
  GroupArgs a = g;
  const int cus = device_cu_count(s);
  a.slots = KERNEL == kTilePingPong || g.mode != kModeWgrad ? cus : 0;
  if (tile_grid<C>(g) > 0x7fffffff - 2 * (long long)cus) return (int)hipErrorInvalidValue;
  if (tile_grid<C>(g) == 0) return 0;
  if constexpr (KERNEL == kTilePingPong) {
    hipLaunchKernelGGL((group_tile_pp<C>), dim3((unsigned)cus), dim3(C::THREADS), 0, s, a);
  } else {
    // The last tiles are cut into parts, at most one more round of workgroups of one a CU (of as many as fit a CU, 80 x 8192 x
    // 8192 fp8 took 42 us for 30: the parts read their columns of B once each).
    const long long grid = tile_grid<C>(g) + a.slots + (g.zero_rest ? kRestBlocks : 0);
    hipLaunchKernelGGL((group_tile_dma<C>), dim3((unsigned)grid), dim3(C::THREADS), 0, s, a);
  }
  return (int)hipGetLastError();
}

// What amdgo_gemm_group answers, having launched nothing, where the operands have to be laid out first
// (amdgo_gemm_group_packed): see dma_ready.
constexpr int kNeedsPacking = -1;

// Whether a tile's lane offsets fit a buffer's 2 GiB.
bool offsets_fit(const GroupArgs& g) {
  const long long es = g.dtype == kFp8 ? 1 : 2, kb = g.red / kScaleBlock + 1;
  const long long across = ((long long)(g.rows > g.cols ? g.rows : g.cols) + g.red) * es;
  return g.lda * es * 256 + across < 0x7fffffffll && g.ldb * es * 256 + across < 0x7fffffffll &&
         (g.scale == kScaleNone || ((g.as_row * 256 + g.as_k * kb) * 4 < 0x7fffffffll &&
                                    (g.bs_row * 4 + g.bs_k * kb) * 4 < 0x7fffffffll));
}

// Whether every 16-byte chunk that a tile reads is whole and aligned too: what LDS-DMA needs. (A K-major operand's
// chunks lie along the reduction, a reduction-major one's along its rows.)
bool dma_ready(const GroupArgs& g) {
  const long long es = g.dtype == kFp8 ? 1 : 2;
  const bool a_tr = g.mode == kModeWgrad, b_tr = g.mode != kModeForward;
  const auto whole = [&](const void* p, long long ld, long long batch, bool tr, long long width) {
    const long long along = tr ? (g.padded ? 0 : width) : g.red;
    return (((uintptr_t)p | (uintptr_t)(ld * es) | (uintptr_t)(batch * es) | (uintptr_t)(along * es)) & 15) == 0;
  };
  return whole(g.a, g.lda, 0, a_tr, g.rows) && whole(g.b, g.ldb, g.b_expert, b_tr, g.cols) && offsets_fit(g);
}

// A matrix [batches, rows, row_bytes] of any strides to [batches, to_rows, to_bytes] (to_bytes a multiple of 16, rows to_ld
// apart), zeros where the source has nothing.
struct PackMatrix {
  const char* from;
  char* to;
  long long ld, batch, to_ld, row_bytes, to_bytes;
  int batches, rows, to_rows;

  __host__ __device__ long long blocks() const { return (long long)batches * to_rows; }
};

// Both operands in one launch: a workgroup takes whole rows, 16 bytes a lane.
__global__ void __launch_bounds__(256) pack_rows(const PackMatrix a, const PackMatrix b) {
  const unsigned in_a = (unsigned)a.blocks(), block = blockIdx.x < in_a ? blockIdx.x : blockIdx.x - in_a;
  const PackMatrix m = blockIdx.x < in_a ? a : b;
  const int batch = block / (unsigned)m.to_rows, r = block - batch * (unsigned)m.to_rows;
  const char* src = m.from + (size_t)batch * m.batch + (size_t)r * m.ld;
  char* dst = m.to + (size_t)block * m.to_ld;
  for (long long at = threadIdx.x * 16ll; at < m.to_bytes; at += 256 * 16) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < m.rows) v = __builtin_bit_cast(uint4, load_chunk<1>(src, (int)at, (int)m.row_bytes));
    *(uint4*)(dst + at) = v;
  }
}

// What has to be laid out for a product whose operands are not dma_ready, and the product on it. A reduction along the rows is
// filled up with zeros to whole 16-byte pieces, in both operands, so that they add nothing; the rows start on lines.
struct PackPlan {
  PackMatrix a, b;
  GroupArgs g;
  long long bytes;

  explicit PackPlan(const GroupArgs& from) : a{}, b{}, g(from), bytes(0) {
    const long long es = g.dtype == kFp8 ? 1 : 2, unit = 16 / es, full = (g.red + unit - 1) / unit * unit;
    const bool a_tr = g.mode == kModeWgrad, b_tr = g.mode != kModeForward;
    const auto lay = [&](PackMatrix& m, const void*& p, long long& ld, long long* batch, int batches, long long rows, long long width,
                         long long to_rows) {
      const long long to = (width + unit - 1) / unit * unit, pitch = (to * es + 127) / 128 * 128;
      const long long strides = (long long)(uintptr_t)p | ld * es | (batch ? *batch * es : 0) | width * es;
      const long long across = ((long long)(g.rows > g.cols ? g.rows : g.cols) + g.red) * es;
      if ((strides & 15) == 0 && to_rows == rows && ld * es * 256 + across < 0x7fffffffll) return;
      m = PackMatrix{(const char*)p, nullptr, ld * es, batch ? *batch * es : 0, pitch, width * es, to * es, batches, (int)rows, (int)to_rows};
      m.to = (char*)(uintptr_t)bytes;                     // its place in the workspace
      bytes += batches * to_rows * pitch;
      ld = pitch / es;
      if (batch) *batch = to_rows * ld;
    };
    lay(a, g.a, g.lda, nullptr, 1, a_tr ? g.red : g.rows, a_tr ? g.rows : g.red, a_tr ? g.red : g.rows);
    const long long b_rows = b_tr ? g.red : g.cols;
    lay(b, g.b, g.ldb, g.mode == kModeWgrad ? nullptr : &g.b_expert, g.mode == kModeWgrad ? 1 : g.experts, b_rows, b_tr ? g.cols : g.red,
        g.mode == kModeDgrad ? full : b_rows);
    if (g.mode != kModeWgrad) g.red = (int)full;
    g.padded = 1;
  }
  bool fits() const { return g.red >= 0 && a.blocks() + b.blocks() <= 0x7fffffffll && offsets_fit(g); }
  int launch(char* space, hipStream_t s) {
    for (PackMatrix* m : {&a, &b}) m->to = space + (uintptr_t)m->to;
    if (a.blocks()) g.a = a.to;
    if (b.blocks()) g.b = b.to;
    if (bytes == 0) return 0;
    hipLaunchKernelGGL(pack_rows, dim3((unsigned)(a.blocks() + b.blocks())), dim3(256), 0, s, a, b);
    return (int)hipGetLastError();
  }
};

template <class C>
int launch_skinny(const GroupArgs& g, long long tiles_m, hipStream_t s) {
  const long long grid = tiles_m * (((long long)g.cols + C::COLS - 1) / C::COLS) + (g.zero_rest ? kRestBlocks : 0);
  if (grid > 0x7fffffff) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL((group_skinny<C>), dim3((unsigned)grid), dim3(C::THREADS), 0, s, g);
  return (int)hipGetLastError();
}

// MT 16-row tiles a workgroup. 64 columns and 4 waves where that leaves more than two workgroups a CU, else
// narrower columns and the reduction over more waves (8192 x 8192 fp8, 16 rows: 128 workgroups of 64 columns
// 23.0 us, 256 of 32 with 8 waves 17.5; 1024 x 2048 bf16 over 4 experts: 32 columns 7.5, 16 columns 6.5; 64 experts of
// 4096 x 2048 fp8: 64 columns and 4 waves 54.3, 32 and 8 58.0; the weights at a copy's rate: 13.3, 2.2, 58.0). 16-bit
// weights of a few rows each are narrower still, down to 16 columns from 4096 of K on (16 rows over 16 experts, 4096 x 4096
// bf16: 64 columns 65.1, 32 62.1, 16 54.1; 64 over 64, 4096 x 2048: 108.9, 100.3, 110.3; but 64 rows over 8: 48.8, 52.3, 51.4).
template <int DT, int SC, int MT>
int skinny_columns(const GroupArgs& g, hipStream_t s) {
  const long long tiles_m = group_tile_bound(g.rows, g.experts, g.offsets != nullptr, 16 * MT);
  const long long busy = g.experts < g.rows ? g.experts : g.rows;
  const bool narrow = DT != kFp8 && g.rows <= 4 * busy;
  if (!narrow && tiles_m * ((g.cols + 63) / 64) > 512) return launch_skinny<SkinnyCfg<DT, SC, MT, 4, 4>>(g, tiles_m, s);
  if constexpr (MT == 1)
    if ((narrow && g.red >= 4096) || tiles_m * ((g.cols + 31) / 32) < 256)
      return launch_skinny<SkinnyCfg<DT, SC, 1, 1, 8>>(g, tiles_m, s);
  return launch_skinny<SkinnyCfg<DT, SC, MT, 2, 8>>(g, tiles_m, s);
}

// The same for operands without whole aligned chunks: rows that start on 4 bytes are loaded as they lie, others in words (8192
// x 8190 fp8, 16 rows: 43.3 us as they lie, 23.8; 12 groups of 57 rows, 1184 x 3471 bf16: 51.0, 34.6; but x 3470: 28.8, 34.7).
template <int DT, int SC, int MT>
int skinny_unaligned(const GroupArgs& g, hipStream_t s) {
  if (!offsets_fit(g)) return kNeedsPacking;
  const long long tiles_m = group_tile_bound(g.rows, g.experts, g.offsets != nullptr, 16 * MT), es = DT == kFp8 ? 1 : 2;
  if ((((uintptr_t)g.a | (uintptr_t)g.b | (uintptr_t)(g.lda * es) | (uintptr_t)(g.ldb * es) | (uintptr_t)(g.b_expert * es)) & 3) == 0)
    return launch_skinny<SkinnyCfg<DT, SC, MT, 2, 8, 4>>(g, tiles_m, s);
  return launch_skinny<SkinnyCfg<DT, SC, MT, 2, 8, 1>>(g, tiles_m, s);
}

// Few rows: the skinny kernel with tiles of 16 rows, or of 32 for a single group of 17 to 64 (8192 x 8192 fp8, 32 rows:
// 16-row tiles 30 us, 32-row ones 22.5; 64 rows of 4096 x 4096: 15.6, 12.2). Groups of more than 12 rows on average
// are for the tiled kernel (16 of 16 rows, 4096 x 2048: 65.5 us, Low 60.4; 64 of 8 rows: 93.8, Small 110.5); of more than
// 20 where the operands are not `ready`, since that one needs a copy of the weights then (16 of 15 rows, 2048 x 1537 bf16:
// 42.9, 59.1; of 25: 58.4, 59.5; fp8 29.8, 33.6 and 40.0, 34.4). The offsets are on the device, so the mean is all that there is
// to go by, padding and idle experts included: 700 rows over 64 experts of 4096 x 2048 bf16 take 208 us evenly and 103 where one
// expert has all of them, which as a product of one expert's take 21 (fp8: 109, 63, 14). 0: not here.
int skinny_rows(const GroupArgs& g, bool ready) {
  if (g.mode != kModeForward) return 0;
  if (g.offsets == nullptr) return g.rows <= 16 ? 1 : g.rows <= 64 ? 2 : 0;
  const long long busy = g.experts < g.rows ? g.experts : g.rows;
  return g.rows <= (ready ? 12 : 20) * busy ? 1 : 0;
}

// The tile, by how many there are and how many rows a group has:
//
//   Large    256 x 256, ping-pong, one a CU: groups that fill it and a grid that nearly fills the CUs (16 groups of
//            250 rows, 2048 x 1024: 248 tiles 27.0 us, 128 x 128 36.1); from 7/16 of the CUs on where the groups are
//            long, since a part of a tile is most of its width still (1792 x 4096 x 4096 fp8, 112 tiles as 224 parts:
//            37.3 us, Small 39.4; 2304 rows, 144 tiles: 51.3, 57.3; 1536 rows, 96 tiles: 36.0, 33.5). Not where a fifth or
//            more of its columns would be empty (64 groups of 256 rows, 384 x 384: 16.1, Small 11.3; 4 of 8192 rows, 128
//            x 4096 fp8: 64.5, 50.6)
//   Small    128 x 128, two a CU, so that one's prologue and epilogue run under the other's loop: one round to about
//            two of groups that fill most of it (16 groups of 128 rows, 2048 x 2048: 41.3 us, Low 47.5, Deep 44.9;
//            700 x 8192 x 2048 fp8: 17.8, 23.3, 25.5; 32 groups of 94 rows, 880 tiles: 83.7, 70.6, 73.7). Not compared between
//            40 and 90 rows a group: 28 of 73, 1032 x 2056 fp16, take 57 us here, and their dgrad, of the same weights, 35 by Low
//   Deep     128 x 128, 8 waves, a ring of four: most of one round, where a workgroup's own latency is the time (fp8
//            512 x 8192 x 8192: 52.9 us, Low 59.7, Small 60.2; 16 groups of 125 rows, 1024 x 2048: 23.4, 26.2, 32.6)
//   Low      64 x 128, a ring of three: few rows a group, or fewer tiles than that (fp8 128 x 4096 x 4096: 13.5 us,
//            Deep 16.7, Small 21.9; 4 groups of 250 rows, 2048 x 2048: 18.8, 22.7, 24.7; 20 groups of 30 rows, 1024 x
//            1024: 10.6, 13.1, 14.3; 32 fp8 groups of 32, 2048 x 2048: 26.1, 33.5, 28.7)
//
// A weight gradient has whole tiles whatever the groups are, as long as their groups: from two rounds on Large, where
// the next tile starts under the stores and the rounds even out (32 groups of 65 rows, 1024 x 2048: 35.9 us, Small 44.3;
// 64 of 16 rows: 57.1, 99.3), unless a fifth of it would be empty (64 of 640 x 640: 53.6, 38.9); below Small, whose tiles
// find a free CU (16 groups of 40 to 3000 rows, 1024 x 1024: 50.7, Large 64.2); below one round Deep (4 groups of 8192
// rows, 1024 x 1024: 118, Small 169).
template <int DT, int SC, bool ATR, bool BTR>
int dispatch_tile(const GroupArgs& g, hipStream_t s) {
  using Large = TileCfg<DT, SC, ATR, BTR, 256, 256, 2, 4, 2>;
  using Small = TileCfg<DT, SC, ATR, BTR, 128, 128, 2, 2, 2>;
  using Deep = TileCfg<DT, SC, ATR, BTR, 128, 128, 2, 4, 4>;
  const bool ready = dma_ready(g);
  if constexpr (!ATR && !BTR) {
    switch (skinny_rows(g, ready)) {
      case 1: return ready ? skinny_columns<DT, SC, 1>(g, s) : skinny_unaligned<DT, SC, 1>(g, s);
      case 2:                                        // (a product without groups is an fp8 one)
        if constexpr (DT == kFp8) return ready ? skinny_columns<DT, SC, 2>(g, s) : skinny_unaligned<DT, SC, 2>(g, s);
    }
  }
  if (!ready) return kNeedsPacking;
  const int cus = device_cu_count(s);
  // (a Large tile's stores are 32-bit offsets in it)
  const long long large = g.ldc * 2 * 256 < 0x7fffffffll ? tile_grid<Large>(g) : 0;
  const long long small = tile_grid<Small>(g);
  if constexpr (ATR) {
    if (large >= 2 * cus && 16 * large < 5 * small) return launch_tile<Large, kTilePingPong>(g, s);
    if (small > cus) return launch_tile<Small, kTileDma>(g, s);
    return launch_tile<Deep, kTileDma>(g, s);
  } else {
    using Low = TileCfg<DT, SC, ATR, BTR, 64, 128, 1, 4, 3>;
    const long long per_group = g.rows / g.experts;
    const bool fills_columns = 10 * ((g.cols + 255ll) / 256) < 6 * ((g.cols + 127ll) / 128);
    if (fills_columns && ((5 * large >= 4 * cus && per_group > 128) || (16 * large >= 7 * cus && per_group >= 512)))
      return launch_tile<Large, kTilePingPong>(g, s);
    if (small > cus && per_group > 40 && (small <= 3 * cus || per_group > 128)) return launch_tile<Small, kTileDma>(g, s);
    if (small > cus || 4 * small <= 3 * cus || per_group <= 64) return launch_tile<Low, kTileDma>(g, s);
    return launch_tile<Deep, kTileDma>(g, s);
  }
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

namespace {

// The arguments as the caller packs them, up to `slots`.
GroupArgs group_args(const void* args) {
  GroupArgs g = {};
  __builtin_memcpy(&g, args, offsetof(GroupArgs, slots));
  if (g.offsets == nullptr || g.mode == kModeWgrad) g.zero_rest = 0;
  return g;
}

constexpr int kMostExtent = 0x7fffffff - 4096;                // (a tile's own indices may go past the end)

bool valid(const GroupArgs& g) {
  if (g.rows < 0 || g.cols < 0 || g.red < 0 || g.experts < 1) return false;
  if (g.rows > kMostExtent || g.cols > kMostExtent || g.red > kMostExtent) return false;
  if (g.dtype == kFp8) return g.mode == kModeForward && (g.scale == kScaleF32 || g.scale == kScaleE8);
  return (g.dtype == kBf16 || g.dtype == kFp16) && g.scale == kScaleNone && g.mode >= kModeForward && g.mode <= kModeWgrad;
}

// Whether c may share memory with an operand.
bool may_share(const GroupArgs& g) {
  const int es = g.dtype == kFp8 ? 1 : 2, ss = g.scale == kScaleF32 ? 4 : 1;
  const bool wgrad = g.mode == kModeWgrad, b_tr = g.mode != kModeForward;
  const long long kb = ((long long)g.red + kScaleBlock - 1) / kScaleBlock, nb = ((long long)g.cols + kScaleBlock - 1) / kScaleBlock;
  const auto reach = [](const void* p, int size, __int128 n0, __int128 s0, __int128 n1, __int128 s1, __int128 n2, __int128 s2) {
    return MemoryReach(p, n0 <= 0 || n1 <= 0 || n2 <= 0, (n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2, size);
  };
  const MemoryReach c = reach(g.c, 2, wgrad ? g.experts : 1, g.c_expert, g.rows, g.ldc, g.cols, 1);
  const long long a_rows = wgrad ? g.red : g.rows, a_cols = wgrad ? g.rows : g.red;
  if (c.meets(reach(g.a, es, 1, 0, a_rows, g.lda, a_cols, 1))) {
    // side by side in rows of one pitch, none of them shared
    const __int128 pitch = (__int128)g.lda * es, d = pitch > 0 ? ((__int128)(uintptr_t)g.a - (uintptr_t)g.c) % pitch : 0;
    const __int128 at = d < 0 ? d + pitch : d;
    if (wgrad || pitch != (__int128)g.ldc * 2 || at < 2ll * g.cols || at + a_cols * es > pitch) return true;
  }
  if (c.meets(reach(g.b, es, wgrad ? 1 : g.experts, g.b_expert, b_tr ? g.red : g.cols, g.ldb, b_tr ? g.cols : g.red, 1))) return true;
  if (g.offsets != nullptr && c.meets(reach(g.offsets, 4, 1, 0, 1, 0, (__int128)g.experts + 1, 1))) return true;
  return g.scale != kScaleNone && (c.meets(reach(g.a_scale, ss, 1, 0, g.rows, g.as_row, kb, g.as_k)) ||
                                   c.meets(reach(g.b_scale, ss, g.experts, g.bs_expert, nb, g.bs_row, kb, g.bs_k)));
}

int dispatch(const GroupArgs& g, hipStream_t s) {
  if (g.rows == 0 || g.cols == 0) return 0;
  if (g.dtype == kFp8) return g.scale == kScaleF32 ? dispatch_tile<kFp8, kScaleF32, false, false>(g, s)
                                                   : dispatch_tile<kFp8, kScaleE8, false, false>(g, s);
  return g.dtype == kBf16 ? dispatch16<kBf16>(g, s) : dispatch16<kFp16>(g, s);
}

}  // namespace

extern "C" {

int amdgo_gemm_group(const void* args, hipStream_t s) {
  if (!args) return (int)hipErrorInvalidValue;
  const GroupArgs g = group_args(args);
  if (!valid(g)) return (int)hipErrorInvalidValue;
  return may_share(g) ? kMayShare : dispatch(g, s);
}

// The same where the caller knows that c shares no memory with an operand.
int amdgo_gemm_group_apart(const void* args, hipStream_t s) {
  if (!args) return (int)hipErrorInvalidValue;
  const GroupArgs g = group_args(args);
  return valid(g) ? dispatch(g, s) : (int)hipErrorInvalidValue;
}

// Bytes of the workspace that amdgo_gemm_group_packed needs; negative: an argument is invalid, or no copy would do.
long long amdgo_group_workspace(const void* args) {
  if (!args || !valid(group_args(args))) return -1;
  const PackPlan plan(group_args(args));
  return plan.fits() ? plan.bytes : -1;
}

// `space`: 16-byte aligned, of that many bytes.
int amdgo_gemm_group_packed(const void* args, void* space, hipStream_t s) {
  if (!args || !valid(group_args(args)) || ((uintptr_t)space & 15)) return (int)hipErrorInvalidValue;
  PackPlan plan(group_args(args));
  if (!plan.fits() || (plan.bytes && !space)) return (int)hipErrorInvalidValue;
  const int err = plan.launch((char*)space, s);
  return err ? err : dispatch(plan.g, s);
}

}  // extern "C"
