// The tiled kernels of the grouped products: a BM x BN output tile per workgroup, WM x WN waves, operand panels
// of PB bytes along the reduction (128: 64 elements of 16 bits, or 128 of fp8, one scale block) staged through
// LDS.
#pragma once

#include "group_common.h"

template <int DT_, int SC_, bool ATR_, bool BTR_, int BM_, int BN_, int WM_, int WN_, int PB_ = 128, int NBUF_ = 1>
struct TileCfg {
  static constexpr int DT = DT_, SC = SC_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ATR = ATR_, BTR = BTR_;
  static constexpr int ES = DT == kFp8 ? 1 : 2;          // bytes an element
  static constexpr int PB = PB_, NBUF = NBUF_;            // bytes a panel is wide; panels in the ring
  static constexpr int KT = PB / ES;                      // reduction steps a panel
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int TM = BM / WM, TN = BN / WN;        // a wave's part
  static constexpr int NI = TM / 16, NJ = TN / 16;
  static constexpr int OPA = BM * PB, OPB = BN * PB;      // bytes of a panel
  static constexpr int SCB = SC == kScaleNone ? 0 : THREADS * 4;

  static constexpr int STAGE = OPA + OPB + SCB;
  static constexpr int LDS = NBUF * STAGE;
  static_assert(LDS <= 160 * 1024, "one CU's LDS");
  static constexpr int EU = WM * WN / 4 * (160 * 1024 / LDS >= 2 ? 2 : 1);   // waves a SIMD that the ring leaves room for
  static_assert(!(DT == kFp8 && (ATR || BTR)), "fp8 operands are K-major");
  static_assert((DT == kFp8) == (SC != kScaleNone), "fp8 has scales");
  static_assert(PB == 128 || (PB == 64 && DT != kFp8), "an fp8 panel is one scale block");
};

// Byte of 16-byte chunk q of row r in a K-major panel: rows of PB bytes, chunks permuted by the row so that
// the fragment reads (16 rows, one chunk) spread over the banks.
template <int PB>
__device__ __forceinline__ int km_swizzle(int r) { return PB == 128 ? r & 7 : (r >> 1) & 3; }
template <int PB>
__device__ __forceinline__ int km_at(int r, int q) { return r * PB + ((q ^ km_swizzle<PB>(r)) << 4); }

// Byte of 16-byte chunk q of row r in a reduction-major panel of W columns (2 W bytes a row): 32-byte slots
// permuted by the row. A transposing read takes 16 columns (one slot) of rows 8 g + 4 h + 0..3, so the rows
// that one read touches together are told apart by r & 3 and by bit 3 of r.
__device__ __forceinline__ int rm_swizzle(int r) { return (r & 3) | (((r >> 3) & 1) << 2); }
template <int W>
__device__ __forceinline__ int rm_at(int r, int q) {
  return r * (2 * W) + (((q >> 1) ^ rm_swizzle(r)) << 5) + ((q & 1) << 4);
}

// 16 bytes of a row from element `from`, elements at or past `upto` as zeros; any alignment.
template <int ES>
__device__ __forceinline__ gi4 load_chunk(const char* row, int from, int upto) {
  constexpr int N = 16 / ES;
  gi4 v = {0, 0, 0, 0};
  if (from + N <= upto) {
    __builtin_memcpy(&v, row + (size_t)from * ES, 16);
  } else {
    union { unsigned char b[16]; unsigned short h[8]; gi4 v; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (from + i < upto) {
        if constexpr (ES == 1) u.b[i] = ((const unsigned char*)row)[from + i];
        else u.h[i] = ((const unsigned short*)row)[from + i];
      }
    v = u.v;
  }
  return v;
}

// Where a tile's operands are and how far they go.
struct TileOperands {
  const char* a;          // first row (K-major) or first reduction row (reduction-major) of the tile
  const char* b;
  long long lda_b, ldb_b; // bytes
  int a_rows, b_rows;     // rows / columns of the tile that exist
  int a_col0, b_col0;     // reduction-major: the tile's first column
  int a_cols, b_cols;     // reduction-major: columns that exist
  int red;                // reduction steps
  const char* as;         // scales of the tile's rows and columns
  const char* bs;
};

// One panel: acc += A panel x B panel^T (fp8: times the scales of the panel's block).
template <class C>
__device__ __forceinline__ void tile_compute(const char* lds, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  const int lane = threadIdx.x & 63, j16 = lane & 15, g = lane >> 4;
  const char* la = lds;
  const char* lb = lds + C::OPA;
  if constexpr (C::DT == kFp8) {
    gi8 bf[C::NJ];
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      const int r = wn * C::TN + j * 16 + j16;
      const gi4 x = *(const gi4*)(lb + km_at<C::PB>(r, g)), y = *(const gi4*)(lb + km_at<C::PB>(r, g + 4));
      bf[j] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const char* ls = lds + C::OPA + C::OPB;
    if constexpr (C::SC == kScaleF32) {
      const float sb = *(const float*)(ls + C::BM * 4 + (wn * C::TN / kScaleBlock) * 4);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const int r = wm * C::TM + i * 16 + j16;
        const gi4 x = *(const gi4*)(la + km_at<C::PB>(r, g)), y = *(const gi4*)(la + km_at<C::PB>(r, g + 4));
        const gi8 af = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        const float s = *(const float*)(ls + r * 4) * sb;
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          const gf4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af, gf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(p[q], s, acc[i][j][q]);
        }
      }
    } else {
      const int sb = *(const int*)(ls + C::BM * 4 + (wn * C::TN / kScaleBlock) * 4);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const int r = wm * C::TM + i * 16 + j16;
        const gi4 x = *(const gi4*)(la + km_at<C::PB>(r, g)), y = *(const gi4*)(la + km_at<C::PB>(r, g + 4));
        const gi8 af = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        const int sa = *(const int*)(ls + r * 4);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af, acc[i][j], 0, 0, 0, sb, 0, sa);
      }
    }
  } else {
    auto frag = [&](auto TR, const char* base, int row0, int s) -> gi4 {
      if constexpr (decltype(TR)::value > 0) {
        constexpr int W = decltype(TR)::value;
        const int r = s * 32 + g * 8 + (j16 >> 2);
        const int at = rm_at<W>(r, row0 >> 3) + (j16 & 3) * 8;
        const gs4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gs4_lds)(base + at));
        const gs4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gs4_lds)(base + at + 4 * 2 * W));
        const gi2 l2 = __builtin_bit_cast(gi2, lo), h2 = __builtin_bit_cast(gi2, hi);
        return gi4{l2[0], l2[1], h2[0], h2[1]};
      } else {
        return *(const gi4*)(base + km_at<C::PB>(row0 + j16, s * 4 + g));
      }
    };
    constexpr std::integral_constant<int, C::ATR ? C::BM : 0> ta;
    constexpr std::integral_constant<int, C::BTR ? C::BN : 0> tb;
#pragma unroll
    for (int s = 0; s < C::PB / 64; ++s) {
      gi4 bf[C::NJ];
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) bf[j] = frag(tb, lb, wn * C::TN + j * 16, s);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const gi4 af = frag(ta, la, wm * C::TM + i * 16, s);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          if constexpr (C::DT == kFp16)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gh8, bf[j]), __builtin_bit_cast(gh8, af),
                                                                acc[i][j], 0, 0, 0);
          else
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gbf8, bf[j]), __builtin_bit_cast(gbf8, af),
                                                                acc[i][j], 0, 0, 0);
        }
      }
    }
  }
}

// A panel into LDS through registers: any alignment, any leading dimension, what lies outside reads as zero.
template <class C, bool TR, int ROWS>
__device__ __forceinline__ void stage_regs(char* lds, const char* base, long long ld_b, int rows, int col0, int cols, int red,
                                           int kt) {
  constexpr int ES = C::ES;
  if constexpr (TR) {
    constexpr int CPR = ROWS * 2 / 16;                 // chunks a reduction row
    for (int i = threadIdx.x; i < C::KT * CPR; i += C::THREADS) {
      const int r = i / CPR, q = i % CPR, k = kt * C::KT + r;
      gi4 v = {0, 0, 0, 0};
      if (k < red) v = load_chunk<ES>(base + (size_t)k * ld_b, col0 + q * 8, cols);
      *(gi4*)(lds + rm_at<ROWS>(r, q)) = v;
    }
  } else {
    constexpr int CPR = C::PB / 16;
    for (int i = threadIdx.x; i < ROWS * CPR; i += C::THREADS) {
      const int r = i / CPR, q = i % CPR;
      gi4 v = {0, 0, 0, 0};
      if (r < rows) v = load_chunk<ES>(base + (size_t)r * ld_b, kt * C::KT + q * (16 / ES), red);
      *(gi4*)(lds + km_at<C::PB>(r, q)) = v;
    }
  }
}

// The scales of a panel's block into LDS: one 32-bit word for each row of the tile, then one for each 128
// columns (float32, or the e8m0 byte). Rows and columns that do not exist get zero.
template <class C>
__device__ __forceinline__ void stage_scales(char* lds, const GroupArgs& g, const TileOperands& t, int kt) {
  if constexpr (C::SC != kScaleNone) {
    for (int i = threadIdx.x; i < C::BM + C::BN / kScaleBlock; i += C::THREADS) {
      int v = 0;
      if (i < C::BM) {
        const long long at = i * g.as_row + kt * g.as_k;
        if (i < t.a_rows) v = C::SC == kScaleF32 ? ((const int*)t.as)[at] : (int)((const unsigned char*)t.as)[at];
      } else {
        const int n = i - C::BM;
        const long long at = n * g.bs_row + kt * g.bs_k;
        if (n * kScaleBlock < t.b_rows) v = C::SC == kScaleF32 ? ((const int*)t.bs)[at] : (int)((const unsigned char*)t.bs)[at];
      }
      *(int*)(lds + i * 4) = v;
    }
  }
}

// The tile of this workgroup: what it reads and where it writes. False: nothing to do.
template <class C>
__device__ __forceinline__ bool tile_setup(const GroupArgs& g, int block, TileOperands& t, char*& c_tile, int& c_rows, int& c_cols) {
  const int tiles_n = (g.cols + C::BN - 1) / C::BN;
  if (g.mode == kModeWgrad) {
    const int tiles_m = (g.rows + C::BM - 1) / C::BM, per = tiles_m * tiles_n;
    // an expert's tiles over all XCDs: whole experts to an XCD would leave those with the short ones idle
    const int place = block / per, e = group_by_size(g, g.red, place);
    int tm, tn, begin = 0, end = g.red;
    tile_coords(xcd_remap(block - place * per, per), tiles_m, tiles_n, tm, tn);
    if (g.offsets) group_rows(g.offsets, e, g.red, begin, end);
    t.a = (const char*)g.a + (size_t)begin * g.lda * C::ES;
    t.b = (const char*)g.b + (size_t)begin * g.ldb * C::ES;
    t.a_col0 = tm * C::BM;
    t.b_col0 = tn * C::BN;
    t.a_cols = g.rows;
    t.b_cols = g.cols;
    t.red = end - begin;
    c_rows = min(C::BM, g.rows - tm * C::BM);
    c_cols = min(C::BN, g.cols - tn * C::BN);
    c_tile = (char*)g.c + 2 * ((size_t)e * g.c_expert + (size_t)tm * C::BM * g.ldc + (size_t)tn * C::BN);
  } else {
    const int tiles_m = group_tile_count(g, g.rows, C::BM);
    if (block >= tiles_m * tiles_n) return false;
    int tm, tn;
    tile_coords(xcd_remap(block, tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
    RowTile rt;
    if (!group_find_tile(g, g.rows, C::BM, tm, rt)) return false;
    t.a = (const char*)g.a + (size_t)rt.row0 * g.lda * C::ES;
    t.a_rows = min(C::BM, rt.row_end - rt.row0);
    t.b_rows = min(C::BN, g.cols - tn * C::BN);
    t.b_col0 = tn * C::BN;
    t.b_cols = g.cols;
    t.b = (const char*)g.b + ((size_t)rt.expert * g.b_expert + (C::BTR ? 0 : (size_t)tn * C::BN * g.ldb)) * C::ES;
    t.red = g.red;
    if constexpr (C::SC != kScaleNone) {
      constexpr int S = C::SC == kScaleF32 ? 4 : 1;
      t.as = (const char*)g.a_scale + (size_t)rt.row0 * g.as_row * S;
      t.bs = (const char*)g.b_scale + ((size_t)rt.expert * g.bs_expert + (size_t)(tn * C::BN / kScaleBlock) * g.bs_row) * S;
    }
    c_rows = t.a_rows;
    c_cols = t.b_rows;
    c_tile = (char*)g.c + 2 * ((size_t)rt.row0 * g.ldc + (size_t)tn * C::BN);
  }
  t.lda_b = g.lda * C::ES;
  t.ldb_b = g.ldb * C::ES;
  return true;
}

// Accumulator [i][j] of a lane: row 16 i + (lane & 15), columns 16 j + 4 (lane >> 4) + 0..3 of the wave's part
// (B is the matrix instruction's first operand, so a lane's four values lie along a row of C).
template <class C>
__device__ __forceinline__ void tile_store(const GroupArgs& g, char* c_tile, int c_rows, int c_cols, int wm, int wn,
                                           const gf4 (&acc)[C::NI][C::NJ]) {
  constexpr int OUT = C::DT == kFp16 ? kFp16 : kBf16;
  const int lane = threadIdx.x & 63;
  const bool wide = ((uintptr_t)g.c & 7) == 0 && (g.ldc & 3) == 0 && (g.c_expert & 3) == 0;
#pragma unroll
  for (int i = 0; i < C::NI; ++i) {
    const int r = wm * C::TM + i * 16 + (lane & 15);
    if (r >= c_rows) continue;
    unsigned short* row = (unsigned short*)c_tile + (size_t)r * g.ldc;
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      const int c = wn * C::TN + j * 16 + (lane >> 4) * 4;
      unsigned short v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = to_out<OUT>(acc[i][j][q]);
      if (wide && c + 4 <= c_cols) {
        *(uint2*)(row + c) = make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (c + q < c_cols) row[c + q] = v[q];
      }
    }
  }
}

// What an LDS-DMA lane that has nothing to load asks for: past every buffer's end, so it gets zeros.
constexpr unsigned kNowhere = 0x80000000u;

typedef __attribute__((address_space(3))) void* g_lds_ptr;

// One operand's panels by LDS-DMA (buffer_load ... lds): a wave instruction fills 1 KiB of LDS in lane order,
// so the permutation of the chunks goes on the addresses that the lanes read. Each lane keeps the offsets of its
// pieces; the panel's place is the descriptor's base. Rows or columns that do not exist, and in the last panel
// the reduction steps past the end, are offsets past the buffer: zeros, whatever lies there.
template <class C, bool TR, int ROWS>
struct PanelDma {
  static constexpr int WAVES = C::THREADS / 64;
  static constexpr int PIECES = ROWS * C::PB / 1024 / WAVES;
  static_assert(PIECES * WAVES * 1024 == ROWS * C::PB, "whole pieces");
  unsigned off[PIECES];

  __device__ __forceinline__ static int row_of(int piece, int wave, int lane) {
    if constexpr (TR) return (piece * WAVES + wave) * (1024 / (2 * ROWS)) + lane / (ROWS / 8);
    else return (piece * WAVES + wave) * (1024 / C::PB) + lane / (C::PB / 16);
  }
  // the 16-byte chunk of its row that the lane reads
  __device__ __forceinline__ static int chunk_of(int row, int lane) {
    if constexpr (TR) {
      const int q = lane % (ROWS / 8);
      return (((q >> 1) ^ rm_swizzle(row)) << 1) | (q & 1);
    } else {
      return (lane % (C::PB / 16)) ^ km_swizzle<C::PB>(row);
    }
  }
  __device__ __forceinline__ void init(int wave, int lane, unsigned ld, int rows, int col0, int cols) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int r = row_of(i, wave, lane), q = chunk_of(r, lane);
      if constexpr (TR) off[i] = col0 + q * 8 < cols ? (unsigned)r * ld + (unsigned)(col0 + q * 8) * 2 : kNowhere;
      else off[i] = r < rows ? (unsigned)r * ld + q * 16 : kNowhere;
    }
  }
  // the last panel: `left` reduction steps of it exist
  __device__ __forceinline__ void cut(int wave, int lane, int left) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int r = row_of(i, wave, lane);
      if constexpr (TR) off[i] = r < left ? off[i] : kNowhere;
      else off[i] = chunk_of(r, lane) * 16 < left * C::ES ? off[i] : kNowhere;
    }
  }
  __device__ __forceinline__ void load(char* lds, const char* panel, int wave) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)panel, 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (g_lds_ptr)(lds + (i * WAVES + wave) * 1024), 16, off[i], 0, 0, 0);
  }
};

template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// One panel's work: the next panel's DMA goes into `into` while `from` is multiplied. Two pointers that do not
// alias, so that the compiler puts no wait for the DMA before the fragment reads.
template <class C, class F>
__device__ __forceinline__ void tile_step(char* __restrict__ into, const char* __restrict__ from, int wm, int wn,
                                          gf4 (&acc)[C::NI][C::NJ], F&& issue) {
  issue(into);
  tile_compute<C>(from, wm, wn, acc);
}

// The same tile with its panels in a ring of NBUF, NBUF - 1 of them in flight. At panel t a counted wait
// retires t's pieces only, a bare s_barrier publishes them, and panel t + NBUF - 1 goes into the buffer that
// every wave left at t - 1.
template <class C>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::EU, C::EU)))
group_tile_dma(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[C::LDS];     // the only LDS object: see tile_step
  zero_rest_rows(g, g.cols, blockIdx.x, gridDim.x, C::THREADS);
  TileOperands t;
  char* c_tile;
  int c_rows, c_cols;
  if (!tile_setup<C>(g, blockIdx.x, t, c_tile, c_rows, c_cols)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WN, wn = wave % C::WN;
  using DmaA = PanelDma<C, C::ATR, C::BM>;
  using DmaB = PanelDma<C, C::BTR, C::BN>;
  DmaA da;
  DmaB db;
  da.init(wave, lane, (unsigned)t.lda_b, t.a_rows, t.a_col0, t.a_cols);
  db.init(wave, lane, (unsigned)t.ldb_b, t.b_rows, t.b_col0, t.b_cols);
  const size_t step_a = C::ATR ? (size_t)C::KT * t.lda_b : C::PB, step_b = C::BTR ? (size_t)C::KT * t.ldb_b : C::PB;
  // scales: waves 0 .. BM / 64 - 1 fetch a row's each lane, the next wave the columns', the others nothing
  constexpr int SB = C::SC == kScaleF32 ? 4 : 1;
  unsigned soff = kNowhere;
  const char* sbase = t.as;
  long long sstep = 0;
  if constexpr (C::SC != kScaleNone) {
    if (wave < C::BM / 64) {
      const int r = wave * 64 + lane;
      if (r < t.a_rows) soff = (unsigned)r * (unsigned)(g.as_row * SB);
      sstep = g.as_k * SB;
    } else if (wave == C::BM / 64) {
      if (lane < C::BN / kScaleBlock && lane * kScaleBlock < t.b_rows) soff = (unsigned)lane * (unsigned)(g.bs_row * SB);
      sbase = t.bs;
      sstep = g.bs_k * SB;
    }
  }
  constexpr int PT = DmaA::PIECES + DmaB::PIECES + (C::SC != kScaleNone ? 1 : 0);
  const int nk = (t.red + C::KT - 1) / C::KT, left = t.red - (nk - 1) * C::KT;
  const char *pa = t.a, *pb = t.b;
  auto issue = [&](int kt, char* base) {
    if (kt == nk - 1 && left < C::KT) {
      da.cut(wave, lane, left);
      db.cut(wave, lane, left);
    }
    da.load(base, pa, wave);
    db.load(base + C::OPA, pb, wave);
    if constexpr (C::SC != kScaleNone) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)sbase, 0, 0x7fffffff, 0x00020000);
      g_lds_ptr const at = (g_lds_ptr)(base + C::OPA + C::OPB + wave * 256);
      if constexpr (C::SC == kScaleF32) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at, 4, soff, 0, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at, 1, soff, 0, 0, 0);      // a byte to a word each
      sbase += sstep;
    }
    pa += step_a;
    pb += step_b;
  };
  gf4 acc[C::NI][C::NJ];
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = gf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < C::NBUF - 1; ++p)
    if (p < nk) issue(p, lds + p * C::STAGE);
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const int ahead = nk - 1 - kt;
    if constexpr (C::NBUF >= 4) {
      if (ahead >= C::NBUF - 2) wait_vm<PT * (C::NBUF - 2)>();
      else if (ahead == 1) wait_vm<PT>();
      else if (ahead == 0) wait_vm<0>();
      else wait_vm<2 * PT>();
    } else if constexpr (C::NBUF == 3) {
      if (ahead >= 1) wait_vm<PT>();
      else wait_vm<0>();
    } else {
      wait_vm<0>();
    }
    bar();
    tile_step<C>(lds + (buf == 0 ? C::NBUF - 1 : buf - 1) * C::STAGE, lds + buf * C::STAGE, wm, wn, acc,
                 [&](char* into) {
                   if (kt + C::NBUF - 1 < nk) issue(kt + C::NBUF - 1, into);
                 });
    buf = buf == C::NBUF - 1 ? 0 : buf + 1;
  }
  tile_store<C>(g, c_tile, c_rows, c_cols, wm, wn, acc);
}

template <class C>
__global__ void __launch_bounds__(C::THREADS) group_tile_regs(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[C::STAGE];
  zero_rest_rows(g, g.cols, blockIdx.x, gridDim.x, C::THREADS);
  TileOperands t;
  char* c_tile;
  int c_rows, c_cols;
  if (!tile_setup<C>(g, blockIdx.x, t, c_tile, c_rows, c_cols)) return;
  const int wave = threadIdx.x >> 6, wm = wave / C::WN, wn = wave % C::WN;
  gf4 acc[C::NI][C::NJ];
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = gf4{0.f, 0.f, 0.f, 0.f};
  const int nk = (t.red + C::KT - 1) / C::KT;
  for (int kt = 0; kt < nk; ++kt) {
    stage_regs<C, C::ATR, C::BM>(lds, t.a, t.lda_b, t.a_rows, t.a_col0, t.a_cols, t.red, kt);
    stage_regs<C, C::BTR, C::BN>(lds + C::OPA, t.b, t.ldb_b, t.b_rows, t.b_col0, t.b_cols, t.red, kt);
    stage_scales<C>(lds + C::OPA + C::OPB, g, t, kt);
    __syncthreads();
    tile_compute<C>(lds, wm, wn, acc);
    __syncthreads();
  }
  tile_store<C>(g, c_tile, c_rows, c_cols, wm, wn, acc);
}
