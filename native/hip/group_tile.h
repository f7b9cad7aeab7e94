// The tiled kernel of the grouped products: a BM x BN output tile per workgroup, WM x WN waves, operand panels
// of 128 bytes along the reduction (64 elements of 16 bits, 128 of fp8: one scale block) staged through LDS.
#pragma once

#include "group_common.h"

template <int DT_, int SC_, bool ATR_, bool BTR_, int BM_, int BN_, int WM_, int WN_>
struct TileCfg {
  static constexpr int DT = DT_, SC = SC_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ATR = ATR_, BTR = BTR_;
  static constexpr int ES = DT == kFp8 ? 1 : 2;          // bytes an element
  static constexpr int KT = 128 / ES;                     // reduction steps a panel
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int TM = BM / WM, TN = BN / WN;        // a wave's part
  static constexpr int NI = TM / 16, NJ = TN / 16;
  static constexpr int OPA = BM * 128, OPB = BN * 128;    // bytes of a panel
  static constexpr int SCB = SC == kScaleNone ? 0 : (BM + 4) * 4;
  static constexpr int STAGE = OPA + OPB + SCB;
  static_assert(!(DT == kFp8 && (ATR || BTR)), "fp8 operands are K-major");
  static_assert((DT == kFp8) == (SC != kScaleNone), "fp8 has scales");
};

// Byte of 16-byte chunk q of row r in a K-major panel: rows of 128 bytes, chunks permuted by the row so that
// the fragment reads (16 rows, one chunk) spread over the banks.
__device__ __forceinline__ int km_at(int r, int q) { return r * 128 + ((q ^ (r & 7)) << 4); }

// Byte of 16-byte chunk q of row r in a reduction-major panel of W columns (2 W bytes a row): 32-byte slots
// permuted by the row. A transposing read takes 16 columns (one slot) of rows 8 g + 4 h + 0..3, so the rows
// that one read touches together are told apart by r & 3 and by bit 3 of r.
template <int W>
__device__ __forceinline__ int rm_at(int r, int q) {
  const int f = (r & 3) | (((r >> 3) & 1) << 2);
  return r * (2 * W) + (((q >> 1) ^ f) << 5) + ((q & 1) << 4);
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

// One reduction step of 128 bytes: acc += A panel x B panel^T (fp8: times the scales of the panel's block).
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
      const gi4 x = *(const gi4*)(lb + km_at(r, g)), y = *(const gi4*)(lb + km_at(r, g + 4));
      bf[j] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const char* ls = lds + C::OPA + C::OPB;
    if constexpr (C::SC == kScaleF32) {
      const float sb = *(const float*)(ls + C::BM * 4 + (wn * C::TN / kScaleBlock) * 4);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const int r = wm * C::TM + i * 16 + j16;
        const gi4 x = *(const gi4*)(la + km_at(r, g)), y = *(const gi4*)(la + km_at(r, g + 4));
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
        const gi4 x = *(const gi4*)(la + km_at(r, g)), y = *(const gi4*)(la + km_at(r, g + 4));
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
        return *(const gi4*)(base + km_at(row0 + j16, s * 4 + g));
      }
    };
    constexpr std::integral_constant<int, C::ATR ? C::BM : 0> ta;
    constexpr std::integral_constant<int, C::BTR ? C::BN : 0> tb;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
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
    for (int i = threadIdx.x; i < ROWS * 8; i += C::THREADS) {
      const int r = i >> 3, q = i & 7;
      gi4 v = {0, 0, 0, 0};
      if (r < rows) v = load_chunk<ES>(base + (size_t)r * ld_b, kt * C::KT + q * (16 / ES), red);
      *(gi4*)(lds + km_at(r, q)) = v;
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
    const int id = xcd_remap(block, per * g.experts);
    const int e = id / per;
    int tm, tn, begin = 0, end = g.red;
    tile_coords(id - e * per, tiles_m, tiles_n, tm, tn);
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
