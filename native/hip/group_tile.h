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
  // a wave's part: TN columns, and of the 16-row blocks every WM-th, so that all waves share what rows there are
  static constexpr int TN = BN / WN, NI = BM / WM / 16, NJ = TN / 16;
  static constexpr int OPA = BM * PB, OPB = BN * PB;      // bytes of a panel
  static constexpr int SCB = SC == kScaleNone ? 0 : THREADS * 4;

  static constexpr int STAGE = OPA + OPB + SCB;
  static constexpr int LDS = NBUF * STAGE;
  static_assert(LDS <= 160 * 1024, "one CU's LDS");
  static constexpr int RESIDENT = 160 * 1024 / LDS;                          // workgroups a CU that the ring leaves room for
  static constexpr int EU = WM * WN / 4 * (RESIDENT < 2 ? 1 : RESIDENT > 3 ? 4 : RESIDENT);   // waves a SIMD to plan registers for
  static_assert(!(DT == kFp8 && (ATR || BTR)), "fp8 operands are K-major");
  static_assert((DT == kFp8) == (SC != kScaleNone), "fp8 has scales");
  static_assert(NBUF <= 4, "the ring's counted waits");
  static_assert(BN >= 128 && (!ATR || BM >= 128), "the chunk permutations reach over 256 bytes of a row");
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

typedef const __attribute__((address_space(3))) char* lds_in;      // a panel to read: 32-bit addresses, constant offsets
__device__ __forceinline__ gi4 lds_chunk(lds_in p) { return *(const __attribute__((address_space(3))) gi4*)p; }
__device__ __forceinline__ int lds_word(lds_in p) { return *(const __attribute__((address_space(3))) int*)p; }

// A 64-byte step's fragments of a wave (16-bit operands), and its matrix instructions.
template <class C>
struct TileFrags {
  gi4 a[C::NI], b[C::NJ];
};

template <class C, int W>     // 16-row block `blk`; W: a reduction-major panel's columns, 0: K-major
__device__ __forceinline__ gi4 tile_frag(lds_in base, int blk0, int blk, int s) {
  const int lane = threadIdx.x & 63, j16 = lane & 15, g = lane >> 4;
  if constexpr (W > 0) {
    // rows s 32 + 8 g + 4 h + 0..3 of the panel: their swizzle depends on the lane alone
    const int r = g * 8 + (j16 >> 2), slot = (blk0 + blk) ^ rm_swizzle(r);
    const lds_in at = base + r * (2 * W) + (slot << 5) + (j16 & 3) * 8 + s * 32 * 2 * W;
    const gs4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gs4_lds)at);
    const gs4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gs4_lds)(at + 4 * 2 * W));
    const gi2 l2 = __builtin_bit_cast(gi2, lo), h2 = __builtin_bit_cast(gi2, hi);
    return gi4{l2[0], l2[1], h2[0], h2[1]};
  } else {
    return lds_chunk(base + blk0 * 16 * C::PB + km_at<C::PB>(j16, s * 4 + g) + blk * 16 * C::PB);
  }
}

template <class C>
__device__ __forceinline__ gf4 tile_mfma(const gi4& b, const gi4& a, const gf4& c) {
  if constexpr (C::DT == kFp16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gh8, b), __builtin_bit_cast(gh8, a), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gbf8, b), __builtin_bit_cast(gbf8, a), c, 0, 0, 0);
}

// NA of the wave's NI row blocks exist.
template <class C, int NA>
__device__ __forceinline__ void tile_read(lds_in lds, int wm, int wn, int s, TileFrags<C>& f) {
#pragma unroll
  for (int j = 0; j < C::NJ; ++j) f.b[j] = tile_frag<C, C::BTR ? C::BN : 0>(lds + C::OPA, wn * C::NJ, j, s);
#pragma unroll
  for (int i = 0; i < NA; ++i) f.a[i] = tile_frag<C, C::ATR ? C::BM : 0>(lds, wm, i * C::WM, s);
}

template <class C, int NA>
__device__ __forceinline__ void tile_mul(const TileFrags<C>& f, gf4 (&acc)[C::NI][C::NJ]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = tile_mfma<C>(f.b[j], f.a[i], acc[i][j]);
}

// One panel: acc += A panel x B panel^T (fp8: times the scales of the panel's block).
template <class C>
__device__ __forceinline__ gi8 tile_frag8(lds_in base, int blk0, int blk) {
  const int lane = threadIdx.x & 63, j16 = lane & 15, g = lane >> 4;
  const gi4 x = lds_chunk(base + blk0 * 2048 + km_at<128>(j16, g) + blk * 2048);
  const gi4 y = lds_chunk(base + blk0 * 2048 + km_at<128>(j16, g + 4) + blk * 2048);
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// fp8: one matrix instruction of 128 steps for each accumulator, weighted with the block's scales. e8m0 scales
// go into the instruction. float32 ones need its sum apart (16 x 16 of it: 4 registers) and 4 multiply-adds, which
// take half its time on the vector unit: the sums of 16 rows are kept while the next 16 rows' instructions run, so the
// vector unit works under the matrix unit (one scale for a lane's 4 values, since they lie along a row of A).
template <class C, int NA>
__device__ __forceinline__ void tile_compute8(lds_in lds, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  const int j16 = threadIdx.x & 15;
  const lds_in la = lds, lb = lds + C::OPA, ls = lds + C::OPA + C::OPB;
  gi8 bf[C::NJ];
#pragma unroll
  for (int j = 0; j < C::NJ; ++j) bf[j] = tile_frag8<C>(lb, wn * C::NJ, j);
  const int sb = lds_word(ls + C::BM * 4 + (wn * C::TN / kScaleBlock) * 4);
  const lds_in lsa = ls + (wm * 16 + j16) * 4;
  if constexpr (C::SC == kScaleE8) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const gi8 af = tile_frag8<C>(la, wm, i * C::WM);
      const int sa = lds_word(lsa + i * C::WM * 64);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af, acc[i][j], 0, 0, 0, sb, 0, sa);
    }
  } else {
    gf4 part[2][C::NJ];
    float s[2];
#pragma unroll
    for (int i = 0; i <= NA; ++i) {
      if (i < NA) {
        const gi8 af = tile_frag8<C>(la, wm, i * C::WM);
        s[i & 1] = __builtin_bit_cast(float, lds_word(lsa + i * C::WM * 64)) * __builtin_bit_cast(float, sb);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
          part[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af, gf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
      }
      if (i > 0) {
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i - 1][j][q] = fmaf(part[(i - 1) & 1][j][q], s[(i - 1) & 1], acc[i - 1][j][q]);
      }
    }
  }
}

template <class C, int NA>
__device__ __forceinline__ void tile_compute(lds_in lds, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  if constexpr (C::DT == kFp8) {
    tile_compute8<C, NA>(lds, wm, wn, acc);
  } else {
#pragma unroll
    for (int s = 0; s < C::PB / 64; ++s) {
      TileFrags<C> f;
      tile_read<C, NA>(lds, wm, wn, s, f);
      tile_mul<C, NA>(f, acc);
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
    RowTiles row_tiles(g, g.rows, C::BM);
    const int tiles_m = row_tiles.tiles, tiles = tiles_m * tiles_n;
    // The tiles past the last whole round of the `slots` workgroups that run at once would keep few of them busy for a
    // whole tile's time: they are cut into 2 or 4 parts by rows, as many as still fit one round.
    const int over = g.slots > 0 ? tiles % g.slots : 0, whole = tiles - over;
    const int parts = over == 0 ? 1 : 4 * over <= g.slots ? 4 : 2 * over <= g.slots ? 2 : 1;
    int tm, tn, tile, part = 0;
    if (block < whole) {
      tile = xcd_remap(block, whole);
    } else {
      if (block - whole >= over * parts) return false;
      const int item = xcd_remap(block - whole, over * parts);
      tile = whole + item / parts;
      part = item % parts;
    }
    tile_coords(tile, tiles_m, tiles_n, tm, tn);
    RowTile rt = row_tiles.find(tm);
    if (parts > 1 && block >= whole) {
      const int rows = C::BM / parts;
      rt.row0 += part * rows;
      rt.row_end = min(rt.row_end, rt.row0 + rows);
      if (rt.row0 >= rt.row_end) return false;
    }
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

// The result through LDS, which the loop has left: whole rows of the tile at a time, 16 bytes a lane (straight from
// the accumulators a store would write 32 bytes of each of 16 rows). Accumulator [i][j] of a lane holds row
// 16 (i WM + wm) + (lane & 15), columns 16 j + 4 (lane >> 4) + 0..3 of the wave's part: B is the matrix instruction's
// first operand, so a lane's four values lie along a row. 16-byte chunk c of row r lies at c ^ (r & 15): neither side
// conflicts. Rows that do not start on 16 bytes are stored by the same unaligned vector stores.
template <class C>
__device__ __forceinline__ void tile_store_rows(const GroupArgs& g, char* lds, char* c_tile, int c_rows, int c_cols, int wm, int wn,
                                                const gf4 (&acc)[C::NI][C::NJ]) {
  static_assert(C::BM * C::BN * 2 <= C::LDS, "the tile fits the ring");
  constexpr int OUT = C::DT == kFp16 ? kFp16 : kBf16;
  const bool wide = (((uintptr_t)g.c | (uintptr_t)(g.ldc * 2) | (uintptr_t)(g.c_expert * 2)) & 15) == 0;
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  bar();                                                 // every wave has read its last fragments
#pragma unroll
  for (int i = 0; i < C::NI; ++i) {
    const int r = (i * C::WM + wm) * 16 + l16;
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      unsigned short v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to_out<OUT>(acc[i][j][e]);
      const int c = (wn * C::TN + j * 16) / 8 + (q >> 1);
      *(uint2*)(lds + r * (C::BN * 2) + ((c ^ l16) << 4) + (q & 1) * 8) =
          make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
    }
  }
  __syncthreads();
  constexpr int CPR = C::BN / 8, RPI = C::THREADS / CPR;  // chunks a row, rows a step of the workgroup
  const int c = threadIdx.x % CPR;
  for (int r = threadIdx.x / CPR; r < c_rows; r += RPI) {
    const uint4 v = *(const uint4*)(lds + r * (C::BN * 2) + ((c ^ (r & 15)) << 4));
    unsigned short* at = (unsigned short*)c_tile + (size_t)r * g.ldc + c * 8;
    if (c * 8 + 8 <= c_cols) {
      if (wide) store_c16(at, v);
      else __builtin_memcpy(at, &v, 16);
    } else {
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c * 8 + e < c_cols) at[e] = (unsigned short)(w[e >> 1] >> ((e & 1) * 16));
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

// The scales of a panel by LDS-DMA: waves 0 .. BM / 64 - 1 fetch a row's each lane, the next wave the columns', the
// others nothing.
template <class C>
__device__ __forceinline__ void scale_lanes(const GroupArgs& g, const TileOperands& t, int wave, int lane, unsigned& soff,
                                            const char*& base, long long& step) {
  constexpr int SB = C::SC == kScaleF32 ? 4 : 1;
  if (wave < C::BM / 64) {
    const int r = wave * 64 + lane;
    if (r < t.a_rows) soff = (unsigned)r * (unsigned)(g.as_row * SB);
    base = t.as;
    step = g.as_k * SB;
  } else if (wave == C::BM / 64) {
    if (lane < C::BN / kScaleBlock && lane * kScaleBlock < t.b_rows) soff = (unsigned)lane * (unsigned)(g.bs_row * SB);
    base = t.bs;
    step = g.bs_k * SB;
  }
}

template <class C>
__device__ __forceinline__ void scale_load(char* lds, const char* base, int wave, unsigned soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
  g_lds_ptr const at = (g_lds_ptr)(lds + wave * 256);
  if constexpr (C::SC == kScaleF32) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at, 4, soff, 0, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at, 1, soff, 0, 0, 0);      // a byte to a word each
}

// A tile's panels by LDS-DMA, one after the other: PT pieces a wave for each.
template <class C>
struct TileLoader {
  using DmaA = PanelDma<C, C::ATR, C::BM>;
  using DmaB = PanelDma<C, C::BTR, C::BN>;
  static constexpr int PT = DmaA::PIECES + DmaB::PIECES + (C::SC != kScaleNone ? 1 : 0);
  DmaA da;
  DmaB db;
  const char *pa, *pb, *ps;
  size_t step_a, step_b;
  long long step_s;
  unsigned soff;
  int wave, lane, nk, left;

  __device__ __forceinline__ TileLoader(const GroupArgs& g, const TileOperands& t, int wave_, int lane_)
      : pa(t.a), pb(t.b), ps(t.as), step_a(C::ATR ? (size_t)C::KT * t.lda_b : C::PB),
        step_b(C::BTR ? (size_t)C::KT * t.ldb_b : C::PB), step_s(0), soff(kNowhere), wave(wave_), lane(lane_) {
    nk = (t.red + C::KT - 1) / C::KT;
    left = t.red - (nk - 1) * C::KT;
    da.init(wave, lane, (unsigned)t.lda_b, t.a_rows, t.a_col0, t.a_cols);
    db.init(wave, lane, (unsigned)t.ldb_b, t.b_rows, t.b_col0, t.b_cols);
    if constexpr (C::SC != kScaleNone) scale_lanes<C>(g, t, wave, lane, soff, ps, step_s);
  }
  // panel kt (the next one) into `base`
  __device__ __forceinline__ void issue(int kt, char* base) {
    if (kt == nk - 1 && left < C::KT) {
      da.cut(wave, lane, left);
      db.cut(wave, lane, left);
    }
    da.load(base, pa, wave);
    db.load(base + C::OPA, pb, wave);
    if constexpr (C::SC != kScaleNone) {
      scale_load<C>(base + C::OPA + C::OPB, ps, wave, soff);
      ps += step_s;
    }
    pa += step_a;
    pb += step_b;
  }
};

template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// One panel's work: panel kt goes into `into` (if there is one) while `from` is multiplied. Two pointers that do
// not alias, so that the compiler puts no wait for the DMA before the fragment reads.
template <class C, int NA>
__device__ __forceinline__ void tile_step(char* __restrict__ into, const __attribute__((address_space(3))) char* __restrict__ from,
                                          TileLoader<C>& ld, int kt, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  if (kt < ld.nk) ld.issue(kt, into);
  tile_compute<C, NA>(from, wm, wn, acc);
}

// The loop over the panels with NA of a wave's row blocks.
template <class C, int NA>
__device__ __forceinline__ void tile_loop(char* lds, TileLoader<C>& ld, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  constexpr int PT = TileLoader<C>::PT;
  int buf = 0;
  for (int kt = 0; kt < ld.nk; ++kt) {
    const int ahead = ld.nk - 1 - kt;                 // panels younger than kt that may stay in flight
    if (C::NBUF >= 4 && ahead >= 2) wait_vm<2 * PT>();
    else if (C::NBUF >= 3 && ahead >= 1) wait_vm<PT>();
    else wait_vm<0>();
    bar();
    tile_step<C, NA>(lds + (buf == 0 ? C::NBUF - 1 : buf - 1) * C::STAGE, (lds_in)lds + buf * C::STAGE, ld, kt + C::NBUF - 1,
                     wm, wn, acc);
    buf = buf == C::NBUF - 1 ? 0 : buf + 1;
  }
}

// The same tile with its panels in a ring of NBUF, NBUF - 1 of them in flight. At panel t a counted wait
// retires t's pieces only, a bare s_barrier publishes them, and panel t + NBUF - 1 goes into the buffer that
// every wave left at t - 1.
template <class C>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::EU, C::EU)))
group_tile_dma(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[C::LDS];     // the only LDS object: see tile_step
  if (zero_rest_rows(g, C::THREADS)) return;
  TileOperands t;
  char* c_tile;
  int c_rows, c_cols;
  if (!tile_setup<C>(g, blockIdx.x, t, c_tile, c_rows, c_cols)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WN, wn = wave % C::WN;
  TileLoader<C> ld(g, t, wave, lane);
  gf4 acc[C::NI][C::NJ];
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = gf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < C::NBUF - 1; ++p)
    if (p < ld.nk) ld.issue(p, lds + p * C::STAGE);
  // a group's last tile, or a part of a tile, is as long as its rows, in quarters
  if (C::NI < 4 || c_rows > C::BM / 2) tile_loop<C, C::NI>(lds, ld, wm, wn, acc);
  else if (c_rows > C::BM / 4) tile_loop<C, (C::NI + 1) / 2>(lds, ld, wm, wn, acc);
  else tile_loop<C, (C::NI + 3) / 4>(lds, ld, wm, wn, acc);
  tile_store_rows<C>(g, lds, c_tile, c_rows, c_cols, wm, wn, acc);
}

// The ping-pong form of the 256 x 256 tile. Its 8 waves are two groups of 4 (a SIMD has one wave of each), one
// interval apart: while one group runs matrix instructions, the other reads its next fragments from LDS and issues
// DMA; a barrier ends every interval. A panel takes a group four of them:
//
//   read B and the upper half's A | multiply the upper half | read the lower half's A | multiply the lower half
//
// (the wave's 64 columns of B are kept for both halves: 64 registers of fragments, 128 of sums). With two panels in
// LDS the parts of a buffer are refilled as soon as they are free: B, the upper half of A and the scales of panel t
// have been read by both groups when the first one reads the lower half, and there it issues those of panel
// t + 2; the lower half of panel t + 1 is issued where panel t's first read is. So a piece has 4 to 5 intervals (about
// 2500 cycles) to land, where the plain ring of two gives it 4 at most and leaves the matrix pipes idle while
// all waves read.
template <class C>
struct PingPong {
  static constexpr int HM = C::BM / 2, NH = C::NI / 2;                    // rows and a wave's blocks in a half
  static constexpr int HALF = HM * C::PB;
  static constexpr int LO = 0, HI = HALF, B = 2 * HALF, STAGE = B + C::OPB;      // where they are in a stage
  static constexpr int SCALES = 2 * STAGE, LDS = SCALES + 4 * C::SCB;             // the scales' ring
  using DmaA = PanelDma<C, C::ATR, HM>;
  using DmaB = PanelDma<C, C::BTR, C::BN>;
  static constexpr int P1 = DmaA::PIECES + DmaB::PIECES + (C::SC != kScaleNone ? 1 : 0), P2 = DmaA::PIECES;
  static_assert(C::WM == 2 && C::WN == 4 && C::NBUF == 2 && C::PB == 128, "two groups of four waves, two panels");
};

template <class C>
struct PingPongLoader {
  using P = PingPong<C>;
  typename P::DmaA lo, hi;
  typename P::DmaB b;
  const char *pa, *pb, *ps;
  size_t step_a, step_b;
  long long step_s;
  unsigned soff;
  int wave, lane, nk, left;

  __device__ __forceinline__ PingPongLoader(const GroupArgs& g, const TileOperands& t, int wave_, int lane_)
      : pa(t.a), pb(t.b), ps(t.as), step_a(C::ATR ? (size_t)C::KT * t.lda_b : C::PB),
        step_b(C::BTR ? (size_t)C::KT * t.ldb_b : C::PB), step_s(0), soff(kNowhere), wave(wave_), lane(lane_) {
    nk = (t.red + C::KT - 1) / C::KT;
    left = t.red - (nk - 1) * C::KT;
    lo.init(wave, lane, (unsigned)t.lda_b, t.a_rows, t.a_col0, t.a_cols);
    if constexpr (C::ATR) {
      hi.init(wave, lane, (unsigned)t.lda_b, 0, t.a_col0 + P::HM, t.a_cols);
    } else {
      hi.init(wave, lane, (unsigned)t.lda_b, t.a_rows - P::HM, 0, 0);
#pragma unroll
      for (int i = 0; i < P::DmaA::PIECES; ++i)
        if (hi.off[i] != kNowhere) hi.off[i] += (unsigned)P::HM * (unsigned)t.lda_b;
    }
    b.init(wave, lane, (unsigned)t.ldb_b, t.b_rows, t.b_col0, t.b_cols);
    if constexpr (C::SC != kScaleNone) scale_lanes<C>(g, t, wave, lane, soff, ps, step_s);
  }
  // B, A's upper half and the scales of panel kt into the stage at `base`
  __device__ __forceinline__ void issue_lo(int kt, char* base, char* ring) {
    if (kt == nk - 1 && left < C::KT) {
      lo.cut(wave, lane, left);
      b.cut(wave, lane, left);
    }
    b.load(base + P::B, pb + (size_t)kt * step_b, wave);
    lo.load(base + P::LO, pa + (size_t)kt * step_a, wave);
    if constexpr (C::SC != kScaleNone) scale_load<C>(ring + (kt & 3) * C::SCB, ps + kt * step_s, wave, soff);
  }
  __device__ __forceinline__ void issue_hi(int kt, char* base) {
    if (kt == nk - 1 && left < C::KT) hi.cut(wave, lane, left);
    hi.load(base + P::HI, pa + (size_t)kt * step_a, wave);
  }
};

// A wave's fragments of 16 rows or columns of a whole panel: 8 registers, for fp8 one matrix instruction's operand, for
// 16 bits two steps'.
template <class C, int W>
__device__ __forceinline__ gi8 panel_frag(lds_in base, int blk0, int blk) {
  if constexpr (C::DT == kFp8) {
    return tile_frag8<C>(base, blk0, blk);
  } else {
    const gi4 x = tile_frag<C, W>(base, blk0, blk, 0), y = tile_frag<C, W>(base, blk0, blk, 1);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <class C>
struct PingPongFrags {
  gi8 a[PingPong<C>::NH], b[C::NJ];
  int s[C::SC == kScaleNone ? 1 : PingPong<C>::NH];    // float32: the product of the scales; e8m0: the row's byte
  int sb;
};

// The scales of a half's rows. They have a ring of four panels apart, so that both halves can read them while the
// stage's next ones land.
template <class C, int NA, int HALF>
__device__ __forceinline__ void pp_scales(lds_in ring, int kt, int wm, int wn, PingPongFrags<C>& f) {
  if constexpr (C::SC != kScaleNone) {
    const lds_in at = ring + (kt & 3) * C::SCB;
    f.sb = lds_word(at + C::BM * 4 + (wn * C::TN / kScaleBlock) * 4);
    const lds_in rows = at + (HALF * PingPong<C>::HM + wm * 16 + (threadIdx.x & 15)) * 4;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      f.s[i] = lds_word(rows + i * C::WM * 64);
      if constexpr (C::SC == kScaleF32)
        f.s[i] = __builtin_bit_cast(int, __builtin_bit_cast(float, f.s[i]) * __builtin_bit_cast(float, f.sb));
    }
  }
}

// B and the upper half's A (NA of the wave's blocks).
template <class C, int NA>
__device__ __forceinline__ void pp_frags_lo(lds_in from, int wm, int wn, PingPongFrags<C>& f) {
  using P = PingPong<C>;
#pragma unroll
  for (int j = 0; j < C::NJ; ++j) f.b[j] = panel_frag<C, C::BTR ? C::BN : 0>(from + P::B, wn * C::NJ, j);
#pragma unroll
  for (int i = 0; i < NA; ++i) f.a[i] = panel_frag<C, C::ATR ? P::HM : 0>(from + P::LO, wm, i * C::WM);
}

// (Two pointers that do not alias, as in tile_step.)
template <class C>
__device__ __forceinline__ void pp_read_lo(char* __restrict__ into, const __attribute__((address_space(3))) char* __restrict__ from,
                                           lds_in ring, PingPongLoader<C>& ld, int kt, int wm, int wn, PingPongFrags<C>& f) {
  pp_frags_lo<C, PingPong<C>::NH>(from, wm, wn, f);
  pp_scales<C, PingPong<C>::NH, 0>(ring, kt, wm, wn, f);
  if (kt + 1 < ld.nk) ld.issue_hi(kt + 1, into);
}

template <class C>
__device__ __forceinline__ void pp_read_hi(char* __restrict__ into, const __attribute__((address_space(3))) char* __restrict__ from,
                                           char* ring, PingPongLoader<C>& ld, int kt, int wm, int wn, PingPongFrags<C>& f) {
  using P = PingPong<C>;
#pragma unroll
  for (int i = 0; i < P::NH; ++i) f.a[i] = panel_frag<C, C::ATR ? P::HM : 0>(from + P::HI, wm, i * C::WM);
  pp_scales<C, P::NH, 1>((lds_in)ring, kt, wm, wn, f);
  if (kt + 2 < ld.nk) ld.issue_lo(kt + 2, into, ring);
}

// The products of NA blocks of the wave, from its block I0 on.
template <class C, int I0, int NA>
__device__ __forceinline__ void pp_mul(const PingPongFrags<C>& f, gf4 (&acc)[C::NI][C::NJ]) {
  if constexpr (C::SC == kScaleF32) {
    // Accumulator k's sum is weighted after instruction k + 2 has been issued: by then it is there without a wait
    // (an instruction takes 32 cycles, its result 12 more), and 4 multiply-adds fit under each instruction. The
    // order is pinned: the scheduler would gather them and wait.
    constexpr int STEPS = NA * C::NJ;
    gf4 part[3];
#pragma unroll
    for (int k = 0; k < STEPS + 2; ++k) {
      if (k < STEPS)
        part[k % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f.b[k % C::NJ], f.a[k / C::NJ], gf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
                                                                     0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (k >= 2) {
        const int i = (k - 2) / C::NJ, j = (k - 2) % C::NJ;
        const float s = __builtin_bit_cast(float, f.s[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[I0 + i][j][q] = fmaf(part[(k - 2) % 3][q], s, acc[I0 + i][j][q]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if constexpr (C::SC == kScaleE8) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
        acc[I0 + i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f.b[j], f.a[i], acc[I0 + i][j], 0, 0, 0, f.sb, 0, f.s[i]);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          const gi8 b = f.b[j], a = f.a[i];
          acc[I0 + i][j] = h == 0 ? tile_mfma<C>(__builtin_shufflevector(b, b, 0, 1, 2, 3), __builtin_shufflevector(a, a, 0, 1, 2, 3), acc[I0 + i][j])
                                  : tile_mfma<C>(__builtin_shufflevector(b, b, 4, 5, 6, 7), __builtin_shufflevector(a, a, 4, 5, 6, 7), acc[I0 + i][j]);
        }
  }
  // the sums are done here: the compiler may not sink work past the barrier that follows
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) asm volatile("" : "+v"(acc[I0 + i][j]));
}

template <class C>
__device__ __forceinline__ void pp_loop(char* lds, PingPongLoader<C>& ld, int wave, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  using P = PingPong<C>;
  const int nk = ld.nk;
  if (nk == 0) return;
  char* const ring = lds + P::SCALES;
  ld.issue_lo(0, lds, ring);
  ld.issue_hi(0, lds);
  if (nk > 1) {
    ld.issue_lo(1, lds + P::STAGE, ring);
    wait_vm<P::P1 + P::P2>();
  } else {
    wait_vm<P::P2>();
  }
  bar();
  if (wave >= 4) bar();
  for (int kt = 0; kt < nk; ++kt) {
    char* const here = lds + (kt & 1) * P::STAGE;
    char* const there = lds + (~kt & 1) * P::STAGE;
    PingPongFrags<C> f;
    pp_read_lo<C>(there, (lds_in)here, (lds_in)ring, ld, kt, wm, wn, f);
    if (kt + 1 < nk) wait_vm<P::P1 + P::P2>();       // this wave's pieces of the lower half have landed
    else wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
    pp_mul<C, 0, P::NH>(f, acc);
    __builtin_amdgcn_s_setprio(0);
    bar();
    // (the stage's upper half, B and scales have been read by both groups: panel kt + 2's go there)
    pp_read_hi<C>(here, (lds_in)here, ring, ld, kt, wm, wn, f);
    if (kt + 2 < nk) wait_vm<P::P1 + P::P2>();       // and of the next panel's first part
    else wait_vm<P::P2>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
    pp_mul<C, P::NH, P::NH>(f, acc);
    __builtin_amdgcn_s_setprio(0);
    bar();
  }
  if (wave < 4) bar();
}

// A tile of at most half the rows: its upper half alone, NA of a wave's blocks, all waves in step.
template <class C, int NA>
__device__ __forceinline__ void pp_half_step(char* __restrict__ into, const __attribute__((address_space(3))) char* __restrict__ from,
                                             char* ring, PingPongLoader<C>& ld, int kt, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  if (kt + 1 < ld.nk) ld.issue_lo(kt + 1, into, ring);
  PingPongFrags<C> f;
  pp_frags_lo<C, NA>(from, wm, wn, f);
  pp_scales<C, NA, 0>((lds_in)ring, kt, wm, wn, f);
  pp_mul<C, 0, NA>(f, acc);
}

template <class C, int NA>
__device__ __forceinline__ void pp_half_loop(char* lds, PingPongLoader<C>& ld, int wm, int wn, gf4 (&acc)[C::NI][C::NJ]) {
  using P = PingPong<C>;
  char* const ring = lds + P::SCALES;
  if (ld.nk > 0) ld.issue_lo(0, lds, ring);
  for (int kt = 0; kt < ld.nk; ++kt) {
    wait_vm<0>();
    bar();
    pp_half_step<C, NA>(lds + (~kt & 1) * P::STAGE, (lds_in)lds + (kt & 1) * P::STAGE, ring, ld, kt, wm, wn, acc);
  }
}

template <class C>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) group_tile_pp(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[PingPong<C>::LDS];     // the only LDS object: see tile_step
  if (zero_rest_rows(g, C::THREADS)) return;
  TileOperands t;
  char* c_tile;
  int c_rows, c_cols;
  if (!tile_setup<C>(g, blockIdx.x, t, c_tile, c_rows, c_cols)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WN, wn = wave % C::WN;
  PingPongLoader<C> ld(g, t, wave, lane);
  gf4 acc[C::NI][C::NJ];
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = gf4{0.f, 0.f, 0.f, 0.f};
  if (c_rows > C::BM / 2) pp_loop<C>(lds, ld, wave, wm, wn, acc);
  else if (c_rows > C::BM / 4) pp_half_loop<C, PingPong<C>::NH>(lds, ld, wm, wn, acc);
  else pp_half_loop<C, PingPong<C>::NH / 2>(lds, ld, wm, wn, acc);
  tile_store_rows<C>(g, lds, c_tile, c_rows, c_cols, wm, wn, acc);
}
